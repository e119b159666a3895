"""Run by test_gpu_feedforward.py in a process of its own (torch has to be imported before beam): the feed-forward operators on
torch tensors.  The compiled binding and the general path give the same bits and the same errors; a training step and a served
layer, as a program strings them together, against float64; other streams; graphs that replay beside each other's workspaces."""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "general-nvgpu-testing_amd"))
import beam  # noqa: E402
from beam import _C  # noqa: E402

native = _C._native
assert native is not None
calls = []


class Counting:
    def __getattr__(self, name):
        def call(*args):
            status = getattr(native, name)(*args)
            calls.append((name, status))
            return status
        return call


def both(what, f, outs, handled=True):
    got = []
    for binding in (Counting(), None):
        _C._native = binding
        for o in outs:
            o.view(torch.uint8).fill_(0xFF)
        calls.clear()
        f()
        torch.cuda.synchronize()
        if binding is not None:
            assert bool(calls and calls[-1][1] >= 0) == handled, (what, calls)
        got.append([o.clone() for o in outs])
    _C._native = native
    assert all((x.view(torch.uint8) == y.view(torch.uint8)).all() for x, y in zip(*got)), what


def same_error(what, f):
    said = []
    for binding in (Counting(), None):
        _C._native = binding
        try:
            f()
        except Exception as e:  # noqa: BLE001
            said.append((type(e), str(e)))
    _C._native = native
    assert len(said) == 2 and said[0] == said[1], (what, said)


def randn(*shape, dtype, scale=1.0):
    return torch.randn(*shape, device="cuda", dtype=dtype) * scale


def held(rows, K, dtype, scale=1.0):
    w = randn(rows, K, dtype=dtype, scale=scale)
    q = torch.empty(rows, K // 2, device="cuda", dtype=torch.uint8)
    s = torch.empty(beam.mxfp4_scales_shape(rows, K), device="cuda", dtype=torch.uint8)
    beam.mxfp4_quantize(w, q, s)
    return q, s


for dtype in (torch.float16, torch.bfloat16):
    e = torch.finfo(dtype).eps / 2
    for M, N, K in ((65, 72, 200), (1, 1000, 96), (300, 501, 256), (17, 64, 1001)):
        a, b = randn(M, K, dtype=dtype), randn(2 * N, K, dtype=dtype, scale=K ** -0.5)
        h, gu = torch.empty(M, N, device="cuda", dtype=dtype), torch.empty(M, 2 * N, device="cuda", dtype=dtype)
        both("gated", lambda: beam.gemmrc_gated(a, b, h), [h])
        both("gated, kept", lambda: beam.gemmrc_gated(a, torch.nn.Parameter(b), h, gu=gu), [h, gu])
        dh, da, db = randn(M, N, dtype=dtype), torch.empty_like(a), torch.empty_like(b)
        both("backward", lambda: beam.gemmrc_gated_backward(dh, gu, a, b, da, db), [da, db])
        both("backward of a", lambda: beam.gemmrc_gated_backward(dh, gu, a, b, da=da), [da])
        both("backward of b", lambda: beam.gemmrc_gated_backward(dh, gu, a, b, db=db), [db])
        # the step's gradients against float64 autograd (loss: sum of dh * h); a value's rounding on the way (gu, D) is e of it,
        # and their sums over tokens or features are of independent parts: norms are within 4 e
        A, B = a.double().requires_grad_(), b.double().requires_grad_()
        z = A @ B.t()
        (torch.nn.functional.silu(z[:, :N]) * z[:, N:] * dh.double()).sum().backward()
        for got, want in ((da, A.grad), (db, B.grad)):
            assert (got.double() - want).norm() <= 4 * e * want.norm(), (M, N, K, dtype)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            both("another stream", lambda: (beam.gemmrc_gated(a, b, h, gu), beam.gemmrc_gated_backward(dh, gu, a, b, da, db)), [h, gu, da, db])
        torch.cuda.synchronize()
    for M, N, K in ((1, 500, 96), (16, 64, 1024), (40, 333, 288), (300, 1001, 4096)):
        a, (q, s) = randn(M, K, dtype=dtype), held(N, K, dtype, K ** -0.5)
        qa, sa = torch.empty(M, K // 2, device="cuda", dtype=torch.uint8), torch.empty(beam.mxfp4_scales_shape(M, K), device="cuda", dtype=torch.uint8)
        x, c, c2 = torch.empty_like(a), torch.empty(M, N, device="cuda", dtype=dtype), torch.empty(M, N, device="cuda", dtype=dtype)
        both("quantize", lambda: beam.mxfp4_quantize(a, qa, sa), [qa, sa])
        both("dequantize", lambda: beam.mxfp4_dequantize(qa, sa, x), [x])
        both("product", lambda: beam.gemmrc_mxfp4(qa, sa, q, s, c), [c])
        both("linear", lambda: beam.linear_mxfp4(a, q, s, c2), [c2])
        assert (c == c2).all()
        w = torch.empty(N, K, device="cuda", dtype=dtype)
        beam.mxfp4_dequantize(q, s, w)
        want = x.double() @ w.double().t()
        assert ((c.double() - want).abs() <= e * want.abs() + K * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()) + 1e-7).all()
        if hasattr(torch, "float4_e2m1fn_x2"):
            both("4-bit types", lambda: beam.gemmrc_mxfp4(qa.view(torch.float4_e2m1fn_x2), sa.view(torch.float8_e8m0fnu), q, s, c), [c], handled=False)
        both("rows from the middle", lambda: beam.linear_mxfp4(a[M // 2:], q, s, c[M // 2:]), [c[M // 2:]])

    a, b, h, gu = randn(8, 64, dtype=dtype), randn(12, 64, dtype=dtype), randn(8, 6, dtype=dtype), randn(8, 12, dtype=dtype)
    (q, s), c = held(6, 64, dtype), randn(8, 6, dtype=dtype)
    other = torch.float16 if dtype == torch.bfloat16 else torch.bfloat16
    same_error("odd rows", lambda: beam.gemmrc_gated(a, b[:-1], h))
    same_error("K differs", lambda: beam.gemmrc_gated(a[:, :-1].contiguous(), b, h))
    same_error("rows apart", lambda: beam.gemmrc_gated(randn(8, 128, dtype=dtype)[:, :64], b, h))
    same_error("two types", lambda: beam.gemmrc_gated(a, b.to(other), h))
    same_error("on the CPU", lambda: beam.gemmrc_gated(a, b.cpu(), h))
    same_error("fp32", lambda: beam.gemmrc_gated(a, b, h.float()))
    same_error("gu", lambda: beam.gemmrc_gated(a, b, h, gu[:, :6].contiguous()))
    same_error("no h", lambda: beam.gemmrc_gated(a, b, None))
    same_error("dh", lambda: beam.gemmrc_gated_backward(gu, gu, a, b, a, b))
    same_error("db", lambda: beam.gemmrc_gated_backward(h, gu, a, b, a, a))
    same_error("scales as rows", lambda: beam.linear_mxfp4(a, q, s.view(6, 8), c))
    same_error("scales of another", lambda: beam.linear_mxfp4(a, q, s[:, :-1].contiguous(), c))
    same_error("elements in 16 bits", lambda: beam.linear_mxfp4(a, q.view(torch.int16), s, c))
    same_error("elements apart", lambda: beam.linear_mxfp4(a, torch.zeros(6, 64, device="cuda", dtype=torch.uint8)[:, :32], s, c))
    same_error("elements off 16 bytes", lambda: beam.linear_mxfp4(a, torch.zeros(6 * 32 + 8, device="cuda", dtype=torch.uint8)[8:].view(6, 32), s, c))
    same_error("K not in blocks", lambda: beam.mxfp4_quantize(randn(4, 40, dtype=dtype), q, s))
    same_error("c's type", lambda: beam.linear_mxfp4(a, q, s, c.to(other)))

# Two graphs whose calls need workspace, replayed beside each other on two streams, with eager calls in between.
M, N, K = 333, 416, 520
b = randn(2 * N, K, dtype=torch.bfloat16, scale=K ** -0.5)
q, s = held(K, N, torch.bfloat16, N ** -0.5)
_C._native = native


def step(t):
    beam.gemmrc_gated(t["a"], b, t["h"], t["gu"])
    beam.linear_mxfp4(t["h"], q, s, t["y"])
    beam.gemmrc_gated_backward(t["dh"], t["gu"], t["a"], b, t["da"], t["db"])


def tensors():
    bf = torch.bfloat16
    t = {"a": randn(M, K, dtype=bf), "dh": randn(M, N, dtype=bf)}
    for name, shape in (("h", (M, N)), ("gu", (M, 2 * N)), ("y", (M, K)), ("da", (M, K)), ("db", (2 * N, K))):
        t[name] = torch.empty(shape, device="cuda", dtype=bf)
    return t


outs = ("h", "gu", "y", "da", "db")
sets, graphs, streams = [tensors(), tensors()], [], [torch.cuda.Stream(), torch.cuda.Stream()]
for t in sets:
    step(t)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(t)
    graphs.append(g)
for replay in range(5):
    want = []
    for t in sets:
        t["a"].copy_(randn(M, K, dtype=torch.bfloat16))
        t["dh"].copy_(randn(M, N, dtype=torch.bfloat16))
        step(t)
        torch.cuda.synchronize()
        want.append({n: t[n].clone() for n in outs})
        for n in outs:
            t[n].fill_(float("nan"))
    torch.cuda.synchronize()
    for g, stream in zip(graphs, streams):
        with torch.cuda.stream(stream):
            for _ in range(3):
                g.replay()
    extra = tensors()
    step(extra)  # eager, on a third stream
    torch.cuda.synchronize()
    for t, w in zip(sets, want):
        assert all((t[n] == w[n]).all() for n in outs), (replay, [n for n in outs if not (t[n] == w[n]).all()])
print("feed-forward OK")
