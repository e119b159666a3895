"""What the gated layer's entry points refuse, before anything is launched: no GPU is needed to be told."""
import ctypes

import pytest

F16, F32 = 0, 2
INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
P = 0x10000  # never dereferenced


def refused(beamc, rc, status, text):
    assert rc == status, (rc, beamc.lib.beam_last_error())
    assert text in beamc.lib.beam_last_error().decode()


def test_forward(beamc):
    f = beamc.lib.beam_gemmrc_gated
    refused(beamc, f(P, P, P, P, -1, 8, 8, F16, None), INVALID, "negative")
    refused(beamc, f(P, P, P, P, 8, -8, 8, F16, None), INVALID, "negative")
    refused(beamc, f(P, P, P, P, 8, 8, 8, F32, None), UNSUPPORTED, "dtype")
    refused(beamc, f(None, P, P, P, 8, 8, 8, F16, None), INVALID, "null input")
    refused(beamc, f(P, None, P, P, 8, 8, 8, F16, None), INVALID, "null input")
    refused(beamc, f(P, P, None, P, 8, 8, 8, F16, None), INVALID, "null output")
    refused(beamc, f(P + 1, P, P, P, 8, 8, 8, F16, None), INVALID, "aligned")
    refused(beamc, f(P, P, P, P + 1, 8, 8, 8, F16, None), INVALID, "aligned")
    refused(beamc, f(P, P, P, P, 8, 1 << 30, 8, F16, None), UNSUPPORTED, "too large")
    refused(beamc, f(P, P, P, P, 1 << 30, 8, 8, F16, None), UNSUPPORTED, "too large")


def test_overlaps(beamc):
    """M 100, N 60, K 60: one byte of an output in something else."""
    M, N, K = 100, 60, 60
    sizes = {"a": M * K * 2, "b": N * K * 4, "h": M * N * 2, "gu": M * N * 4, "dh": M * N * 2, "da": M * K * 2, "db": N * K * 4}
    ws_bytes = beamc.lib.beam_gemmrc_gated_backward_workspace_bytes(M, N, K, 1, 1)
    sizes["ws"] = ws_bytes
    apart, at = {}, P
    for k, n in sizes.items():
        apart[k] = at
        at += (n + 511) // 256 * 256
    last = {k: apart[k] + sizes[k] - 2 for k in sizes}

    def forward(**kw):
        v = {**apart, **kw}
        return beamc.lib.beam_gemmrc_gated(v["a"], v["b"], v["h"], v["gu"], M, N, K, F16, None)

    def backward(**kw):
        v = {**apart, **kw}
        return beamc.lib.beam_gemmrc_gated_backward(v["dh"], v["gu"], v["a"], v["b"], v["da"], v["db"], M, N, K, F16, v["ws"], ws_bytes, None)

    for x in ("a", "b"):
        for out in ("h", "gu"):
            refused(beamc, forward(**{out: last[x]}), INVALID, "overlap")
    refused(beamc, forward(h=last["gu"]), INVALID, "overlap")
    for x in ("dh", "gu", "a", "b"):
        for out in ("da", "db"):
            refused(beamc, backward(**{out: last[x]}), INVALID, "overlap")
        refused(beamc, backward(**{x: apart["ws"]}), INVALID, "overlap")
    refused(beamc, backward(da=last["db"]), INVALID, "overlap")
    refused(beamc, backward(da=last["ws"]), INVALID, "overlap")


def test_backward(beamc):
    f, need = beamc.lib.beam_gemmrc_gated_backward, beamc.lib.beam_gemmrc_gated_backward_workspace_bytes
    n = need(100, 60, 8, 1, 1)
    assert n <= need(100, 60, 8, 1, 0) + need(100, 60, 8, 0, 1) and min(need(100, 60, 8, 1, 0), need(100, 60, 8, 0, 1)) >= 100 * 120 * 2 and n % 256 == 0
    assert need(0, 60, 8, 1, 1) == need(100, 0, 8, 1, 1) == need(100, 60, 8, 0, 0) == 0
    good = [P, P, P, P, P, P, 100, 60, 8, F16, P, n, None]

    def but(**kw):
        names = ["dh", "gu", "a", "b", "da", "db", "M", "N", "K", "dtype", "ws", "bytes", "stream"]
        return f(*[kw.get(k, v) for k, v in zip(names, good)])

    refused(beamc, but(M=-1), INVALID, "negative")
    refused(beamc, but(dtype=F32), UNSUPPORTED, "dtype")
    for k in ("dh", "gu", "a", "b"):
        refused(beamc, but(**{k: None}), INVALID, "null input")
        refused(beamc, but(**{k: P + 1}), INVALID, "aligned")
    for k in ("da", "db"):
        refused(beamc, but(**{k: P + 1}), INVALID, "aligned")
    refused(beamc, but(ws=None), WORKSPACE, "workspace")
    refused(beamc, but(ws=P + 128), WORKSPACE, "workspace")
    refused(beamc, but(bytes=n - 1), WORKSPACE, "workspace")
    refused(beamc, but(M=1 << 28, N=1 << 18), UNSUPPORTED, "too large")
    refused(beamc, but(N=1 << 23), UNSUPPORTED, "too large")
    assert but(da=None, db=None) == 0  # nothing asked for


def test_python_layer(beamc):
    class Fake(beamc.DeviceArray):
        def __init__(self, shape, dtype=F16):
            self.shape, self.dtype, self.itemsize, self.ptr = shape, dtype, 2, 0

    def raises(text, f, *args):
        with pytest.raises(beamc.BeamError) as e:
            f(*args)
        assert text in str(e.value), e.value

    a, b, h, gu = Fake((4, 16)), Fake((12, 16)), Fake((4, 6)), Fake((4, 12))
    f = beamc.gemmrc_gated
    raises("rows", f, a, Fake((11, 16)), h)
    raises("b has shape", f, a, Fake((12, 8)), h)
    raises("h has shape", f, a, b, Fake((4, 12)))
    raises("gu has shape", f, a, b, h, Fake((4, 6)))
    raises("must be 2-D", f, Fake((4, 2, 8)), b, h)
    raises("must be fp16", f, a, Fake((12, 16), 1), h)
    raises("too large", f, Fake((1 << 31, 16)), b, h)
    g = beamc.gemmrc_gated_backward
    raises("dh has shape", g, Fake((4, 5)), gu, a, b, a, b)
    raises("gu has shape", g, h, h, a, b, a, b)
    raises("da has shape", g, h, gu, a, b, b, b)
    raises("db has shape", g, h, gu, a, b, a, a)
    raises("db must be", g, h, gu, a, b, a, Fake((12, 16), 1))
    with pytest.raises(TypeError):
        f(a, b, None)
