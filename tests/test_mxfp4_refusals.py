"""What the MXFP4 entry points refuse, before anything is launched: no GPU is needed to be told."""
import pytest

from test_gated_refusals import F16, F32, INVALID, P, UNSUPPORTED, WORKSPACE, refused


def test_scale_bytes(beamc):
    f = beamc.lib.beam_mxfp4_scale_bytes
    assert [f(r, k) for r, k in ((1, 32), (1, 256), (3, 288), (0, 32), (5, 0), (-1, 32))] == [8, 8, 48, 0, 0, 0]
    assert f(1 << 20, 1 << 22) == (1 << 14) * (1 << 20) * 8  # beyond 32 bits
    for r, k in ((1, 32), (7, 4096), (3, 288)):
        shape = beamc.mxfp4_scales_shape(r, k)
        assert shape[0] * shape[1] * shape[2] == f(r, k)


def test_quantize_and_dequantize(beamc):
    L = beamc.lib
    for f, first in ((L.beam_mxfp4_quantize, lambda x, q, s: (x, q, s)), (L.beam_mxfp4_dequantize, lambda x, q, s: (q, s, x))):
        def call(x=P, q=P, s=P, rows=4, K=64, dtype=F16):
            return f(*first(x, q, s), rows, K, dtype, None)
        refused(beamc, call(rows=-1), INVALID, "negative")
        refused(beamc, call(K=-32), INVALID, "negative")
        refused(beamc, call(K=48), INVALID, "blocks of 32")
        refused(beamc, call(K=(1 << 22) + 32), UNSUPPORTED, "beyond")
        refused(beamc, call(dtype=F32), UNSUPPORTED, "dtype")
        refused(beamc, call(rows=(1 << 31) - 1, K=1 << 22), UNSUPPORTED, "too many")
        refused(beamc, call(x=None), INVALID, "null")
        refused(beamc, call(q=None), INVALID, "null")
        refused(beamc, call(s=None), INVALID, "null")
        refused(beamc, call(x=P + 1), INVALID, "aligned")
        refused(beamc, call(q=P + 8), INVALID, "16 bytes")
        refused(beamc, call(s=P + 4), INVALID, "scales on 8")
        assert call(rows=0, x=None, q=None, s=None) == 0 and call(K=0, x=None) == 0


def test_products(beamc):
    L = beamc.lib
    need = L.beam_linear_mxfp4_workspace_bytes(100, 64)
    assert need >= 100 * 34 and need % 256 == 0
    assert L.beam_linear_mxfp4_workspace_bytes(16, 10240) == 0 == L.beam_linear_mxfp4_workspace_bytes(0, 64)
    assert L.beam_linear_mxfp4_workspace_bytes(17, 64) > 0 < L.beam_linear_mxfp4_workspace_bytes(1, 10272)

    def held(**kw):
        v = dict(a=P, sa=P, b=P, sb=P, c=P, M=100, N=8, K=64, dtype=F16)
        v.update(kw)
        return L.beam_gemmrc_mxfp4(*v.values(), None)

    def linear(**kw):
        v = dict(a=P, b=P, sb=P, c=P, M=100, N=8, K=64, dtype=F16, ws=P, bytes=need)
        v.update(kw)
        return L.beam_linear_mxfp4(*v.values(), None)

    for call in (held, linear):
        refused(beamc, call(M=-1), INVALID, "negative")
        refused(beamc, call(N=-1), INVALID, "negative")
        refused(beamc, call(K=40), INVALID, "blocks of 32")
        refused(beamc, call(dtype=F32), UNSUPPORTED, "dtype")
        for k in ("a", "b", "sb", "c"):
            refused(beamc, call(**{k: None}), INVALID, "null")
        refused(beamc, call(b=P + 8), INVALID, "16 bytes")
        refused(beamc, call(sb=P + 2), INVALID, "scales on 8")
        refused(beamc, call(c=P + 1), INVALID, "aligned")
        refused(beamc, call(M=1 << 30, N=1 << 30), UNSUPPORTED, "too large")
        assert call(M=0, a=None) == 0 and call(N=0, b=None) == 0
    refused(beamc, held(sa=None), INVALID, "null")
    refused(beamc, held(a=P + 1), INVALID, "16 bytes")
    refused(beamc, linear(a=P + 1), INVALID, "aligned")
    refused(beamc, linear(ws=None), WORKSPACE, "workspace")
    refused(beamc, linear(ws=P + 16), WORKSPACE, "workspace")
    refused(beamc, linear(bytes=need - 1), WORKSPACE, "workspace")


def test_overlaps(beamc):
    M, N, K = 100, 64, 64
    need = beamc.lib.beam_linear_mxfp4_workspace_bytes(M, K)
    sizes = {"x": M * K * 2, "a": M * K // 2, "sa": M * 8, "b": N * K // 2, "sb": N * 8, "c": M * N * 2, "ws": need}
    apart, at = {}, P
    for k, n in sizes.items():
        apart[k] = at
        at += (n + 511) // 256 * 256
    back = {k: apart[k] + sizes[k] - 8 for k in sizes}  # on 8 bytes, the last of what is there
    L = beamc.lib

    def quantize(**kw):
        v = {**apart, **kw}
        return L.beam_mxfp4_quantize(v["x"], v["a"], v["sa"], M, K, F16, None)

    def dequantize(**kw):
        v = {**apart, **kw}
        return L.beam_mxfp4_dequantize(v["a"], v["sa"], v["x"], M, K, F16, None)

    def product(**kw):
        v = {**apart, **kw}
        return L.beam_gemmrc_mxfp4(v["a"], v["sa"], v["b"], v["sb"], v["c"], M, N, K, F16, None)

    def linear(**kw):
        v = {**apart, **kw}
        return L.beam_linear_mxfp4(v["x"], v["b"], v["sb"], v["c"], M, N, K, F16, v["ws"], need, None)

    for call, out, others in ((quantize, "sa", ("x", "a")), (dequantize, "x", ("a", "sa")), (product, "c", ("a", "sa", "b", "sb")),
                              (linear, "c", ("x", "b", "sb", "ws"))):
        for k in others:
            refused(beamc, call(**{out: back[k]}), INVALID, "overlap")
    for k in ("x", "b", "sb"):
        refused(beamc, linear(**{k: apart["ws"]}), INVALID, "overlap")


def test_python_layer(beamc):
    class Fake(beamc.DeviceArray):
        def __init__(self, shape, dtype=F16, itemsize=2):
            self.shape, self.dtype, self.itemsize, self.ptr = shape, dtype, itemsize, 0

    def b(*shape):
        return Fake(shape, itemsize=1)

    def raises(text, f, *args):
        with pytest.raises(beamc.BeamError) as e:
            f(*args)
        assert text in str(e.value), e.value

    x, q, s = Fake((4, 288)), b(4, 144), b(2, 4, 8)
    raises("blocks of 32", beamc.mxfp4_quantize, Fake((4, 40)), b(4, 20), s)
    raises("one byte", beamc.mxfp4_quantize, x, Fake((4, 144)), s)
    raises("q has shape", beamc.mxfp4_quantize, x, b(4, 288), s)
    raises("scales has shape", beamc.mxfp4_quantize, x, q, b(4, 9))
    raises("must be 2-D", beamc.mxfp4_dequantize, q, s, Fake((4,)))
    c, w, ws = Fake((4, 6)), b(6, 144), b(2, 6, 8)
    raises("b has shape", beamc.gemmrc_mxfp4, q, s, b(6, 128), ws, c)
    raises("b's scales has shape", beamc.gemmrc_mxfp4, q, s, w, s, c)
    raises("c has shape", beamc.gemmrc_mxfp4, q, s, w, ws, Fake((6, 4)))
    raises("a must be 2-D", beamc.gemmrc_mxfp4, b(4), s, w, ws, c)
    raises("b has shape", beamc.linear_mxfp4, Fake((4, 256)), w, ws, c)
    raises("c must be", beamc.linear_mxfp4, x, w, ws, Fake((4, 6), 1))
    with pytest.raises(TypeError):
        beamc.gemmrc_mxfp4(q, s, w, None, c)
