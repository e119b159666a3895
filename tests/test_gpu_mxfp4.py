"""MXFP4 against its definition in float64 on the CPU: quantising (every bit pattern of a 16-bit value, exact), the values held
(every byte under every scale, exact) and products (every kind of tile, K tiles that end anywhere, operands between guards).

Bounds of the products, derived before the first run: the held values are exact on both sides; a sum of K products in fp32, in
any order, each addition off by at most one step: K 2^-23 sum |a| |b|; half a step of the type for the result (2^-11 of the
value in fp16, 2^-8 in bf16), and a smallest subnormal."""
import ctypes

import numpy as np
import pytest

from test_gpu_gated import BF16, F16, HALF_STEP, TINY, Guarded, f64

pytestmark = pytest.mark.gpu

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
NAN_SCALE = 255


class Bytes:
    """Bytes on the GPU with a guard on both sides."""
    GUARD = 512

    def __init__(self, beamc, content):
        self.out = not isinstance(content, np.ndarray)
        self.shape = content if self.out else content.shape
        self.n = int(np.prod(self.shape))
        host = np.full(self.n + 2 * self.GUARD, 0xAB if self.out else 0xFF, np.uint8)
        if not self.out:
            host[self.GUARD:self.GUARD + self.n] = content.ravel()
        self.fill = host[0]
        self.buf = beamc.DeviceArray.from_numpy(host)
        self.ptr = self.buf.ptr + self.GUARD

    def read(self):
        got = self.buf.to_numpy(np.uint8)
        assert (got[:self.GUARD] == self.fill).all() and (got[self.GUARD + self.n:] == self.fill).all(), "written outside"
        return got[self.GUARD:self.GUARD + self.n].reshape(self.shape)

    def free(self):
        self.buf.free()


def scales_shape(rows, K):
    return ((K + 255) // 256, rows, 8)


def to_tiles(biased, behind=0):
    """[rows, K / 32] -> the layout of the scales, with `behind` where there is no block."""
    rows, blocks = biased.shape
    out = np.full(((blocks + 7) // 8 * 8, rows), behind, np.uint8)
    out[:blocks] = biased.T
    return np.ascontiguousarray(out.reshape(-1, 8, rows).transpose(0, 2, 1))


def quantized(x):
    """Codes [rows, K] and biased exponents [rows, K / 32] of float64 values, by the definition."""
    rows, K = x.shape
    v = x.reshape(rows, K // 32, 32)
    with np.errstate(invalid="ignore"):
        top = np.abs(v).max(2)
    bad = ~np.isfinite(v).all(2)
    e = np.where(bad | (top == 0), -127, np.frexp(np.where(bad, 1.0, top))[1] - 1 - 2)
    e = np.maximum(e, -127)
    y = np.abs(np.where(bad[:, :, None], 0.0, v)) / 2.0 ** e[:, :, None].astype(np.float64)
    gap = np.abs(y[..., None] - LEVELS)
    near = gap.min(-1, keepdims=True) == gap
    # of two as near the one with an even code
    code = np.where(near[..., ::2].any(-1), 2 * near[..., ::2].argmax(-1), near.argmax(-1))
    code = np.where(y > 6, 7, code) + 8 * np.signbit(v)
    return code.reshape(rows, K).astype(np.uint8), np.where(bad, NAN_SCALE, e + 127).astype(np.uint8)


def packed(code):
    return code[:, 0::2] | code[:, 1::2] << 4


def held(code, biased):
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    rows, K = code.shape
    with np.errstate(over="ignore"):
        return (v.reshape(rows, K // 32, 32) * 2.0 ** (biased.astype(np.float64) - 127)[:, :, None]).reshape(rows, K)


def run_quantize(beamc, bits, dtype, offset=0):
    rows, K = bits.shape
    x = Guarded(beamc, bits, offset, dtype)
    q, s = Bytes(beamc, (rows, K // 2)), Bytes(beamc, scales_shape(rows, K))
    beamc._check(beamc.lib.beam_mxfp4_quantize(x.ptr, q.ptr, s.ptr, rows, K, dtype, None))
    out = q.read(), s.read()
    for t in (x, q, s):
        t.free()
    return out


def check_quantize(beamc, oracle, bits, dtype, offset=0):
    q, s = run_quantize(beamc, bits, dtype, offset)
    code, biased = quantized(f64(oracle, bits, dtype))
    assert (s == to_tiles(biased)).all()
    whole = np.repeat(biased != NAN_SCALE, 16, axis=1)  # bytes of blocks that are values
    assert (q == packed(code))[whole].all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_quantize_every_pattern(gpu, beamc, oracle, dtype):
    rng = np.random.default_rng(1)
    every = np.arange(65536, dtype=np.uint16)
    for order in (every, rng.permutation(every), rng.permutation(every & 0xBFFF)):  # neighbours in magnitude, and anything beside anything
        check_quantize(beamc, oracle, order.reshape(64, 1024), dtype)
    # every pattern as the smaller part of a block whose largest value is 1 to 8 times a power of two
    finite = every[np.isfinite(oracle.to_f32(every, dtype))]
    x = oracle.to_f32(finite, dtype).astype(np.float64)
    top = 2.0 ** np.clip(np.frexp(np.where(x == 0, 1.0, x))[1] + 1, -100 if dtype == BF16 else -14, 100 if dtype == BF16 else 14)
    block = np.repeat(finite[:, None], 32, 1)
    block[:, 5] = oracle.from_f32((top * 1.5).astype(np.float32), dtype)
    pad = (-len(block)) % 16
    block = np.concatenate([block, block[:pad]])
    check_quantize(beamc, oracle, np.ascontiguousarray(block.reshape(-1, 512)), dtype)


@pytest.mark.parametrize("rows,K", [(1, 32), (1, 4096), (3, 96), (33, 256), (31, 288), (70, 2016), (5, 8192), (1000, 64)])
def test_quantize_sizes(gpu, beamc, oracle, rows, K):
    for dtype, offset in ((F16, 0), (BF16, 1), (F16, 3)):
        bits = beamc.host_normal((rows, K), dtype, 11, rows + K, 0.0, 2.0)
        bits[rows // 2, :32] = 0
        check_quantize(beamc, oracle, bits, dtype, offset)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_dequantize_every_byte_and_scale(gpu, beamc, oracle, dtype):
    K = 512  # 256 bytes: every pair of codes
    code = np.stack([np.arange(256) & 15, np.arange(256) >> 4], 1).reshape(1, K).astype(np.uint8).repeat(256, 0)
    biased = np.arange(256, dtype=np.uint8)[:, None].repeat(K // 32, 1)
    q, s = Bytes(beamc, packed(code)), Bytes(beamc, to_tiles(biased))
    x = Guarded(beamc, (256, K), 1, dtype)
    beamc._check(beamc.lib.beam_mxfp4_dequantize(q.ptr, s.ptr, x.ptr, 256, K, dtype, None))
    got = x.read()
    with np.errstate(over="ignore"):
        want = oracle.from_f32(held(code, biased).astype(np.float32), dtype)
    assert (got[:255] == want[:255]).all()
    assert np.isnan(oracle.to_f32(got[255], dtype)).all()
    for t in (q, s, x):
        t.free()


def test_quantized_and_back(gpu, beamc, oracle):
    """What is read back is within half a step of the block's elements of what went in, and is held as it stands."""
    for dtype in (F16, BF16):
        bits = beamc.host_normal((37, 1056), dtype, 12, 0, 0.0, 3.0)
        q, s = run_quantize(beamc, bits, dtype)
        gq, gs, x = Bytes(beamc, q), Bytes(beamc, s), Guarded(beamc, bits.shape, 0, dtype)
        beamc._check(beamc.lib.beam_mxfp4_dequantize(gq.ptr, gs.ptr, x.ptr, *bits.shape, dtype, None))
        back = x.read()
        code, biased = quantized(f64(oracle, bits, dtype))
        assert (f64(oracle, back, dtype) == held(code, biased)).all()
        again = run_quantize(beamc, back, dtype)
        code2, biased2 = quantized(held(code, biased))
        assert (again[0] == packed(code2)).all() and (again[1] == to_tiles(biased2)).all()
        for t in (gq, gs, x):
            t.free()


# ---- products -------------------------------------------------------------------------------------


def operand(rng, rows, K):
    """Random codes and scales over a range in which no sum overflows fp16."""
    code = rng.integers(0, 16, (rows, K), dtype=np.uint8)
    biased = rng.integers(117, 124, (rows, K // 32), dtype=np.uint8)
    return code, biased


def check_product(oracle, A, B, got, dtype, what):
    want = A @ B.T
    bound = HALF_STEP[dtype] * np.abs(want) + A.shape[1] * 2.0 ** -23 * (np.abs(A) @ np.abs(B).T) + TINY[dtype]
    err = np.abs(f64(oracle, got, dtype) - want)
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:5].tolist(), float(np.nanmax(err)))


def run_product(beamc, a, b, dtype, offset=0, behind=0xFF):
    """behind: what lies in the scales behind the last block, which nobody may look at."""
    M, K = a[0].shape
    N = b[0].shape[0]
    bufs = [Bytes(beamc, x) for x in (packed(a[0]), to_tiles(a[1], behind), packed(b[0]), to_tiles(b[1], behind))]
    c = Guarded(beamc, (M, N), offset, dtype)
    beamc._check(beamc.lib.beam_gemmrc_mxfp4(*[t.ptr for t in bufs], c.ptr, M, N, K, dtype, None))
    got = c.read()
    for t in bufs + [c]:
        t.free()
    return got


# (rows, columns, kwave) of beam_dbg_mx_tile -> (M, N) that it names at K = 1024, for the walking kernel 4096
TILES = {
    (16, 16, 1): [(1, 1), (1, 300), (16, 4096), (77, 100)],
    (16, 32, 1): [(9, 4133), (200, 345)],
    (16, 64, 1): [(1, 9001), (16, 20000), (40, 4500)],
    (32, 32, 1): [(500, 493)],
    (32, 64, 1): [(500, 1003)],
    (64, 32, 1): [(9000, 20)],
    (64, 64, 0): [(135, 8316), (1433, 1383)],
    (64, 64, 3): [(1000, 1001), (1024, 1024), (33, 8532)],
    (128, 64, 3): [(68, 8403), (1080, 1100)],
    (128, 128, 0): [(263, 9967), (1780, 1781)],
    (128, 128, 3): [(409, 8215), (2060, 2070)],
    (256, 128, 0): [(399, 8292), (2053, 2060)],
    (256, 256, 0): [(1154, 7748), (7033, 1293)],
    (256, 256, 2): [(944, 8416), (7714, 1040), (8200, 4104)],
}


def tile_of(beamc, M, N, K):
    out = [ctypes.c_int() for _ in range(3)]
    beamc._check(beamc.lib.beam_dbg_mx_tile(M, N, K, *map(ctypes.byref, out)))
    return tuple(v.value for v in out)


def test_problems_reach_the_tiles_that_they_are_listed_under(gpu, beamc):
    for tile, problems in TILES.items():
        for M, N in problems:
            K = 4096 if tile in ((256, 128, 0), (256, 256, 2)) else 1024
            assert tile_of(beamc, M, N, K) == tile, (M, N, tile_of(beamc, M, N, K))


@pytest.mark.parametrize("tile", sorted(TILES), ids=lambda t: "x".join(map(str, t)))
@pytest.mark.parametrize("K", [32, 224, 256, 288, 544, 1024, 2016])
def test_product(gpu, beamc, oracle, tile, K):
    rng = np.random.default_rng(K)
    beamc.lib.beam_dbg_set_mx_tile(*tile)  # at every K, not only where it is the best
    try:
        for i, (M, N) in enumerate(TILES[tile]):
            if M * N > 1 << 22 and K > 1024 or tile[2] == 2 and K != 1024:
                continue  # (the walking kernel is for whole K tiles, three and more)
            dtype, offset = ((F16, 0), (BF16, 0 if tile[2] == 2 else 1))[(i + K // 32) % 2]
            a, b = operand(rng, M, K), operand(rng, N, K)
            assert tile_of(beamc, M, N, K) == tile
            got = run_product(beamc, a, b, dtype, offset)
            check_product(oracle, held(*a), held(*b), got, dtype, (tile, M, N, K, dtype))
    finally:
        beamc.lib.beam_dbg_set_mx_tile(0, 0, 0)


def test_product_of_nothing(gpu, beamc):
    c = Guarded(beamc, (3, 5))
    L = beamc.lib
    assert L.beam_gemmrc_mxfp4(None, None, None, None, c.ptr, 3, 5, 0, F16, None) == 0
    assert (c.read() == 0).all()
    assert L.beam_linear_mxfp4(None, None, None, c.ptr, 3, 5, 0, F16, None, 0, None) == 0
    assert L.beam_gemmrc_mxfp4(None, None, None, None, None, 0, 5, 32, F16, None) == 0
    c.free()


def test_extreme_scales(gpu, beamc, oracle):
    """Scales from end to end whose products are in range, and blocks that hold NaN: their row or column, and nothing else."""
    rng = np.random.default_rng(5)
    M, N, K = 70, 90, 320
    a, b = operand(rng, M, K), operand(rng, N, K)
    a[1][::2], b[1][:] = 250, 3  # 2^123 x 2^-124
    a[1][1::2] = 254 - 7
    check_product(oracle, held(*a), held(*b), run_product(beamc, a, b, BF16), BF16, "extreme")
    for M, N in ((70, 90), (2000, 2100)):
        a, b = operand(rng, M, K), operand(rng, N, K)
        clean = run_product(beamc, a, b, F16)
        a[1][7, 9] = b[1][3, 0] = NAN_SCALE
        nan = np.isnan(oracle.to_f32(run_product(beamc, a, b, F16), F16))
        got = run_product(beamc, a, b, F16)
        assert nan[7].all() and nan[:, 3].all() and nan.sum() == M + N - 1
        keep = ~nan
        assert (got[keep] == clean[keep]).all()


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 100])
def test_linear(gpu, beamc, oracle, M):
    L = beamc.lib
    for i, (N, K) in enumerate(((33, 32), (500, 288), (1003, 2016), (4200, 1024), (9000, 544), (40, 10240), (40, 10272))):
        dtype, offset = ((F16, 1), (BF16, 0))[(i + M) % 2]
        rng = np.random.default_rng(M + N)
        bits = beamc.host_normal((M, K), dtype, 13, i, 0.0, 1.0)
        bits[0, K // 2 - K // 2 % 32] = oracle.from_f32(np.float32([300.0]), dtype)[0]
        b = operand(rng, N, K)
        x, q, s, c = Guarded(beamc, bits, offset, dtype), Bytes(beamc, packed(b[0])), Bytes(beamc, to_tiles(b[1], 0xFF)), Guarded(beamc, (M, N), 1, dtype)
        need = L.beam_linear_mxfp4_workspace_bytes(M, K)
        assert (need == 0) == (M <= 16 and K <= 10240)
        ws = beamc.DeviceArray((need + 256,), itemsize=1)
        ws.fill_bytes(0xFF)
        beamc._check(L.beam_linear_mxfp4(x.ptr, q.ptr, s.ptr, c.ptr, M, N, K, dtype, ws.ptr if need else None, need, None))
        assert (ws.to_numpy(np.uint8)[need:] == 0xFF).all()
        got = c.read()
        a = quantized(f64(oracle, bits, dtype))
        check_product(oracle, held(*a), held(*b), got, dtype, (M, N, K, dtype))
        assert (run_product(beamc, a, b, dtype) == got).all(), "quantised first, the same bits"
        for t in (x, q, s, c, ws):
            t.free()


def test_linear_is_not_misled_by_a_named_tile(gpu, beamc, oracle):
    """beam_dbg_set_mx_tile names tiles for operands in MXFP4; 16-bit rows keep to those that take them."""
    M, N, K = 5, 300, 256
    bits = beamc.host_normal((M, K), BF16, 16, 0, 0.0, 1.0)
    b = operand(np.random.default_rng(4), N, K)
    x, q, s, c = Guarded(beamc, bits, 0, BF16), Bytes(beamc, packed(b[0])), Bytes(beamc, to_tiles(b[1])), Guarded(beamc, (M, N), 0, BF16)
    for tile in ((64, 64, 0), (32, 64, 1), (16, 16, 1), (16, 64, 1)):
        beamc.lib.beam_dbg_set_mx_tile(*tile)
        try:
            beamc._check(beamc.lib.beam_linear_mxfp4(x.ptr, q.ptr, s.ptr, c.ptr, M, N, K, BF16, None, 0, None))
        finally:
            beamc.lib.beam_dbg_set_mx_tile(0, 0, 0)
        check_product(oracle, held(*quantized(f64(oracle, bits, BF16))), held(*b), c.read(), BF16, tile)
    for t in (x, q, s, c):
        t.free()


def test_linear_of_a_token_with_a_nan(gpu, beamc, oracle):
    M, N, K = 3, 100, 512
    bits = beamc.host_normal((M, K), BF16, 14, 0, 0.0, 1.0)
    bits[1, 77], bits[2, 300] = 0x7FC0, 0xFF80  # a NaN, an infinity
    b = operand(np.random.default_rng(2), N, K)
    x, q, s, c = Guarded(beamc, bits, 0, BF16), Bytes(beamc, packed(b[0])), Bytes(beamc, to_tiles(b[1])), Guarded(beamc, (M, N), 0, BF16)
    beamc._check(beamc.lib.beam_linear_mxfp4(x.ptr, q.ptr, s.ptr, c.ptr, M, N, K, BF16, None, 0, None))
    nan = np.isnan(oracle.to_f32(c.read(), BF16))
    assert not nan[0].any() and nan[1:].all()
    for t in (x, q, s, c):
        t.free()


def test_elements_beyond_32_bits(gpu, beamc, oracle):
    """B of 2.3 GB: its last rows, and C behind 2^31 bytes, are where they belong."""
    M, N, K = 20, 70001, 65536
    L, chk = beamc.lib, beamc._check
    b, sb = beamc.DeviceArray((N, K // 2), itemsize=1), beamc.DeviceArray(scales_shape(N, K), itemsize=1)
    b.fill_bytes(0x22)   # 1.0 throughout
    sb.fill_bytes(127)
    last = np.full((1, K // 2), 0x44, np.uint8)  # 2.0 in the last row
    chk(L.beam_memcpy_h2d(b.ptr + (N - 1) * (K // 2), last.ctypes.data, K // 2))
    code, biased = operand(np.random.default_rng(3), M, K)
    biased[:] = 118
    a, sa, c = Bytes(beamc, packed(code)), Bytes(beamc, to_tiles(biased)), Guarded(beamc, (M, N), 0, BF16)
    chk(L.beam_gemmrc_mxfp4(a.ptr, sa.ptr, b.ptr, sb.ptr, c.ptr, M, N, K, BF16, None))
    got = f64(oracle, c.read(), BF16)
    sums = held(code, biased).sum(1, keepdims=True)
    bound = HALF_STEP[BF16] * np.abs(sums) + K * 2.0 ** -23 * np.abs(held(code, biased)).sum(1, keepdims=True)
    assert (np.abs(got[:, :-1] - sums) <= bound).all() and (np.abs(got[:, -1:] - 2 * sums) <= 2 * bound).all()
    for t in (a, sa, b, sb, c):
        t.free()


def test_served_layer_in_a_graph(gpu, beamc, oracle):
    """A feed-forward layer as it is served, gated projection in 16 bits and the second one in 4: captured, replayed with other
    tokens and eager calls in between."""
    L, chk = beamc.lib, beamc._check
    M, N, K = 24, 704, 320
    x = beamc.DeviceArray((M, K), BF16)
    w1 = beamc.DeviceArray.from_numpy(beamc.host_normal((2 * N, K), BF16, 15, 1, 0.0, K ** -0.5), BF16)
    w2_bits = beamc.host_normal((K, N), BF16, 15, 2, 0.0, N ** -0.5)
    w2 = beamc.DeviceArray.from_numpy(w2_bits, BF16)
    q, s = beamc.DeviceArray((K, N // 2), itemsize=1), beamc.DeviceArray(scales_shape(K, N), itemsize=1)
    beamc.mxfp4_quantize(w2, q, s)
    need = L.beam_linear_mxfp4_workspace_bytes(M, N)

    def results():
        return beamc.DeviceArray((M, N), BF16), beamc.DeviceArray((M, K), BF16), beamc.DeviceArray((need,), itemsize=1)

    def layer(r, stream):
        h, y, ws = r
        chk(L.beam_gemmrc_gated(x.ptr, w1.ptr, h.ptr, None, M, N, K, BF16, stream))
        chk(L.beam_linear_mxfp4(h.ptr, q.ptr, s.ptr, y.ptr, M, K, N, BF16, ws.ptr, need, stream))
        chk(L.beam_linear_mxfp4(h.ptr, q.ptr, s.ptr, y.ptr, 1, K, N, BF16, None, 0, stream))  # one token, over its own row

    mine, eager = results(), results()
    layer(mine, None)
    beamc.sync()
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    chk(L.beam_stream_create(ctypes.byref(stream)))
    chk(L.beam_graph_begin_capture(stream))
    layer(mine, stream)
    chk(L.beam_graph_end_capture(stream, ctypes.byref(graph)))
    for replay in range(4):
        host = beamc.host_normal((M, K), BF16, 40 + replay, 0, 0.0, 1.0)
        chk(L.beam_memcpy_h2d(x.ptr, host.ctypes.data, host.nbytes))
        for r in mine:
            r.fill_bytes(0xFF)
        chk(L.beam_graph_launch(graph, stream))
        chk(L.beam_sync(stream))
        layer(eager, None)
        beamc.sync()
        h, y = mine[0].to_numpy(), mine[1].to_numpy()
        assert (h == eager[0].to_numpy()).all() and (y == eager[1].to_numpy()).all(), replay
        check_product(oracle, held(*quantized(f64(oracle, h, BF16))), held(*quantized(f64(oracle, w2_bits, BF16))), y, BF16, replay)
    chk(L.beam_graph_destroy(graph))
    chk(L.beam_stream_destroy(stream))
