"""The gated layer, forward and backward, against float64 on the CPU: every kind of tile, rows on and off 16 bytes and 128-byte
lines, operands at any element's address inside buffers of NaNs, outputs inside buffers whose other bytes must stay.

Bounds, derived before the first run (e: half a step of the type relative to a value, 2^-11 fp16, 2^-8 bf16):
  * a sum of K products in fp32, in any order, each addition off by at most one step (2^-23): K 2^-23 sum |a| |b|;
  * G and U: that, and e of the value;
  * H = silu(G) U: |silu'| <= 1.1, so 1.1 dG |U| + |silu(G)| dU + 1.1 dG dU, 2^-18 of the value for the hardware's exp2 and
    reciprocal (its argument, up to 2^5 here, is off by 2^-24 of itself), e of the value, and a smallest subnormal;
  * dA and dB: the operands D are rounded to 16 bits, each by a part of e of its own that does not depend on the others, so that
    by Hoeffding's inequality their sum is beyond 8 e sqrt(sum D^2 B^2) with a probability below 2 e^-32; the sum itself in
    fp32; 2^-17 of D for exp2, reciprocal and five products, which may add up; e of the result."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F16, BF16 = 0, 1
HALF_STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F16: 2.0 ** -24, BF16: 2.0 ** -126}

# (rows, rows of B, kind) as in beam_dbg_gated_tile -> problems that are run on it
TILES = {
    (8, 32, 4): [(1, 8, 9), (3, 70, 200), (8, 333, 64), (1, 1, 8), (1, 4135, 12), (5, 4267, 64)],
    (16, 32, 4): [(9, 9, 15), (16, 300, 513), (10, 8, 64), (10, 4365, 10), (9, 4447, 64), (16, 5000, 200)],
    (16, 64, 4): [(40, 2700, 64), (37, 2125, 100)],
    (32, 32, 4): [(4144, 8, 13), (31, 4000, 64)],
    (32, 64, 4): [(4627, 17, 9), (17, 4167, 8), (19, 4697, 64)],
    (64, 32, 4): [(4469, 39, 17), (4193, 37, 64)],
    (64, 64, 4): [(34, 4497, 17), (34, 4128, 8), (35, 4294, 64)],
    (64, 64, 5): [(65, 2757, 1320)],
    (16, 32, 5): [(9, 9, 1736)],
    (16, 64, 5): [(37, 2125, 984)],
    (32, 32, 5): [(18, 2496, 1248)],
    (32, 64, 5): [(34, 2810, 992)],
    (64, 32, 5): [(926, 262, 840)],
    (64, 128, 0): [(70, 4112, 20), (69, 4297, 8), (83, 4097, 64)],
    (64, 128, 2): [(68, 4226, 282), (147, 2903, 850), (340, 1377, 768)],
    (64, 128, 3): [(105, 4682, 480)],
    (96, 128, 3): [(84, 4113, 424), (275, 1447, 1152)],
    (128, 128, 0): [(833, 2378, 22), (774, 2547, 8), (536, 3732, 64)],
    (128, 128, 2): [(1626, 611, 2404), (315, 3309, 1122), (715, 1380, 1152)],
    (160, 128, 3): [(1390, 1489, 144), (1827, 1090, 72), (398, 4726, 256)],
    (192, 128, 3): [(544, 4260, 480), (806, 1008, 960)],
    (192, 256, 0): [(4395, 948, 346), (1098, 3863, 344), (881, 4704, 384)],
    (224, 256, 0): [(1570, 3791, 122), (3592, 1699, 112), (2440, 2686, 128)],
    (256, 256, 0): [(3956, 1827, 164), (2246, 2957, 144), (2939, 2606, 192)],
    (256, 256, 1): [(1812, 3992, 192), (4096, 2048, 192), (3877, 1944, 192)],
    (256, 128, 0): [(1930, 1105, 1487), (1062, 2005, 1472)],
}
# ... -> problems that the library picks it for
PICKED = {
    (8, 32, 4): [(1, 4135, 12), (5, 4267, 64)],
    (16, 32, 4): [(10, 8, 64), (9, 4447, 64)],
    (16, 64, 4): [(40, 2700, 64), (37, 2125, 100)],
    (32, 32, 4): [(4144, 8, 13), (31, 4000, 64)],
    (32, 64, 4): [(4627, 17, 9), (17, 4167, 8), (19, 4697, 64)],
    (64, 32, 4): [(4469, 39, 17), (4193, 37, 64)],
    (16, 32, 5): [(9, 9, 1736)],
    (16, 64, 5): [(37, 2125, 984)],
    (32, 32, 5): [(18, 2496, 1248)],
    (32, 64, 5): [(34, 2810, 992)],
    (64, 32, 5): [(926, 262, 840)],
    (64, 64, 4): [(33, 4223, 10), (34, 4215, 8), (33, 4144, 64)],
    (64, 64, 5): [(34, 4216, 1360), (65, 2757, 1320)],
    (64, 128, 0): [(68, 4166, 9), (72, 4141, 8), (65, 4125, 64)],
    (64, 128, 2): [(68, 4226, 282), (69, 4102, 448)],
    (64, 128, 3): [(65, 4241, 464)],
    (96, 128, 3): [(4175, 194, 280), (275, 3447, 1152)],
    (128, 128, 0): [(4763, 403, 10), (404, 4687, 8), (386, 4677, 64)],
    (128, 128, 2): [(274, 3307, 2468), (4929, 261, 464), (4627, 195, 512)],
    (160, 128, 3): [(1827, 1090, 72), (398, 4726, 256)],
    (192, 128, 3): [(519, 4231, 480), (806, 3008, 960)],
    (192, 256, 0): [(781, 4771, 721), (772, 5022, 8), (4353, 898, 64)],
    (224, 256, 0): [(3935, 1035, 10), (1161, 4766, 8), (1190, 4723, 64)],
    (256, 128, 0): [(529, 3678, 327), (495, 4103, 280), (485, 4627, 640)],
    (256, 256, 0): [(4092, 1714, 130), (2033, 3252, 136), (1827, 3626, 256)],
    (256, 256, 1): [(4096, 11008, 4096)],
}


def row_starts(K):
    return 0 if K % 8 else 2 if K % 64 == 0 else 1


def tile_of(beamc, M, N, K):
    out = [ctypes.c_int() for _ in range(3)]
    beamc._check(beamc.lib.beam_dbg_gated_tile(M, N, K, row_starts(K), *map(ctypes.byref, out)))
    return tuple(v.value for v in out)


class Guarded:
    """16-bit elements on the GPU, `offset` elements behind a 256-byte boundary, with a guard on both sides: NaNs around an
    input, a pattern around an output that has to be there afterwards."""
    GUARD = 256

    def __init__(self, beamc, content, offset=0, dtype=F16):
        self.out = not isinstance(content, np.ndarray)
        self.shape = content if self.out else content.shape
        self.n = int(np.prod(self.shape))
        self.at = self.GUARD + offset
        host = np.full(self.n + 2 * self.GUARD + offset, 0xABCD if self.out else 0xFFFF, np.uint16)
        if not self.out:
            host[self.at:self.at + self.n] = content.ravel()
        self.host = host
        self.buf = beamc.DeviceArray.from_numpy(host, dtype)
        self.ptr = self.buf.ptr + 2 * self.at

    def read(self):
        got = self.buf.to_numpy()
        rest = np.concatenate([got[:self.at], got[self.at + self.n:]])
        assert (rest == (0xABCD if self.out else 0xFFFF)).all(), "written outside"
        return got[self.at:self.at + self.n].reshape(self.shape)

    def free(self):
        self.buf.free()


def inputs(beamc, M, N, K, dtype, seed=7):
    a = beamc.host_normal((M, K), dtype, seed, 0, 0.0, 1.0)
    b = beamc.host_normal((2 * N, K), dtype, seed, 1, 0.0, max(K, 1) ** -0.5)
    return a, b


def f64(oracle, bits, dtype):
    return oracle.to_f32(bits, dtype).astype(np.float64)


def sigmoid(x):
    return 1 / (1 + np.exp(-x))


def check_forward(oracle, a, b, h, gu, dtype, what):
    A, B = f64(oracle, a, dtype), f64(oracle, b, dtype)
    N, K, e = B.shape[0] // 2, A.shape[1], HALF_STEP[dtype]
    want = A @ B.T
    d = K * 2.0 ** -23 * (np.abs(A) @ np.abs(B).T)
    if gu is not None:
        err = np.abs(f64(oracle, gu, dtype) - want)
        assert (err <= e * np.abs(want) + d * (1 + e) + TINY[dtype]).all(), (what, "gu", np.nanmax(err))
        assert not np.isnan(err).any()
    G, U, dG, dU = want[:, :N], want[:, N:], d[:, :N], d[:, N:]
    H = G * sigmoid(G) * U
    bound = (e + 2.0 ** -18) * np.abs(H) + (1 + e) * (1.1 * dG * np.abs(U) + np.abs(G * sigmoid(G)) * dU + 1.1 * dG * dU) + TINY[dtype]
    err = np.abs(f64(oracle, h, dtype) - H)
    bad = ~(err <= bound)
    assert not bad.any(), (what, "h", int(bad.sum()), np.argwhere(bad)[:5].tolist(), float(np.nanmax(err)))


def run_forward(beamc, a, b, dtype, offsets=(0, 0, 0, 0), train=True):
    M, K = a.shape
    N = b.shape[0] // 2
    ga, gb = Guarded(beamc, a, offsets[0], dtype), Guarded(beamc, b, offsets[1], dtype)
    gh, gg = Guarded(beamc, (M, N), offsets[2], dtype), Guarded(beamc, (M, 2 * N), offsets[3], dtype)
    beamc._check(beamc.lib.beam_gemmrc_gated(ga.ptr, gb.ptr, gh.ptr, gg.ptr if train else None, M, N, K, dtype, None))
    h, gu = gh.read(), gg.read()
    if not train:
        assert (gu == 0xABCD).all()
    for t in (ga, gb, gh, gg):
        t.free()
    return h, (gu if train else None)


def test_the_library_picks_every_tile(gpu, beamc):
    assert set(PICKED) == set(TILES)
    for tile, problems in PICKED.items():
        for M, N, K in problems:
            assert tile_of(beamc, M, N, K) == tile, (M, N, K)


@pytest.mark.parametrize("tile", sorted(TILES), ids=lambda t: "x".join(map(str, t)))
def test_forward(gpu, beamc, oracle, tile):
    beamc.lib.beam_dbg_set_gated_tile(*tile)
    try:
        for i, (M, N, K) in enumerate(TILES[tile]):
            assert tile_of(beamc, M, N, K) == tile
            dtype = (F16, BF16)[i % 2]
            a, b = inputs(beamc, M, N, K, dtype)
            h, gu = run_forward(beamc, a, b, dtype)
            check_forward(oracle, a, b, h, gu, dtype, (tile, M, N, K, dtype))
            again, _ = run_forward(beamc, a, b, dtype, train=False)
            assert (again == h).all(), "h depends on whether gu is asked for"
            other = 1 - dtype
            a, b = inputs(beamc, M, N, K, other)
            h, gu = run_forward(beamc, a, b, other, offsets=(1, 3, 8, 16) if tile[2] == 1 else (1, 3, 1, 5) if i % 2 else (8, 24, 2, 4))
            check_forward(oracle, a, b, h, gu, other, (tile, M, N, K, other, "anywhere"))
    finally:
        beamc.lib.beam_dbg_set_gated_tile(0, 0, 0)


@pytest.mark.parametrize("K", [1, 2, 7])
def test_forward_of_short_sums(gpu, beamc, oracle, K):
    a, b = inputs(beamc, 37, 51, K, BF16)
    h, gu = run_forward(beamc, a, b, BF16, offsets=(1, 1, 1, 1))
    check_forward(oracle, a, b, h, gu, BF16, K)


def test_forward_of_nothing(gpu, beamc):
    h, gu = run_forward(beamc, np.zeros((5, 0), np.uint16), np.zeros((14, 0), np.uint16), F16)
    assert (h == 0).all() and (gu == 0).all()
    L = beamc.lib
    assert L.beam_gemmrc_gated(None, None, None, None, 0, 8, 8, F16, None) == 0
    assert L.beam_gemmrc_gated(None, None, None, None, 8, 0, 8, F16, None) == 0


def test_forward_keeps_signs_and_large_values(gpu, beamc, oracle):
    """silu far out on both sides; a factor that fp16 cannot hold is infinite in gu and still right in h, where h fits."""
    K = 64
    a = np.zeros((4, K), np.float32)
    a[:, 0] = [200.0, -200.0, 30.0, -30.0]
    b = np.zeros((2 * 16, K), np.float32)
    b[:16, 0] = 400.0   # gate: 80000 is beyond fp16
    b[16:, 0] = np.linspace(-1, 1, 16) * 2.0 ** -9
    bits = lambda x: oracle.from_f32(x.astype(np.float32), F16)
    a16, b16 = bits(a), bits(b)
    h, gu = run_forward(beamc, a16, b16, F16)
    want = f64(oracle, a16, F16) @ f64(oracle, b16, F16).T
    G, U = want[:, :16], want[:, 16:]
    H = np.where(G < -100, 0.0, G) * U
    got = f64(oracle, h, F16)
    assert np.isfinite(got).all() and (np.abs(got - H) <= 2.0 ** -10 * np.abs(H) + 2.0 ** -24).all()
    assert np.isposinf(oracle.to_f32(gu, F16)[0, :16]).all() and np.isneginf(oracle.to_f32(gu, F16)[1, :16]).all()


def test_a_row_of_nans_stays_in_its_row(gpu, beamc, oracle):
    for M, N, K in ((33, 100, 200), (700, 1500, 96)):
        a, b = inputs(beamc, M, N, K, F16)
        clean, _ = run_forward(beamc, a, b, F16)
        a[M // 2] = 0x7E00
        b2 = b.copy()
        b2[N + 3] = 0x7E00  # an up row: column 3
        h, gu = run_forward(beamc, a, b2, F16)
        nan = np.isnan(oracle.to_f32(h, F16))
        assert nan[M // 2].all() and nan[:, 3].all()
        nan[M // 2], nan[:, 3] = False, False
        assert not nan.any()
        keep = np.ones((M, N), bool)
        keep[M // 2], keep[:, 3] = False, False
        assert (h[keep] == clean[keep]).all()


# ---- backward ------------------------------------------------------------------------------------


def run_backward(beamc, dh, gu, a, b, dtype, offsets=(0,) * 6, want=(True, True)):
    M, K = a.shape
    N = b.shape[0] // 2
    ins = [Guarded(beamc, x, o, dtype) for x, o in zip((dh, gu, a, b), offsets)]
    da, db = Guarded(beamc, (M, K), offsets[4], dtype), Guarded(beamc, (2 * N, K), offsets[5], dtype)
    need = beamc.lib.beam_gemmrc_gated_backward_workspace_bytes(M, N, K, *want)
    ws = beamc.DeviceArray((need + 256,), itemsize=1)
    ws.fill_bytes(0xFF)
    beamc._check(beamc.lib.beam_gemmrc_gated_backward(*[t.ptr for t in ins], da.ptr if want[0] else None, db.ptr if want[1] else None,
                                                       M, N, K, dtype, ws.ptr, need, None))
    assert (ws.to_numpy(np.uint8)[need:] == 0xFF).all()
    out = da.read(), db.read()
    for t in ins + [da, db, ws]:
        t.free()
    return out


def gradients(oracle, dh, gu, dtype):
    """D in float64."""
    d, g = f64(oracle, dh, dtype), f64(oracle, gu, dtype)
    N = d.shape[1]
    G, U = g[:, :N], g[:, N:]
    s = sigmoid(G)
    return np.concatenate((d * U * s * (1 + G * (1 - s)), d * G * s), 1)


def check_products(D, B, got, e, tiny, what):
    """got = D @ B with D rounded to 16 bits in between."""
    want = D @ B
    bound = (8 * e * np.sqrt((D * D) @ (B * B)) + (D.shape[1] * 2.0 ** -23 + 2.0 ** -17) * (np.abs(D) @ np.abs(B))) * (1 + e)
    bound += e * np.abs(want) + tiny * (1 + np.abs(B).sum(0))
    err = np.abs(got - want)
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:5].tolist(), float(np.nanmax(err)))


def backward_inputs(beamc, M, N, K, dtype, seed=8):
    a, b = inputs(beamc, M, N, K, dtype, seed)
    return beamc.host_normal((M, N), dtype, seed, 2, 0.0, 0.5), beamc.host_normal((M, 2 * N), dtype, seed, 3, 0.0, 1.5), a, b


BACKWARD = [(1, 1, 1), (1, 1, 8), (1, 300, 200), (7, 9, 5), (64, 64, 64), (65, 63, 72), (200, 333, 130), (129, 500, 257), (512, 256, 640),
            (1000, 72, 96), (77, 1030, 333), (1001, 501, 500)]


@pytest.mark.parametrize("M,N,K", BACKWARD)
def test_backward(gpu, beamc, oracle, M, N, K):
    for dtype, offsets in ((F16, (0,) * 6), (BF16, (1, 3, 5, 7, 1, 3))):
        dh, gu, a, b = backward_inputs(beamc, M, N, K, dtype)
        da, db = run_backward(beamc, dh, gu, a, b, dtype, offsets)
        D = gradients(oracle, dh, gu, dtype)
        e, tiny = HALF_STEP[dtype], TINY[dtype]
        check_products(D, f64(oracle, b, dtype), f64(oracle, da, dtype), e, tiny, ("da", M, N, K, dtype))
        check_products(D.T, f64(oracle, a, dtype), f64(oracle, db, dtype), e, tiny, ("db", M, N, K, dtype))
        only_a = run_backward(beamc, dh, gu, a, b, dtype, offsets, (True, False))
        only_b = run_backward(beamc, dh, gu, a, b, dtype, offsets, (False, True))
        assert (only_a[0] == da).all() and (only_b[1] == db).all()
        assert (only_a[1] == 0xABCD).all() and (only_b[0] == 0xABCD).all()


def test_backward_against_differences(gpu, beamc, oracle):
    """What the layer's sum of dh * h changes by along a direction, by central differences in float64, and what the gradients
    that came from the forward call's own gu say."""
    M, N, K, dtype = 130, 150, 96, F16
    e = HALF_STEP[dtype]
    a, b = inputs(beamc, M, N, K, dtype, 9)
    dh = beamc.host_normal((M, N), dtype, 9, 2, 0.0, 0.5)
    _, gu = run_forward(beamc, a, b, dtype)
    da, db = run_backward(beamc, dh, gu, a, b, dtype)
    A, B, W = f64(oracle, a, dtype), f64(oracle, b, dtype), f64(oracle, dh, dtype)

    def loss(x, y):
        z = x @ y.T
        return float((W * z[:, :N] * sigmoid(z[:, :N]) * z[:, N:]).sum())

    rng = np.random.default_rng(3)
    for which in range(4):
        va = rng.standard_normal(A.shape) * (which != 1)
        vb = rng.standard_normal(B.shape) * (which != 0) * K ** -0.5
        t = 1e-4
        slope = (loss(A + t * va, B + t * vb) - loss(A - t * va, B - t * vb)) / (2 * t)
        got = float((f64(oracle, da, dtype) * va).sum() + (f64(oracle, db, dtype) * vb).sum())
        # gu, D and the results are rounded, each value by a part of e of its own: independent parts, eight times their root sum
        # of squares (|d^2 h| <= 1.1 |U| + 1 per unit of either factor), and the differences' own t^2 |third derivative|
        D = gradients(oracle, dh, gu, dtype)
        Z = A @ B.T
        spread = np.abs(W) * (1.1 * np.abs(Z[:, N:]) + 1.1) * e
        per_z = np.concatenate((spread * np.abs(Z[:, :N]), spread * np.abs(Z[:, N:])), 1) + e * np.abs(D)
        move = np.abs(va @ B.T + A @ vb.T)
        rough = np.sqrt(((per_z * move) ** 2).sum() * 2)
        rough += e * np.sqrt(((f64(oracle, da, dtype) * va) ** 2).sum() + ((f64(oracle, db, dtype) * vb) ** 2).sum())
        assert abs(got - slope) <= 8 * rough + 1e-4 * abs(slope), (which, got, slope, rough)
        assert 8 * rough < 0.2 * np.sqrt((f64(oracle, da, dtype) ** 2).sum() * (va ** 2).mean() + (f64(oracle, db, dtype) ** 2).sum() * (vb ** 2).mean()), "the test can tell"


def test_backward_of_nothing(gpu, beamc):
    none = np.zeros((0, 6), np.uint16)
    _, db = run_backward(beamc, none[:, :3], none, np.zeros((0, 5), np.uint16), np.ones((6, 5), np.uint16), F16)
    assert (db == 0).all()  # no tokens: an empty sum
    da, _ = run_backward(beamc, np.zeros((4, 0), np.uint16), np.zeros((4, 0), np.uint16), np.ones((4, 5), np.uint16), np.zeros((0, 5), np.uint16), F16)
    assert (da == 0).all()


def test_backward_far_out(gpu, beamc, oracle):
    """Large and very negative gates: the slope is 1 or 0, nothing is NaN."""
    M, N, K = 16, 16, 16
    g = np.zeros((M, 2 * N), np.float32)
    g[:, :N] = np.linspace(-60000, 60000, N)
    g[:, N:] = 1.0
    gu = oracle.from_f32(g, F16)
    dh = oracle.from_f32(np.full((M, N), 2.0 ** -12, np.float32), F16)
    eye = oracle.from_f32(np.vstack([np.eye(16, dtype=np.float32)] * 2), F16)  # da = dg + du
    da, db = run_backward(beamc, dh, gu, oracle.from_f32(np.eye(16, dtype=np.float32), F16), eye, F16)
    D = gradients(oracle, dh, gu, F16)
    got = f64(oracle, da, F16)
    assert np.abs(got - (D[:, :N] + D[:, N:])).max() <= 2 * HALF_STEP[F16] * 15
    assert np.isfinite(got).all() and (f64(oracle, db, F16)[:8] == 0).all()


def test_graph_of_a_training_step(gpu, beamc):
    """Forward and backward captured once, replayed with new inputs and eager calls in between, each with workspace of its own."""
    L, chk = beamc.lib, beamc._check
    M, N, K = 203, 310, 264
    a, b, dh = (beamc.DeviceArray(s, BF16) for s in ((M, K), (2 * N, K), (M, N)))
    need = L.beam_gemmrc_gated_backward_workspace_bytes(M, N, K, 1, 1)

    def results():
        return [beamc.DeviceArray(s, BF16) for s in ((M, N), (M, 2 * N), (M, K), (2 * N, K))] + [beamc.DeviceArray((need,), itemsize=1)]

    def step(r, stream):
        h, gu, da, db, ws = r
        chk(L.beam_gemmrc_gated(a.ptr, b.ptr, h.ptr, gu.ptr, M, N, K, BF16, stream))
        chk(L.beam_gemmrc_gated_backward(dh.ptr, gu.ptr, a.ptr, b.ptr, da.ptr, db.ptr, M, N, K, BF16, ws.ptr, need, stream))

    mine, eager = results(), results()
    step(mine, None)
    beamc.sync()
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    chk(L.beam_stream_create(ctypes.byref(stream)))
    chk(L.beam_graph_begin_capture(stream))
    step(mine, stream)
    chk(L.beam_graph_end_capture(stream, ctypes.byref(graph)))
    for replay in range(4):
        for d, i, scale in ((a, 0, 1.0), (b, 1, K ** -0.5), (dh, 2, 0.5)):
            host = beamc.host_normal(d.shape, BF16, 30 + replay, i, 0.0, scale)
            chk(L.beam_memcpy_h2d(d.ptr, host.ctypes.data, host.nbytes))
        for r in mine:
            r.fill_bytes(0xFF)
        chk(L.beam_graph_launch(graph, stream))
        chk(L.beam_sync(stream))
        step(eager, None)
        beamc.sync()
        for x, y in zip(mine[:4], eager[:4]):
            assert (x.to_numpy() == y.to_numpy()).all(), replay
    chk(L.beam_graph_destroy(graph))
    chk(L.beam_stream_destroy(stream))


def test_backward_of_infinities_in_the_last_row(gpu, beamc, oracle):
    """The last row's gradients are not finite: they reach its row of da and all of db's rows that they belong to, and nothing
    comes from behind the last row, which is a whole line of the workspace away."""
    M, N, K = 70, 40, 64
    dh, gu, a, b = backward_inputs(beamc, M, N, K, F16)
    clean = run_backward(beamc, dh, gu, a, b, F16)
    gu2 = gu.copy()
    gu2[M - 1, N + 5] = 0x7C00  # u of column 5 is infinite: dg of column 5 is, in the last row
    da, db = run_backward(beamc, dh, gu2, a, b, F16)
    bad = ~np.isfinite(oracle.to_f32(da, F16))
    assert bad[M - 1].all() and not bad[:M - 1].any() and (da[:M - 1] == clean[0][:M - 1]).all()
    bad = ~np.isfinite(oracle.to_f32(db, F16))
    assert bad[5].all() and bad.sum() == K
    keep = np.arange(2 * N) != 5
    assert (db[keep] == clean[1][keep]).all()


@pytest.mark.parametrize("rows,slices", [(64, 2), (64, 7), (128, 3), (128, 16)])
@pytest.mark.parametrize("M,N,K", [(1, 65, 8), (65, 63, 72), (200, 333, 136), (777, 256, 320), (1001, 501, 504), (1, 65, 9), (65, 63, 75), (200, 333, 137),
                                   (777, 256, 318), (1001, 501, 503), (129, 64, 12)])
def test_backward_in_slices(gpu, beamc, oracle, rows, slices, M, N, K):
    """Sums cut into slices, whatever the problem: more than there are K tiles, and a last one that is short."""
    beamc.lib.beam_dbg_set_nn_split(rows, slices)
    try:
        for dtype, offsets in ((F16, (0,) * 6), (BF16, (1, 3, 5, 7, 1, 3))):
            dh, gu, a, b = backward_inputs(beamc, M, N, K, dtype)
            da, db = run_backward(beamc, dh, gu, a, b, dtype, offsets)
            D = gradients(oracle, dh, gu, dtype)
            check_products(D, f64(oracle, b, dtype), f64(oracle, da, dtype), HALF_STEP[dtype], TINY[dtype], ("da", M, N, K, dtype))
            check_products(D.T, f64(oracle, a, dtype), f64(oracle, db, dtype), HALF_STEP[dtype], TINY[dtype], ("db", M, N, K, dtype))
    finally:
        beamc.lib.beam_dbg_set_nn_split(-1, 0)


def test_backward_of_a_few_tokens_through_a_wide_layer(gpu, beamc, oracle):
    """What the library cuts into slices by itself; the same bits again."""
    for M, N, K in ((3, 4100, 264), (130, 2200, 136)):
        dh, gu, a, b = backward_inputs(beamc, M, N, K, BF16)
        da, db = run_backward(beamc, dh, gu, a, b, BF16)
        D = gradients(oracle, dh, gu, BF16)
        check_products(D, f64(oracle, b, BF16), f64(oracle, da, BF16), HALF_STEP[BF16], TINY[BF16], ("da", M, N, K))
        check_products(D.T, f64(oracle, a, BF16), f64(oracle, db, BF16), HALF_STEP[BF16], TINY[BF16], ("db", M, N, K))
        again = run_backward(beamc, dh, gu, a, b, BF16)
        assert (again[0] == da).all() and (again[1] == db).all()


def test_walking_tiles_of_several_rounds(gpu, beamc, oracle):
    """More 256 x 256 tiles than twice the CUs: every workgroup carries its sums through several tile boundaries."""
    M, N, K = 6147, 2920, 320
    beamc.lib.beam_dbg_set_gated_tile(256, 256, 1)
    try:
        assert tile_of(beamc, M, N, K) == (256, 256, 1)
        a, b = inputs(beamc, M, N, K, BF16)
        h, gu = run_forward(beamc, a, b, BF16)
        check_forward(oracle, a, b, h, gu, BF16, (M, N, K))
        assert (run_forward(beamc, a, b, BF16, train=False)[0] == h).all()
        # outputs off 16 bytes, and K tiles that are not whole: not that kernel's
        h, gu = run_forward(beamc, a[:300], b, BF16, offsets=(0, 0, 1, 0))
        check_forward(oracle, a[:300], b, h, gu, BF16, "off 16 bytes")
    finally:
        beamc.lib.beam_dbg_set_gated_tile(0, 0, 0)
