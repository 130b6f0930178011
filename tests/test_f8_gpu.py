"""GPU parity of the 8-bit operators (f8_pack, f8_norm, f8_rows, f8_gemm) with their CPU restatement.

Packed weights and ungated rows are exact: scales and codes are fp32 operations with one result each. Elsewhere the bounds count
roundings, u = 2^-24 an fp32 one, for each value by itself:
 * a code stands for a value within half a step, 2^-4 of it, or s 2^-10 below the least normal code (2^-6 s);
 * gated values: exp2 of an argument rounded to fp32 (|z| log2 e 2^-24, z up to 40 here), the exponential, a sum, a quotient, two
   products and z's own four roundings: (60 + 60 + 10) u < 2^-16 of the value;
 * a norm: sums of up to 2^15 squares in fp32, each lane's in order, 8 to 40 of them, then up to 22 levels: 62 u, halved by the
   root, the mean of an LN likewise 62 u of the mean magnitude, and 10 roundings a value: 2^-17 of the value and 2^-17 of the
   row's mean magnitude times rstd |g|; a t that is normalised first is within 2^-18 of itself;
 * a product: sums of 128 products inside the matrix instructions (at most one rounding or cut of 2^-23 each), one fma per block:
   (128 + 2 K / 128) 2^-23 of the sum of magnitudes; then one rounding to the type. 16-bit results of many rows are taken on the
   8-bit instruction: of each 8 consecutive k, 7 products may each lose up to 2^-13 of the largest one's leading bit.
"""
import numpy as np
import pytest

from oracle import f8
from p0pc0rn_amd import capi
from tests.test_kv_gpu import from_type, size_of, to_type

pytestmark = pytest.mark.gpu
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step, relative
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}
FILL = 0xA5


class Rows:
    """a device matrix of `n` rows of `width` values, `ld` apart, with bytes around and between that must stay as they are"""

    def __init__(self, dtype, n, width, ld=None, raw=None, lead=64):
        self.dtype, self.n, self.width, self.ld = np.dtype(dtype), n, width, ld or width
        self.lead = lead
        self.host = np.full(lead + (n * self.ld + 64) * self.dtype.itemsize, FILL, np.uint8)
        if raw is not None:
            self.view(self.host)[:] = raw
        self.buf = capi.to_device(self.host)
        self.ptr = self.buf.ptr + lead

    def view(self, host):
        flat = host[self.lead:self.lead + self.n * self.ld * self.dtype.itemsize].view(self.dtype)
        return flat.reshape(self.n, self.ld)[:, :self.width]

    def read(self):
        now = self.buf.read(np.uint8, self.host.size)
        kept = self.host.copy()
        self.view(kept)[:] = self.view(now)
        assert np.array_equal(kept, now), "written past its rows"
        return self.view(now).copy()

    def free(self):
        self.buf.free()


RAW = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


def values_in(type_, x, ld=None, lead=64):
    raw, v = to_type(x, type_)
    return Rows(RAW[type_], x.shape[0], x.shape[1], ld, raw, lead), v


def activations(rng, M, D, sigma=1.0):
    x = rng.standard_normal((M, D)) * np.exp(0.7 * rng.standard_normal((1, D))) * sigma
    return x.astype(np.float32)


def codes_near(codes, s, want, slack):
    """codes and scales against values in float64, `slack` their own possible error; the scale is the largest magnitude's"""
    M, D = want.shape
    v = f8.values(codes, s)
    assert not codes[:, D:].any(), "padding"
    full, sl = f8.padded(want), f8.padded(np.broadcast_to(slack, want.shape))
    most = np.abs(full).reshape(M, -1, 128).max(2)
    err = sl.reshape(M, -1, 128).max(2)
    assert (np.abs(s.T.astype(np.float64) * 448 - np.maximum(most, 448 * 2.0 ** -126)) <= err + 2.0 ** -22 * most + 2.0 ** -140).all(), "scales"
    step = np.maximum(2.0 ** -4 * (np.abs(full) + sl) * (1 + 2.0 ** -20), np.repeat(s.T.astype(np.float64), 128, 1) * 2.0 ** -10 * (1 + 2.0 ** -20))
    bad = np.abs(v - full) > step + sl
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:3], v[bad][:3], full[bad][:3])


# ------------------------------------------------------------------------------------------------ weights
@pytest.mark.parametrize("N,K", [(1, 1), (1, 128), (127, 129), (128, 128), (129, 255), (300, 1000), (16, 2048), (513, 384)])
@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
def test_pack(dev, N, K, type_):
    rng = np.random.default_rng(N * 7 + K)
    x = (0.05 * rng.standard_normal((N, K)) * np.exp(rng.standard_normal((N, 1)))).astype(np.float32)
    if N > 2 and K > 2:
        x[1, 2], x[2, 1], x[0, 0] = np.inf, np.nan, -np.inf
    if N > 200:
        x[128:256] = 0
    K8 = 128 * f8.blocks(K)
    for ldx, ldw, lds, lead in ((None, None, None, 64), (K + 3, K8 + 32, f8.blocks(K) + 1, 64), (K + 8, None, None, 64 + size_of(type_))):
        xr, v = values_in(type_, x, ldx, lead)
        w, s = Rows(np.uint8, N, K8, ldw), Rows(np.float32, f8.blocks(N), f8.blocks(K), lds)
        capi.f8_pack(capi.f8_pack_args(x=xr.ptr, ldx=ldx or 0, type=capi.TYPE[type_], N=N, K=K, w=w.ptr, ldw=ldw or 0, s=s.ptr, lds=lds or 0))
        wc, ws = f8.pack(v.astype(np.float32))
        got, gs = w.read(), s.read()
        assert np.array_equal(gs, ws)
        nan = np.isnan(f8.VALUES[wc])
        assert np.array_equal(np.isnan(f8.VALUES[got]), nan) and np.array_equal(got[~nan], wc[~nan])
        xr.read()
        for r in (xr, w, s):
            r.free()


# ------------------------------------------------------------------------------------------------ activations
@pytest.mark.parametrize("M,D", [(1, 1), (1, 8192), (3, 65), (5, 128), (17, 1000), (64, 136), (300, 72), (1021, 520), (4, 6144), (2100, 2056)])
@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
def test_rows(dev, M, D, type_):
    rng = np.random.default_rng(M * 7 + D)
    x = activations(rng, M, D)
    x[M // 2] = 0
    if M > 2:
        x[0, D // 3], x[1, 0] = np.nan, -np.inf
    K8 = 128 * f8.blocks(D)
    for ldx, ldy, lds, lead in ((None, None, None, 64), (D + 5, K8 + 16, M + 3, 64 + size_of(type_))):
        xr, v = values_in(type_, x, ldx, lead)
        y, s = Rows(np.uint8, M, K8, ldy), Rows(np.float32, f8.blocks(D), M, lds)
        capi.f8_rows(capi.f8_rows_args(x=xr.ptr, ldx=ldx or 0, type=capi.TYPE[type_], M=M, D=D, y=y.ptr, ldy=ldy or 0, s=s.ptr, lds=lds or 0))
        wc, ws = f8.quantise(v.astype(np.float32))
        got, gs = y.read(), s.read()
        assert np.array_equal(gs, ws)
        nan = np.isnan(f8.VALUES[wc])
        assert np.array_equal(np.isnan(f8.VALUES[got]), nan) and np.array_equal(got[~nan], wc[~nan])
        for r in (xr, y, s):
            r.free()


@pytest.mark.parametrize("glu", ["silu", "gelu"])
@pytest.mark.parametrize("M,D,up", [(1, 8192, 0), (1, 1, 0), (5, 100, 128), (64, 136, 0), (257, 1000, 1008), (2100, 1536, 0)])
@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
def test_gated_rows(dev, glu, M, D, up, type_):
    rng = np.random.default_rng(M * 7 + D)
    x = activations(rng, M, (up or D) + D, 2.0)
    x[:, :D] = np.clip(x[:, :D], -6, 6) if glu == "gelu" else np.clip(x[:, :D], -40, 40)   # z up to 40 (gelu: 1.6 (6 + 0.045 216) = 25)
    xr, v = values_in(type_, x)
    y, s = Rows(np.uint8, M, 128 * f8.blocks(D)), Rows(np.float32, f8.blocks(D), M)
    capi.f8_rows(capi.f8_rows_args(x=xr.ptr, type=capi.TYPE[type_], glu=capi.GLU[glu], up=up, M=M, D=D, y=y.ptr, s=s.ptr))
    want = f8.glu(glu, v[:, :D], v[:, (up or D):])
    codes_near(y.read(), s.read(), want, 2.0 ** -16 * np.abs(want))
    for r in (xr, y, s):
        r.free()


def test_gates_far_from_zero(dev):
    """exp's ends: a gate far below zero gives zero, far above it passes its partner on; infinities as the formula has them"""
    g = np.float32([[-1e30, -200, -104, -88, 88, 104, 200, 1e30] + [1.0] * 120])
    x = np.concatenate([g, np.full((1, 128), 0.5, np.float32)], 1)
    for glu in ("silu", "gelu"):
        xr, _ = values_in("f32", x)
        y, s = Rows(np.uint8, 1, 128), Rows(np.float32, 1, 1)
        capi.f8_rows(capi.f8_rows_args(x=xr.ptr, type=0, glu=capi.GLU[glu], M=1, D=128, y=y.ptr, s=s.ptr))
        v = f8.values(y.read(), s.read())[0]
        most = np.float64(s.read()[0, 0]) * 448
        assert np.isclose(most, 5e29, rtol=1e-5) and v[7] == most and (v[:7] == 0).all()
        for r in (xr, y, s):
            r.free()


# ------------------------------------------------------------------------------------------------ the stream's norm
def norm_check(rng, M, D, xt, tt, mode, post, w_one, bias, weight, scale, add, in_place, pad):
    x = activations(rng, M, D)
    K8 = 128 * f8.blocks(D)
    ld = D + pad if pad else None
    xr, xv = values_in(xt, x, ld)
    tr, tv = values_in(tt, (0.3 * rng.standard_normal((M, D))).astype(np.float32), ld) if add else (None, None)
    vec = lambda on, c: (1 * c + 0.2 * rng.standard_normal(D)).astype(np.float32) if on else None  # noqa: E731
    w, b, tw = vec(weight, 0 if w_one else 1), vec(bias, 0), vec(post, 1)
    dv = [None if v is None else capi.to_device(v) for v in (w, b, tw)]
    y, s = Rows(np.uint8, M, K8, K8 + 16 if pad else None), Rows(np.float32, f8.blocks(D), M, M + pad if pad else None)
    o = None if in_place else Rows(RAW[xt], M, D, ld)
    a = capi.f8_norm_args(x=xr.ptr, ldx=ld or 0, type=capi.TYPE[xt], t=tr.ptr if add else None, ldt=ld or 0, t_type=capi.TYPE[tt], tw=dv[2],
                          x_out=None if in_place else o.ptr, ldo=ld or 0, scale=scale, mode=mode, w_one=w_one, w=dv[0], b=dv[1], M=M, D=D,
                          y=y.ptr, ldy=K8 + 16 if pad else 0, s=s.ptr, lds=M + pad if pad else 0)
    capi.f8_norm(a)
    keep = {}
    half = HALF[xt]

    def rounded(r):
        """what the GPU's stream holds, once it is as near to r as a rounding lets it be"""
        if add or scale or not in_place:
            got = (o if not in_place else xr).read()
            got = from_type(got, xt) if xt != "f32" else got.astype(np.float64)
            part = 2.0 ** -21 * np.abs(xv)
            if post:   # the normalised t: its sum of squares and four roundings more
                part = part + 2.0 ** -18 * np.abs(tv / np.sqrt((tv ** 2).mean(1, keepdims=True) + 1e-6) * tw)
            elif add:
                part = part + 2.0 ** -21 * np.abs(tv)
            assert (np.abs(got - r) <= half * np.abs(r) + part * abs(scale or 1) + TINY[xt]).all(), np.abs(got - r).max()
            return got
        keep["as it was"] = True
        return r

    r, want = f8.norm(xv, tv, tw, w, b, bool(w_one), mode, scale or 1.0, rounded=rounded)
    d = r - r.mean(1, keepdims=True) if mode == 0 else r
    rstd = 1 / np.sqrt((d ** 2).mean(1, keepdims=True) + 1e-6)
    g = np.abs((0.0 if w_one else 1.0) if w is None else w) + (1.0 if w_one else 0.0)
    slack = 2.0 ** -17 * (np.abs(want) + (0 if b is None else np.abs(b)) + np.abs(r).mean(1, keepdims=True) * rstd * g)
    codes_near(y.read(), s.read(), want, slack)
    if keep:
        assert np.array_equal(xr.read(), xr.view(xr.host))
    for q in (xr, tr, y, s, o):
        if q:
            q.free()
    for q in dv:
        if q:
            q.free()


@pytest.mark.parametrize("M,D", [(1, 1), (1, 2048), (3, 100), (5, 1536), (64, 2560), (300, 65), (256, 512), (700, 1025), (259, 2560), (2, 4096),
                                 (3, 8192), (2, 8200), (1, 16384), (2, 20000), (1, 32768), (300, 2568)])
@pytest.mark.parametrize("mode", [0, 1])
def test_norm_sizes(dev, M, D, mode):
    rng = np.random.default_rng(M * 11 + D + mode)
    norm_check(rng, M, D, "f32", "f32", mode, False, mode == 0, mode == 0, True, 0, True, False, 0)
    norm_check(rng, M, D, "bf16", "bf16", mode, True, 0, False, True, 0, True, True, 5)


@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,D", [(3, 1000), (300, 520)])
def test_norm_types(dev, xt, tt, M, D):
    norm_check(np.random.default_rng(D), M, D, xt, tt, 1, False, 0, True, True, 0, True, False, 0)
    norm_check(np.random.default_rng(D), M, D, xt, tt, 0, True, 1, True, False, 0.5, True, True, 8)


@pytest.mark.parametrize("weight,bias,w_one,scale,add,in_place", [(False, False, 0, 0, False, True), (True, False, 0, 0, False, True),
                                                                  (True, True, 1, 0, False, False), (False, True, 1, 0.25, False, True),
                                                                  (False, False, 1, 2.0, True, False)])
def test_norm_forms(dev, weight, bias, w_one, scale, add, in_place):
    for M, D in ((2, 384), (300, 200)):
        for mode in (0, 1):
            norm_check(np.random.default_rng(D), M, D, "f16", "f32", mode, False, w_one, bias, weight, scale, add, in_place, 0)


def test_norm_rows_that_are_not_finite_or_nothing(dev):
    """a row with a NaN or an infinity is NaN, a row of zeros is b; their neighbours are theirs alone"""
    rng = np.random.default_rng(4)
    for M, D in ((4, 2048), (256, 300)):
        for mode in (0, 1):
            x = activations(rng, M, D)
            x[1], x[2, 7], x[3, 9] = 0, np.nan, np.inf
            xr, v = values_in("bf16", x)
            y, s = Rows(np.uint8, M, 128 * f8.blocks(D)), Rows(np.float32, f8.blocks(D), M)
            capi.f8_norm(capi.f8_norm_args(x=xr.ptr, type=2, mode=mode, M=M, D=D, y=y.ptr, s=s.ptr))
            got = f8.values(y.read(), s.read())
            assert (got[1] == 0).all() and np.isnan(got[2, :D]).all()
            assert np.isnan(got[3, 9]) and (np.isnan(got[3, :D]) | (got[3, :D] == 0)).all()
            rest = np.r_[0, 4:M]
            _, want = f8.norm(v[rest], mode=mode)
            codes_near(y.read()[rest], s.read()[:, rest], want, 2.0 ** -17 * (np.abs(want) + np.abs(want).mean(1, keepdims=True) * 2))
            for r in (xr, y, s):
                r.free()


# ------------------------------------------------------------------------------------------------ the product
def operands(rng, M, N, K):
    xc, xs = f8.quantise(activations(rng, M, K))
    wc, ws = f8.pack((0.05 * rng.standard_normal((N, K)) * np.exp(0.5 * rng.standard_normal((N, 1)))).astype(np.float32))
    return xc, xs, wc, ws


def product_near(got, type_, xc, xs, wc, ws, K):
    x, w = f8.values(xc, xs), f8.weight(wc, ws)
    want, total = x @ w.T, np.abs(x) @ np.abs(w).T
    bound = (128 + 2 * K / 128) * 2.0 ** -23 * total
    if type_ != "f32":
        for k in range(0, K, 8):
            bound += 7 * 2.0 ** -13 * (np.abs(x[:, None, k:k + 8]) * np.abs(w[None, :, k:k + 8])).max(2)
    err = np.abs(got - want)
    ok = err <= bound + HALF[type_] * (np.abs(want) + bound) + TINY[type_]
    assert ok.all(), (np.argwhere(~ok)[:4], got[~ok][:4], want[~ok][:4], (~ok).sum())


def product(M, N, K, type_, seed, pads=None, spoil=None):
    rng = np.random.default_rng(seed)
    xc, xs, wc, ws = operands(rng, M, N, K)
    if spoil:
        spoil(xc, xs, wc, ws)
    pads = pads or {}
    ld = lambda name, n: n + pads[name] if name in pads else None  # noqa: E731
    x, w = Rows(np.uint8, M, K, ld("x", K), xc), Rows(np.uint8, N, K, ld("w", K), wc)
    xsr, wsr = Rows(np.float32, K // 128, M, ld("xs", M), xs), Rows(np.float32, f8.blocks(N), K // 128, ld("ws", K // 128), ws)
    y = Rows(RAW[type_], M, N, ld("y", N), lead=64 + size_of(type_) * pads.get("lead", 0))
    a = capi.f8_gemm_args(x=x.ptr, ldx=x.ld, xs=xsr.ptr, ldxs=xsr.ld, w=w.ptr, ldw=w.ld, ws=wsr.ptr, ldws=wsr.ld, M=M, N=N, K=K,
                          type=capi.TYPE[type_], y=y.ptr, ldy=y.ld)
    capi.f8_gemm(a)
    got = y.read()
    capi.f8_gemm(a)
    assert np.array_equal(y.read().view(np.uint8), got.view(np.uint8)), "the same bits each time"
    for r in (x, w, xsr, wsr, y):
        r.free()
    return from_type(got, type_), (xc, xs, wc, ws)


SIZES = [(1, 1, 128), (1, 64, 256), (1, 2048, 8192), (2, 17, 384), (5, 300, 1024), (15, 129, 640), (16, 128, 128), (17, 16, 2048), (31, 257, 512),
         (33, 1000, 384), (64, 512, 4096), (65, 127, 1280), (100, 2048, 640), (128, 128, 128), (129, 640, 256), (200, 1025, 1152),
         (256, 256, 512), (257, 255, 640), (300, 2048, 2048), (513, 1300, 384), (1021, 520, 1024), (1100, 2300, 256), (40, 5000, 128),
         (7, 9, 16384), (130, 70, 9216)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_gemm_sizes(dev, M, N, K):
    got, ops = product(M, N, K, "f32", M + N + K)
    product_near(got, "f32", *ops, K)


# rows, outputs and k that take each tile, in one and in more slices of k, ragged at both ends
@pytest.mark.parametrize("M,N,K,type_", [(23, 4327, 2560, "f16"), (27, 33, 2048, "bf16"), (94, 21, 5120, "f32"), (17, 6123, 2048, "f32"),
                                         (77, 8820, 128, "f32"), (17, 8431, 5120, "bf16"), (17, 4191, 5120, "f32"),
                                         (195, 8757, 128, "f16"), (195, 8757, 128, "f32"), (69, 8194, 5120, "bf16"), (65, 4395, 8192, "f32"),
                                         (390, 8346, 128, "bf16"), (522, 7318, 128, "f32"), (387, 8171, 8192, "f16"), (200, 8694, 8192, "f32"),
                                         (1025, 7295, 384, "f16"), (1025, 7295, 384, "bf16"), (1021, 16383, 2048, "bf16"), (1537, 9217, 1280, "f16"),
                                         # the same again for the figures of each tile as they are now; over 64 blocks of k in one go; 7 slices
                                         (1537, 1282, 9216, "f16"), (1025, 906, 16640, "f32"), (259, 6531, 128, "f32"), (2050, 905, 128, "bf16"),
                                         (1025, 975, 5120, "bf16"), (1537, 2435, 9216, "f16"), (1537, 2435, 9216, "f32"), (1537, 2561, 128, "bf16"),
                                         (1537, 2562, 640, "f32"), (1537, 1281, 16640, "bf16"), (1537, 1292, 8192, "f32"), (1537, 1155, 9216, "f16"),
                                         (1537, 1155, 9216, "f32"), (65, 8197, 128, "f32"), (700, 710, 5120, "f16"), (2050, 130, 16640, "f32"),
                                         (2050, 3849, 9216, "f16"), (1537, 4993, 640, "bf16"), (130, 70, 4224, "f32"), (130, 70, 4224, "f16"),
                                         (1025, 996, 5120, "bf16"), (1025, 867, 5120, "f16"), (130, 4097, 16640, "f32"), (1025, 1282, 16640, "f32"),
                                         (17, 24, 25600, "f32"), (17, 24, 26880, "bf16"), (387, 1249, 128, "bf16"), (1025, 938, 9216, "f16"),
                                         (1537, 2306, 9216, "f32"), (387, 307, 9216, "bf16"), (17, 20, 9216, "f16"), (195, 577, 128, "f32"),
                                         (522, 875, 1024, "bf16"), (522, 835, 1024, "f32"), (1025, 801, 2048, "f16"), (1025, 839, 2048, "f32"),
                                         (1021, 1793, 5120, "bf16"), (1025, 1474, 5120, "f32"), (387, 306, 53760, "f16"), (130, 321, 53760, "f32"),
                                         (1025, 642, 128, "bf16"), (387, 1699, 128, "f32"), (1537, 642, 128, "f32"), (387, 2306, 128, "f16")])
def test_gemm_tiles(dev, M, N, K, type_):
    """a sample of the rows and outputs, the first and the last among them (the whole product is the GPU's work)"""
    rng = np.random.default_rng(M)
    xc, wc = rng.integers(0, 254, (M, K)).astype(np.uint8), rng.integers(0, 254, (N, K)).astype(np.uint8)
    xc[(xc & 127) == 127], wc[(wc & 127) == 127] = 0, 0
    xs, ws = np.exp(rng.standard_normal((K // 128, M))).astype(np.float32) * 1e-3, np.exp(rng.standard_normal((f8.blocks(N), K // 128))).astype(np.float32) * 1e-4
    x, w, xsr, wsr = (Rows(a.dtype, a.shape[0], a.shape[1], raw=a) for a in (xc, wc, xs, ws))
    y = Rows(RAW[type_], M, N)
    capi.f8_gemm(capi.f8_gemm_args(x=x.ptr, xs=xsr.ptr, w=w.ptr, ws=wsr.ptr, M=M, N=N, K=K, type=capi.TYPE[type_], y=y.ptr))
    got = from_type(y.read(), type_).reshape(M, N)
    m = np.unique(np.r_[0, M - 1, rng.integers(0, M, 40)])
    n = np.unique(np.r_[0, N - 1, np.arange(0, N, 128), rng.integers(0, N, 60)])
    full = f8.weight(wc, ws)[n]
    a = f8.values(xc[m], np.ascontiguousarray(xs[:, m]))
    want, total = a @ full.T, np.abs(a) @ np.abs(full).T
    bound = (128 + 2 * K / 128) * 2.0 ** -23 * total
    if type_ != "f32":
        for k in range(0, K, 8):
            bound += 7 * 2.0 ** -13 * (np.abs(a[:, None, k:k + 8]) * np.abs(full[None, :, k:k + 8])).max(2)
    err = np.abs(got[np.ix_(m, n)] - want)
    assert (err <= bound + HALF[type_] * (np.abs(want) + bound) + TINY[type_]).all(), (err / np.maximum(bound, 1e-30)).max()
    for r in (x, w, xsr, wsr, y):
        r.free()


@pytest.mark.parametrize("M,N,K", [(1, 100, 512), (13, 500, 640), (70, 390, 256), (300, 770, 384), (600, 2050, 640)])
@pytest.mark.parametrize("type_", ["f16", "bf16"])
def test_gemm_types(dev, M, N, K, type_):
    got, ops = product(M, N, K, type_, M)
    product_near(got, type_, *ops, K)


@pytest.mark.parametrize("M,N,K", [(1, 100, 512), (13, 500, 640), (70, 390, 256), (300, 770, 384), (1030, 770, 384)])
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_gemm_strides(dev, M, N, K, type_):
    """rows apart in every operand; outputs that are not aligned to four of them"""
    got, ops = product(M, N, K, type_, N, dict(x=16, w=48, xs=3, ws=1, y=3, lead=1))
    product_near(got, type_, *ops, K)


@pytest.mark.parametrize("M,N,K", [(3, 200, 512), (70, 300, 512), (600, 700, 512)])
def test_gemm_values_that_are_not_finite(dev, M, N, K):
    """a NaN code makes its row of outputs NaN, a NaN in the weight its column, an infinite scale its row; the others are theirs alone"""
    def spoil(xc, xs, wc, ws):
        xc[1, 300], wc[150, 130] = 0x7F, 0xFF
        xs[2, 2] = np.inf

    got, (xc, xs, wc, ws) = product(M, N, K, "f32", 5, spoil=spoil)
    assert np.isnan(got[1]).all() and np.isnan(got[:, 150]).all() and not np.isfinite(got[2]).any()
    m, n = np.delete(np.arange(M), [1, 2]), np.delete(np.arange(N), 150)
    fine = wc.copy()
    fine[150] = 0
    x, w = f8.values(xc[m], xs[:, m]), f8.weight(fine, ws)[n]
    err = np.abs(got[np.ix_(m, n)] - x @ w.T)
    assert (err <= (128 + 2 * K / 128) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T) * 1.01 + 1e-30).all()


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K", [(130, 300, 640), (300, 600, 384), (9, 40, 1024), (40, 300, 512), (1100, 530, 256)])
def test_gemm_of_one_code_finds_every_place(dev, M, N, K, type_):
    """x has one code a row: each output is one weight's value times powers of two and the block's number, exact in every type"""
    for _ in range(1):
        xc, xs = np.zeros((M, K), np.uint8), np.ones((K // 128, M), np.float32)
        at = (np.arange(M) * 37) % K
        xc[np.arange(M), at] = f8.encode(1.0)
        xs[:] = (1 + np.arange(K // 128) % 4)[:, None]
        rng = np.random.default_rng(M)
        wc = rng.integers(0, 254, (N, K)).astype(np.uint8)                # any code, the least ones among them
        wc[(wc & 127) == 127] = 1
        ws = (2.0 ** rng.integers(-3, 4, (f8.blocks(N), K // 128))).astype(np.float32)
        x, w, xsr, wsr = Rows(np.uint8, M, K, raw=xc), Rows(np.uint8, N, K, raw=wc), Rows(np.float32, K // 128, M, raw=xs), Rows(np.float32, f8.blocks(N), K // 128, raw=ws)
        y = Rows(RAW[type_], M, N)
        capi.f8_gemm(capi.f8_gemm_args(x=x.ptr, xs=xsr.ptr, w=w.ptr, ws=wsr.ptr, M=M, N=N, K=K, type=capi.TYPE[type_], y=y.ptr))
        assert np.array_equal(from_type(y.read(), type_), f8.gemm(xc, xs, wc, ws))
        for r in (x, w, xsr, wsr, y):
            r.free()


def test_nothing_to_do(dev):
    """no rows: nothing is read or written"""
    y = Rows(np.float32, 4, 128)
    capi.f8_gemm(capi.f8_gemm_args(M=0, N=128, K=128, type=0, y=y.ptr))
    capi.f8_gemm(capi.f8_gemm_args(M=4, N=0, K=128, type=0, y=y.ptr))
    capi.f8_rows(capi.f8_rows_args(M=0, D=128, type=0))
    capi.f8_norm(capi.f8_norm_args(M=0, D=128, type=0))
    capi.f8_pack(capi.f8_pack_args(N=0, K=128, type=0))
    assert (y.read().view(np.uint8) == FILL).all()
    y.free()


def test_recorded_calls_replay(dev):
    """pack, norm, product, gated rows and their product in a recording, replayed with the program's own calls between"""
    rng = np.random.default_rng(9)
    M, D, F = 70, 512, 640
    xr, _ = values_in("bf16", activations(rng, M, D))
    w1, _ = values_in("bf16", (0.05 * rng.standard_normal((2 * F, D))).astype(np.float32))
    w2, _ = values_in("bf16", (0.05 * rng.standard_normal((D, F))).astype(np.float32))
    c1, s1, c2, s2 = Rows(np.uint8, 2 * F, D), Rows(np.float32, 10, 4), Rows(np.uint8, D, F), Rows(np.float32, 4, 5)
    a, as_, h, g, gs, y = (Rows(np.uint8, M, D), Rows(np.float32, 4, M), Rows(np.uint16, M, 2 * F), Rows(np.uint8, M, F), Rows(np.float32, 5, M),
                           Rows(np.float32, M, D))

    def step():
        capi.f8_pack(capi.f8_pack_args(x=w1.ptr, type=2, N=2 * F, K=D, w=c1.ptr, s=s1.ptr))
        capi.f8_pack(capi.f8_pack_args(x=w2.ptr, type=2, N=D, K=F, w=c2.ptr, s=s2.ptr))
        capi.f8_norm(capi.f8_norm_args(x=xr.ptr, type=2, M=M, D=D, y=a.ptr, s=as_.ptr))
        capi.f8_gemm(capi.f8_gemm_args(x=a.ptr, xs=as_.ptr, w=c1.ptr, ws=s1.ptr, M=M, N=2 * F, K=D, type=2, y=h.ptr))
        capi.f8_rows(capi.f8_rows_args(x=h.ptr, type=2, glu=1, M=M, D=F, y=g.ptr, s=gs.ptr))
        capi.f8_gemm(capi.f8_gemm_args(x=g.ptr, xs=gs.ptr, w=c2.ptr, ws=s2.ptr, M=M, N=D, K=F, type=0, y=y.ptr))

    step()
    want = y.read()
    rec = capi.record(step)
    for _ in range(4):
        y.buf.fill_u32(0xA5A5A5A5)
        rec.replay()
        assert np.array_equal(y.read(), want)
        step()
        assert np.array_equal(y.read(), want)
    rec.free()
    for r in (xr, w1, w2, c1, s1, c2, s2, a, as_, h, g, gs, y):
        r.free()


def test_calls_refused_in_a_chain(dev):
    import ctypes
    capi.check(capi.lib().p0_chain_begin())
    try:
        for call, args in (("f8_gemm", capi.f8_gemm_args(M=0, N=1, K=128)), ("f8_rows", capi.f8_rows_args(M=0, D=1)), ("rope", capi.rope_args(rows=0, hq=1, dim=2))):
            with pytest.raises(capi.P0Error, match=call + ": only gemv"):
                getattr(capi, call)(args)
    finally:
        h = ctypes.c_void_p()
        capi.lib().p0_chain_end(ctypes.byref(h))
        if h.value:
            capi.lib().p0_chain_free(h)


def test_rows_far_apart(dev):
    """rows 2 GiB apart: offsets past 32 bits in what each operator reads and writes"""
    ld, rows = (1 << 30) + 64, 3
    rng = np.random.default_rng(3)
    far = capi.Buffer(2 * (2 * ld + 1024))
    x = to_type(rng.standard_normal((rows, 256)).astype(np.float32), "bf16")
    put = lambda: [far.upload(x[0][i], 2 * i * ld) for i in range(rows)]  # noqa: E731
    get = lambda n: np.stack([far.read(np.uint16, n, 2 * i * ld) for i in range(rows)])  # noqa: E731
    put()
    y, s = Rows(np.uint8, rows, 256), Rows(np.float32, 2, rows)
    capi.f8_rows(capi.f8_rows_args(x=far, ldx=ld, type=2, M=rows, D=256, y=y.ptr, s=s.ptr))
    wc, ws = f8.quantise(x[1].astype(np.float32))
    assert np.array_equal(y.read(), wc) and np.array_equal(s.read(), ws)
    capi.f8_pack(capi.f8_pack_args(x=far, ldx=ld, type=2, N=rows, K=256, w=y.ptr, s=s.ptr, lds=2))
    assert np.array_equal(y.read(), f8.pack(x[1].astype(np.float32))[0])
    capi.f8_norm(capi.f8_norm_args(x=far, ldx=ld, type=2, t=far, t_type=2, ldt=ld, x_out=far.ptr + 512, ldo=ld, M=rows, D=256, y=y.ptr, s=s.ptr))
    assert np.array_equal(np.stack([far.read(np.uint16, 256, 2 * i * ld + 512) for i in range(rows)]), to_type((2 * x[1]).astype(np.float32), "bf16")[0])
    put()
    pos = capi.to_device(np.zeros(rows, np.int32))
    capi.rope(capi.rope_args(x=far, ldr=ld, y=far, y_ldr=ld, type=2, rows=rows, hq=4, dim=64, pos=pos))
    assert np.array_equal(get(256), x[0])
    for M in (rows, 20):   # a product whose rows are far apart: the kernel for few rows, and one of tiles into columns of one buffer
        n = 24
        ops = operands(rng, M, n, 128)
        dv = [capi.to_device(o) for o in ops]
        out = capi.Buffer(4 * ((M - 1) * (1 << 28) + n)) if M == rows else capi.Buffer(4 * M * (1 << 26))
        ldy = (1 << 28) if M == rows else (1 << 26)
        capi.f8_gemm(capi.f8_gemm_args(x=dv[0], xs=dv[1], w=dv[2], ws=dv[3], M=M, N=n, K=128, type=0, y=out, ldy=ldy))
        product_near(np.stack([out.read(np.float32, n, 4 * i * ldy) for i in range(M)]).astype(np.float64), "f32", *ops, 128)
        for b in dv + [out]:
            b.free()
    for b in (far, y, s, pos):
        b.free()
