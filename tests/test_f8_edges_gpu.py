"""The 8-bit operators and the rotation at the ends of what their calls allow: the longest rows and sums, a matrix by itself, a caller's
stream, recordings that share the workspace of K slices, the first and last positions of int32. Bounds as in test_f8_gpu.py and test_rope_gpu.py."""
import ctypes

import numpy as np
import pytest

from oracle import f8
from p0pc0rn_amd import capi
from tests.test_f8_gpu import RAW, Rows, activations, codes_near, operands, product, product_near, values_in
from tests.test_kv_gpu import from_type, to_type

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,type_", [(1, 8, "f32"), (16, 9, "f32"), (17, 8, "f32"), (17, 8, "bf16")])
def test_longest_product(dev, M, N, type_):
    got, ops = product(M, N, 1 << 20, type_, M)
    product_near(got, type_, *ops, 1 << 20)


@pytest.mark.parametrize("call", ["rows", "gated", "pack"])
def test_longest_rows(dev, call):
    D = (1 << 20) - 3
    rng = np.random.default_rng(4)
    xr, v = values_in("bf16", activations(rng, 3, D * (2 if call == "gated" else 1)))
    y, s = Rows(np.uint8, 3, D + 3), Rows(np.float32, *((1, 8192) if call == "pack" else (8192, 3)))
    if call == "pack":
        capi.f8_pack(capi.f8_pack_args(x=xr.ptr, type=2, N=3, K=D, w=y.ptr, s=s.ptr))
        want = f8.pack(v.astype(np.float32))
    else:
        capi.f8_rows(capi.f8_rows_args(x=xr.ptr, type=2, glu=1 if call == "gated" else 0, M=3, D=D, y=y.ptr, s=s.ptr))
        want = f8.quantise(v.astype(np.float32))
    if call == "gated":
        g, u = v[:, :D].astype(np.float64), v[:, D:].astype(np.float64)
        value = g / (1 + np.exp(-g)) * u
        codes_near(y.read(), s.read(), value, 2.0 ** -16 * np.abs(value))
    else:
        assert np.array_equal(y.read(), want[0]) and np.array_equal(s.read(), want[1])
    for r in (xr, y, s):
        r.free()


def test_a_matrix_by_itself(dev):
    """both operands one buffer, and one run of scales: a block's are those of 128 rows and of 128 x 128"""
    rng = np.random.default_rng(6)
    for n, type_ in ((12, "f32"), (128, "f32"), (128, "f16")):
        xc, xs = f8.quantise(activations(rng, n, 128))
        xs[:] = xs.max()
        x, s = Rows(np.uint8, n, 128, raw=xc), Rows(np.float32, 1, n, raw=xs)
        y = Rows(RAW[type_], n, n)
        capi.f8_gemm(capi.f8_gemm_args(x=x.ptr, xs=s.ptr, w=x.ptr, ws=s.ptr, M=n, N=n, K=128, type=capi.TYPE[type_], y=y.ptr))
        product_near(from_type(y.read(), type_), type_, xc, xs, xc, xs[:, :1], 128)
        for r in (x, s, y):
            r.free()


class Product:
    """a product on the device, its operands and its call"""

    def __init__(self, M, N, K, type_, seed):
        self.ops = operands(np.random.default_rng(seed), M, N, K)
        self.K, self.type = K, type_
        self.dv = [Rows(o.dtype, o.shape[0], o.shape[1], raw=o) for o in self.ops]
        self.y = Rows(RAW[type_], M, N)
        p = [d.ptr for d in self.dv]
        self.args = capi.f8_gemm_args(x=p[0], xs=p[1], w=p[2], ws=p[3], M=M, N=N, K=K, type=capi.TYPE[type_], y=self.y.ptr)

    def call(self):
        capi.f8_gemm(self.args)

    def read(self):
        return self.y.read()

    def clear(self):
        raw = np.full(self.y.host.size, 0xA5, np.uint8)
        self.y.buf.upload(raw)

    def free(self):
        for r in self.dv + [self.y]:
            r.free()


def test_recordings_that_share_the_slices_workspace(dev):
    """products in slices of K, each in a recording of its own, replayed in turn and beside an eager one"""
    many = [Product(17, 24, 25600, "bf16", 1), Product(18, 24, 26880, "f32", 2), Product(20, 30, 28160, "f16", 3)]
    want = []
    for p in many:
        p.call()
        want.append(p.read())
        product_near(from_type(want[-1], p.type), p.type, *p.ops, p.K)
    recs = [capi.record(p.call) for p in many]
    both = capi.record(lambda: [p.call() for p in many])
    for order in ((0, 1, 2), (2, 0, 1), (1, 1, 0, 2)):
        for p in many:
            p.clear()
        for i in order:
            recs[i].replay()
            many[(i + 1) % 3].call()
        for p, w in zip(many, want):
            assert np.array_equal(p.read(), w)
            p.clear()
        both.replay()
        both.replay()
        for p, w in zip(many, want):
            assert np.array_equal(p.read(), w)
    for r in recs + [both] + many:
        r.free()


def test_a_callers_stream(dev):
    """every operator on a stream that the caller made, behind work of that stream; then on the library's again"""
    rng = np.random.default_rng(8)
    p = Product(40, 130, 4096, "f32", 5)
    xr, v = values_in("f32", activations(rng, 40, 256))
    y, s = Rows(np.uint8, 40, 256), Rows(np.float32, 2, 40)
    w, ws = Rows(np.uint8, 40, 256), Rows(np.float32, 1, 2)
    pos = capi.to_device(np.full(40, 3, np.int32))
    turned = capi.Buffer(40 * 256 * 4)

    def all_of_them(x):
        capi.f8_rows(capi.f8_rows_args(x=x, type=0, M=40, D=256, y=y.ptr, s=s.ptr))
        capi.f8_pack(capi.f8_pack_args(x=x, type=0, N=40, K=256, w=w.ptr, s=ws.ptr))
        capi.rope(capi.rope_args(x=x, y=turned, type=0, rows=40, hq=4, dim=64, pos=pos))
        p.call()
        return y.read(), s.read(), w.read(), ws.read(), turned.read(np.float32, 40 * 256), p.read()

    want = all_of_them(xr.ptr)
    hip, stream = capi.lib(), ctypes.c_void_p()      # the runtime that the library has loaded
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    late, big = capi.Buffer(40 * 256 * 4), [capi.Buffer(1 << 28) for _ in range(2)]
    late.fill_u32(0x7FC00000)
    capi.done()
    capi.check(capi.lib().p0_set_stream(stream))
    try:
        for _ in range(8):
            capi.copy(big[0], 0, big[1], 0, 1 << 28)         # work ahead of the operators' input on that stream
        capi.copy(xr.ptr, 0, late, 0, 40 * 256 * 4)
        got = all_of_them(late)
    finally:
        capi.done()
        capi.check(capi.lib().p0_set_stream(None))
        assert hip.hipStreamDestroy(stream) == 0
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    for a, b in zip(all_of_them(xr.ptr), want):
        assert np.array_equal(a, b)
    for r in (p, xr, y, s, w, ws, pos, turned, late, *big):
        r.free()


@pytest.mark.parametrize("mode", ["inter", "half"])
def test_first_and_last_positions(dev, mode):
    """the ends of int32: 2^31 positions times a frequency off by 10 roundings of 2^-53 are 2.4e-6 rad, and the oracle's own as much"""
    pos = np.array([[-(1 << 31), (1 << 31) - 1, 1 << 30, -1, 0]], np.int32)
    rng = np.random.default_rng(2)
    x = rng.standard_normal((5, 2, 128)).astype(np.float32)
    xb, yb, pb = capi.to_device(x), capi.Buffer(x.nbytes), capi.to_device(pos)
    capi.rope(capi.rope_args(x=xb, y=yb, type=0, rows=5, hq=1, hk=1, dim=128, mode=capi.ROPE[mode], pos=pb))
    got = yb.read(np.float32, x.size).reshape(x.shape)
    e = np.arange(64, dtype=np.longdouble) / 64
    angle = pos[0].astype(np.longdouble)[:, None, None] * np.longdouble(10000) ** -e
    u, v = (x[..., 0::2], x[..., 1::2]) if mode == "inter" else (x[..., :64], x[..., 64:])
    a, b = u * np.cos(angle) - v * np.sin(angle), v * np.cos(angle) + u * np.sin(angle)
    ga, gb = (got[..., 0::2], got[..., 1::2]) if mode == "inter" else (got[..., :64], got[..., 64:])
    bound = (1e-6 + 2.4e-6) * (np.abs(u) + np.abs(v))
    assert (np.abs(ga - a) <= bound).all() and (np.abs(gb - b) <= bound).all()
    for r in (xb, yb, pb):
        r.free()


@pytest.mark.parametrize("mode", ["inter", "half"])
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_channels_that_do_not_turn_beside_infinities(dev, mode, type_):
    """what lies past the turning channels keeps its bits, beside infinities and NaN too"""
    raw, v = to_type(np.random.default_rng(1).standard_normal((6, 2, 80)).astype(np.float32), type_)
    inf, nan = (np.uint16(0x7F80), np.uint16(0x7FC0)) if type_ == "bf16" else (np.float32(np.inf), np.float32(np.nan))
    raw = raw.copy()
    raw[0, 0, 61], raw[1, 1, 60], raw[2, 0, 79], raw[3, 1, 62:70] = inf, inf, nan, inf
    raw[4, 0, 60:] = 0
    raw[4, 0, 61::2] = np.uint16(0x8000) if type_ == "bf16" else -0.0
    xb, yb, pb = capi.to_device(raw), capi.Buffer(raw.nbytes), capi.to_device(np.arange(6, dtype=np.int32))
    capi.rope(capi.rope_args(x=xb, y=yb, type=capi.TYPE[type_], rows=6, hq=1, hk=1, dim=80, mode=capi.ROPE[mode], axis_dim=[60], pos=pb))
    bits = np.uint16 if type_ == "bf16" else np.uint32
    got = yb.read(bits, raw.size).reshape(raw.shape)
    assert np.array_equal(got[..., 60:], raw.view(bits)[..., 60:])
    assert np.isfinite(from_type(got[..., :60].view(RAW[type_]), type_)).all()
    for b in (xb, yb, pb):
        b.free()


@pytest.mark.parametrize("shift", [1, 3, 5])
@pytest.mark.parametrize("D", [1001, 2056, 4099])
def test_rows_at_any_alignment(dev, D, shift):
    """rows of 16-bit values that begin at any element: the norm's, the gated rows' and the weight's inputs and the stream's output"""
    M, ld = 9, D + shift
    rng = np.random.default_rng(D)
    xr, v = values_in("bf16", activations(rng, M, D), ld, 64 + 2 * shift)
    tr, t = values_in("f16", activations(rng, M, D), ld + 2, 64 + 2 * shift)
    out = Rows(np.uint16, M, D, ld, lead=64 + 2 * shift)
    gr, gv = values_in("bf16", activations(rng, M, 2 * D), 2 * D + shift, 64 + 2 * shift)
    wv = (1 + 0.3 * rng.standard_normal(D)).astype(np.float32)
    w = Rows(np.float32, 1, D, raw=wv[None], lead=64 + 4 * shift)
    y, s = Rows(np.uint8, M, 128 * f8.blocks(D)), Rows(np.float32, f8.blocks(D), M)
    capi.f8_norm(capi.f8_norm_args(x=xr.ptr, ldx=ld, type=2, t=tr.ptr, t_type=1, ldt=ld + 2, x_out=out.ptr, ldo=ld, w=w.ptr, mode=1, M=M, D=D, y=y.ptr, s=s.ptr))
    stream = to_type((v.astype(np.float32) + t.astype(np.float32)), "bf16")
    assert np.array_equal(out.read(), stream[0])
    want = stream[1] / np.sqrt((stream[1] ** 2).mean(1, keepdims=True) + 1e-6) * wv
    codes_near(y.read(), s.read(), want, 2.0 ** -17 * (np.abs(want) + np.abs(want).mean(1, keepdims=True)))
    capi.f8_rows(capi.f8_rows_args(x=gr.ptr, ldx=gr.ld, type=2, glu=1, M=M, D=D, y=y.ptr, s=s.ptr))
    g, u = gv[:, :D].astype(np.float64), gv[:, D:].astype(np.float64)
    value = g / (1 + np.exp(-g)) * u
    codes_near(y.read(), s.read(), value, 2.0 ** -16 * np.abs(value))
    pw, ps = Rows(np.uint8, M, 128 * f8.blocks(D)), Rows(np.float32, 1, f8.blocks(D))
    capi.f8_pack(capi.f8_pack_args(x=xr.ptr, ldx=ld, type=2, N=M, K=D, w=pw.ptr, s=ps.ptr))
    codes, scales = f8.pack(v.astype(np.float32))
    assert np.array_equal(pw.read(), codes) and np.array_equal(ps.read(), scales)
    for r in (xr, tr, out, gr, w, y, s, pw, ps):
        r.free()


@pytest.mark.parametrize("M", [1, 3, 8, 9, 16, 17, 40])
@pytest.mark.parametrize("blocks", [1, 3, 17, 31, 65])
def test_scales_that_are_infinite(dev, M, blocks):
    """an infinite scale of the last block makes that row infinite, not NaN, and no other: nothing is added twice with it"""
    N, K = 20, 128 * blocks
    codes = lambda n: np.full((n, K), 0x38, np.uint8)  # noqa: E731  (1.0)
    xs, ws = np.full((blocks, M), 0.5, np.float32), np.full((1, blocks), 0.25, np.float32)
    xs[-1, M // 2] = np.inf
    x, w, s, r = Rows(np.uint8, M, K, raw=codes(M)), Rows(np.uint8, N, K, raw=codes(N)), Rows(np.float32, blocks, M, raw=xs), Rows(np.float32, 1, blocks, raw=ws)
    for type_ in ("f32", "bf16"):
        y = Rows(RAW[type_], M, N)
        capi.f8_gemm(capi.f8_gemm_args(x=x.ptr, xs=s.ptr, w=w.ptr, ws=r.ptr, M=M, N=N, K=K, type=capi.TYPE[type_], y=y.ptr))
        got = from_type(y.read(), type_).reshape(M, N)
        want = np.full((M, N), 16.0 * blocks)
        want[M // 2] = np.inf
        assert np.array_equal(got, want if type_ == "f32" else to_type(want, "bf16")[1])
        y.free()
    for b in (x, w, s, r):
        b.free()
