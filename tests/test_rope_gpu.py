"""GPU parity of the rotation of heads (rope) with its CPU restatement in float64.

The angle's fraction of a turn is rounded to fp32 (2 pi 2^-25 rad at most), its sine and cosine are within 2 units in the last
place, and the frequency in 64 bits is off by less than 2^-52 of itself, so at positions up to 2^20 each of cos, sin is within 6e-7;
two products and a sum are three roundings more: 1e-6 (|u| + |v|) holds a pair. A norm's sum of up to 512 squares and its
factor add 2^-18 of the value. Then one rounding to the type.
"""
import numpy as np
import pytest

from oracle import f8
from p0pc0rn_amd import capi
from tests.test_f8_gpu import HALF, RAW, TINY, Rows
from tests.test_kv_gpu import from_type, to_type

pytestmark = pytest.mark.gpu


def check(rows, hq, hk, dim, axis_dim, type_, mode="inter", freq="own", norm="", theta=1e4, far=0, gap=0, in_place=False, seed=0, lead=64):
    rng = np.random.default_rng(seed + rows * 13 + dim)
    heads, ldh = hq + hk, dim + gap
    width = (heads - 1) * ldh + dim
    ldr = heads * ldh + 2 * gap
    raw, v = to_type(rng.standard_normal((rows, heads, dim)).astype(np.float32), type_)
    full = np.zeros((rows, heads, ldh), RAW[type_])
    full[:, :, dim:] = np.uint8(1)
    full[:, :, :dim] = raw
    full = full.reshape(rows, -1)[:, :width]
    x = Rows(RAW[type_], rows, width, ldr, full, lead)
    y = x if in_place else Rows(RAW[type_], rows, heads * dim, None, None, lead)
    pos = rng.integers(0, 300, (len(axis_dim), rows)) + far
    pos[:, rows // 2] = 0 if far == 0 else far
    if rows > 2:
        pos[0, 1] = -7
    pr = Rows(np.int32, len(axis_dim), rows, rows + gap, pos.astype(np.int32))
    qw, kw = ((1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) if c in norm else None for c in "qk")
    dv = [None if w is None else capi.to_device(w) for w in (qw, kw)]
    strides = dict(y_ldr=ldr, y_ldh=ldh) if in_place else {}
    capi.rope(capi.rope_args(x=x.ptr, ldr=ldr, ldh=ldh, y=y.ptr, type=capi.TYPE[type_], rows=rows, hq=hq, hk=hk, dim=dim, mode=capi.ROPE[mode],
                             axis_dim=axis_dim, freq=capi.FREQ[freq], pos=pr.ptr, pos_ld=rows + gap, theta=theta, qw=dv[0], kw=dv[1], **strides))
    got = y.read()
    if in_place:
        padded = np.zeros((rows, heads * ldh), got.dtype)
        padded[:, :width] = got
        padded = padded.reshape(rows, heads, ldh)
        if gap:
            assert (padded[:, :-1, dim:] == full[0, dim]).all(), "between the heads"
        got = padded[:, :, :dim]
    got = from_type(np.ascontiguousarray(got), type_).reshape(rows, heads, dim)
    want = f8.rope(v, pos, axis_dim, theta, mode, freq, hq, qw, kw)
    plain = f8.rope(v, np.zeros_like(pos), axis_dim, theta, mode, freq, hq, qw, kw)     # normed, not turned
    R = sum(axis_dim)
    size = np.abs(plain)
    pair = size.copy()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if mode == "inter" else (slice(0, R // 2), slice(R // 2, R))
    pair[..., a] = pair[..., b] = size[..., a] + size[..., b]
    err = np.abs(got - want)
    ok = err <= 1e-6 * pair + (2.0 ** -18 * pair if norm else 0) + HALF[type_] * (np.abs(want) + 1e-5 * pair) + TINY[type_]
    assert ok.all(), (np.argwhere(~ok)[:3], got[~ok][:3], want[~ok][:3], (~ok).sum())
    if not norm:
        assert np.array_equal(got[..., R:], v[..., R:]), "channels that do not turn"
    for r in {id(r): r for r in (x, y, pr)}.values():
        r.free()
    for w in dv:
        if w:
            w.free()


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mode", ["inter", "half"])
@pytest.mark.parametrize("dim,axis_dim", [(128, [44, 42, 42]), (128, [32, 32, 32, 32]), (64, [64]), (256, [256]), (512, [172, 170, 170]), (16, [16]),
                                          (96, [96]), (80, [40, 40]), (100, [34, 32, 32]), (2, [2]), (128, [32, 32]), (66, [22, 22]), (48, [4, 2, 2])])
def test_dims_and_axes(dev, dim, axis_dim, mode, type_):
    check(5, 3, 2, dim, axis_dim, type_, mode)
    check(3, 2, 1, dim, axis_dim, type_, mode, freq="shared", norm="qk")


@pytest.mark.parametrize("rows,hq,hk", [(1, 1, 0), (1, 8, 2), (1, 0, 3), (1, 64, 8), (2, 1, 1), (17, 20, 20), (70, 33, 1), (1000, 8, 2), (3001, 2, 2), (400, 130, 7)])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_and_heads(dev, rows, hq, hk, dim):
    check(rows, hq, hk, dim, [dim // 2, dim // 4], "bf16", "inter")
    check(rows, hq, hk, dim, [dim], "f32", "half", norm="q" if hq else "k")


@pytest.mark.parametrize("norm", ["q", "k", "qk"])
@pytest.mark.parametrize("mode", ["inter", "half"])
def test_norms(dev, norm, mode):
    for dim in (256, 72, 34):
        check(4, 3, 2, dim, [dim], "f16", mode, norm=norm)


@pytest.mark.parametrize("gap,lead", [(8, 64), (3, 64), (0, 68), (16, 72)])
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_strides_and_in_place(dev, gap, lead, type_):
    for mode in ("inter", "half"):
        for in_place in (False, True):
            check(19, 4, 2, 64, [32, 32], type_, mode, gap=gap, in_place=in_place, lead=lead, norm="qk")


@pytest.mark.parametrize("far", [4000, 131071, 1 << 20])
@pytest.mark.parametrize("theta", [100.0, 1e4, 1e6])
def test_far_positions(dev, far, theta):
    check(40, 2, 1, 128, [64, 64], "f32", "half", theta=theta, far=far)
    check(40, 2, 1, 128, [128], "f32", "inter", freq="shared", theta=theta, far=far)


def test_a_head_of_zeros_or_nan(dev):
    """a norm of nothing is nothing; a NaN stays in its head"""
    x = np.ones((1, 4, 64), np.float32)
    x[0, 1], x[0, 2, 5] = 0, np.nan
    xr, pr, w = Rows(np.float32, 1, 256, raw=x.reshape(1, -1)), Rows(np.int32, 1, 1, raw=[[3]]), capi.to_device(np.ones(64, np.float32))
    y = Rows(np.float32, 1, 256)
    capi.rope(capi.rope_args(x=xr.ptr, y=y.ptr, type=0, rows=1, hq=4, dim=64, pos=pr.ptr, qw=w))
    got = y.read().reshape(4, 64)
    assert (got[1] == 0).all() and np.isnan(got[2]).all() and np.isfinite(got[[0, 3]]).all()
    for r in (xr, pr, y, w):
        r.free()


def test_recorded_rotation_replays(dev):
    """a copy and a rotation in place, recorded; the program's own calls between the replays"""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((30, 256)).astype(np.float32)
    src, buf, pr, y = capi.to_device(x), capi.Buffer(x.nbytes), capi.to_device(np.arange(30, dtype=np.int32)), capi.Buffer(x.nbytes)

    def step():
        capi.copy(src, 0, buf, 0, x.nbytes)
        capi.rope(capi.rope_args(x=buf, y=buf, type=0, rows=30, hq=4, dim=64, mode=1, pos=pr))

    rec = capi.record(step)
    capi.rope(capi.rope_args(x=src, y=y, type=0, rows=30, hq=4, dim=64, mode=1, pos=pr))
    want = y.read(np.uint8, x.nbytes)
    for _ in range(4):
        buf.fill_u32(0xA5A5A5A5)
        rec.replay()
        assert np.array_equal(buf.read(np.uint8, x.nbytes), want)
        step()
        assert np.array_equal(buf.read(np.uint8, x.nbytes), want)
    rec.free()
    for b in (src, buf, pr, y):
        b.free()
