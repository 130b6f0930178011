"""Gated rows (f8_rows) gate by gate: each has a row, and so a scale, of its own, which is the value / 448 in fp32.

Bound: in units u = 2^-24 of a value the exponential is off by 2 (one in its last place), and the factor that puts back what its argument
rounds off, the sum of the sigmoid's divisor, its reciprocal, the two products and the scale's quotient by one each: 8 u. An error of
the argument z would come z times as large."""
import numpy as np
import pytest

from oracle import f8
from p0pc0rn_amd import capi
from tests.test_f8_gpu import Rows, values_in

pytestmark = pytest.mark.gpu


def formula(glu, g, u):
    """g u sigmoid(z) in float64: without the 1 + tanh(z / 2) that cancels below zero"""
    g = g.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        z = g if glu == "silu" else 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)
        return g / (1 + np.exp(-z)) * u.astype(np.float64)


def gated(glu, type_, g, u):
    """rows [M, D] of gates and of their partners -> codes, scales [M, D / 128], and both as the type holds them"""
    M, D = g.shape
    x, v = values_in(type_, np.concatenate([g, u], 1))
    y, s = Rows(np.uint8, M, 128 * f8.blocks(D)), Rows(np.float32, f8.blocks(D), M)
    capi.f8_rows(capi.f8_rows_args(x=x.ptr, type=capi.TYPE[type_], glu=capi.GLU[glu], M=M, D=D, y=y.ptr, s=s.ptr))
    out = y.read(), s.read().T.copy(), v[:, :D], v[:, D:]
    for r in (x, y, s):
        r.free()
    return out


@pytest.mark.parametrize("glu,low", [("silu", -87.0), ("gelu", -9.9)])
@pytest.mark.parametrize("type_", ["f32", "bf16", "f16"])
def test_each_gate_to_the_last_places(dev, glu, low, type_):
    """gates from where the sigmoid is the least normal value up to where it is 1, partners that make the value a normal one"""
    rng = np.random.default_rng(3)
    M = 4096
    g = np.concatenate([rng.uniform(low, 0, 3 * M // 4), rng.uniform(0, 40, M // 4)]).astype(np.float32)[:, None]
    at = np.log2(np.abs(formula(glu, g, np.ones_like(g))))
    most = 14 if type_ == "f16" else 126
    u = np.exp2(np.clip(np.rint(rng.uniform(-20, 20, (M, 1)) - at), -14, most)) * rng.choice([-1.0, 1.0], (M, 1))
    codes, s, gv, uv = gated(glu, type_, np.repeat(g, 128, 1), np.repeat(u.astype(np.float32), 128, 1))
    want = formula(glu, gv[:, 0], uv[:, 0])
    normal = np.abs(want) >= 448 * 2.0 ** -126
    assert normal.mean() > 0.5 and (type_ == "f16" or normal.all())
    off = np.abs(s[:, 0].astype(np.float64) * 448 - np.abs(want))[normal] / np.abs(want[normal])
    assert (off <= 8.01 * 2.0 ** -24).all(), (off.max() * 2 ** 24, gv[normal, 0][off.argmax()])
    assert (f8.VALUES[codes[normal]] == np.where(want < 0, -448.0, 448.0)[normal, None]).all()


@pytest.mark.parametrize("glu", ["silu", "gelu"])
@pytest.mark.parametrize("type_", ["f32", "bf16", "f16"])
def test_gates_and_partners_that_are_not_finite(dev, glu, type_):
    """a code is NaN where the formula's value is not finite, and nothing beside it changes; a gate far below zero gives 0, far above it its partner's multiple"""
    big = 1e4 if type_ == "f16" else 1e30
    pairs = [(a, b) for a in (np.inf, -np.inf, np.nan, big, -big, -300.0, -200.0, -140.0, 0.0, 1.0) for b in (np.inf, -np.inf, np.nan, 0.0, 2.0)]
    M = len(pairs)
    g, u = np.ones((M, 256), np.float32), np.full((M, 256), 0.5, np.float32)
    where = (np.arange(M) * 37) % 256
    g[np.arange(M), where], u[np.arange(M), where] = np.float32(pairs).T
    codes, s, gv, uv = gated(glu, type_, g, u)
    want = formula(glu, gv, uv)
    got = f8.values(codes, s.T)
    assert np.array_equal(np.isnan(got), ~np.isfinite(want))
    full = np.where(np.isfinite(want), want, 0.0)
    step = np.repeat(np.abs(full).reshape(M, 2, 128).max(2), 128, 1) / 448 * 2.0 ** -10
    fine = np.isfinite(want)
    assert (np.abs(got - full)[fine] <= (np.maximum(2.0 ** -4 * np.abs(full), step) * (1 + 2.0 ** -20) + 2.0 ** -20 * np.abs(full))[fine]).all()
    ones = formula(glu, np.ones(1), np.full(1, 0.5))[0]
    assert np.allclose(s[np.arange(M), 1 - where // 128] * 448, ones, rtol=2.0 ** -20, atol=0)
