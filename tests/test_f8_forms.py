"""Every form of the 8-bit product (f8_gemm): the kernels for few rows, the tiles, each in as many slices of K as the rule (f8_choice.hpp) gives it.

The rule is built by itself, on the CPU, and asked: SHAPES says which form takes each, and no form that any shape finds is missing from it. The
GPU's results are held against float64 with the bounds of test_f8_gpu.py on a sample of rows and outputs, each tile's edges among them."""
import os
import random
import subprocess

import numpy as np
import pytest

from oracle import f8
from p0pc0rn_amd import capi
from tests.test_f8_gpu import HALF, RAW, TINY, Rows
from tests.test_kv_gpu import from_type

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "p0pc0rn_amd", "csrc")
CUS, PART = 256, 16 << 20   # the MI355X's CUs, the workspace's floats
FORMS = ["small", "low", "half", "long", "wide", "few32", "few32w", "few32x", "few64", "few8", "pairs4", "pairs", "few16b", "few16"]

# form, slices: rows, outputs, blocks of k; 16-bit results, then fp32 ones
SHAPES = [
    ("few8", 1, (7, 133, 16), (3, 4617, 5)), ("few16b", 1, (9, 133, 16), (15, 4101, 1)), ("few16", 1, (13, 261, 17), (11, 135, 63)),
    ("pairs", 1, (8, 133, 17), (5, 4607, 33)), ("pairs", 1, (1, 4617, 65), (7, 17, 64)), ("pairs4", 1, (5, 4617, 17), (1, 4621, 31)),
    ("pairs4", 1, (8, 4625, 63), (8, 4617, 44)),
    ("few32", 1, (29, 133, 9), (17, 1027, 5)), ("few32w", 1, (33, 2111, 1), (33, 2061, 7)), ("few32x", 1, (579, 771, 8), (877, 485, 8)),
    ("few64", 1, (1149, 737, 16), (961, 933, 15)),
    ("small", 1, (65, 7511, 1), (97, 5583, 1)), ("small", 4, (17, 4021, 131), None), ("small", 8, (135, 331, 241), (133, 323, 366)),
    ("small", 15, (17, 37, 177), (17, 35, 177)), ("small", 16, (17, 61, 182), (17, 33, 169)),
    ("low", 1, (129, 5921, 1), (97, 8219, 1)), ("low", 2, (19, 8739, 60), None), ("low", 4, (557, 807, 332), None), ("low", 8, (361, 339, 232), (365, 343, 494)),
    ("low", 16, (277, 193, 542), (129, 339, 377)),
    ("half", 1, (199, 8249, 1), (195, 8383, 1)), ("half", 2, (1351, 745, 46), (1219, 1257, 31)), ("half", 4, (963, 625, 124), (299, 2067, 641)),
    ("half", 8, (683, 577, 225), (699, 583, 327)), ("half", 16, (343, 329, 782), (401, 305, 557)),
    ("long", 1, (385, 8245, 2), (705, 5425, 1)), ("long", 2, (1735, 1159, 100), (1683, 1179, 48)), ("long", 4, (1227, 803, 164), (1467, 975, 83)),
    ("long", 8, (647, 789, 576), (715, 869, 333)),
    ("wide", 1, (899, 8373, 1), None), ("wide", 1, (1021, 16383, 16), None),
]
LISTED = [(form, n, shape, types) for form, n, half, full in SHAPES for shape, types in ((half, ("f16", "bf16")), (full, ("f32",))) if shape]


@pytest.fixture(scope="module")
def choice(tmp_path_factory):
    """(M, N, blocks, fp32) of many -> (form, slices) of each"""
    d = tmp_path_factory.mktemp("choice")
    (d / "ask.cc").write_text('#include "f8_choice.hpp"\n#include <cstdio>\nint main() {\n  long long M, N; int b, f;\n'
                              '  while (scanf("%%lld %%lld %%d %%d", &M, &N, &b, &f) == 4) {\n    const auto c = p0::f8_choice(M, N, b, f, %d, %d);\n'
                              '    printf("%%d %%d\\n", c.form, c.slices);\n  }\n}\n' % (CUS, PART))
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I" + CSRC, str(d / "ask.cc"), "-o", str(d / "ask")], check=True)

    def ask(shapes):
        out = subprocess.run([str(d / "ask")], input="".join("%d %d %d %d\n" % s for s in shapes), capture_output=True, text=True, check=True).stdout
        return [(FORMS[f] if f >= 0 else None, n) for f, n in (map(int, line.split()) for line in out.splitlines())]
    return ask


def test_each_shape_takes_the_form_that_it_stands_for(choice):
    got = choice([(*shape, int("f32" in types)) for _, _, shape, types in LISTED])
    assert [(form, n) for form, n, _, _ in LISTED] == got


def test_no_form_is_left_out(choice):
    """of shapes over the whole range, each form with its type of results and one, two or three, or more slices is listed"""
    rng = random.Random(5)

    def log(lo, hi):
        return int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))
    shapes = [(log(1, 2600), log(1, 18432), log(1, 1000), rng.randint(0, 1)) for _ in range(40000)]
    kind = lambda form, n, f32: (form, bool(f32), min(n, 4) // 2)  # noqa: E731
    listed = {kind(form, n, "f32" in types) for form, n, _, types in LISTED}
    missing = {kind(*c, s[3]): s for c, s in zip(choice(shapes), shapes)}
    assert not [(k, missing[k]) for k in missing if k not in listed]


def test_slices_have_blocks_of_their_own_and_fit_the_workspace(choice):
    rng = random.Random(6)
    bn, bm = dict(small=64, low=128, half=128, long=128), dict(small=64, low=64, half=128, long=256)
    shapes = [(rng.randint(17, 2600), rng.randint(1, 9300), rng.randint(1, 1000), rng.randint(0, 1)) for _ in range(20000)]
    for (M, N, blocks, _), (form, n) in zip(shapes, choice(shapes)):
        assert n >= 1 and (n - 1) * -(-blocks // n) < blocks
        if n > 1:
            assert -(-M // bm[form]) * -(-N // bn[form]) * n * bm[form] * bn[form] <= PART


def test_the_largest_products_have_a_form(choice):
    """rows and outputs at their limits, as far as an operand and the result fit the card (288 GB)"""
    rng = random.Random(7)
    for f32 in (0, 1):
        shapes = [(1 << 30, 64, 1, f32), (1 << 30, 100, 1, f32), (1, 1 << 26, 33, f32), (16, 1 << 26, 33, f32), (17, 1 << 26, 33, f32), (1000, 1 << 26, 16, f32)]
        while len(shapes) < 2000:
            M, N, b = (int(2 ** rng.uniform(0, k)) for k in (30, 26, 13))
            if M * N * (4 if f32 else 2) + (M + N) * b * 128 < 288e9:
                shapes.append((M, N, b, f32))
        assert None not in [form for form, _ in choice(shapes)]


def operands(rng, M, N, K):
    xc, wc = rng.integers(0, 254, (M, K), np.uint8), rng.integers(0, 254, (N, K), np.uint8)
    xc[(xc & 127) == 127], wc[(wc & 127) == 127] = 0, 0
    xs = (np.exp(rng.standard_normal((K // 128, M))) * 1e-3).astype(np.float32)
    ws = (np.exp(rng.standard_normal((f8.blocks(N), K // 128))) * 1e-4).astype(np.float32)
    return xc, xs, wc, ws


def product(ops, N, type_):
    xc, xs, wc, ws = ops
    M, K = xc.shape
    dv = [Rows(o.dtype, *o.shape, raw=o) for o in ops]
    y = Rows(RAW[type_], M, N)
    capi.f8_gemm(capi.f8_gemm_args(x=dv[0].ptr, xs=dv[1].ptr, w=dv[2].ptr, ws=dv[3].ptr, M=M, N=N, K=K, type=capi.TYPE[type_], y=y.ptr))
    got = from_type(y.read(), type_).reshape(M, N)
    for r in dv + [y]:
        r.free()
    return got


def sample_near(got, ops, type_, m, n):
    """rows m and outputs n of a product against float64"""
    xc, xs, wc, ws = ops
    K = xc.shape[1]
    x = f8.values(xc[m], np.ascontiguousarray(xs[:, m]))
    w = (f8.VALUES[wc[n]].reshape(len(n), -1, 128) * ws.astype(np.float64)[n // 128][..., None]).reshape(len(n), K)
    want, total = x @ w.T, np.abs(x) @ np.abs(w).T
    bound = (128 + 2 * K / 128) * 2.0 ** -23 * total
    if type_ != "f32":
        bound += 7 * 2.0 ** -13 * largest_of_8(x, w)
    err = np.abs(got[np.ix_(m, n)] - want)
    assert (err <= bound + HALF[type_] * (np.abs(want) + bound) + TINY[type_]).all(), (err / np.maximum(bound, 1e-30)).max()


def largest_of_8(x, w):
    """the sum over groups of 8 consecutive k of a group's largest product"""
    out = np.zeros((len(x), len(w)))
    a, b = np.abs(x).reshape(len(x), -1, 8), np.abs(w).reshape(len(w), -1, 8)
    for k in range(a.shape[1]):
        out += (a[:, None, k] * b[None, :, k]).max(2)
    return out


def sample(rng, n, tile):
    """the first and the last, both sides of each 8th tile's border, and some between"""
    edges = np.arange(tile, n, tile)[::8]
    return np.unique(np.clip(np.r_[0, n - 1, edges, edges - 1, rng.integers(0, n, 24)], 0, n - 1))


@pytest.mark.gpu
@pytest.mark.parametrize("form,slices,shape,type_", [(f, n, s, t) for f, n, s, types in LISTED for t in types])
def test_form(dev, form, slices, shape, type_):
    M, N, blocks = shape
    rng = np.random.default_rng(M + N)
    ops = operands(rng, M, N, 128 * blocks)
    sample_near(product(ops, N, type_), ops, type_, sample(rng, M, 64), sample(rng, N, 64))


@pytest.mark.gpu
@pytest.mark.parametrize("form,slices,shape,type_", [(f, n, s, t) for f, n, s, types in LISTED for t in types if t != "f16" or f == "wide"])
def test_values_that_are_not_finite(dev, form, slices, shape, type_):
    """a NaN code makes its row of the results NaN, one of the weight its column, in the first, a middle and the last block of k and at the lowest and the highest
    place of 8; no other value changes, though the matrix instructions take 16 rows and columns, and 8 k, together"""
    M, N, blocks = shape
    K = 128 * blocks
    rng = np.random.default_rng(M + N)
    ops = operands(rng, M, N, K)
    clean = product(ops, N, type_)
    at = [0, 7, (blocks // 2) * 128 + 63, (blocks - 1) * 128, K - 1]
    rows, cols = np.unique(rng.integers(0, M, 5))[:max(1, M // 2)], np.unique(rng.integers(0, N, 5))[:max(1, N // 2)]
    for i, r in enumerate(rows):
        ops[0][r, at[i]] = (0x7F, 0xFF)[i % 2]
    for i, r in enumerate(cols):
        ops[2][r, at[4 - i]] = (0xFF, 0x7F)[i % 2]
    got = product(ops, N, type_)
    nan = np.zeros((M, N), bool)
    nan[rows], nan[:, cols] = True, True
    assert np.array_equal(np.isnan(got), nan) and np.isfinite(clean).all()
    assert np.array_equal(got[~nan], clean[~nan])


CUT = [("few32", (29, 133, 9)), ("few32w", (33, 2111, 1)), ("few64", (1149, 737, 16)), ("small", (135, 331, 241)), ("low", (129, 5921, 1)), ("half", (199, 8249, 1)),
       ("long", (1735, 1159, 100)), ("wide", (1021, 16383, 16))]


@pytest.mark.gpu
@pytest.mark.parametrize("form,shape", CUT)
@pytest.mark.parametrize("cancel", [False, True])
def test_outliers_beside_small_values(dev, form, shape, cancel):
    """one large product and seven small ones in each 8 consecutive k, the large ones of two neighbouring 8s the same with opposite signs (cancel) or not. 16-bit
    results lose at most 7 * 2^-13 of the largest of each 8 (sample_near's bound), where that is more than a share of the result; fp32 results lose none"""
    M, N, blocks = shape
    K = 128 * blocks
    rng = np.random.default_rng(M)
    small = rng.choice([15.0, 13.0, 0.9375, 7.5, 2.0], (M, K))
    x = small.copy()
    x[:, 0::8] = rng.choice([448.0, 256.0, 240.0], (M, K // 16)).repeat(2, 1)
    w = np.ones((N, K))
    w[:, 0::8] = rng.choice([448.0, 256.0], (N, K // 16)).repeat(2, 1)
    if cancel:
        w[:, 8::16] *= -1
    ops = f8.encode(x), np.full((blocks, M), 2.0 ** -10, np.float32), f8.encode(w), np.full((f8.blocks(N), blocks), 2.0 ** -10, np.float32)
    m, n = sample(rng, M, 64), sample(rng, N, 64)
    for type_ in ("f16", "bf16", "f32"):
        sample_near(product(ops, N, type_), ops, type_, m, n)
