"""GPU parity of the 4-bit cache (kv_put, kv_get) and its attention (kv_attn) with their CPU restatement in float64.

The cache's bytes and the values read back are exact. Attention: f32 queries and probabilities are pairs of fp16 values, 22
bits each, the scores here stay below 32, and a probability's exponent is rounded in fp32 (32 * 1.44 * 2^-24 = 3e-6 at the
most): 5e-6 relative L2 holds all of it. f16 and bf16 outputs are rounded once, at most half a unit in 11 and 8 bits
(2^-12, 2^-9), and f16 / bf16 probabilities may be held in fp16: 2 * 2^-11 and 2 * 2^-8 bound both.
"""
import numpy as np
import pytest

from oracle import kvcache as KV
from p0pc0rn_amd import capi
from tests.conftest import rel_l2

pytestmark = pytest.mark.gpu
BOUND = {"f32": 5e-6, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}
NAN = 0x7FC00000


def to_type(x, type_):
    """float array -> (the bytes of a type, the values they stand for)"""
    x = np.ascontiguousarray(x, np.float32)
    if type_ == "f32":
        return x, x.astype(np.float64)
    if type_ == "f16":
        h = x.astype(np.float16)
        return h, h.astype(np.float64)
    u = x.view(np.uint32).astype(np.uint64)
    h = ((u + 0x7FFF + (u >> 16 & 1)) >> 16).astype(np.uint16)
    h = np.where(np.isnan(x), np.uint16(0x7FC0), h).astype(np.uint16)
    return h, (h.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def from_type(raw, type_):
    if type_ == "bf16":
        return (raw.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return raw.view(np.float16 if type_ == "f16" else np.float32).astype(np.float64)


def size_of(type_):
    return 4 if type_ == "f32" else 2


class Held:
    """a cache on the device and the same on the host: random bytes everywhere, rows for every sequence's tokens"""

    def __init__(self, lens, D, H, page, seed, spare=3, sigma=1.0, cols=None, special=None):
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lens]
        self.cols = cols or max(need + [1]) + 1
        P = sum(need) + spare
        self.c = KV.Cache(P, page, H, D, seed=seed)
        order = rng.permutation(P)
        self.table = np.full((len(lens), self.cols), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.len = np.array(lens, np.int32)
        for b, n in enumerate(lens):
            for h in range(H):
                k, v = (rng.standard_normal((n, D)).astype(np.float32) * sigma for _ in "kv")
                if special:
                    special(b, h, k, v)
                for t in range(n):
                    self.c.write(self.table[b, t // page], t % page, h, k[t], v[t])
        self.send()

    def send(self):
        self.pool_b, self.table_b, self.len_b = capi.to_device(self.c.pool), capi.to_device(self.table), capi.to_device(self.len)

    def kv(self, **kw):
        c = self.c
        base = dict(pages=self.pool_b, n_pages=c.n_pages, page=c.page, heads=c.heads, dim=c.dim, table=self.table_b, cols=self.cols,
                    len=self.len_b)
        base.update(kw)
        return capi.kv(**base)

    def free(self):
        for b in (self.pool_b, self.table_b, self.len_b):
            b.free()


def run_attn(c, q, type_, rows=None, pad=(0, 0, 0), shift=0, **kw):
    """attention of q [B, M, heads, D] with gaps of `pad` elements after each head, row and sequence, the buffers `shift` elements
    past their start -> (values, the raw output with its gaps left out checked to be untouched)"""
    B, M, Hq, D = q.shape
    ldh = D + pad[0]
    ldm = Hq * ldh + pad[1]
    ldb = M * ldm + pad[2]
    raw, exact = to_type(q, type_)
    size = size_of(type_)
    idx = shift + (np.arange(B)[:, None, None, None] * ldb + np.arange(M)[:, None, None] * ldm + np.arange(Hq)[:, None] * ldh + np.arange(D))
    flat = np.zeros(shift + B * ldb + 8, raw.dtype)
    flat[idx] = raw
    qb = capi.to_device(flat)
    yb = capi.Buffer((flat.nbytes + 15) // 16 * 16).fill_u32(NAN)
    rb = None if rows is None else capi.to_device(np.asarray(rows, np.int32))
    capi.kv_attn(capi.kv_attn_args(kv=c.kv(), B=B, M=M, rows=rb, heads=Hq, type=capi.KV_TYPE[type_], q=qb.ptr + shift * size,
                                   q_ldb=ldb, q_ldm=ldm, q_ldh=ldh, y=yb.ptr + shift * size, y_ldb=ldb, y_ldm=ldm, y_ldh=ldh, **kw))
    got = yb.read(flat.dtype, flat.size)
    gaps = np.ones(flat.size, bool)
    gaps[idx] = False
    fresh = np.full(flat.nbytes // 4 + 1, NAN, np.uint32).view(flat.dtype)[:flat.size]
    assert np.array_equal(got[gaps].view(np.uint8), fresh[gaps].view(np.uint8)), "written outside the rows"
    for b in (qb, yb, rb):
        if b:
            b.free()
    return from_type(np.ascontiguousarray(got[idx]), type_), exact


def check(got, want, type_):
    assert np.all(np.isfinite(got))
    assert rel_l2(got, want) <= BOUND[type_], rel_l2(got, want)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
def test_put_writes_the_bytes_and_get_reads_the_values(dev, D, type_):
    H, page, lens, rows, M = 3, 64, [70, 0, 33, 130], [41, 0, 33, 2], 41
    c = Held(lens, D, H, page, seed=D)
    rng = np.random.default_rng(D + 1)
    k, v = (rng.standard_normal((4, M, H, D)) * np.exp(2 * rng.standard_normal((4, M, H, 1))) for _ in "kv")
    k[0, 3, 1, 7], v[0, 5, 2, D - 1], k[2, 0, 0, 40] = np.inf, np.nan, -np.inf    # tokens that are no numbers
    k[0, 0, 0, :], v[3, 0, 1, 32:64] = 0.0, 1e-12                                 # blocks of nothing, of next to nothing
    v[0, 1, 0, 3] = 60000.0 if type_ == "f16" else 1e7                            # past the largest that is held
    raw = [to_type(x, type_) for x in (k, v)]
    kb, vb = (capi.to_device(r) for r, _ in raw)
    rb = capi.to_device(np.array(rows, np.int32))
    args = dict(kv=c.kv(), B=4, M=M, rows=rb, type=capi.KV_TYPE[type_])
    capi.kv_put(capi.kv_rows_args(k=kb, v=vb, **args))
    for b, n in enumerate(rows):
        for i in range(n):
            t = lens[b] - n + i
            for h in range(H):
                c.c.write(c.table[b, t // page], t % page, h, raw[0][1][b, i, h], raw[1][1][b, i, h])
    assert np.array_equal(c.pool_b.read(np.uint8, c.c.pool.size).reshape(c.c.pool.shape), c.c.pool)
    ko, vo = (capi.Buffer(r.nbytes).fill_u32(NAN) for r, _ in raw)
    capi.kv_get(capi.kv_rows_args(k=ko, v=vo, **args))
    with np.errstate(invalid="ignore"):
        hk, hv = KV.held(raw[0][1], raw[1][1])
    for buf, want in ((ko, hk), (vo, hv)):
        got = from_type(buf.read(raw[0][0].dtype), type_).reshape(4, M, H, D)
        for b, n in enumerate(rows):
            assert np.array_equal(got[b, :n], want[b, :n], equal_nan=True)
            assert not got[b, n:].any()
    for b in (kb, vb, rb, ko, vo):
        b.free()
    c.free()


def test_rows_at_given_tokens_with_strides_and_pages_that_are_none(dev):
    D, H, page, M = 128, 2, 32, 40
    c = Held([100, 64], D, H, page, seed=5)
    c.table[0, 1], c.table[1, 0] = -1, 99999            # the pages of tokens 32-63, 0-31
    c.send()
    before = c.pool_b.read(np.uint8, c.c.pool.size)
    rng = np.random.default_rng(6)
    ldh, ldm, ldb = D + 4, H * (D + 4) + 6, M * (H * (D + 4) + 6) + 10
    flat = [rng.standard_normal(2 * ldb).astype(np.float32) for _ in "kv"]
    at = np.array([20, -3], np.int32)                   # two calls' worth of tokens before the first and past the last page
    kb, vb, ab = capi.to_device(flat[0]), capi.to_device(flat[1]), capi.to_device(at)
    args = dict(kv=c.kv(), B=2, M=M, at=ab, ldb=ldb, ldm=ldm, ldh=ldh)
    capi.kv_put(capi.kv_rows_args(k=kb, v=vb, **args))
    view = lambda x, b, i, h: x[b * ldb + i * ldm + h * ldh:][:D]  # noqa: E731
    want = np.zeros((2, 2, M, H, D))
    c.c.pool = before.reshape(c.c.pool.shape).copy()
    for b in range(2):
        for i in range(M):
            t = at[b] + i
            if t < 0 or t >= c.len[b] or not 0 <= c.table[b, t // page] < c.c.n_pages:
                continue
            for h in range(H):
                c.c.write(c.table[b, t // page], t % page, h, view(flat[0], b, i, h), view(flat[1], b, i, h))
                want[:, b, i, h] = KV.held(view(flat[0], b, i, h), view(flat[1], b, i, h))
    assert np.array_equal(c.pool_b.read(np.uint8, before.size), c.c.pool.ravel())
    ko, vo = capi.to_device(np.full(2 * ldb, 7, np.float32)), capi.to_device(np.full(2 * ldb, 7, np.float32))
    capi.kv_get(capi.kv_rows_args(k=ko, v=vo, **args))
    for n, buf in enumerate((ko, vo)):
        got = buf.read(np.float32, 2 * ldb)
        for b in range(2):
            for i in range(M):
                for h in range(H):
                    assert np.array_equal(view(got, b, i, h), want[n, b, i, h])
                    view(got, b, i, h)[:] = 7
        assert np.all(got == 7)                         # nothing between the rows
    for b in (kb, vb, ab, ko, vo):
        b.free()
    c.free()


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
def test_one_row_over_ragged_lengths(dev, D, type_):
    lens = [1, 0, 31, 32, 33, 64, 100, 517]
    c = Held(lens, D, 2, 64, seed=D + 7)
    q = 1.5 * np.random.default_rng(D).standard_normal((len(lens), 1, 8, D))
    got, exact = run_attn(c, q, type_)
    want = KV.attention(c.c, c.table, c.len, exact)
    assert not got[1].any()                             # a sequence of no tokens
    check(got, want, type_)
    c.free()


@pytest.mark.parametrize("M,G,H,page", [(5, 4, 2, 32), (5, 8, 1, 128), (16, 1, 3, 64), (2, 16, 1, 256), (37, 4, 1, 64), (70, 3, 2, 32),
                                        (150, 1, 1, 1024)])
def test_many_rows_are_causal(dev, M, G, H, page):
    D, lens = 128, [M, M + 133, M // 2]                 # the last has fewer tokens than rows: the rows before its first see nothing
    c = Held(lens, D, H, page, seed=M)
    q = np.random.default_rng(M).standard_normal((3, M, G * H, D))
    got, exact = run_attn(c, q, "f32")
    want = KV.attention(c.c, c.table, c.len, exact)
    assert not got[2, :M - M // 2].any()
    check(got, want, "f32")
    c.free()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (32, 4), (64, 40), (100, 200), (500, 0), (3, 100000), (1 << 40, 0)])
@pytest.mark.parametrize("D,M", [(64, 1), (256, 5), (128, 40)])
def test_windows_and_first_tokens(dev, window, sinks, D, M):
    lens = [300, 60, 45, M]
    c = Held(lens, D, 1, 32, seed=window % 1000 + M)
    q = np.random.default_rng(sinks % 1000).standard_normal((4, M, 4, D))
    rows = [M, min(M, 3), 0, M]
    got, exact = run_attn(c, q, "f32", rows=rows, window=window, sinks=sinks)
    want = KV.attention(c.c, c.table, c.len, exact, rows=rows, window=window, sinks=sinks)
    assert not got[2].any() and not got[1, rows[1]:].any()
    check(got, want, "f32")
    c.free()


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,M,G,H", [(64, 64, 4, 2), (64, 300, 1, 1), (128, 86, 3, 2), (128, 64, 8, 1), (128, 257, 1, 2)])
def test_rows_that_share_converted_runs(dev, D, type_, M, G, H):
    """256 rows of a key head and more, over lengths of which some are in parts"""
    lens = [M, M + 333, M // 2, 0, 1500]
    c = Held(lens, D, H, 64, seed=M + D, cols=2000)          # room for lengths at which sharing pays
    rows = [M, M - 1, M, M, M]
    q = np.random.default_rng(M).standard_normal((5, M, G * H, D))
    got, exact = run_attn(c, q, type_, rows=rows)
    again, _ = run_attn(c, q, type_, rows=rows)
    assert np.array_equal(got, again)
    want = KV.attention(c.c, c.table, c.len, exact, rows=rows)
    assert not got[2, :M - M // 2].any() and not got[3].any() and not got[1, M - 1:].any()
    check(got, want, type_)
    c.free()


@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 3), (100, 200), (333, 4), (3, 100000)])
@pytest.mark.parametrize("D", [64, 128])
def test_windows_of_rows_that_share_converted_runs(dev, D, window, sinks):
    M = 130
    c = Held([900, 140, 60], D, 1, 32, seed=window + D, cols=5000)
    c.table[0, 3], c.table[0, 26] = -1, c.c.n_pages          # tokens 96-127 and 832-863 have no page
    c.send()
    G = 2 if sinks > 1000 else 320                           # of short windows the rows have to be many
    q = np.random.default_rng(sinks % 1000).standard_normal((3, M, G, D))
    got, exact = run_attn(c, q, "f16", window=window, sinks=sinks, pad=(8, 3, 0), shift=2)
    check(got, KV.attention(c.c, c.table, c.len, exact, window=window, sinks=sinks), "f16")
    c.free()


def test_a_token_that_is_no_number_among_shared_runs(dev):
    M, n, D = 256, 420, 128

    def special(b, h, k, v):
        k[n - 40, 5] = np.inf                               # rows 216.. see it
    c = Held([n], D, 1, 32, seed=5, special=special, cols=13000)
    q = np.random.default_rng(5).standard_normal((1, M, 1, D))
    got, exact = run_attn(c, q, "f32")
    with np.errstate(invalid="ignore"):
        want = KV.attention(c.c, c.table, c.len, exact)
    assert np.isnan(got[0, M - 40:]).all() and not np.isnan(got[0, :M - 40]).any()
    check(got[~np.isnan(got)], want[~np.isnan(want)], "f32")
    c.free()


@pytest.mark.parametrize("D,M,G,n,type_", [(64, 1, 4, 9000, "f32"), (128, 3, 8, 5000, "f16"), (256, 1, 16, 9000, "bf16"), (64, 256, 1, 3000, "f32"),
                                           (128, 128, 2, 3000, "f16"), (512, 1, 8, 9000, "f32"), (512, 3, 8, 3000, "f16"), (512, 10, 8, 3000, "bf16")])
def test_many_parts_of_one_item(dev, D, M, G, n, type_):
    c = Held([n], D, 1, 128, seed=D + M, cols=3200 if M > 100 else None)
    q = np.random.default_rng(D + M).standard_normal((1, M, G, D))
    for most in (0, n):
        got, exact = run_attn(c, q, type_, max_len=most)
        check(got, KV.attention(c.c, c.table, c.len, exact), type_)
    c.free()


@pytest.mark.parametrize("B,H,D", [(150, 2, 64), (70, 3, 128), (33, 4, 256)])
def test_many_sequences_of_very_different_lengths(dev, B, H, D):
    """few long ones in parts beside short ones and empty ones"""
    rng = np.random.default_rng(B)
    lens = np.where(rng.random(B) < 0.5, 0, rng.integers(1, 40, B))
    lens[[0, B // 2, B - 1]] = 1700, 900, 1333
    c = Held(lens.tolist(), D, H, 64, seed=B)
    q = rng.standard_normal((B, 1, 2 * H, D))
    got, exact = run_attn(c, q, "f32")
    assert not got[lens == 0].any()
    check(got, KV.attention(c.c, c.table, c.len, exact), "f32")
    c.free()


def test_pages_outside_the_window_may_be_given_up(dev):
    D, window, sinks = 128, 50, 5
    c = Held([400, 333], D, 2, 32, seed=3)
    q = np.random.default_rng(3).standard_normal((2, 2, 4, D))
    want_full = KV.attention(c.c, c.table, c.len, q.astype(np.float32), window=window, sinks=sinks)
    for b in range(2):
        j = np.arange(c.cols)
        c.table[b, ((j + 1) * 32 <= c.len[b] - 2 - window + 1) & (j * 32 >= sinks)] = -1
    assert (c.table[0] == -1).sum() > 5
    c.send()
    got, _ = run_attn(c, q, "f32", window=window, sinks=sinks)
    check(got, want_full, "f32")
    c.free()


def test_tokens_of_no_page_are_seen_by_no_row(dev):
    D = 256
    c = Held([200, 90], D, 1, 32, seed=11)
    c.table[0, 2], c.table[0, 6], c.table[1, :] = -5, c.c.n_pages, -1
    c.send()
    q = np.random.default_rng(4).standard_normal((2, 3, 2, D))
    got, exact = run_attn(c, q, "f32")
    assert not got[1].any()
    check(got, KV.attention(c.c, c.table, c.len, exact), "f32")
    c.free()


def test_a_length_past_the_table_counts_as_the_table(dev):
    c = Held([96], 64, 1, 32, seed=2, cols=3)
    c.len[0] = 1000
    c.send()
    q = np.random.default_rng(4).standard_normal((1, 2, 2, 64))
    got, exact = run_attn(c, q, "f32")
    check(got, KV.attention(c.c, c.table, c.len, exact), "f32")
    c.free()


@pytest.mark.parametrize("D,type_", [(128, "f32"), (256, "f16"), (64, "bf16")])
@pytest.mark.parametrize("pad,shift", [((0, 0, 0), 1), ((1, 0, 0), 0), ((8, 3, 0), 0), ((8, 16, 8), 8), ((0, 0, 5), 3)])
def test_strides_and_alignments(dev, D, type_, pad, shift):
    c = Held([75, 130], D, 2, 64, seed=9)
    q = np.random.default_rng(shift).standard_normal((2, 3, 4, D))
    got, exact = run_attn(c, q, type_, pad=pad, shift=shift)
    check(got, KV.attention(c.c, c.table, c.len, exact), type_)
    c.free()


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_a_token_that_is_no_number_reaches_the_rows_that_see_it_alone(dev, D):
    M, n = 6, 80

    def special(b, h, k, v):
        if h == 0:
            k[n - 3, 5] = np.nan                        # rows 3.. see it
        else:
            v[10, D - 1] = np.inf                       # outside the window of 40: no row does
    c = Held([n], D, 2, 32, seed=D, special=special)
    q = np.random.default_rng(D).standard_normal((1, M, 4, D))
    got, exact = run_attn(c, q, "f32", window=40, sinks=2)
    with np.errstate(invalid="ignore"):
        want = KV.attention(c.c, c.table, c.len, exact, window=40, sinks=2)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got).any()
    assert np.isnan(got[0, 3:, :2]).all() and not np.isnan(got[0, :3]).any() and not np.isnan(got[0, :, 2:]).any()
    check(got[~np.isnan(got)], want[~np.isnan(want)], "f32")
    c.free()


def test_queries_of_any_magnitude(dev):
    """one row that is 0, one with an infinity, one with a NaN, very large and very small ones beside ordinary ones"""
    D = 128
    c = Held([90], D, 1, 32, seed=1)
    q = np.random.default_rng(1).standard_normal((1, 8, 2, D))
    q[0, 0], q[0, 1] = 0.0, q[0, 1] * 1e-30
    q[0, 2] *= 50.0
    q[0, 3, 0, 5], q[0, 4, 1, 9] = np.nan, np.inf
    got, exact = run_attn(c, q, "f32")
    with np.errstate(invalid="ignore", over="ignore"):
        want = KV.attention(c.c, c.table, c.len, exact)
    assert np.isnan(got[0, 3, 0]).all() and np.isnan(got[0, 4, 1]).all()
    fine = np.ones((1, 8, 2, D), bool)
    fine[0, 3, 0] = fine[0, 4, 1] = False
    fine[0, 2] = False                                  # scores of some hundreds: their own bound, 300 * 1.44 * 2^-22
    check(got[fine], want[fine], "f32")
    assert rel_l2(got[0, 2], want[0, 2]) <= 1.1e-4
    c.free()


def test_a_scale_of_the_callers(dev):
    c = Held([70], 64, 1, 64, seed=8)
    q = np.random.default_rng(2).standard_normal((1, 1, 8, 64))
    got, exact = run_attn(c, q, "f32", scale=0.5)
    check(got, KV.attention(c.c, c.table, c.len, exact, scale=0.5), "f32")
    c.free()


@pytest.mark.parametrize("D,M,G", [(256, 1, 4), (512, 5, 8), (128, 3, 2)])
def test_a_long_sequence_in_parts_and_twice_the_same(dev, D, M, G):
    """the work over many workgroups, joined; any max_len is right, and a call's repetition is the same bit for bit"""
    n = 3000
    c = Held([n, 40], D, 1, 64, seed=D)
    q = np.random.default_rng(D).standard_normal((2, M, G, D))
    want = None
    for most in (0, 1, 64, 3000, 1 << 20):
        got, exact = run_attn(c, q, "f32", max_len=most)
        again, _ = run_attn(c, q, "f32", max_len=most)
        assert np.array_equal(got, again)
        if want is None:
            want = KV.attention(c.c, c.table, c.len, exact)
        check(got, want, "f32")
    c.free()


def test_a_pool_past_four_gigabytes(dev):
    """pages whose bytes lie beyond 32-bit offsets"""
    D, H, page = 256, 2, 64
    size = capi.kv_page_bytes(page, H, D)
    P = (5 << 30) // size
    pool = capi.Buffer(P * size)
    pool.fill_u32(0x41414141, P * size // 4)
    c = Held([150], D, H, page, seed=21)
    far = [P - 1, 7, P - 130]
    for j, pg in enumerate(far):
        pool.upload(c.c.pool[c.table[0, j]], off=pg * size)
    table = capi.to_device(np.array(far, np.int32))
    q = np.random.default_rng(5).standard_normal((1, 2, 4, D)).astype(np.float32)
    qb, yb = capi.to_device(q), capi.Buffer(q.nbytes)
    kv = c.kv(pages=pool, n_pages=P, table=table, cols=3)
    capi.kv_attn(capi.kv_attn_args(kv=kv, B=1, M=2, heads=4, q=qb, y=yb))
    check(yb.read(np.float32, q.size).reshape(q.shape), KV.attention(c.c, c.table, c.len, q), "f32")
    new = np.random.default_rng(6).standard_normal((2, 2, H, D)).astype(np.float32)
    kb, vb, ko, vo = capi.to_device(new[0]), capi.to_device(new[1]), capi.Buffer(new[0].nbytes), capi.Buffer(new[0].nbytes)
    capi.kv_put(capi.kv_rows_args(kv=kv, B=1, M=2, k=kb, v=vb))
    capi.kv_get(capi.kv_rows_args(kv=kv, B=1, M=2, k=ko, v=vo))
    hk, hv = KV.held(new[0], new[1])
    assert np.array_equal(ko.read(np.float32, hk.size), hk.ravel()) and np.array_equal(vo.read(np.float32, hv.size), hv.ravel())
    for b in (pool, table, qb, yb, kb, vb, ko, vo):
        b.free()
    c.free()


def test_recorded_calls_replay(dev):
    """a token's put and attention in a recording, replayed with other work between, each time against the eager result"""
    D, H, n = 128, 2, 200
    c = Held([n, n - 70], D, H, 64, seed=13)
    rng = np.random.default_rng(13)
    k, v = (rng.standard_normal((2, 1, H, D)).astype(np.float32) for _ in "kv")
    q = rng.standard_normal((2, 1, 8, D)).astype(np.float32)
    kb, vb, qb, yb = capi.to_device(k), capi.to_device(v), capi.to_device(q), capi.Buffer(q.nbytes)
    put = capi.kv_rows_args(kv=c.kv(), B=2, M=1, k=kb, v=vb)
    att = capi.kv_attn_args(kv=c.kv(), B=2, M=1, heads=8, q=qb, y=yb)
    capi.kv_put(put)
    capi.kv_attn(att)
    want = yb.read(np.float32, q.size)
    rec = capi.record(lambda: (capi.kv_put(put), capi.kv_attn(att)))
    for _ in range(4):
        yb.fill_u32(NAN)
        rec.replay()
        assert np.array_equal(yb.read(np.float32, q.size), want)
        capi.kv_attn(att)
        capi.done()
    rec.free()
    for b in (kb, vb, qb, yb):
        b.free()
    c.free()


def test_no_rows_and_no_sequences_do_nothing(dev):
    c = Held([10], 64, 1, 32, seed=1)
    yb = capi.Buffer(1024).fill_u32(NAN)
    for B, M in ((0, 1), (1, 0)):
        capi.kv_attn(capi.kv_attn_args(kv=c.kv(), B=B, M=M, heads=1, q=yb, y=yb))
        capi.kv_put(capi.kv_rows_args(kv=c.kv(), B=B, M=M, k=yb, v=yb))
        capi.kv_get(capi.kv_rows_args(kv=c.kv(), B=B, M=M, k=yb, v=yb))
    assert np.all(yb.read(np.uint32) == NAN)
    assert np.array_equal(c.pool_b.read(np.uint8, c.c.pool.size), c.c.pool.ravel())
    yb.free()
    c.free()


def test_a_chain_being_built_refuses_them(dev):
    c = Held([10], 64, 1, 32, seed=1)
    capi.check(capi.lib().p0_chain_begin())
    try:
        with pytest.raises(capi.P0Error, match="kv_attn: only gemv"):
            capi.kv_attn(capi.kv_attn_args(kv=c.kv(), B=1, M=1, heads=1, q=c.pool_b, y=c.pool_b))
        with pytest.raises(capi.P0Error, match="kv_put: only gemv"):
            capi.kv_put(capi.kv_rows_args(kv=c.kv(), B=1, M=1, k=c.pool_b, v=c.pool_b))
    finally:
        h = capi.vp()
        capi.lib().p0_chain_end(capi.C.byref(h))
        if h.value:
            capi.lib().p0_chain_free(h)
    c.free()


@pytest.mark.parametrize("type_,most,rest,sigma", [("f32", 1e3, 1, 1), ("f32", 1e6, 1, 1), ("f32", 100, 0.01, 100), ("f16", 1000, 0.01, 100),
                                                   ("f16", 60000, 0.01, 100), ("f16", 60000, 3e-5, 1e4), ("bf16", 1e4, 1, 1), ("bf16", 1e7, 1, 1)])
@pytest.mark.parametrize("D,M,G,cols", [(64, 2, 2, None), (128, 3, 1, None), (256, 2, 2, None), (512, 2, 1, None), (64, 256, 1, 13000), (128, 256, 1, 13000)])
def test_a_channel_far_above_the_rest_of_its_row(dev, D, M, G, cols, type_, most, rest, sigma):
    """the keys are 0 in the large channel, so the scores are the small ones' alone, each of which has to be held to its own bits;
    256 rows are those that share converted runs"""
    def special(b, h, k, v):
        k *= sigma
        k[:, 5] = 0.0
    c = Held([90], D, 1, 32, seed=D, special=special, cols=cols)
    q = rest * np.random.default_rng(D + M).standard_normal((1, M, G, D))
    q[..., 5] = most
    got, exact = run_attn(c, q, type_)
    check(got, KV.attention(c.c, c.table, c.len, exact), type_)
    c.free()


@pytest.mark.parametrize("scale,size", [(1e-10, 1e-35), (1e-44, 1.0), (1e30, 1e30), (3e38, 1.0)])
@pytest.mark.parametrize("D,M,cols", [(128, 3, None), (512, 2, None), (64, 256, 13000)])
def test_scales_past_what_fp32_holds(dev, scale, size, D, M, cols):
    """scale times a query's power of two may be under the least fp32 number, or over the largest: rows whose scores are all next to
    nothing are means of what they see, and a score of exactly 0 stays one (the rows of zeros)"""
    c = Held([90], D, 1, 32, seed=D, cols=cols)
    q = size * np.random.default_rng(D).standard_normal((1, M, 2 if M < 9 else 1, D))
    if scale > 1:
        q[0, 0] = 0.0
    got, exact = run_attn(c, q, "f32", scale=scale)
    want = KV.attention(c.c, c.table, c.len, exact, scale=scale)
    if scale > 1:
        got, want = got[0, 0], want[0, 0]
    check(got, want, "f32")
    c.free()


@pytest.mark.parametrize("D,M,cols", [(64, 2, None), (128, 2, None), (256, 2, None), (512, 2, None), (64, 256, 13000), (128, 256, 13000)])
def test_f16_outputs_are_off_by_their_own_rounding(dev, D, M, cols):
    """whichever kernel takes the rows. An output is the rounding of a value off by d, |d| <= 5e-6 as f32's are: where that rounds as
    the exact value does the error is the exact value's own, else the exact value lies within d of the middle and the error is over
    its own by 2 d at the most"""
    c = Held([700], D, 1, 32, seed=D, cols=cols)
    q = 0.1 * np.random.default_rng(D + M).standard_normal((1, M, 16 if M < 9 else 1, D))
    got, exact = run_attn(c, q, "f16")
    want = KV.attention(c.c, c.table, c.len, exact)
    assert rel_l2(got, want) <= rel_l2(want.astype(np.float16), want) + 2 * BOUND["f32"]
    c.free()


def test_tables_of_more_runs_than_32_bits_count(dev):
    """34 groups of rows over a table of 2^31 tokens, of which 1300 are there: no parts, whose deal would count past 32 bits if they all were"""
    D, M, n = 256, 1060, 1300
    c = Held([n], D, 1, 1024, seed=3, cols=(1 << 21) - 1)
    q = np.random.default_rng(3).standard_normal((1, M, 1, D))
    got, exact = run_attn(c, q, "f32")
    check(got, KV.attention(c.c, c.table, c.len, exact), "f32")
    c.free()


@pytest.mark.parametrize("type_,size", [("f32", 1e4), ("f32", 1e6), ("f32", 1e8), ("f32", 1e15), ("f32", -1e30), ("f16", 6e4), ("bf16", 1e20)])
@pytest.mark.parametrize("D,M,cols", [(128, 3, None), (512, 2, None), (64, 256, 13000)])
def test_scores_of_any_magnitude(dev, D, M, cols, type_, size):
    """past 2^24 an fp32 score's neighbours are whole powers of two apart: a row is then its best token's value, and no NaN"""
    def special(b, h, k, v):
        k *= 1e3
    c = Held([90], D, 1, 32, seed=D + 1, cols=cols, special=special)
    q = size * np.random.default_rng(D).uniform(0.5, 1.0, (1, M, 2 if M < 9 else 1, D))
    got, exact = run_attn(c, q, type_)
    want = KV.attention(c.c, c.table, c.len, exact)
    check(got, want, type_)
    c.free()
