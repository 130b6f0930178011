"""kv_update and kv_compact against their CPU restatement (oracle/kvcache.py): every table entry, length, count, status word and
byte of the pool, in one workgroup and over the chip."""
import numpy as np
import pytest

from oracle import kvcache as KV
from p0pc0rn_amd import capi
from tests.test_kv_gpu import run_attn

pytestmark = pytest.mark.gpu
FRESH = 0x77777777


class Pool:
    """tables over a pool of random bytes, on both sides"""

    def __init__(self, table, length, page, n_pages, layers=1, H=1, D=64, seed=0, extra=0):
        self.table, self.len = np.ascontiguousarray(table, np.int32), np.asarray(length, np.int32)
        self.page, self.P, self.layers, self.H, self.D = page, n_pages, layers, H, D
        self.size = capi.kv_page_bytes(page, H, D) + extra
        self.pool = np.random.default_rng(seed).integers(0, 256, (layers, n_pages, self.size), np.uint8)
        self.bufs = [capi.to_device(x) for x in (self.pool, self.table, self.len)]

    def kv(self):
        return capi.kv(pages=self.bufs[0], n_pages=self.P, page_bytes=self.size, page=self.page, heads=self.H, dim=self.D,
                       table=self.bufs[1], cols=self.table.shape[1], len=self.bufs[2])

    def out(self, Bo, gap=0):
        cols = self.table.shape[1]
        self.outs = [capi.Buffer(max(16, 4 * n)).fill_u32(FRESH) for n in (Bo * (cols + gap), Bo, self.P, 4)]
        return self.outs

    def moved(self, moves):
        want = self.pool.copy()
        used = capi.kv_page_bytes(self.page, self.H, self.D)
        for a, b in moves:
            want[:, b, :used] = self.pool[:, a, :used]
        got = self.bufs[0].read(np.uint8, self.pool.size).reshape(self.pool.shape)
        assert np.array_equal(got, want)

    def free(self):
        for b in self.bufs + self.outs:
            b.free()


def check_update(pool, Bo, gap=0, ref=True, **kw):
    dev = {k: capi.to_device(np.asarray(v, np.int32)) for k, v in kw.items() if k in ("src", "keep", "grow") and v is not None}
    rest = {k: v for k, v in kw.items() if k not in ("src", "keep", "grow")}
    t, n, r, s = pool.out(Bo, gap)
    cols = pool.table.shape[1]
    capi.kv_update(capi.kv_update_args(kv=pool.kv(), B=len(pool.len), Bo=Bo, layers=pool.layers, table_out=t, out_ld=cols + gap, len_out=n,
                                       ref=r if ref else None, status=s, **dev, **rest))
    wt, wn, wr, ws, moves = KV.update(pool.table, pool.len, pool.page, pool.P, Bo, **kw)
    got = t.read(np.int32, Bo * (cols + gap)).reshape(Bo, cols + gap)
    assert s.read(np.int32, 4).tolist() == ws
    assert np.array_equal(got[:, :cols], wt)
    assert np.all(got[:, cols:] == FRESH)
    assert np.array_equal(n.read(np.int32, Bo), wn)
    count = r.read(np.int32, pool.P)
    assert np.array_equal(count, wr) if ref and wr is not None else np.all(count == FRESH)
    pool.moved(moves)
    for b in dev.values():
        b.free()
    return ws, moves


def beams(rng, groups, W, page, cols, P, longest):
    """searches whose beams share their first pages -> table, lengths"""
    B = groups * W
    table, length = np.full((B, cols), -1, np.int32), np.zeros(B, np.int32)
    pages = iter(rng.permutation(P))
    for s in range(groups):
        n = int(rng.integers(1, longest + 1))
        need = -(-n // page)
        split = int(rng.integers(0, need + 1))
        shared = [next(pages) for _ in range(split)]
        for w in range(W):
            b = s * W + w
            length[b] = n
            table[b, :need] = shared + [next(pages) for _ in range(need - split)]
    return table, length


@pytest.mark.parametrize("groups,W,page,longest,P", [(1, 1, 32, 1, 3), (1, 4, 64, 500, 80), (3, 5, 32, 200, 200), (8, 8, 64, 700, 900),
                                                     (2, 300, 32, 90, 2500), (40, 30, 32, 33, 3000), (2, 3, 32, 300, 20000)])
@pytest.mark.parametrize("seed", [0, 1])
def test_beams_go_on_from_their_parents(dev, groups, W, page, longest, P, seed):
    """small pools are one workgroup's, 1200 sequences and 20000 pages the chip's"""
    rng = np.random.default_rng(seed)
    cols = -(-(longest + 2) // page) + 1
    table, length = beams(rng, groups, W, page, cols, P, longest)
    src = (rng.integers(0, W, (groups, W)) + np.arange(groups)[:, None] * W).ravel()
    pool = Pool(table, length, page, P, layers=2 if P < 1000 else 1, seed=seed, extra=48 * seed)
    check_update(pool, groups * W, gap=seed * 3, src=src, grow_n=1)
    pool.free()


@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("seed", range(6))
def test_any_mix_of_forks_cuts_growth_and_windows(dev, big, seed):
    rng = np.random.default_rng(100 + seed)
    page, B, cols, P = 32, 12, 14, 13000 if big else 160
    table, length = beams(rng, 4, 3, page, cols, P, 300)
    table[rng.random(table.shape) < 0.05] = -1           # pages given up, entries that are no page
    table[rng.random(table.shape) < 0.03] = P + 5
    Bo = [12, 20, 5, 12, 1, 30][seed]
    src = rng.integers(-2, B + 2, Bo)
    keep = rng.integers(-5, 330, Bo)
    grow = rng.integers(-3, 90, Bo)
    pool = Pool(table, length, page, P, seed=seed)
    check_update(pool, Bo, ref=seed != 4, src=src, keep=keep, grow=grow, window=[0, 40, 1, 100, 64, 1 << 40][seed], sinks=[0, 4, 0, 70, 32, 5][seed])
    pool.free()


@pytest.mark.parametrize("big", [False, True])
def test_a_page_still_read_past_its_cut_is_copied(dev, big):
    """sequence 1 is sequence 0 cut in its second page and goes on there; 0 stays whole and does not grow"""
    P = 12500 if big else 9
    pool = Pool([[4, 2, 7, -1]], [90], 32, P)
    ws, moves = check_update(pool, 2, src=[0, 0], keep=[90, 40], grow=[0, 3])
    assert len(moves) == 1 and moves[0][0] == 2
    pool.free()


@pytest.mark.parametrize("big", [False, True])
def test_too_few_pages_or_columns_change_nothing(dev, big):
    P = 12300 if big else 8
    table = [[0, 1, 2, -1], [3, 4, -1, -1]] if not big else [list(range(4)), list(range(4, 8))]
    pool = Pool(table, [70, 64], 32, P)
    check_update(pool, 2, grow=[1, 300])                 # past the columns
    check_update(pool, 3, src=[0, 1, 0], grow=[1, 65, 0])
    check_update(pool, 1, src=[0], grow=[0x7FFFFFFF])
    pool.free()
    if not big:
        pool = Pool([[0, 1, 2, -1], [3, 4, -1, -1]], [70, 64], 32, 6)
        ws, _ = check_update(pool, 2, grow=[40, 33])     # three pages more, one there
        assert ws == [2, 1, 0, 0]
        pool.free()


def test_no_sequences(dev):
    pool = Pool([[1, 0]], [40], 32, 5)
    ws, _ = check_update(pool, 1, src=[-1])
    assert ws[1] == 5
    pool.free()


@pytest.mark.parametrize("B,page,longest,P", [(1, 32, 40, 2), (4, 64, 700, 96), (9, 32, 300, 97), (64, 64, 2000, 4096), (3, 32, 400, 12288),
                                              (5, 32, 300, 12289), (1100, 32, 1000, 36000), (2, 128, 5000, 50000)])
@pytest.mark.parametrize("seed", [0, 1])
def test_compact(dev, B, page, longest, P, seed):
    rng = np.random.default_rng(seed)
    cols = -(-longest // page) + seed
    length = rng.integers(0, longest + 1, B)
    order = rng.permutation(P)
    table = np.full((B, cols), -1, np.int32)
    at = 0
    for b in range(B):
        need = -(-int(length[b]) // page)
        table[b, :need] = order[np.arange(at, at + need) % P]
        at += need
    table[rng.random(table.shape) < 0.04] = -1
    if B > 2:
        table[1] = table[0]                              # shared pages move once
        length[1] = length[0]
    pool = Pool(table, length, page, P, layers=2 if P < 5000 else 1, seed=seed, extra=16 * seed)
    t, _, _, s = pool.out(B, 2)
    capi.kv_compact(capi.kv_compact_args(kv=pool.kv(), B=B, layers=pool.layers, table_out=t, out_ld=cols + 2, status=s))
    wt, ws, moves = KV.compact(table, length, page, P)
    got = t.read(np.int32, B * (cols + 2)).reshape(B, cols + 2)
    assert s.read(np.int32, 2).tolist() == ws
    assert np.array_equal(got[:, :cols], wt) and np.all(got[:, cols:] == FRESH)
    pool.moved(moves)
    pool.free()


def test_a_full_and_an_empty_pool_do_not_move(dev):
    pool = Pool([[2, 0], [1, 3]], [64, 50], 32, 4)
    t, _, _, s = pool.out(2)
    capi.kv_compact(capi.kv_compact_args(kv=pool.kv(), B=2, table_out=t, status=s))
    assert s.read(np.int32, 2).tolist() == [4, 0] and np.array_equal(t.read(np.int32, 4), pool.table.ravel())
    capi.kv_compact(capi.kv_compact_args(kv=pool.kv(), B=0, table_out=t, status=s))
    assert s.read(np.int32, 2).tolist() == [0, 0]
    pool.moved([])
    pool.free()


def test_attention_is_the_same_after_a_fork_and_a_compaction(dev):
    """two sequences of a shared prompt, forked, extended, compacted: the rows of each attend to what was put for it"""
    H, D, page = 2, 64, 32
    rng = np.random.default_rng(7)
    cache = KV.Cache(40, page, H, D, seed=1)
    pool = Pool([[30, 12, 25, -1, -1]], [70], page, 40, H=H, D=D)
    pool.bufs[0].upload(cache.pool)
    bufs = []

    def dev_of(x):
        bufs.append(capi.to_device(x))
        return bufs[-1]
    kv = lambda t, n: capi.kv(pages=pool.bufs[0], n_pages=40, page=page, heads=H, dim=D, table=t, cols=5, len=n)  # noqa: E731
    prompt = rng.standard_normal((2, 1, 70, H, D)).astype(np.float32)
    capi.kv_put(capi.kv_rows_args(kv=kv(pool.bufs[1], pool.bufs[2]), B=1, M=70, k=dev_of(prompt[0]), v=dev_of(prompt[1])))
    t, n, r, s = pool.out(2)
    capi.kv_update(capi.kv_update_args(kv=kv(pool.bufs[1], pool.bufs[2]), B=1, Bo=2, src=dev_of(np.zeros(2, np.int32)), grow_n=3,
                                       table_out=t, len_out=n, ref=r, status=s))
    new = rng.standard_normal((2, 2, 3, H, D)).astype(np.float32)
    capi.kv_put(capi.kv_rows_args(kv=kv(t, n), B=2, M=3, k=dev_of(new[0]), v=dev_of(new[1])))
    t2, s2 = capi.Buffer(64), capi.Buffer(16)
    bufs.extend([t2, s2])
    capi.kv_compact(capi.kv_compact_args(kv=kv(t, n), B=2, table_out=t2, status=s2))
    assert s2.read(np.int32, 2).tolist() == [4, 3]      # 30, 12 and 25 go; the copy took page 0
    k = [np.concatenate([KV.held(prompt[0, 0], prompt[1, 0])[i], KV.held(new[0, b], new[1, b])[i]]) for b in range(2) for i in range(2)]
    q = rng.standard_normal((2, 3, 4, D))

    class C:
        pass
    C.kv = staticmethod(lambda: kv(t2, n))
    got, exact = run_attn(C, q, "f32")
    for b in range(2):
        for i in range(3):
            for h in range(4):
                kk, vv = k[2 * b][:71 + i, h // 2], k[2 * b + 1][:71 + i, h // 2]
                w = np.exp((x := kk @ exact[b, i, h] / 8.0) - x.max())
                assert np.allclose(got[b, i, h], w @ vv / w.sum(), rtol=0, atol=5e-6 * 4)
    for b in bufs:
        b.free()
    pool.free()


def test_recorded_updates_replay(dev):
    rng = np.random.default_rng(3)
    table, length = beams(rng, 4, 4, 32, 12, 300, 300)
    pool = Pool(table, length, 32, 300, seed=3)
    src = capi.to_device((rng.integers(0, 4, (4, 4)) + np.arange(4)[:, None] * 4).ravel().astype(np.int32))
    t, n, r, s = pool.out(16)
    args = capi.kv_update_args(kv=pool.kv(), B=16, src=src, grow_n=1, table_out=t, len_out=n, ref=r, status=s)
    capi.kv_update(args)
    want = [b.read(np.int32) for b in (t, n, r, s)]
    bytes_ = pool.bufs[0].read(np.uint8)
    rec = capi.record(lambda: capi.kv_update(args))
    for _ in range(4):
        for b in (t, n, r, s):
            b.fill_u32(FRESH)
        pool.bufs[0].upload(pool.pool)
        rec.replay()
        for b, w in zip((t, n, r, s), want):
            assert np.array_equal(b.read(np.int32)[:w.size], w)
        assert np.array_equal(pool.bufs[0].read(np.uint8), bytes_)
    rec.free()
    src.free()
    pool.free()


@pytest.mark.parametrize("big", [False, True])
def test_a_sequence_does_not_go_on_in_a_page_that_is_gone(dev, big):
    """a window's sequence cut back into pages that it has given up: refused as a whole, also beside one that could go on; a cut
    where a page ends goes on, and its new row sees what has been put alone, in a pool of random bytes"""
    H, D, page, P = 1, 64, 32, 12400 if big else 12
    table = [[-1, -1, 7, 8], [1, 2, -1, -1]]
    pool = Pool(table, [100, 40], page, P, H=H, D=D, seed=2)
    ws, moves = check_update(pool, 2, keep=[50, 40], grow=[1, 1], window=16)
    assert ws == [0, P - 2, 0, 1] and not moves
    ws, _ = check_update(pool, 2, keep=[50, 40], grow=[300, 1], window=16)   # too long and gone: one sequence
    assert ws == [0, P - 2, 0, 1]
    ws, _ = check_update(pool, 2, keep=[50, 40], grow=[0, 1], window=16)
    assert ws == [0, P - 2, 0, 0]
    ws, _ = check_update(pool, 2, keep=[64, 40], grow=[1, 1], window=16)
    assert ws == [0, P - 3, 0, 0]
    t, n, _, _ = pool.outs
    kv = capi.kv(pages=pool.bufs[0], n_pages=P, page_bytes=pool.size, page=page, heads=H, dim=D, table=t, cols=4, len=n)
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((2, 1, H, D)).astype(np.float32) for _ in "kv")
    bufs = [capi.to_device(x) for x in (k, v)]
    capi.kv_put(capi.kv_rows_args(kv=kv, B=2, M=1, k=bufs[0], v=bufs[1]))

    class C:
        pass
    C.kv = staticmethod(lambda: kv)
    got, _ = run_attn(C, rng.standard_normal((2, 1, 2, D)), "f32", window=16)
    want = KV.held(k, v)[1]
    assert np.allclose(got[0], want[0], rtol=1e-6, atol=0)   # its window's other tokens are on no page
    for b in bufs:
        b.free()
    pool.free()


@pytest.mark.parametrize("P", [90, 12400])
def test_two_tables_in_each_others_gaps(dev, P):
    """one array with a row of the old table and a row of the new one in turn, which then change places"""
    rng = np.random.default_rng(P)
    table, length = beams(rng, 3, 3, 32, 7, P, 150)
    pool = Pool(table, length, 32, P, seed=4)
    both = np.full((9, 2, 7), FRESH, np.int32)
    both[:, 0] = table
    t, s, n = capi.to_device(both), capi.Buffer(16), [pool.bufs[2], capi.Buffer(48)]
    for turn in range(2):
        src = (rng.integers(0, 3, (3, 3)) + np.arange(3)[:, None] * 3).ravel()
        sb = capi.to_device(src.astype(np.int32))
        kv = capi.kv(pages=pool.bufs[0], n_pages=P, page_bytes=pool.size, page=32, heads=1, dim=64, table=t.ptr + 28 * turn, table_ld=14, cols=7,
                     len=n[turn])
        capi.kv_update(capi.kv_update_args(kv=kv, B=9, src=sb, grow_n=1, table_out=t.ptr + 28 * (1 - turn), out_ld=14, len_out=n[1 - turn], status=s))
        want, length, _, ws, _ = KV.update(table, length, 32, P, 9, src=src, grow_n=1)
        got = t.read(np.int32).reshape(9, 2, 7)
        assert s.read(np.int32, 4).tolist() == ws and np.array_equal(got[:, 1 - turn], want) and np.array_equal(got[:, turn], table)
        assert np.array_equal(n[1 - turn].read(np.int32, 9), length)
        table = want
        sb.free()
    for b in (t, s, n[1]):
        b.free()
    pool.outs = []
    pool.free()


@pytest.mark.parametrize("groups,W,cols,P", [(6, 4, 9, 8192), (6, 4, 9, 8193), (256, 4, 32, 3000), (1, 1025, 5, 3000), (205, 5, 31, 3000), (256, 4, 33, 3000)])
def test_updates_on_both_sides_of_one_workgroups_reach(dev, groups, W, cols, P):
    """8192 pages, 1024 sequences, 32768 entries are one workgroup's; one more of any is the chip's"""
    rng = np.random.default_rng(cols + P)
    table, length = beams(rng, groups, W, 32, cols, P, 60 if groups * W > 100 else 200)
    src = (rng.integers(0, W, (groups, W)) + np.arange(groups)[:, None] * W).ravel()
    pool = Pool(table, length, 32, P, seed=cols)
    ws, _ = check_update(pool, groups * W, src=src, grow_n=1)
    assert ws[0] == ws[3] == 0
    pool.free()


@pytest.mark.parametrize("B,longest,P", [(40, 3000, 8192), (40, 3000, 8193), (1024, 1000, 8000), (1024, 1030, 8000)])
def test_compact_on_both_sides_of_one_workgroups_reach(dev, B, longest, P):
    rng = np.random.default_rng(B + P)
    cols = -(-longest // 32)
    length = rng.integers(0, longest // (8 if B > 100 else 1), B)
    need = -(-length // 32)
    order = rng.permutation(P)
    table = np.full((B, cols), -1, np.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[np.arange(at, at + need[b]) % P]
        at += need[b]
    pool = Pool(table, length, 32, P, seed=B)
    t, _, _, s = pool.out(B)
    capi.kv_compact(capi.kv_compact_args(kv=pool.kv(), B=B, table_out=t, status=s))
    wt, ws, moves = KV.compact(table, length, 32, P)
    assert s.read(np.int32, 2).tolist() == ws and ws[1] > 100
    assert np.array_equal(t.read(np.int32, B * cols).reshape(B, cols), wt)
    pool.moved(moves)
    pool.free()


@pytest.mark.parametrize("length", [64, 40])
def test_too_few_pages_over_the_chip_change_nothing(dev, length):
    """1030 sequences on two pages want one each, or a copy of the second each but the first's"""
    pool = Pool(np.tile(np.array([[3, 1, -1, -1]]), (1030, 1)), np.full(1030, length), 32, 6, seed=length)
    ws, moves = check_update(pool, 1030, grow_n=1)
    assert ws == [1030 - 4 if length == 64 else 1029 - 4, 4, 0, 0] and not moves
    pool.free()
