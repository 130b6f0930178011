"""The beam search's step against its CPU restatement (oracle/kvcache.py, float64): tokens, parents and marks exactly, scores to
2^-22 of the largest magnitude in their sums (three fp32 roundings and a logarithm of a sum that is off by under 2^-21)."""
import numpy as np
import pytest

from oracle import kvcache as KV
from p0pc0rn_amd import capi

pytestmark = pytest.mark.gpu
FRESH = 0x77777777


def step(logits, score, W, k, done=None, eos=-1, hist=None, hist_n=0, ld=None, shift=0):
    rows, V = logits.shape
    n = rows // W
    ld = ld or V
    flat = np.full(shift + rows * ld, 1e30, np.float32)    # what lies between the rows would win
    flat[shift:].reshape(rows, ld)[:, :V] = logits
    dev = [capi.to_device(flat), capi.to_device(np.asarray(score, np.float32))]
    db = capi.to_device(np.asarray(done, np.int32)) if done is not None else None
    hb = capi.to_device(hist) if hist is not None else None
    outs = [capi.Buffer(n * k * 4 + 16).fill_u32(FRESH) for _ in range(4)]
    ho = capi.Buffer(n * k * hist.shape[1] * 4).fill_u32(FRESH) if hist is not None else None
    capi.beam(capi.beam_args(logits=dev[0].ptr + 4 * shift, ld=ld, n=n, W=W, V=V, k=k, score=dev[1], done=db, eos=eos, token=outs[0],
                             parent=outs[1], score_out=outs[2], done_out=outs[3], hist=hb, hist_out=ho, hist_n=hist_n,
                             hist_ld=hist.shape[1] if hist is not None else 0))
    got = [b.read(np.float32 if i == 2 else np.int32)[:n * k].reshape(n, k) for i, b in enumerate(outs)]
    for b in outs:
        assert np.all(b.read(np.uint32)[n * k:n * k + 4] == FRESH)
    h = ho.read(np.int32).reshape(n * k, -1) if ho else None
    for b in dev + outs + [db, hb, ho]:
        if b:
            b.free()
    return got, h


def check(got, want):
    for i in (0, 1, 3):
        assert np.array_equal(got[i], want[i]), i
    fine = np.isfinite(want[2])
    assert np.array_equal(np.isfinite(got[2]), fine) and np.all(got[2][~fine] == want[2][~fine])
    if fine.any():
        assert np.abs(got[2][fine] - want[2][fine]).max() <= 2.0 ** -22 * max(32.0, np.abs(want[2][fine]).max() + 32.0)


@pytest.mark.parametrize("n,W,k,V", [(1, 1, 1, 1), (1, 1, 8, 8), (2, 3, 5, 7), (1, 4, 4, 500), (3, 1, 32, 33), (2, 8, 8, 8191), (2, 5, 16, 8193),
                                     (1, 40, 32, 1000), (4, 4, 4, 30000), (1, 8, 32, 262144), (70, 3, 2, 100), (1, 2, 32, 600001)])
def test_the_best_continuations(dev, n, W, k, V):
    rng = np.random.default_rng(V + k)
    x = (3 * rng.standard_normal((n * W, V))).astype(np.float32)
    score = (-20 * rng.random(n * W)).astype(np.float32)
    want, gap = KV.beam(x, score, W, k)
    assert gap > 5e-5 or V * W * k > 200, "inputs whose order fp32 decides"
    got, _ = step(x, score, W, k)
    if gap > 5e-5:
        check(got, want)
    else:                                                  # neighbours that fp32 may order either way: the same set of scores
        assert np.abs(got[2] - want[2]).max() <= 5e-5
        assert all(len(set(zip(t, p))) == k for t, p in zip(got[0].tolist(), got[1].tolist()))
        at = got[1].ravel(), got[0].ravel()
        s = score[at[0]].astype(np.float64) + x[at] - np.log(np.exp(x.astype(np.float64)).sum(1))[at[0]]
        assert np.abs(s.reshape(n, k) - got[2]).max() <= 5e-5


@pytest.mark.parametrize("n,W,k,V", [(300, 4, 4, 100), (300, 4, 20, 100), (40, 16, 16, 17000), (1100, 1, 1, 3)])
def test_rows_enough_for_a_join_of_its_own(dev, n, W, k, V):
    """among so many searches some scores lie within a rounding: each place's score, then that its token has it"""
    rng = np.random.default_rng(n + k)
    x = (3 * rng.standard_normal((n * W, V))).astype(np.float32)
    score = (-20 * rng.random(n * W)).astype(np.float32)
    want, _ = KV.beam(x, score, W, k)
    got, _ = step(x, score, W, k)
    assert np.abs(got[2] - want[2]).max() <= 2.0 ** -22 * 96
    at = got[1].ravel(), got[0].ravel()
    s = score[at[0]].astype(np.float64) + x[at] - np.log(np.exp(x.astype(np.float64)).sum(1))[at[0]]
    assert np.abs(s.reshape(n, k) - got[2]).max() <= 2.0 ** -22 * 96
    assert all(len(set(zip(t, p))) == k for t, p in zip(got[0].tolist(), got[1].tolist()))


@pytest.mark.parametrize("ld,shift", [(501, 0), (512, 1), (504, 4), (600, 3)])
def test_strides_and_alignments(dev, ld, shift):
    rng = np.random.default_rng(ld)
    x = (3 * rng.standard_normal((6, 499))).astype(np.float32)
    score = (-5 * rng.random(6)).astype(np.float32)
    want, gap = KV.beam(x, score, 3, 4)
    assert gap > 5e-5
    check(step(x, score, 3, 4, ld=ld, shift=shift)[0], want)


def test_ties_go_to_the_lower_beam_and_token(dev):
    V, W, k = 9000, 4, 16
    x = np.zeros((W, V), np.float32)
    x[:, 5::7] = -0.0                                      # as large as the others
    got, _ = step(x, np.zeros(W, np.float32), W, k)
    assert np.array_equal(got[0], np.arange(k)[None]) and not got[1].any()
    x[:] = -1.0
    x[2, [8999, 8200, 4, 4000]] = 1.0
    x[0, 10] = 1.0
    x[1] = x[2]
    got, _ = step(x, np.full(W, -1.0, np.float32), W, 6)
    assert got[0].tolist() == [[10, 4, 4000, 8200, 8999, 4]] and got[1].tolist() == [[0, 1, 1, 1, 1, 2]]


@pytest.mark.parametrize("V", [40, 20000])
def test_values_in_any_order(dev, V):
    """ascending, descending, all of the best in one lane's reach"""
    k = 32
    rows = np.stack([np.arange(V), np.arange(V)[::-1], np.where(np.arange(V) % 1024 < 4, 100.0, 0.0) + np.arange(V) % 97 / 97]).astype(np.float32) / 50
    score = np.array([0.0, -300.0, -900.0], np.float32)
    want, gap = KV.beam(rows, score, 1, k)
    got, _ = step(rows, score, 1, k)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_ended_beams_stay_as_they_are(dev):
    rng = np.random.default_rng(1)
    n, W, k, V = 3, 4, 6, 300
    x = (2 * rng.standard_normal((n * W, V))).astype(np.float32)
    score = (-6 * rng.random(n * W)).astype(np.float32)
    done = np.zeros(n * W, int)
    done[[1, 2, 4, 5, 6, 7]] = 1                           # some of the first search, all of the second
    x[9, 17] = 30.0                                        # the third search ends one
    want, gap = KV.beam(x, score, W, k, done, eos=17)
    assert gap > 5e-5
    got, _ = step(x, score, W, k, done, eos=17)
    check(got, want)
    assert got[3][1].all() and np.all(got[2][1, 4:] == -np.inf) and got[3][2].any()


def test_scores_and_logits_that_are_no_numbers(dev):
    rng = np.random.default_rng(2)
    W, k, V = 5, 4, 400
    x = (2 * rng.standard_normal((W, V))).astype(np.float32)
    x[0, 3], x[0, 100:300] = np.nan, -np.inf
    x[1] = -np.inf
    x[2, 7] = np.inf
    score = np.array([-1.0, 0.0, 0.0, -np.inf, np.nan], np.float32)
    want, gap = KV.beam(x, score, W, k)
    assert gap > 5e-5
    got, _ = step(x, score, W, k)
    check(got, want)
    got, _ = step(x[1:], score[1:], 4, k)                  # nothing but -infinity: the first beam's first tokens
    assert np.all(got[2] == -np.inf) and not got[1].any() and got[0].tolist() == [[0, 1, 2, 3]]


@pytest.mark.parametrize("hist_n,ld", [(0, 1), (1, 2), (37, 50), (1500, 1501)])
def test_histories_follow_their_parents(dev, hist_n, ld):
    rng = np.random.default_rng(hist_n)
    n, W, k, V = 2, 3, 5, 200
    x = (2 * rng.standard_normal((n * W, V))).astype(np.float32)
    hist = rng.integers(0, V, (n * W, ld)).astype(np.int32)
    got, h = step(x, np.zeros(n * W), W, k, hist=np.vstack([hist, np.zeros((n * (k - W), ld), np.int32)]), hist_n=hist_n)
    token, parent = got[0].ravel(), got[1].ravel()
    assert np.array_equal(h[:, :hist_n], hist[parent, :hist_n]) and np.array_equal(h[:, hist_n], token)
    assert np.all(h[:, hist_n + 1:] == FRESH)


def test_recorded_steps_replay(dev):
    rng = np.random.default_rng(4)
    x = (2 * rng.standard_normal((8, 30000))).astype(np.float32)
    b = [capi.to_device(x), capi.to_device(np.zeros(8, np.float32))] + [capi.Buffer(64) for _ in range(3)]
    args = capi.beam_args(logits=b[0], n=2, W=4, V=30000, k=4, score=b[1], token=b[2], parent=b[3], score_out=b[4])
    capi.beam(args)
    want = [o.read(np.uint32, 8) for o in b[2:]]
    rec = capi.record(lambda: capi.beam(args))
    for _ in range(4):
        for o in b[2:]:
            o.fill_u32(FRESH)
        rec.replay()
        for o, w in zip(b[2:], want):
            assert np.array_equal(o.read(np.uint32, 8), w)
        capi.beam(args)
    rec.free()
    for o in b:
        o.free()
