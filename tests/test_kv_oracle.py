"""The CPU restatement of the 4-bit cache (oracle/kvcache.py), and what the kv_* calls refuse before they touch a device."""
import json
import subprocess
import sys

import numpy as np
import pytest

from oracle import kvcache as KV
from p0pc0rn_amd import capi
from tests.conftest import ROOT

DIMS = [64, 128, 256, 512]


@pytest.mark.parametrize("D", DIMS)
def test_every_byte_of_a_run_has_one_owner(D):
    kc, ke, vc, ve = KV.offsets(D)
    assert np.array_equal(kc[:, 0::2], kc[:, 1::2]) and np.array_equal(vc[:, 0::2], vc[:, 1::2])   # two codes a byte
    used = np.concatenate([kc[:, 0::2].ravel(), ke.ravel(), vc[:, 0::2].ravel(), ve.ravel()])
    assert np.array_equal(np.sort(used), np.arange(34 * D))


def test_codes_are_the_nearest_and_ties_go_to_the_even_one():
    y = np.array([0.0, 0.25, 0.26, 0.75, 0.74, 1.25, 1.26, 1.75, 2.5, 2.51, 3.5, 3.49, 5.0, 5.01, 6.0, 7.0])
    want = np.array([0, 0, 1, 2, 1, 2, 3, 4, 4, 5, 6, 5, 6, 7, 7, 7])
    assert np.array_equal(KV.codes(y), want)
    assert np.array_equal(KV.codes(-y)[1:], want[1:] + 8)
    v = np.concatenate([KV.GRID, -KV.GRID])
    assert np.array_equal(KV.values(KV.codes(v).repeat(2), np.zeros(1, int)), v.repeat(2))


def test_the_exponent_is_the_least_that_holds_the_largest():
    x = np.zeros((6, 32))
    x[:, 5] = [6.0, -6.000001, 3.0, 3.0001, 1e-30, 1e9]
    assert KV.exponents(x).tolist() == [0, 1, -1, 0, KV.E_MIN, KV.E_MAX]
    rng = np.random.default_rng(0)
    y = rng.standard_normal((500, 32)) * np.exp(3 * rng.standard_normal((500, 1)))
    c, e = KV.quantise(y.reshape(500, 32))
    held = np.clip(y, -49152, 49152)                           # 6 * 2^13, the largest there is
    assert np.all(np.abs(KV.values(c, e) - held) <= 2.0 ** e)  # half the widest step, 4 to 6


def _kv(**kw):
    base = dict(pages=4096, n_pages=4, page=64, heads=2, dim=128, table=16, cols=4, len=16)
    base.update(kw)
    return capi.kv(**base)


BAD_CACHE = [(dict(page=48), "no pages of 48 tokens, 2 heads of 128"), (dict(page=2048), "no pages of 2048 tokens, 2 heads of 128"),
             (dict(dim=96), "no pages of 64 tokens, 2 heads of 96"), (dict(heads=0), "no pages of 64 tokens, 0 heads of 128"),
             (dict(n_pages=0), "0 pages"), (dict(page_bytes=64), "page_bytes 64 (a page is 17408)"),
             (dict(page_bytes=17416), "page_bytes 17416 (a page is 17408)"), (dict(pages=None), "missing pages, table or len buffer"),
             (dict(table=None), "missing pages, table or len buffer"), (dict(len=None), "missing pages, table or len buffer"),
             (dict(pages=4104), "pages must be 16-byte aligned"), (dict(cols=0), "table of 0 columns, stride 0"),
             (dict(table_ld=3), "table of 4 columns, stride 3"), (dict(cols=1 << 26), "table of 67108864 columns, stride 0")]


def _refused(fn, args, msg):
    with pytest.raises(capi.P0Error) as e:
        fn(args)
    assert e.value.code == capi.P0_EINVAL and str(e.value) == msg


@pytest.mark.parametrize("kw,msg", BAD_CACHE)
def test_a_cache_that_is_none_is_refused(kw, msg):
    _refused(capi.kv_put, capi.kv_rows_args(kv=_kv(**kw), B=1, M=1, k=16, v=16), "kv_put: " + msg)
    _refused(capi.kv_get, capi.kv_rows_args(kv=_kv(**kw), B=1, M=1, k=16, v=16), "kv_get: " + msg)
    _refused(capi.kv_attn, capi.kv_attn_args(kv=_kv(**kw), B=1, M=1, heads=2, q=16, y=16), "kv_attn: " + msg)


@pytest.mark.parametrize("kw,msg", [(dict(B=-1), "B -1"), (dict(B=70000), "B 70000"), (dict(M=-2), "M -2"), (dict(type=3), "type 3"),
                                    (dict(k=None), "missing k or v buffer"), (dict(v=None), "missing k or v buffer"),
                                    (dict(k=18), "k or v is not aligned to its type"), (dict(v=17, type=1), "k or v is not aligned to its type")])
def test_rows_that_are_none_are_refused(kw, msg):
    base = dict(kv=_kv(), B=1, M=1, k=16, v=16)
    base.update(kw)
    _refused(capi.kv_put, capi.kv_rows_args(**base), "kv_put: " + msg)
    _refused(capi.kv_get, capi.kv_rows_args(**base), "kv_get: " + msg)


@pytest.mark.parametrize("kw,msg", [(dict(heads=3), "3 heads over 2 key heads"), (dict(heads=0), "0 heads over 2 key heads"),
                                    (dict(type=-1), "type -1"), (dict(window=-1), "window -1, sinks 0, max_len 0"),
                                    (dict(sinks=-4), "window 0, sinks -4, max_len 0"), (dict(scale=-1.0), "scale -1"),
                                    (dict(scale=float("nan")), "scale nan"), (dict(scale=float("inf")), "scale inf"),
                                    (dict(q=None), "missing q or y buffer"), (dict(y=None), "missing q or y buffer"),
                                    (dict(q=18), "q or y is not aligned to its type"), (dict(M=1 << 25), "M 33554432"),
                                    (dict(y=17, type=2), "q or y is not aligned to its type")])
def test_attention_that_is_none_is_refused(kw, msg):
    base = dict(kv=_kv(), B=1, M=1, heads=4, q=16, y=16)
    base.update(kw)
    _refused(capi.kv_attn, capi.kv_attn_args(**base), "kv_attn: " + msg)


def test_page_bytes():
    assert capi.kv_page_bytes(64, 2, 256) == 2 * 2 * 34 * 256
    assert capi.kv_page_bytes(33, 2, 256) == capi.kv_page_bytes(64, 2, 100) == 0


@pytest.mark.parametrize("kw,msg", [(dict(Bo=70000, src=16), "Bo 70000"), (dict(Bo=3), "3 sequences of 2 need src"),
                                    (dict(window=-1), "window -1, sinks 0"), (dict(sinks=-1), "window 0, sinks -1"),
                                    (dict(layers=-1), "-1 layers, 0 B apart"), (dict(layers=2, layer_bytes=64), "2 layers, 64 B apart"),
                                    (dict(layer_bytes=8), "0 layers, 8 B apart"), (dict(table_out=None), "missing table_out or status buffer"),
                                    (dict(status=None), "missing table_out or status buffer"), (dict(len_out=None), "missing len_out buffer"),
                                    (dict(out_ld=3), "out_ld 3 of 4 columns"), (dict(table_out=40), "table_out or len_out overlaps what is read"),
                                    (dict(len_out=1 << 20), "table_out or len_out overlaps what is read"),
                                    (dict(kv=dict(n_pages=(1 << 21) + 1)), "2097153 pages (at most 2097152)"),
                                    (dict(B=40000, kv=dict(cols=1 << 15)), "40000 sequences of 32768 columns")])
def test_updates_that_are_none_are_refused(kw, msg):
    base = dict(B=2, table_out=4096, len_out=8192, status=16, grow_n=1)
    kv = dict(table=16, len=1 << 20)
    base.update(kw)
    kv.update(base.pop("kv", {}))
    _refused(capi.kv_update, capi.kv_update_args(kv=_kv(**kv), **base), "kv_update: " + msg)
    if kw.keys() <= {"layers", "layer_bytes", "table_out", "status", "out_ld", "kv", "B"} and "overlaps" not in msg:
        for gone in ("len_out", "grow_n"):
            base.pop(gone)
        _refused(capi.kv_compact, capi.kv_compact_args(kv=_kv(**kv), **base), "kv_compact: " + msg)
    if kw == dict(table_out=40):
        _refused(capi.kv_compact, capi.kv_compact_args(kv=_kv(**kv), B=2, status=16, table_out=40), "kv_compact: table_out overlaps what is read")


def test_an_update_by_hand():
    """two beams of one parent in the middle of a page: the first writes on in it, the second in a copy"""
    t, n, holders, status, moves = KV.update(np.array([[5, 3, -1], [1, 2, -1]]), np.array([40, 40]), 32, 6, 2, src=[0, 0], grow_n=1)
    assert t.tolist() == [[5, 3, -1], [5, 0, -1]] and n.tolist() == [41, 41] and moves == [(3, 0)]
    assert holders.tolist() == [1, 0, 0, 1, 0, 2] and status == [0, 3, 1, 0]
    out, status, moves = KV.compact(t, n, 32, 6)
    assert out.tolist() == [[2, 1, -1], [2, 0, -1]] and status == [3, 2] and moves == [(3, 1), (5, 2)]


def test_a_sequence_does_not_go_on_in_a_page_that_is_gone():
    """cut back to 50 tokens of a window's 100, the page of tokens 32-63 has been given up: a fresh one would show tokens that nobody put"""
    table = np.array([[-1, -1, 7, 8]])
    t, n, holders, status, moves = KV.update(table, np.array([100]), 32, 12, 1, keep=[50], grow_n=1, window=16)
    assert status == [0, 12, 0, 1] and t.tolist() == table.tolist() and n.tolist() == [100] and holders is None and not moves
    t, n, _, status, _ = KV.update(table, np.array([100]), 32, 12, 1, keep=[64], grow_n=1, window=16)   # where a page ends it can
    assert status == [0, 11, 0, 0] and t.tolist() == [[-1, -1, 0, -1]] and n.tolist() == [65]
    t, n, _, status, _ = KV.update(table, np.array([100]), 32, 12, 1, keep=[50], window=16)             # nor does one that does not grow
    assert status == [0, 12, 0, 0] and t.tolist() == [[-1, -1, -1, -1]] and n.tolist() == [50]


@pytest.mark.parametrize("kw,msg", [(dict(n=-1), "-1 searches of 2 beams"), (dict(W=0), "1 searches of 0 beams"),
                                    (dict(n=700, W=100), "700 searches of 100 beams"), (dict(V=0), "V 0, ld 0"), (dict(ld=99), "V 100, ld 99"),
                                    (dict(k=0), "k 0 (1..32, at most V)"), (dict(k=33), "k 33 (1..32, at most V)"),
                                    (dict(V=3), "k 4 (1..32, at most V)"), (dict(done=16), "done needs an eos token"),
                                    (dict(hist=16), "hist and hist_out go together"), (dict(hist_out=16), "hist and hist_out go together"),
                                    (dict(hist=16, hist_out=4096, hist_n=4, hist_ld=4), "hist of 4 tokens, stride 4"),
                                    (dict(hist=16, hist_out=32, hist_n=4), "hist and hist_out overlap"),
                                    (dict(n=60, W=1000, V=1 << 20), "60000 rows of 1048576 logits need 307200000 B of workspace")])
def test_steps_that_are_none_are_refused(kw, msg):
    base = dict(logits=16, n=1, W=2, V=100, k=4, score=16, token=16, parent=16, score_out=16)
    base.update(kw)
    _refused(capi.beam, capi.beam_args(**base), "beam: " + msg)
    for gone in ("logits", "score", "token", "parent", "score_out"):
        args = dict(base, **{k: v for k, v in dict(n=1, W=2, V=100, k=4, done=None, hist=None, hist_out=None, ld=0).items()})
        args[gone] = None
        _refused(capi.beam, capi.beam_args(**args), "beam: missing logits, score, token, parent or score_out buffer")


def test_a_step_by_hand():
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.125, 0.75, 0.125]]))
    (token, parent, score, done), _ = KV.beam(x, np.log([0.5, 0.5]), 2, 3, eos=1)
    assert token.tolist() == [[1, 0, 1]] and parent.tolist() == [[1, 0, 0]] and done.tolist() == [[True, False, True]]
    assert np.allclose(np.exp(score), [[0.375, 0.25, 0.125]])


@pytest.mark.parametrize("kw,msg", [(dict(cols=1 << 58), "table of 288230376151711744 columns, stride 0"),
                                    (dict(cols=(1 << 25) + 1), "table of 33554433 columns, stride 0"),
                                    (dict(page_bytes=1 << 62), "page_bytes 4611686018427387904 (a page is 17408)")])
def test_a_cache_whose_size_passes_64_bits_is_refused(kw, msg):
    """cols * page and n_pages * page_bytes of these are small again in 64 bits"""
    _refused(capi.kv_put, capi.kv_rows_args(kv=_kv(**kw), B=1, M=1, k=16, v=16), "kv_put: " + msg)
    _refused(capi.kv_attn, capi.kv_attn_args(kv=_kv(**kw), B=1, M=1, heads=2, q=16, y=16), "kv_attn: " + msg)
    args = dict(B=1, layers=2, layer_bytes=16, table_out=4096, status=16)
    _refused(capi.kv_update, capi.kv_update_args(kv=_kv(**kw), len_out=8192, **args), "kv_update: " + msg)
    _refused(capi.kv_compact, capi.kv_compact_args(kv=_kv(**kw), **args), "kv_compact: " + msg)


def _in_a_process_of_its_own(body):
    """`body` in a process that never opens a device, where a call whose arguments are taken ends with P0_ENODEV (3)"""
    code = "from p0pc0rn_amd import capi\nfrom tests.test_kv_oracle import _kv\n" + """
def says(fn, args):
    try:
        fn(args)
    except capi.P0Error as e:
        return "taken" if e.code == 3 else str(e)
""" + body
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return json.loads(r.stdout)


def test_rows_that_lie_between_each_other_do_not_overlap():
    """two tables, two histories of one stride, the one's rows in the other's gaps; and up to the last word of a last row"""
    got = _in_a_process_of_its_own("""
import json
out = []
for at in (4096 + 16, 4096 + 12, 4096 + 20, 4096 + 80, 4096 + 76, 4096 - 80, 4096 - 76):
    kv = _kv(table=4096, table_ld=8, cols=4, len=1 << 20)
    out.append([says(capi.kv_update, capi.kv_update_args(kv=kv, B=3, table_out=at, out_ld=8, len_out=1 << 21, status=1 << 22)),
                says(capi.kv_compact, capi.kv_compact_args(kv=kv, B=3, table_out=at, out_ld=8, status=1 << 22))])
for at in (4096 + 20, 4096 + 16, 4096 + 12, 4096 + 24, 4096 + 20 + 40, 4096 + 56, 4096 - 140, 4096 - 136):
    out.append(says(capi.beam, capi.beam_args(logits=16, n=1, W=2, V=100, k=4, score=16, token=16, parent=16, score_out=16,
                                              hist=4096, hist_out=at, hist_n=4, hist_ld=10)))
print(json.dumps(out))""")
    over = ["kv_update: table_out or len_out overlaps what is read", "kv_compact: table_out overlaps what is read"]
    assert got[:7] == [["taken"] * 2 if fine else over for fine in (True, False, False, True, False, True, False)]
    # rows of 4 words at 10, 5 at 10 into them
    assert got[7:] == ["taken" if fine else "beam: hist and hist_out overlap" for fine in (True, True, False, False, True, True, True, False)]


@pytest.mark.parametrize("kw,msg", [(dict(table_out=(1 << 20) - 4), "table_out or len_out overlaps what is read"),
                                    (dict(len_out=4096 + 28), "table_out or len_out overlaps what is read"),
                                    (dict(src=8192, table_out=8196), "table_out or len_out overlaps what is read"),
                                    (dict(keep=8192, table_out=8196), "table_out or len_out overlaps what is read"),
                                    (dict(grow=8192, table_out=8196), "table_out or len_out overlaps what is read"),
                                    (dict(status=4096 + 16), "ref or status overlaps what is read"), (dict(status=1 << 20), "ref or status overlaps what is read"),
                                    (dict(ref=4096 - 12), "ref or status overlaps what is read"),
                                    (dict(status=(1 << 21) + 4), "two of table_out, len_out, ref and status overlap"),
                                    (dict(ref=(1 << 23) + 8), "two of table_out, len_out, ref and status overlap"),
                                    (dict(table_out=(1 << 22) - 8), "two of table_out, len_out, ref and status overlap")])
def test_outputs_of_an_update_that_overlap_are_refused(kw, msg):
    base = dict(kv=_kv(table=4096, len=1 << 20), B=2, table_out=1 << 23, len_out=1 << 21, status=1 << 22, grow_n=1)
    base.update(kw)
    _refused(capi.kv_update, capi.kv_update_args(**base), "kv_update: " + msg)
    if kw.keys() == {"status"} and "read" in msg:
        _refused(capi.kv_compact, capi.kv_compact_args(kv=base["kv"], B=2, table_out=1 << 23, **kw), "kv_compact: table_out or status overlaps what is read")
