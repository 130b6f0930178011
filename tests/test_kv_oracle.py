"""The CPU restatement of the 4-bit cache (oracle/kvcache.py), and what the kv_* calls refuse before they touch a device."""
import numpy as np
import pytest

from oracle import kvcache as KV
from p0pc0rn_amd import capi

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
