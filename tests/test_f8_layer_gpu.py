"""p0pc0rn_amd.f8_layer: a layer's operators one after the other, each held against the CPU restatement in float64 on what the GPU gave it;
and the same tokens as one prompt, as a prompt and single tokens, and in chunks.

Bounds, relative in the 2-norm: codes are within half a step (2^-4 of a value at the most, 2^-5 on average: 0.04 holds it), 16-bit
results within 2^-8 of a value, one such rounding per operator (a rotation in place makes two); fp32 results 2^-15.
Chunks: rows that take different kernels differ by the 8-bit instruction's cut (1e-4) and a bf16 rounding (2^-9 on average) before values
are rounded to codes; where that moves a value over a border its code moves by a step, 2^-3 of the value, for a share of values of
the differences over the step: sqrt(2^-9 / 2^-3) 2^-3 = 0.016 a product's input, four products a layer and the attention between,
over a stream of the same size as their outputs: 0.05 a layer."""
import numpy as np
import pytest

from oracle import f8
from oracle import kvcache as KV
from p0pc0rn_amd import f8_layer as L
from tests.conftest import rel_l2
from tests.test_kv_gpu import from_type

pytestmark = pytest.mark.gpu


def codes(c, R):
    return c.codes.read(np.uint8, R * c.K).reshape(R, c.K), c.s.read(np.float32, R * (c.K // 128)).reshape(c.K // 128, R)


def weight(w):
    return f8.weight(w.codes.read(np.uint8, w.N * w.K).reshape(w.N, w.K), w.s.read(np.float32, -(-w.N // 128) * (w.K // 128)).reshape(-1, w.K // 128))


def half(buf, *s):
    return from_type(buf.read(np.uint16, int(np.prod(s))), "bf16").reshape(s)


@pytest.mark.parametrize("K,heads,kv_heads,dim,mlp,axis_dim,mode,M", [(512, 8, 2, 64, 1024, [64], "half", 40), (200, 4, 4, 128, 520, [44, 42, 42], "inter", 1),
                                                                     (320, 6, 2, 64, 300, [16, 24, 24], "half", 130)])
def test_each_operator_of_a_layer(dev, K, heads, kv_heads, dim, mlp, axis_dim, mode, M):
    m = L.Decoder(1, K, heads, kv_heads, dim, mlp, axis_dim, 1000.0, mode)
    B, l, rng = 2, m.w[0], np.random.default_rng(M)
    run = L.Run(m, B, 300, 130)
    R, vec = B * M, lambda b, n: b.read(np.float32, n)  # noqa: E731
    pos0 = np.arange(60)
    run.step(rng.standard_normal((B, 60, K)), np.broadcast_to(pos0, (len(axis_dim), B, 60)))            # a prompt ahead of the rows
    x = rng.standard_normal((B, M, K)).astype(np.float32)
    pos = np.stack([60 + rng.integers(0, 50, (B, M)) for _ in axis_dim])

    seen = []                                             # the products in order: their codes, their result in float64
    product = run._product

    def spy(a, w, rows, y, type_):
        product(a, w, rows, y, type_)
        seen.append((codes(a, rows), f8.values(*codes(a, rows)) @ weight(w).T))
    run._product = spy
    out = run.step(x, pos).reshape(R, K)
    x = x.reshape(R, K)
    (ac, asc), qkv = seen[0]
    _, want = f8.norm(x, w=vec(l["norm"][0], K))
    assert rel_l2(f8.values(ac, asc)[:, :K], want) <= 0.04
    # rotated heads and values, the cache and its attention
    got = half(run.qkv, R, m.width)
    turned = f8.rope(qkv[:, :(heads + kv_heads) * dim].reshape(R, heads + kv_heads, dim), pos.reshape(len(axis_dim), R), axis_dim, 1000.0, mode, hq=heads,
                     qw=vec(l["qn"], dim), kw=vec(l["kn"], dim)).reshape(R, -1)
    assert rel_l2(got[:, :turned.shape[1]], turned) <= 2 * 2.0 ** -8
    assert rel_l2(got[:, turned.shape[1]:], qkv[:, turned.shape[1]:]) <= 2.0 ** -8
    c = KV.Cache(run.n_pages, run.page, kv_heads, dim)
    c.pool[:] = run.pages.read(np.uint8, c.pool.size).reshape(c.pool.shape)
    table = run.tables[0].read(np.int32, B * run.cols).reshape(B, run.cols)
    q = got[:, :heads * dim].reshape(B, M, heads, dim).astype(np.float32)
    att = half(run.att, R, heads * dim)
    assert rel_l2(att, KV.attention(c, table, [60 + M] * B, q)) <= 2.0 ** -7
    (oc, osc), t = seen[1]
    assert np.array_equal(oc, f8.quantise(att)[0]) and np.array_equal(osc, f8.quantise(att)[1])
    r, want = f8.norm(x, t, vec(l["norm"][1], K), vec(l["norm"][2], K))
    (hc, hsc), h = seen[2]
    assert rel_l2(f8.values(hc, hsc)[:, :K], want) <= 0.04
    assert rel_l2(half(run.h, R, 2 * mlp), h) <= 2.0 ** -8
    gate = half(run.h, R, 2 * mlp)
    (dc, dsc), t = seen[3]
    assert rel_l2(f8.values(dc, dsc)[:, :mlp], f8.glu("gelu", gate[:, :mlp], gate[:, mlp:])) <= 0.04
    assert rel_l2(run.t.read(np.float32, R * K).reshape(R, K), t) <= 2.0 ** -15
    assert rel_l2(out, f8.norm(r, t, vec(l["norm"][3], K))[0]) <= 2.0 ** -15


@pytest.mark.parametrize("chunks", [[100, 1, 1, 1], [1] * 9 + [94], [33, 70], [17, 17, 69]])
def test_chunks_of_a_prompt(dev, chunks):
    m, B, n = L.Decoder(2), 2, 103
    x = np.random.default_rng(7).standard_normal((B, n, m.K))
    at = np.broadcast_to(np.arange(n), (1, B, n))
    whole = L.Run(m, B, n, n).step(x, at)
    run, got, i = L.Run(m, B, n, n), [], 0
    for c in chunks:
        got.append(run.step(x[:, i:i + c], at[:, :, i:i + c]))
        i += c
    assert i == n and rel_l2(np.concatenate(got, 1), whole) <= 0.1


def test_more_rows_than_there_is_room_for(dev):
    run = L.Run(L.Decoder(1), 1, 10, 4)
    with pytest.raises(ValueError, match="5 rows at a time"):
        run.step(np.zeros((1, 5, 512)), np.zeros((1, 1, 5)))


def test_the_command(dev, capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["f8_layer", "--prompt", "40", "--tokens", "3"])
    L.main()
    assert "3 tokens: last row's rms" in capsys.readouterr().out
