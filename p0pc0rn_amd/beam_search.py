"""Beam search with a small decoder over the 4-bit cache: how the operators of a token go together.

    python -m p0pc0rn_amd.beam_search [--beams 4] [--tokens 24]

A token of every beam is, per layer, the qkv projection (gemvM, rms), its keys and values into the cache (kv_put), the attention
of the new row over all of the sequence's (kv_attn), the o projection, the residual norm (normadd), the gated FFN; then the
head's logits (softcap), the best continuations of each search (beam) and the sequences they continue (kv_update): beams that
share a past share its pages, and only a page two of them write to is copied. Weights are random: the text is noise, the search
is not (tests/test_beam_search_gpu.py scores its results again, token by token). There is no position embedding.
"""
import argparse

import numpy as np

from . import capi

EPS = 1e-6


class Decoder:
    """`layers` layers of random q4 weights: hidden K, `heads` query heads on `kv_heads` key heads of `dim`, FFN `mlp`, `vocab` words."""

    def __init__(self, layers=2, K=512, heads=8, kv_heads=2, dim=64, mlp=1024, vocab=4096, seed=1):
        self.layers, self.K, self.heads, self.kv_heads, self.dim, self.mlp, self.vocab = layers, K, heads, kv_heads, dim, mlp, vocab
        rng = np.random.default_rng(seed)
        self.embed = rng.standard_normal((vocab, K)).astype(np.float32)
        self.width = (heads + 2 * kv_heads) * dim

        def q4(N, k, s):
            w = capi.Buffer(N // 64 * (k // 32) * 1280)
            capi.fill_q4_sym(w, N, k, int(rng.integers(1 << 31)), 0.25 * s / k ** 0.5)
            return w
        self.w = [dict(qkv=q4(self.width, K, 1.0), o=q4(K, heads * dim, 1.0), gu=q4(2 * mlp, K, 1.0), down=q4(K, mlp, 1.0),
                       norm=[capi.to_device((1 + 0.1 * rng.standard_normal(K)).astype(np.float32)) for _ in range(4)])
                  for _ in range(layers)]
        self.head, self.head_norm = q4(vocab, K, 3.0), capi.to_device(np.ones(K, np.float32))


class Search:
    """`n` searches that end as `W` beams each (n * W at most 16: the rows of one gemvM), of up to `longest` tokens."""

    def __init__(self, model, n, W, longest, page=32, window=0, sinks=0):
        m, R = model, n * W
        self.m, self.n, self.W, self.page, self.window, self.sinks = m, n, W, page, window, sinks
        self.rows, self.length = n, 0                     # one beam a search until the first step of the search
        self.cols = -(-longest // page) + 1
        self.n_pages = 2 * R * self.cols
        self.layer_bytes = self.n_pages * capi.kv_page_bytes(page, m.kv_heads, m.dim)
        f32 = lambda *s: capi.Buffer(4 * int(np.prod(s)))  # noqa: E731
        self.pages = capi.Buffer(m.layers * self.layer_bytes)
        self.tables, self.lens = [f32(R, self.cols) for _ in "ab"], [f32(R) for _ in "ab"]
        self.tables[0].fill_u32(0xFFFFFFFF)
        self.lens[0].fill_u32(0)
        self.status, self.ref = f32(4), f32(self.n_pages)
        self.x, self.qkv, self.att, self.t, self.h = f32(R, m.K), f32(R, m.width), f32(R, m.heads * m.dim), f32(R, m.K), f32(R, m.mlp)
        self.stat, self.pairs, self.logits, self.mx = f32(R), f32(R, 2), f32(R, m.vocab), f32(R, m.vocab // 64, 2)
        self.score, self.token, self.parent = [f32(R) for _ in "ab"], f32(R), f32(R)
        self.score[0].fill_u32(0)
        self.hist_ld = longest + 1
        self.hist = [f32(R, self.hist_ld) for _ in "ab"]
        self.steps = 0

    def _cache(self, layer=0):
        m = self.m
        return capi.kv(pages=self.pages.ptr + layer * self.layer_bytes, n_pages=self.n_pages, page=self.page, heads=m.kv_heads, dim=m.dim,
                       table=self.tables[0], cols=self.cols, len=self.lens[0])

    def sequences(self, rows, src=None, keep=None):
        """the sequences of the next token: one token longer, from `src` (kv_update); raises where the pool is too small"""
        capi.kv_update(capi.kv_update_args(kv=self._cache(), B=self.rows, Bo=rows, src=src, keep=keep, grow_n=1, window=self.window,
                                           sinks=self.sinks, layers=self.m.layers, table_out=self.tables[1], len_out=self.lens[1],
                                           ref=self.ref, status=self.status))
        missing, _, _, stuck = self.status.read(np.int32, 4)
        if missing or stuck:
            raise RuntimeError("beam_search: %d pages missing, %d sequences that cannot grow" % (missing, stuck))
        self.tables.reverse()
        self.lens.reverse()
        self.rows, self.length = rows, self.length + 1

    def forward(self, tokens):
        """one token of every sequence -> its logits, in self.logits"""
        m, R = self.m, self.rows
        self.x.upload(m.embed[tokens])
        capi.rowstats(capi.rowstats_args(x=self.x, x_ld=m.K, rows=R, cols=m.K, mode=1, eps=EPS, st=self.pairs))
        stat, off, ld = self.pairs, 1, 2                  # 1 / rms of the embedding; normadd's from then on

        def gemv(w, N, K, x, y, **kw):
            capi.q4_gemvM(capi.gemvm_args(w=w, w_rows=kw.pop("w_rows", N), w_cols=K, x=x, M=R, N=N, K=K, y=y, y_ldm=N, **kw))

        def add(w):
            capi.normadd(capi.normadd_args(t=self.t, t_n=1, t_ld=R * m.K, w=w, x=self.x, st=self.stat, D=m.K, M=R, eps=EPS))
        for i, l in enumerate(m.w):
            rms = dict(pro=capi.PRO["rms"], stat=stat, stat_off=off, stat_ld=ld)
            gemv(l["qkv"], m.width, m.K, self.x, self.qkv, norm=l["norm"][0], **rms)
            kv, size = self._cache(i), 4 * m.dim
            capi.kv_put(capi.kv_rows_args(kv=kv, B=R, M=1, k=self.qkv.ptr + m.heads * size, v=self.qkv.ptr + (m.heads + m.kv_heads) * size,
                                          ldb=m.width, ldm=m.width))
            capi.kv_attn(capi.kv_attn_args(kv=kv, B=R, M=1, heads=m.heads, q=self.qkv, q_ldb=m.width, q_ldm=m.width, y=self.att,
                                           window=self.window, sinks=self.sinks, max_len=self.length))
            gemv(l["o"], m.K, m.heads * m.dim, self.att, self.t)
            add(l["norm"][1])
            stat, off, ld = self.stat, 0, 1
            rms = dict(pro=capi.PRO["rms"], stat=stat, stat_off=off, stat_ld=ld)
            gemv(l["gu"], m.mlp, m.K, self.x, self.h, w_rows=2 * m.mlp, epi=capi.EPI["geglu"], norm=l["norm"][2], **rms)
            gemv(l["down"], m.K, m.mlp, self.h, self.t)
            add(l["norm"][3])
        gemv(m.head, m.vocab, m.K, self.x, self.logits, epi=capi.EPI["softcap"], mx=self.mx, norm=m.head_norm, pro=capi.PRO["rms"],
             stat=stat, stat_off=off, stat_ld=ld)

    def choose(self):
        """each search's W best continuations of its beams -> their tokens; the beams are theirs from then on"""
        before = self.rows // self.n
        capi.beam(capi.beam_args(logits=self.logits, n=self.n, W=before, V=self.m.vocab, k=self.W, score=self.score[0], token=self.token,
                                 parent=self.parent, score_out=self.score[1], hist=self.hist[0], hist_out=self.hist[1],
                                 hist_n=self.steps, hist_ld=self.hist_ld))
        self.score.reverse()
        self.hist.reverse()
        self.steps += 1
        return self.token.read(np.int32, self.n * self.W)

    def run(self, prompts, tokens):
        """prompts [n][at least one token], all of one length -> (tokens [n][W][tokens], scores [n][W]), best first"""
        for column in np.asarray(prompts).T:
            self.sequences(self.n)
            self.forward(column)
        new = self.choose()
        for _ in range(tokens - 1):
            self.sequences(self.n * self.W, src=self.parent)
            self.forward(new)
            new = self.choose()
        hist = self.hist[0].read(np.int32).reshape(-1, self.hist_ld)[:self.n * self.W, :tokens]
        return hist.reshape(self.n, self.W, tokens), self.score[0].read(np.float32, self.n * self.W).reshape(self.n, self.W)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=24)
    a = ap.parse_args()
    capi.open_device(0)
    s = Search(Decoder(), 1, a.beams, longest=8 + a.tokens)
    text, score = s.run([[1, 5, 9, 2]], a.tokens)
    for t, v in zip(text[0], score[0]):
        print("%9.4f  %s" % (v, " ".join(map(str, t))))
    pages = s.ref.read(np.int32, s.n_pages)
    print("%d sequences of %d tokens on %d pages of %d" % (s.rows, s.length, int((pages > 0).sum()), s.page))


if __name__ == "__main__":
    main()
