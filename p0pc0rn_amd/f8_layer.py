"""A decoder's layers in 8-bit floating point over the 4-bit cache: how the operators of a prompt and of its tokens go together.

    python -m p0pc0rn_amd.f8_layer [--prompt 512] [--tokens 16]

The stream is fp32 rows. A layer is: its norm into codes (f8_norm, which also adds the last sub-layer's output), the qkv product
(f8_gemm), the rotation of its query and key heads, each normalised before (rope), keys and values into the cache (kv_put), the new
rows' attention (kv_attn), the result into codes (f8_rows), the o product, the residual update and norm of the FFN (f8_norm), the gate
and up product, its gated activation in codes (f8_rows), the down product. A prompt's rows and a single token's take the same calls.
Weights are random fp32 matrices packed once (f8_pack); positions may have several axes (an image's rows among a text's).
"""
import argparse

import numpy as np

from . import capi

BF16, F32 = capi.TYPE["bf16"], capi.TYPE["f32"]


def width(n):
    """channels rounded up to whole blocks: the bytes of a row of codes"""
    return -(-n // 128) * 128


class Codes:
    """room for codes of `rows` rows of `channels` channels, and their scales"""

    def __init__(self, rows, channels):
        self.K = width(channels)
        self.codes, self.s = capi.Buffer(rows * self.K), capi.Buffer(4 * rows * (self.K // 128))


class Weight:
    """a weight [N, K] (fp32) packed on the device"""

    def __init__(self, w):
        self.N, self.channels = w.shape
        self.K = width(self.channels)
        self.codes, self.s = capi.Buffer(self.N * self.K), capi.Buffer(4 * -(-self.N // 128) * (self.K // 128))
        src = capi.to_device(np.ascontiguousarray(w, np.float32))
        capi.f8_pack(capi.f8_pack_args(x=src, type=F32, N=self.N, K=self.channels, w=self.codes, s=self.s))
        src.free()                                        # waits


class Decoder:
    """`layers` layers of random weights: hidden `K`, `heads` query heads on `kv_heads` key heads of `dim`, FFN `mlp`."""

    def __init__(self, layers=2, K=512, heads=8, kv_heads=2, dim=64, mlp=1024, axis_dim=None, theta=10000.0, mode="half", seed=1):
        if layers < 1:
            raise ValueError("f8_layer: %d layers" % layers)
        self.layers, self.K, self.heads, self.kv_heads, self.dim, self.mlp = layers, K, heads, kv_heads, dim, mlp
        self.axis_dim, self.theta, self.mode = axis_dim or [dim], theta, mode
        self.width = (heads + 2 * kv_heads) * dim
        rng = np.random.default_rng(seed)
        vec = lambda n: capi.to_device((1 + 0.1 * rng.standard_normal(n)).astype(np.float32))  # noqa: E731

        def weight(n, k):
            w = (rng.standard_normal((n, k)) / k ** 0.5).astype(np.float32)
            return Weight(w)
        self.w = [dict(qkv=weight(self.width, K), o=weight(K, heads * dim), gu=weight(2 * mlp, K), down=weight(K, mlp),
                       norm=[vec(K) for _ in range(4)], qn=vec(dim), kn=vec(dim)) for _ in range(layers)]


class Run:
    """`B` sequences of up to `longest` tokens, at most `most` rows of each at a time."""

    def __init__(self, model, B, longest, most, page=64):
        m, R = model, B * most
        self.m, self.B, self.page, self.longest, self.most, self.length = m, B, page, longest, most, 0
        self.cols = -(-longest // page) + 1
        self.n_pages = B * self.cols
        self.layer_bytes = self.n_pages * capi.kv_page_bytes(page, m.kv_heads, m.dim)
        f32 = lambda *s: capi.Buffer(4 * int(np.prod(s)))  # noqa: E731
        bf16 = lambda *s: capi.Buffer(2 * int(np.prod(s)))  # noqa: E731
        self.pages = capi.Buffer(m.layers * self.layer_bytes)
        self.tables, self.lens, self.status = [f32(B, self.cols) for _ in "ab"], [f32(B) for _ in "ab"], f32(4)
        self.tables[0].fill_u32(0xFFFFFFFF)
        self.lens[0].fill_u32(0)
        self.x, self.t, self.pos = f32(R, m.K), f32(R, m.K), f32(len(m.axis_dim), R)
        self.qkv, self.att, self.h = bf16(R, m.width), bf16(R, m.heads * m.dim), bf16(R, 2 * m.mlp)
        self.a, self.ac, self.hc = Codes(R, m.K), Codes(R, m.heads * m.dim), Codes(R, m.mlp)

    def _cache(self, layer=0):
        m = self.m
        return capi.kv(pages=self.pages.ptr + layer * self.layer_bytes, n_pages=self.n_pages, page=self.page, heads=m.kv_heads, dim=m.dim,
                       table=self.tables[0], cols=self.cols, len=self.lens[0])

    def sequences(self, M):
        """M tokens longer"""
        if M > self.most or self.length + M > self.longest:
            raise ValueError("f8_layer: %d rows at a time, %d tokens" % (M, self.length + M))
        capi.kv_update(capi.kv_update_args(kv=self._cache(), B=self.B, grow_n=M, layers=self.m.layers, table_out=self.tables[1], len_out=self.lens[1],
                                           status=self.status))
        self.tables.reverse()
        self.lens.reverse()
        self.length += M

    def _product(self, x, w, R, y, type_):
        capi.f8_gemm(capi.f8_gemm_args(x=x.codes, xs=x.s, w=w.codes, ws=w.s, M=R, N=w.N, K=w.K, type=type_, y=y))

    def forward(self, M):
        """the layers over the rows in self.x at the positions in self.pos, the sequences' newest M tokens; self.x is the stream after them"""
        m, R = self.m, self.B * M
        size, heads = 2 * m.dim, m.heads + m.kv_heads
        last = None                                       # the norm of the sub-layer's output that is still to be added
        for i, l in enumerate(m.w):
            add = dict(t=self.t, t_type=F32, tw=last) if last else {}
            capi.f8_norm(capi.f8_norm_args(x=self.x, type=F32, w=l["norm"][0], M=R, D=m.K, y=self.a.codes, s=self.a.s, **add))
            self._product(self.a, l["qkv"], R, self.qkv, BF16)
            capi.rope(capi.rope_args(x=self.qkv, ldr=m.width, y=self.qkv, y_ldr=m.width, type=BF16, rows=R, hq=m.heads, hk=m.kv_heads, dim=m.dim,
                                     mode=capi.ROPE[m.mode], axis_dim=m.axis_dim, pos=self.pos, theta=m.theta, qw=l["qn"], kw=l["kn"]))
            kv = self._cache(i)
            capi.kv_put(capi.kv_rows_args(kv=kv, B=self.B, M=M, type=BF16, k=self.qkv.ptr + m.heads * size, v=self.qkv.ptr + heads * size,
                                          ldb=M * m.width, ldm=m.width))
            capi.kv_attn(capi.kv_attn_args(kv=kv, B=self.B, M=M, heads=m.heads, type=BF16, q=self.qkv, q_ldb=M * m.width, q_ldm=m.width, y=self.att,
                                           max_len=self.length))
            capi.f8_rows(capi.f8_rows_args(x=self.att, type=BF16, M=R, D=m.heads * m.dim, y=self.ac.codes, s=self.ac.s))
            self._product(self.ac, l["o"], R, self.t, F32)
            capi.f8_norm(capi.f8_norm_args(x=self.x, type=F32, t=self.t, t_type=F32, tw=l["norm"][1], w=l["norm"][2], M=R, D=m.K,
                                           y=self.a.codes, s=self.a.s))
            self._product(self.a, l["gu"], R, self.h, BF16)
            capi.f8_rows(capi.f8_rows_args(x=self.h, type=BF16, glu=capi.GLU["gelu"], M=R, D=m.mlp, y=self.hc.codes, s=self.hc.s))
            self._product(self.hc, l["down"], R, self.t, F32)
            last = l["norm"][3]
        capi.f8_norm(capi.f8_norm_args(x=self.x, type=F32, t=self.t, t_type=F32, tw=last, M=R, D=m.K, y=self.a.codes, s=self.a.s))

    def step(self, rows, pos):
        """rows [B, M, K] (fp32) at positions [axes, B, M]: the sequences' next tokens -> the stream after the layers, [B, M, K]"""
        rows, pos = np.asarray(rows), np.asarray(pos)
        M = rows.shape[1] if rows.ndim == 3 else 0
        if M < 1 or rows.shape != (self.B, M, self.m.K) or pos.shape != (len(self.m.axis_dim), self.B, M):
            raise ValueError("f8_layer: rows %s, positions %s of %d sequences of %d channels, %d axes"
                             % (rows.shape, pos.shape, self.B, self.m.K, len(self.m.axis_dim)))
        self.sequences(M)
        self.x.upload(np.ascontiguousarray(rows, np.float32))
        self.pos.upload(np.ascontiguousarray(pos, np.int32))
        self.forward(M)
        return self.x.read(np.float32, rows.size).reshape(rows.shape)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--tokens", type=int, default=16)
    a = ap.parse_args()
    if a.prompt < 1 or a.tokens < 0:
        ap.error("a prompt has at least one row")
    capi.open_device(0)
    m = Decoder()
    run = Run(m, 1, a.prompt + a.tokens, a.prompt)
    x = np.random.default_rng(2).standard_normal((1, a.prompt + a.tokens, m.K)).astype(np.float32)
    at = np.arange(x.shape[1])[None, None]
    y = run.step(x[:, :a.prompt], at[:, :, :a.prompt])
    print("prompt of %d rows: last row's rms %.4f" % (a.prompt, np.sqrt((y[0, -1] ** 2).mean())))
    for t in range(a.prompt, x.shape[1]):
        y = run.step(x[:, t:t + 1], at[:, :, t:t + 1])
    print("%d tokens: last row's rms %.4f" % (a.tokens, np.sqrt((y[0, -1] ** 2).mean())))


if __name__ == "__main__":
    main()
