"""The serving operators over a cache of keys and values held in 4 bits, through the C ABI as p0pc0rn_amd.capi binds it.

Keys and values lie in pages of 32-256 tokens (mxfp4: blocks of 32 channels share a power of two, each value is a sign,
two bits of exponent and one of mantissa). kv_put quantises new rows into the pages and kv_get reads rows back; kv_attn is
the attention of the newest rows over the pages, causal, with an optional sliding window and first tokens that stay
visible; kv_update forks, truncates, extends and frees the sequences that share a pool of pages; kv_compact moves the live
pages to the pool's front; beam takes a beam search's best continuations from a head's logits.

listed() names the cases, draw() gives more of the same ranges, prepare() makes what a program holds before the call, run()
is one pass, exact() the same outputs in float64 from the definitions.
"""
import math

import torch

own = False   # False: the plain forms; True: the framework's operators

VOCAB = 262144   # the E2B-shaped head
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E_MIN, E_MAX = -23, 13   # exponents a block may have: every value is then an fp16 value


def listed():
    return [
        # the latency of one new token in a short chat: 8 query heads on 2 key heads, as the E2B-shaped layer has them
        dict(name="attn_decode_517", kind="attn", B=1, M=1, Hq=8, H=2, D=256, T=517, page=64, window=0, sinks=0,
             type="f32", ragged=False),
        # a serving batch: 64 sequences of 0-8192 tokens, one new token each
        dict(name="attn_batch_64", kind="attn", B=64, M=1, Hq=8, H=2, D=256, T=8192, page=64, window=0, sinks=0,
             type="f32", ragged=True),
        # a verify pass of 1 + 4 drafted rows deep into a long document: the balanced pack's 512-wide heads, one key head
        dict(name="attn_verify_131071", kind="attn", B=1, M=5, Hq=8, H=1, D=512, T=131071, page=128, window=0, sinks=0,
             type="f32", ragged=False),
        # prompts read in chunks: 1024 new rows each of two sequences, a window of 4096 tokens and 4 first ones
        dict(name="attn_prefill_window", kind="attn", B=2, M=1024, Hq=16, H=4, D=128, T=8100, page=64, window=4096,
             sinks=4, type="bf16", ragged=True),
        # the newest token's key and value into the cache, and back
        dict(name="put_token", kind="put", B=1, M=1, Hq=8, H=2, D=256, T=700, page=64, type="f32"),
        # eight prompts' rows at once
        dict(name="put_prompts", kind="put", B=8, M=1021, Hq=8, H=2, D=256, T=1500, page=64, type="f16"),
        # one beam search's step: 4 beams go on from their parents, one token longer
        dict(name="update_beams_4", kind="update", groups=1, beams=4, T=513, page=64, H=2, D=256, layers=2, spare=16,
             window=0, sinks=0),
        # 8 searches of 8 beams over 30 layers' pages
        dict(name="update_beams_64", kind="update", groups=8, beams=8, T=3000, page=64, H=2, D=256, layers=30, spare=100,
             window=0, sinks=0),
        # a small pool after one of its sequences has gone
        dict(name="compact_4", kind="compact", B=4, T=700, page=64, H=2, D=256, layers=1, pool=96),
        # a server's pool: 64 sequences in 4096 pages, 8 layers
        dict(name="compact_64", kind="compact", B=64, T=4000, page=64, H=2, D=128, layers=8, pool=4096),
        # one search's step over the whole vocabulary
        dict(name="beam_4", kind="beam", n=1, W=4, k=4, V=VOCAB, hist=40),
        # 32 searches of 8 beams, some of them at their end
        dict(name="beam_32x8", kind="beam", n=32, W=8, k=8, V=VOCAB, hist=200),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "attn", "put", "put", "update", "update", "compact", "beam", "beam"])
    page = rng.choice([32, 64, 64, 128, 256])
    D, H, G = rng.choice([64, 128, 256, 256, 512]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
    if kind == "attn":
        M = rng.choice([1, 1, 1, rng.randint(2, 16), _log(rng, 17, 1024)])
        # at most the batch's cache, and at most the prefill's products
        T = _log(rng, max(M, 33), 131071)
        T = max(M, min(T, 64 * 8192 * 512 // (H * D), 2 * 1024 * 16 * 4096 * 128 // (M * H * G * D)))
        B = _log(rng, 1, max(1, min(64, 64 * 8192 * 512 // (T * H * D), 2 * 1024 * 16 * 4096 * 128 // (T * M * H * G * D))))
        window = rng.choice([0, 0, _log(rng, 16, 8192)])
        return dict(kind="attn", B=B, M=M, Hq=H * G, H=H, D=D, T=T, page=page, window=window,
                    sinks=rng.choice([0, 4, rng.randint(1, 200)]) if window else 0, type=rng.choice(["f32", "f32", "f16", "bf16"]),
                    ragged=rng.random() < 0.6)
    if kind == "put":
        M = rng.choice([1, rng.randint(2, 40), _log(rng, 17, 1024)])
        B = _log(rng, 1, max(1, min(64, 8 * 1024 * 512 // (M * H * D))))
        return dict(kind="put", B=B, M=M, Hq=H * G, H=H, D=D, T=M + rng.randint(0, 700), page=page,
                    type=rng.choice(["f32", "f16", "bf16"]))
    if kind == "update":
        groups, beams = _log(rng, 1, 16), rng.randint(1, 8)
        return dict(kind="update", groups=groups, beams=beams, T=_log(rng, 20, 3000 * 64 // (groups * beams * 2)), page=page, H=2,
                    D=rng.choice([64, 128, 256]), layers=_log(rng, 1, 12), spare=rng.randint(0, 100),
                    window=rng.choice([0, rng.randint(20, 600)]), sinks=rng.choice([0, 4]))
    if kind == "compact":
        B = _log(rng, 1, 64)
        T = _log(rng, 40, 4000)
        return dict(kind="compact", B=B, T=T, page=page, H=2, D=rng.choice([64, 128]), layers=_log(rng, 1, 6),
                    pool=B * -(-T // page) + rng.randint(0, 500))
    n, W = _log(rng, 1, 32), rng.randint(1, 8)
    return dict(kind="beam", n=n, W=W, k=rng.choice([W, W, rng.randint(1, 32)]), V=_log(rng, 500, VOCAB), hist=rng.randint(0, 300))


# ------------------------------------------------------------------------------------------------ the cache, plainly
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_tables = {}


def _pairs():
    """the two values of each of the 256 code bytes, the low four bits first"""
    if "pairs" not in _tables:
        v = [x * s for s in (1.0, -1.0) for x in _GRID]
        _tables["pairs"] = torch.tensor([[v[b & 15], v[b >> 4]] for b in range(256)], device="cuda")
    return _tables["pairs"]


def _codes(x):
    """the 4-bit codes of values scaled to [-6, 6]: the nearest, halves to the even code; larger ones to the largest"""
    a = x.abs()
    c = (a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int()
    return c + 8 * torch.signbit(x).int()


def _quantise(x):
    """rows [..., D] in 32 bits -> code bytes [..., D / 2], exponent bytes [..., D / 32]: the smallest power of two under which
    the block's largest value is at most 6"""
    x = x.reshape(*x.shape[:-1], -1, 32)
    most = x.abs().amax(-1).contiguous()
    e = (((most.view(torch.int32) + 0x3FFFFF) >> 23) - 2).clamp(E_MIN + 127, E_MAX + 127)
    c = _codes(x * _power(254 - e).unsqueeze(-1)).flatten(-2)
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8), e.to(torch.uint8)


def _power(e):
    """2^(e - 127) of integers 1 .. 254"""
    return (e.int() << 23).view(torch.float32)


def _values(codes, exps):
    """rows in 32 bits from their code and exponent bytes"""
    v = _pairs()[codes.int()].flatten(-2)
    return (v.reshape(*exps.shape, 32) * _power(exps).unsqueeze(-1)).flatten(-2)


# A page holds, for each head, runs of 32 tokens of 34 D bytes: the keys' codes and exponents, the values' codes and
# exponents, in the orders that the attention's matrix instructions take them in. These views give both row by row.
def _k_codes(x, D):
    if D == 64:
        return x[..., :16 * D].unflatten(-1, (4, 16, 2, 8)).movedim((-2, -3, -4), (-4, -3, -2)), 4
    return x[..., :16 * D].unflatten(-1, (2, D // 128, 4, 16, 16)).movedim(-2, -4), 5


def _k_exps(x, D):
    x = x[..., 16 * D:17 * D]
    if D == 64:
        return x.unflatten(-1, (2, 16, 2)).movedim((-1, -2, -3), (-3, -2, -1)), 3
    return x.unflatten(-1, (4, 16, 2, D // 128)).movedim((-2, -3, -1, -4), (-4, -3, -2, -1)), 4


def _v_codes(x, D):
    return x[..., 17 * D:33 * D].unflatten(-1, (D // 64, 4, 16, 2, 2, 4)).movedim((-2, -5, -1, -6, -3, -4), (-6, -5, -4, -3, -2, -1)), 6


def _v_exps(x, D):
    return x[..., 33 * D:].unflatten(-1, (4, D // 32, 2, 4)).movedim((-2, -4, -1, -3), (-4, -3, -2, -1)), 4


def _rows(view, n):
    """a view above -> [..., 32 tokens, bytes]"""
    x, dims = view
    return x.reshape(*x.shape[:-dims], 32, n)


def _unpack(x, D):
    """runs [..., 34 D] -> keys, values [..., 32, D] in 32 bits"""
    return (_values(_rows(_k_codes(x, D), D // 2), _rows(_k_exps(x, D), D // 32)),
            _values(_rows(_v_codes(x, D), D // 2), _rows(_v_exps(x, D), D // 32)))


def _places(D):
    """where each byte of a token's row lies in its run: [4 kinds][32, bytes]"""
    if D not in _tables:
        at = torch.arange(34 * D, device="cuda")
        _tables[D] = (_rows(_k_codes(at, D), D // 2), _rows(_k_exps(at, D), D // 32), _rows(_v_codes(at, D), D // 2),
                      _rows(_v_exps(at, D), D // 32))
    return _tables[D]


def _cached(t):
    """every sequence's keys and values, [B, H, T, D] in 32 bits"""
    used = -(-t["T"] // t["page"])
    x = t["pages"][t["table"][:, :used].clamp(min=0).long()]        # [B, used, H, page / 32, 34 D]
    k, v = _unpack(x.transpose(1, 2).flatten(2, 3), t["D"])
    return k.flatten(2, 3), v.flatten(2, 3)


def _visible(t, T):
    """[B, M, T]: which tokens each of the newest rows sees"""
    row = torch.arange(t["M"], device="cuda")
    at = t["len"].view(-1, 1) - t["rows"].view(-1, 1) + row          # the row's own position
    j = torch.arange(T, device="cuda")
    seen = (j <= at.unsqueeze(-1)) & (row < t["rows"].view(-1, 1)).unsqueeze(-1)
    if t["window"]:
        seen &= (j > at.unsqueeze(-1) - t["window"]) | (j < t["sinks"])
    return seen


# ------------------------------------------------------------------------------------------------ inputs
def _page_bytes(c):
    return c["H"] * c["page"] // 32 * 34 * c["D"]


def _pool(g, n, H, page, D):
    """n pages of normally distributed keys and values, as they are held"""
    x = torch.empty(n, H, page // 32, 34 * D, dtype=torch.uint8, device="cuda")
    flat = x.view(-1, 34 * D)
    for i in range(0, flat.shape[0], 1 << 14):
        part = flat[i:i + (1 << 14)]
        for at in (0, 17 * D):
            c = _codes(2.2 * torch.randn(part.shape[0], 16 * D, 2, generator=g, device="cuda"))
            part[:, at:at + 16 * D] = (c[..., 0] | (c[..., 1] << 4)).to(torch.uint8)
            e = 126 + (0.8 * torch.randn(part.shape[0], D, generator=g, device="cuda")).round()
            part[:, at + 16 * D:at + 17 * D] = e.clamp(118, 132).to(torch.uint8)
    return x


def _tables_of(g, length, page, cols, n_pages):
    """pages in no order: table [B, cols], -1 where a sequence has none"""
    need = (length + page - 1) // page
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    j = torch.arange(cols, device="cuda")
    held = j < need.view(-1, 1)
    first = (torch.cumsum(need, 0) - need).view(-1, 1)
    return torch.where(held, order[(first + j).clamp(max=n_pages - 1).long()], -1).int().contiguous()


def prepare(case, seed):
    c, g = dict(case), torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = c["kind"]
    if kind in ("attn", "put"):
        B, M, T, page, D, H = c["B"], c["M"], c["T"], c["page"], c["D"], c["H"]
        n = torch.full((B,), T, device="cuda")
        rows = torch.full((B,), M, device="cuda")
        if c.get("ragged") and B > 1:      # the first is the longest; one may be idle
            u = torch.rand(B, generator=g, device="cuda")
            n[1:] = (u[1:] * (T + 1)).long().clamp(max=T)
            rows = torch.minimum(rows, (n * (0.2 + 0.8 * torch.rand(B, generator=g, device="cuda"))).long())
            rows[0] = M
            if M == 1:
                rows = (n > 0).long()
        cols = -(-T // page) + 1
        pages = B * -(-T // page) + 3
        t = dict(c, pages=_pool(g, pages, H, page, D), len=n.int(), rows=rows.int())
        t["table"] = _tables_of(g, n, page, cols, pages)
        width = (c["Hq"] + 2 * H) * D      # a row of the projection: queries, keys, values
        qkv = torch.randn(B, M, width, generator=g, device="cuda")
        if kind == "put":                  # some channels of the keys are far larger than others
            k = qkv[..., c["Hq"] * D:(c["Hq"] + H) * D]
            k *= torch.exp(0.8 * torch.randn(H * D, generator=g, device="cuda"))
        else:
            qkv[..., :c["Hq"] * D] *= 1.5
        t["qkv"] = qkv.to(TYPES[c["type"]])
        if kind == "attn":
            t["out"] = torch.full((B, M, c["Hq"], D), float("nan"), dtype=TYPES[c["type"]], device="cuda")
            if c["window"]:                # a page that no row can see has been given back
                j = torch.arange(cols, device="cuda")
                gone = ((j + 1) * page <= (n - rows - c["window"] + 1).view(-1, 1)) & (j * page >= c["sinks"])
                t["table"] = torch.where(gone, -1, t["table"]).contiguous()
        else:
            t["k"], t["v"] = (torch.full((B, M, H, D), float("nan"), dtype=TYPES[c["type"]], device="cuda") for _ in "kv")
        return t
    if kind == "update":
        groups, W, page, T = c["groups"], c["beams"], c["page"], c["T"]
        B, cols = groups * W, -(-(T + 1) // page) + 1
        # a search's beams share their first pages; from some page on each has its own
        n = torch.full((groups,), T, device="cuda") - torch.randint(0, max(1, T // 4), (groups,), generator=g, device="cuda")
        split = (torch.rand(groups, generator=g, device="cuda") * (n // page + 1)).long()
        j = torch.arange(cols, device="cuda")
        beam = torch.arange(B, device="cuda")
        keys = torch.where(j < split.repeat_interleave(W).view(-1, 1), (beam // W * W).view(-1, 1), beam.view(-1, 1)) * cols + j
        held = j < (-(-n // page)).repeat_interleave(W).view(-1, 1)
        number, back = torch.unique(keys[held], return_inverse=True)
        P = B * cols + B + c["spare"]
        t = dict(c, B=B, cols=cols, n_pages=P, len=n.repeat_interleave(W).int(), table=torch.full((B, cols), -1, dtype=torch.int32, device="cuda"))
        t["table"][held] = torch.randperm(P, generator=g, device="cuda").int()[back]
        t["src"] = (torch.randint(0, W, (groups, W), generator=g, device="cuda") + torch.arange(0, B, W, device="cuda").view(-1, 1)).flatten().int()
        t["pages"] = torch.empty(c["layers"], P, _page_bytes(c) // 4, dtype=torch.int32, device="cuda")
        t["pages"].random_(-(1 << 31), 1 << 31, generator=g)
        t["table_out"], t["len_out"] = torch.full_like(t["table"], -7), torch.full_like(t["len"], -7)
        t["ref"] = torch.full((P,), -7, dtype=torch.int32, device="cuda")
        t["status"] = torch.full((4,), -7, dtype=torch.int32, device="cuda")
        return t
    if kind == "compact":
        B, page, T = c["B"], c["page"], c["T"]
        cols = -(-T // page)
        n = (torch.rand(B, generator=g, device="cuda") * T).long() + 1
        n[0] = T
        t = dict(c, cols=cols, n_pages=c["pool"], len=n.int(), table=_tables_of(g, n, page, cols, c["pool"]))
        t["pages"] = torch.empty(c["layers"], c["pool"], _page_bytes(c) // 4, dtype=torch.int32, device="cuda")
        t["pages"].random_(-(1 << 31), 1 << 31, generator=g)
        t["table_out"] = torch.full_like(t["table"], -7)
        t["status"] = torch.full((2,), -7, dtype=torch.int32, device="cuda")
        return t
    R, V, n, k = c["n"] * c["W"], c["V"], c["n"], c["k"]
    t = dict(c, logits=30 * torch.tanh(torch.randn(R, V, generator=g, device="cuda") * 0.1), eos=1)
    # a head that knows what comes next: a few words stand out
    t["logits"].scatter_add_(1, torch.randint(0, V, (R, 64), generator=g, device="cuda"), 3 * torch.randn(R, 64, generator=g, device="cuda"))
    t["score"] = -20 * torch.rand(R, generator=g, device="cuda")
    t["done"] = (torch.rand(R, generator=g, device="cuda") < 0.1).int()
    t["hist"] = torch.randint(0, V, (R, c["hist"] + 1), generator=g, device="cuda").int()
    i32 = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")  # noqa: E731
    t.update(token=i32(n, k), parent=i32(n, k), done_out=i32(n, k), hist_out=i32(n * k, c["hist"] + 1),
             score_out=torch.full((n, k), float("nan"), device="cuda"))
    return t


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_attn(t):
    B, M, H, D = t["B"], t["M"], t["H"], t["D"]
    G = t["Hq"] // H
    k, v = _cached(t)
    q = t["qkv"][..., :t["Hq"] * D].float().view(B, M, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * M, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(D))
    s = s.view(B, H, G, M, -1).masked_fill_(~_visible(t, k.shape[2]).view(B, 1, 1, M, -1), -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, H, G * M, -1), v).view(B, H, G, M, D) / torch.where(total > 0, total, torch.ones_like(total))
    t["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(B, M, t["Hq"], D))
    return t["out"]


def _plain_put(t):
    B, M, H, D, page = t["B"], t["M"], t["H"], t["D"], t["page"]
    kv = t["qkv"][..., t["Hq"] * D:].float().view(B, M, 2, H, D)
    pos = (t["len"] - t["rows"]).view(-1, 1).long() + torch.arange(M, device="cuda")
    where = t["table"].gather(1, pos // page).long()                        # the page of each row
    run = (where.unsqueeze(-1) * H + torch.arange(H, device="cuda")) * (page // 32) + (pos % page // 32).unsqueeze(-1)
    flat, places = t["pages"].view(-1), _places(D)
    parts = [*_quantise(kv[:, :, 0]), *_quantise(kv[:, :, 1])]
    held = [run.unsqueeze(-1) * (34 * D) + p[pos % 32].unsqueeze(2) for p in places]
    for at, part in zip(held, parts):
        flat[at] = part
    t["k"].copy_(_values(flat[held[0]], flat[held[1]]))
    t["v"].copy_(_values(flat[held[2]], flat[held[3]]))
    return {"k": t["k"], "v": t["v"]}


def _plain_update(t):
    B, P, page, cols = t["B"], t["n_pages"], t["page"], t["cols"]
    src, kept = t["src"].long(), t["len"][t["src"].long()].long()
    new_len = kept + 1
    j = torch.arange(cols, device="cuda")
    held = j < ((kept + page - 1) // page).view(-1, 1)
    if t["window"]:
        held &= ((j + 1) * page > (kept - t["window"] + 1).view(-1, 1)) | (j * page < t["sinks"])
    table = torch.where(held, t["table"][src], -1).long()
    count = lambda x: torch.zeros(P + 1, dtype=torch.long, device="cuda").scatter_add_(0, x.flatten(), torch.ones_like(x.flatten()))  # noqa: E731
    ref = count(torch.where(table >= 0, table, P))
    last = kept // page                                                     # the page the new token goes to
    open_ = torch.where(kept % page > 0, table.gather(1, last.view(-1, 1)).view(-1), P)
    writers = count(open_)
    row = torch.arange(B, device="cuda")
    first = torch.full((P + 1,), B, device="cuda").scatter_reduce_(0, open_, row, "amin")
    copy = (open_ < P) & (ref[open_] > 1) & ~((ref[open_] == writers[open_]) & (first[open_] == row))
    wants = (j == last.view(-1, 1)) & (copy | (open_ == P)).view(-1, 1)
    free = ref[:P] == 0
    rank = torch.cumsum(free, 0) - 1
    listed_ = torch.zeros(P + 1, dtype=torch.long, device="cuda").scatter_(0, torch.where(free, rank, P), torch.arange(P, device="cuda"))
    mine = listed_[(torch.cumsum(wants.flatten(), 0) - 1).clamp(min=0)].view(B, cols)
    out = torch.where(wants, mine, table)
    dst = out.gather(1, last.view(-1, 1)).view(-1)[copy]
    t["pages"][:, dst] = t["pages"][:, open_[copy]]
    t["table_out"].copy_(out)
    t["len_out"].copy_(new_len)
    t["ref"].copy_(count(torch.where(out >= 0, out, P))[:P])
    t["status"].copy_(torch.stack([torch.zeros_like(rank[0]), free.sum() - wants.sum(), copy.sum(), torch.zeros_like(rank[0])]))
    return {"table": t["table_out"], "len": t["len_out"], "ref": t["ref"], "status": t["status"], "pages": t["pages"]}


def _plain_compact(t):
    P = t["n_pages"]
    table = t["table"].long()
    live = torch.zeros(P + 1, dtype=torch.bool, device="cuda")
    live[torch.where(table >= 0, table, P)] = True
    live = live[:P]
    at = torch.arange(P, device="cuda")
    n = live.sum()
    moved, hole = live & (at >= n), ~live & (at < n)
    to = torch.arange(P + 1, device="cuda")
    to[:P][moved] = at[hole]                                                # both in ascending order
    t["pages"][:, at[hole]] = t["pages"][:, at[moved]]
    t["table_out"].copy_(torch.where(table >= 0, to[table], -1))
    t["status"].copy_(torch.stack([n, moved.sum()]))
    return {"table": t["table_out"], "status": t["status"], "pages": t["pages"]}


def _plain_beam(t):
    n, W, k, V = t["n"], t["W"], t["k"], t["V"]
    x = torch.where(torch.isnan(t["logits"]), -math.inf, t["logits"]) + 0.0
    most = x.amax(1, keepdim=True)
    lse = most + torch.log(torch.exp(x - most).sum(1, keepdim=True))
    bits = x.view(torch.int32)
    order = ((bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32) + (0xFFFFFFFF - torch.arange(V, device="cuda"))
    token = 0xFFFFFFFF - (torch.topk(order, k, 1).values & 0xFFFFFFFF)      # by value, equal ones by their index
    s = t["score"].view(-1, 1) + (x.gather(1, token) - lse)
    s = torch.where(torch.isnan(s), -math.inf, s)
    ended = torch.full_like(s, -math.inf)
    ended[:, 0] = t["score"]
    done = t["done"].view(-1, 1) != 0
    s, token = torch.where(done, ended, s).view(n, W * k), torch.where(done, t["eos"], token).view(n, W * k)
    s, at = torch.sort(s, dim=1, descending=True, stable=True)
    at = at[:, :k]
    t["score_out"].copy_(s[:, :k])
    t["token"].copy_(token.gather(1, at))
    t["parent"].copy_(at // k + torch.arange(0, n * W, W, device="cuda").view(-1, 1))
    parent = t["parent"].long().flatten()
    t["done_out"].copy_(((t["done"][parent].view(n, k) != 0) | (t["token"] == t["eos"])).int())
    t["hist_out"].copy_(torch.cat([t["hist"][parent][:, :t["hist"].shape[1] - 1], t["token"].view(-1, 1)], 1))
    return {"token": t["token"], "parent": t["parent"], "score": t["score_out"], "done": t["done_out"], "hist": t["hist_out"]}


# ------------------------------------------------------------------------------------------------ one pass
def _library():
    """the framework's binding, its device opened"""
    if "capi" not in _tables:
        from p0pc0rn_amd import capi
        capi.open_device(0)
        _tables["capi"] = capi
    return _tables["capi"]


def run(t):
    kind = t["kind"]
    if not own:
        return {"attn": _plain_attn, "put": _plain_put, "update": _plain_update, "compact": _plain_compact, "beam": _plain_beam}[kind](t)
    capi = _library()
    if kind in ("attn", "put"):
        D, H, Hq, M = t["D"], t["H"], t["Hq"], t["M"]
        qkv, size = t["qkv"].data_ptr(), t["qkv"].element_size()
        ldm = (Hq + 2 * H) * D
        kv = capi.kv(pages=t["pages"].data_ptr(), n_pages=t["pages"].shape[0], page=t["page"], heads=H, dim=D,
                     table=t["table"].data_ptr(), cols=t["table"].shape[1], len=t["len"].data_ptr())
        if kind == "attn":
            capi.kv_attn(capi.kv_attn_args(kv=kv, B=t["B"], M=M, rows=t["rows"].data_ptr(), heads=Hq, type=capi.KV_TYPE[t["type"]],
                                           q=qkv, q_ldb=M * ldm, q_ldm=ldm, y=t["out"].data_ptr(), window=t["window"],
                                           sinks=t["sinks"], max_len=t["T"]))
            return t["out"]
        args = dict(kv=kv, B=t["B"], M=M, rows=t["rows"].data_ptr(), type=capi.KV_TYPE[t["type"]])
        capi.kv_put(capi.kv_rows_args(k=qkv + Hq * D * size, v=qkv + (Hq + H) * D * size, ldb=M * ldm, ldm=ldm, **args))
        capi.kv_get(capi.kv_rows_args(k=t["k"].data_ptr(), v=t["v"].data_ptr(), **args))
        return {"k": t["k"], "v": t["v"]}
    if kind in ("update", "compact"):
        kv = capi.kv(pages=t["pages"].data_ptr(), n_pages=t["n_pages"], page=t["page"], heads=t["H"], dim=t["D"],
                     table=t["table"].data_ptr(), cols=t["cols"], len=t["len"].data_ptr())
        if kind == "update":
            capi.kv_update(capi.kv_update_args(kv=kv, B=t["B"], src=t["src"].data_ptr(), grow_n=1, window=t["window"], sinks=t["sinks"],
                                               layers=t["layers"], table_out=t["table_out"].data_ptr(), len_out=t["len_out"].data_ptr(),
                                               ref=t["ref"].data_ptr(), status=t["status"].data_ptr()))
            return {"table": t["table_out"], "len": t["len_out"], "ref": t["ref"], "status": t["status"], "pages": t["pages"]}
        capi.kv_compact(capi.kv_compact_args(kv=kv, B=t["B"], layers=t["layers"], table_out=t["table_out"].data_ptr(),
                                             status=t["status"].data_ptr()))
        return {"table": t["table_out"], "status": t["status"], "pages": t["pages"]}
    capi.beam(capi.beam_args(logits=t["logits"].data_ptr(), n=t["n"], W=t["W"], V=t["V"], k=t["k"], score=t["score"].data_ptr(),
                             done=t["done"].data_ptr(), eos=t["eos"], token=t["token"].data_ptr(), parent=t["parent"].data_ptr(),
                             score_out=t["score_out"].data_ptr(), done_out=t["done_out"].data_ptr(), hist=t["hist"].data_ptr(),
                             hist_out=t["hist_out"].data_ptr(), hist_n=t["hist"].shape[1] - 1, hist_ld=t["hist"].shape[1]))
    return {"token": t["token"], "parent": t["parent"], "score": t["score_out"], "done": t["done_out"], "hist": t["hist_out"]}


def work(case):
    c, kind = case, case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}.get(c.get("type"), 0)
    if kind == "attn":
        half = 0.5 if c["ragged"] and c["B"] > 1 else 1.0
        T = c["T"] * (1 + half * (c["B"] - 1)) / c["B"]                     # a sequence's mean length
        M = c["M"] if not c["ragged"] else min(c["M"], T)
        mean = min(T - (M - 1) / 2, c["window"] + min(c["sinks"], T) if c["window"] else T)   # tokens a row sees
        read = min(T, c["window"] + M - 1 + c["sinks"]) if c["window"] else T
        return {"bytes": c["B"] * (read * c["H"] * c["D"] * 17 / 16 + 2 * M * c["Hq"] * c["D"] * size),
                "flops": 4.0 * c["B"] * M * c["Hq"] * c["D"] * mean}
    if kind == "put":   # the rows in, their pages' bytes out and in, the rows out
        n = c["B"] * c["M"] * c["H"] * c["D"]
        return {"bytes": n * (4 * size + 2 * 17 / 16), "flops": 0}
    if kind == "update":
        B, cols = c["groups"] * c["beams"], -(-(c["T"] + 1) // c["page"]) + 1
        share = 1 - (1 - 1 / c["beams"]) ** c["beams"]                      # of a search's beams that have a child
        copies = 0.0 if c["page"] == 1 else B * (1 - share) * (1 - 1 / c["page"])
        return {"bytes": 8 * B * cols + 4 * (B * cols // 2) + 2 * copies * c["layers"] * _page_bytes(c), "flops": 0}
    if kind == "compact":
        held = min(c["pool"], (1 + (c["B"] - 1) / 2) * -(-c["T"] // c["page"]))
        moved = held * (1 - held / c["pool"])
        return {"bytes": 8 * c["B"] * -(-c["T"] // c["page"]) + 2 * moved * c["layers"] * _page_bytes(c), "flops": 0}
    rows = c["n"] * c["W"]
    return {"bytes": 4.0 * rows * c["V"] + 8 * c["n"] * c["k"] * c["hist"], "flops": 3.0 * rows * c["V"]}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _decode64(page_runs, D, what):
    """[32, D] values of runs [n, 34 D], found one byte at a time: token, channel -> its code, its exponent"""
    tok, ch = torch.meshgrid(torch.arange(32, device="cuda"), torch.arange(D, device="cuda"), indexing="ij")
    if what == "k":
        if D == 64:
            at = ((ch // 16) * 16 + tok % 16) * 16 + (tok // 16) * 8 + ch % 16 // 2
            ex = 1024 + (ch // 32 * 16 + tok % 16) * 2 + tok // 16
        else:
            u, lane = ch // 128, (ch % 128 // 32) * 16 + tok % 16
            at = ((tok // 16) * (D // 128) + u) * 1024 + lane * 16 + ch % 32 // 2
            ex = 16 * D + (lane * 2 + tok // 16) * (D // 128) + u
    else:
        lane, j = tok % 16 // 4, tok // 16 * 4 + tok % 4
        at = 17 * D + (ch // 64) * 1024 + (lane * 16 + ch % 32 // 2) * 16 + (ch // 32 % 2) * 8 + j
        ex = 33 * D + (lane * (D // 32) + ch // 32) * 8 + j
    code = page_runs[:, at.flatten()].to(torch.int64) >> (4 * (ch % 2)).flatten() & 15
    two, one = code >> 1 & 3, code & 1
    mag = torch.where(two == 0, 0.5 * one, (1 + 0.5 * one) * 2.0 ** (two - 1).double())
    val = torch.where(code >= 8, -mag, mag).double() * 2.0 ** (page_runs[:, ex.flatten()].double() - 127)
    return val.view(-1, 32, D)


def exact(case, seed):
    kind = case["kind"]
    if kind in ("update", "compact"):
        return None                                                         # whole numbers and moved bytes only
    t = prepare(case, seed)
    if kind == "beam":
        x = t["logits"].double()
        s = t["score"].double().view(-1, 1) + torch.log_softmax(x, 1)
        s = torch.where(t["done"].view(-1, 1) != 0, -math.inf, s)
        s[:, t["eos"]] = torch.where(t["done"] != 0, t["score"].double(), s[:, t["eos"]])
        return {"token": None, "parent": None, "done": None, "hist": None, "score": torch.topk(s.view(t["n"], -1), t["k"], 1).values}
    B, M, H, Hq, D, page = t["B"], t["M"], t["H"], t["Hq"], t["D"], t["page"]
    if kind == "put":
        out = {}
        for name, first in (("k", Hq * D), ("v", (Hq + H) * D)):
            x = t["qkv"][..., first:first + H * D].double().view(B, M, H, D // 32, 32)
            e = torch.ceil(torch.log2((x.abs().amax(-1, keepdim=True) / 6).clamp(min=2.0 ** -40))).clamp(E_MIN, E_MAX)
            y = x.abs() / 2.0 ** e
            step = 2.0 ** (torch.floor(torch.log2(y.clamp(min=1.0))).clamp(max=2) - 1)
            out[name] = (torch.sign(x) * (torch.round(y / step) * step).clamp(max=6) * 2.0 ** e).view(B, M, H, D)
        return out
    out = torch.zeros(B, M, Hq, D, dtype=torch.float64, device="cuda")
    lengths, rows = t["len"].tolist(), t["rows"].tolist()
    for b in range(B):
        n, m = lengths[b], rows[b]
        if m == 0:
            continue
        runs = t["pages"][t["table"][b, :-(-n // page)].clamp(min=0).long()]
        j = torch.arange(n, device="cuda")
        p = torch.arange(n - m, n, device="cuda").view(-1, 1)
        hidden = j > p
        if t["window"]:
            hidden |= (j <= p - t["window"]) & (j >= t["sinks"])
        for h in range(H):
            k, v = (_decode64(runs[:, h].reshape(-1, 34 * D), D, w).reshape(-1, D)[:n] for w in "kv")
            for q in range(h * (Hq // H), (h + 1) * (Hq // H)):
                s = (t["qkv"][b, :m, q * D:(q + 1) * D].double() @ k.t()) / math.sqrt(D)
                out[b, :m, q] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v
    return out
