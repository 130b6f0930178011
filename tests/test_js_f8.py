"""The 8-bit linears and the rotation of heads from Node: refusals (the library's own messages, views against their buffers) without a GPU,
a layer's front on one."""
import json

import numpy as np
import pytest

from oracle import f8
from tests.test_js_host import _save, run_node


def test_refusals(tmp_path):
    out = run_node(tmp_path, r"""
const g = {}, B = { ptr: 4096 }, C = { ptr: 1 << 20 }, D = { ptr: 1 << 21 }, E = { ptr: 1 << 22 }, F = { ptr: 1 << 23 }, small = { ptr: 4096, _pf: 64 };
const codes = (b, s, o) => Object.assign({ buf: b, s: { buf: s } }, o), res = [];
const t = (f) => { try { f(); res.push('no error'); } catch (e) { res.push(e.message); } };
t(() => P.f8Pack(g, { x: { buf: B, type: 'f8' }, N: 4, K: 4, w: codes(C, D) }));
t(() => P.f8Pack(g, { x: { buf: small }, N: 4, K: 5, w: codes(C, D) }));
t(() => P.f8Pack(g, { x: { buf: B }, N: 200, K: 130, w: codes(C, small) }));
t(() => P.f8Norm(g, { x: { buf: B }, t: { buf: small, type: 'f16' }, M: 2, D: 40, y: codes(C, D) }));
t(() => P.f8Norm(g, { x: { buf: B }, mode: 'group', M: 2, D: 40, y: codes(C, D) }));
t(() => P.f8Norm(g, { x: { buf: B }, M: 2, D: 40, y: codes(small, D) }));
t(() => P.f8Rows(g, { x: { buf: small, up: 8 }, glu: 'silu', M: 2, D: 4, y: codes(C, D) }));
t(() => P.f8Rows(g, { x: { buf: B }, glu: 'relu', M: 2, D: 4, y: codes(C, D) }));
t(() => P.f8Gemm(g, { x: codes(B, C), w: codes(D, E), M: 2, N: 4, K: 100, y: { buf: F } }));
t(() => P.f8Gemm(g, { x: codes(B, C), w: codes(D, E), M: 2, N: 40, K: 128, y: { buf: small } }));
t(() => P.f8Gemm(g, { x: codes(B, C), w: codes(D, E), M: 2, N: 40, K: 128, y: { buf: F, ld: 39 } }));
t(() => P.rope(g, { x: { buf: B }, y: { buf: C }, rows: 2, hq: 1, dim: 64, axisDim: [32, 40], pos: { buf: D } }));
t(() => P.rope(g, { x: { buf: B }, rows: 2, hq: 1, dim: 64, axisDim: [], pos: { buf: D } }));
t(() => P.rope(g, { x: { buf: B }, rows: 20, hq: 1, dim: 64, pos: { buf: small } }));
t(() => P.rope(g, { x: { buf: B }, y: { buf: small }, rows: 1, hq: 1, dim: 64, pos: { buf: D } }));
t(() => P.rope(g, { x: { buf: B }, rows: 1, hq: 1, dim: 64, mode: 'third', pos: { buf: D } }));
console.log(JSON.stringify([res, P.f8Width(1), P.f8Width(256)]));
""")
    res, one, two = json.loads(out.strip().splitlines()[-1])
    assert (one, two) == (128, 256)
    assert res == [
        "f8_pack: type f8", "f8_pack: x needs 80 B of a 64 B buffer", "f8_pack: outputs overlap",
        "f8_norm: t needs 160 B of a 64 B buffer", "f8_norm: mode group", "f8_norm: y needs 256 B of a 64 B buffer",
        "f8_rows: x needs 96 B of a 64 B buffer", "f8_rows: glu relu", "f8_gemm: K 100 must be a multiple of 128",
        "f8_gemm: y needs 320 B of a 64 B buffer", "f8_gemm: y has rows of 160 B, 156 B apart",
        "rope: axis 1 of 40 channels (heads of 64)", "rope: 0 axes", "rope: pos needs 80 B of a 64 B buffer", "rope: y needs 256 B of a 64 B buffer",
        "rope: mode third"]


def test_what_is_missing_is_named(tmp_path):
    """an operand, its scales or an output left out: the library's message, not an error of the language"""
    out = run_node(tmp_path, r"""
const g = {}, B = { ptr: 4096 }, C = { ptr: 1 << 20 }, D = { ptr: 1 << 21 }, E = { ptr: 1 << 22 }, F = { ptr: 1 << 23 }, res = [];
const codes = (b, s) => ({ buf: b, s: s && { buf: s } });
const t = (f) => { try { f(); res.push('no error'); } catch (e) { res.push(e.message); } };
t(() => P.f8Pack(g, { N: 4, K: 4, w: codes(C, D) }));
t(() => P.f8Pack(g, { x: { buf: B }, N: 4, K: 4 }));
t(() => P.f8Pack(g, { x: { buf: B }, N: 4, K: 4, w: { buf: C } }));
t(() => P.f8Norm(g, { M: 2, D: 40, y: codes(C, D) }));
t(() => P.f8Norm(g, { x: { buf: B }, M: 2, D: 40 }));
t(() => P.f8Norm(g, { x: { buf: B }, M: 2, D: 40, y: { buf: C } }));
t(() => P.f8Rows(g, { M: 2, D: 4, y: codes(C, D) }));
t(() => P.f8Rows(g, { x: { buf: B }, M: 2, D: 4 }));
t(() => P.f8Rows(g, { x: { buf: B }, M: 2, D: 4, y: codes(C) }));
t(() => P.f8Gemm(g, { w: codes(D, E), M: 2, N: 4, K: 128, y: { buf: F } }));
t(() => P.f8Gemm(g, { x: codes(B), w: codes(D, E), M: 2, N: 4, K: 128, y: { buf: F } }));
t(() => P.f8Gemm(g, { x: codes(B, C), M: 2, N: 4, K: 128, y: { buf: F } }));
t(() => P.f8Gemm(g, { x: codes(B, C), w: codes(D), M: 2, N: 4, K: 128, y: { buf: F } }));
t(() => P.f8Gemm(g, { x: codes(B, C), w: codes(D, E), M: 2, N: 4, K: 128 }));
t(() => P.rope(g, { y: { buf: C }, rows: 2, hq: 1, dim: 64, pos: { buf: D } }));
t(() => P.rope(g, { x: { buf: B }, rows: 2, hq: 1, dim: 64 }));
console.log(JSON.stringify(res));
""")
    assert json.loads(out.strip().splitlines()[-1]) == [
        "f8_pack: missing x buffer", "f8_pack: missing w buffer", "f8_pack: missing s buffer",
        "f8_norm: missing x buffer", "f8_norm: missing y buffer", "f8_norm: missing s buffer",
        "f8_rows: missing x buffer", "f8_rows: missing y buffer", "f8_rows: missing s buffer",
        "f8_gemm: missing x buffer", "f8_gemm: missing xs buffer", "f8_gemm: missing w buffer", "f8_gemm: missing ws buffer", "f8_gemm: missing y buffer",
        "rope: missing x buffer", "rope: missing pos buffer"]


@pytest.mark.gpu
def test_a_layers_front(tmp_path):
    """norm, product, rotation in place, a gate: against the CPU restatement, product and rotation within 2^-15 of the row's largest"""
    M, D, hq, hk, dim = 5, 200, 2, 1, 64
    rng = np.random.default_rng(2)
    x = rng.standard_normal((M, D)).astype(np.float32)
    w = (0.1 * rng.standard_normal(((hq + hk) * dim, D))).astype(np.float32)
    pos = np.stack([np.arange(M), 7 * np.arange(M)]).astype(np.int32)
    _save(tmp_path, x=x, w=w, pos=pos, nw=np.full(D, 0.5, np.float32))
    run_node(tmp_path, r"""
const g = await_gpu();
const up = (name) => { const b = fs.readFileSync(name + '.bin'); return { buf: g.upload(new Uint8Array(b.buffer, b.byteOffset, b.length)) }; };
const [x, w, pos, nw] = ['x', 'w', 'pos', 'nw'].map(up);
const out = (bytes) => ({ buf: g.buffer(bytes) }), codes = (bytes, s) => Object.assign(out(bytes), { s: out(s) });
const wc = codes(192 * 256, 2 * 2 * 4), a = codes(5 * 256, 2 * 5 * 4), gc = codes(5 * 128, 5 * 4), h = out(5 * 192 * 4), r = out(5 * 192 * 4);
P.f8Pack(g, { x: w, N: 192, K: 200, w: wc });
P.f8Norm(g, { x, w: nw, M: 5, D: 200, y: a });
const flops = P.f8Gemm(g, { x: a, w: wc, M: 5, N: 192, K: 256, y: h });
g.runner.copy(h.buf, 0, r.buf, 0, 5 * 192 * 4);
P.rope(g, { x: r, rows: 5, hq: 2, hk: 1, dim: 64, mode: 'half', axisDim: [32, 32], pos, theta: 100 });
P.f8Rows(g, { x: Object.assign({ ld: 192, up: 96 }, h), glu: 'silu', M: 5, D: 96, y: gc });
(async () => {
  await g.done();
  for (const [name, b] of Object.entries({ a, as: a.s, h, r, gc, gs: gc.s })) fs.writeFileSync(name + '.out', Buffer.from(await g.read(b.buf)));
  fs.writeFileSync('flops.out', String(flops));
  g.freeAll(); g.device.destroy();
})();
""")
    got = lambda name, dt, *s: np.fromfile(str(tmp_path / (name + ".out")), dt)[:int(np.prod(s))].reshape(s)  # noqa: E731
    codes, s = got("a", np.uint8, M, 256), got("as", np.float32, 2, M)
    _, want = f8.norm(x, w=np.full(D, 0.5, np.float32))
    assert np.abs(f8.values(codes, s)[:, :D] - want).max() <= 2.0 ** -4 * np.abs(want).max()
    wc, ws = f8.pack(w)
    h = got("h", np.float32, M, 192)
    assert np.abs(h - f8.gemm(codes, s, wc, ws)).max() <= 2.0 ** -15 * np.abs(h).max()
    turned = f8.rope(h.reshape(M, 3, 64), pos, [32, 32], theta=100.0, mode="half", hq=2)
    assert np.abs(got("r", np.float32, M, 3, 64) - turned).max() <= 2.0 ** -15 * np.abs(h).max()
    gate = f8.glu("silu", h[:, :96], h[:, 96:])
    assert np.abs(f8.values(got("gc", np.uint8, M, 128), got("gs", np.float32, 1, M))[:, :96] - gate).max() <= 2.0 ** -4 * np.abs(gate).max()
    assert open(tmp_path / "flops.out").read() == str(2 * M * 192 * 256)
