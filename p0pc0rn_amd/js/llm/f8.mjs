// f8.mjs - a layer's linears in 8-bit floating point and the rotation of its heads, on the MI355X library (include/p0pc0rn.h has each
// call's rules). Buffers are Gpu.buffer handles, views {buf, off}: `off` in bytes; `ld` from row to row, in elements of the view (codes: bytes).
//
// Codes: { buf, off?, ld?, s: { buf, off?, ld? } }: e4m3 bytes and their scales.
'use strict';
import { native } from '../native.mjs';
import { addr, within } from './lops.mjs';

export const F8_TYPE = { f32: 0, f16: 1, bf16: 2 };
const SIZE = { f32: 4, f16: 2, bf16: 2 }, GLU = { none: 0, silu: 1, gelu: 2 }, MODE = { ln: 0, rms: 1 }, ROPE = { inter: 0, half: 1 }, FREQ = { own: 0, shared: 1 };

/** channels rounded up to whole blocks of 128: the bytes of a row of codes */
export const f8Width = (n) => Math.ceil(n / 128) * 128;

const at = (v) => (v && v.buf ? addr(v.buf) + (v.off || 0) : 0);
function pick(op, what, table, v, dflt) {
  const e = table[v === undefined ? dflt : v];
  if (e === undefined) throw new Error(`${op}: ${what} ${v}`);
  return e;
}
/** `rows` rows of `width` elements of `size` bytes fit the view */
function rows(op, name, v, n, width, size, ld) {
  if (v && v.buf && n > 0) within(op, name, v.buf, (v.off || 0) + ((n - 1) * (ld || v.ld || width) + width) * size);
}
/** codes of n rows of d channels with scales (activations: K / 128 rows of n) */
function acts(op, name, v, n, d) {
  const K = f8Width(d);
  rows(op, name, v, n, K, 1);
  rows(op, name + '.s', v.s, n > 0 ? K / 128 : 0, n, 4);
}
function weights(op, name, v, n, d) {
  const K = f8Width(d);
  rows(op, name, v, n, K, 1);
  rows(op, name + '.s', v.s, Math.ceil(n / 128), K / 128, 4);
}

/** a = { x: { buf, off?, ld?, type? }, N, K, w: codes }: a weight into codes */
export function f8Pack(g, a) {
  const op = 'f8_pack', type = pick(op, 'type', F8_TYPE, a.x.type, 'f32');
  rows(op, 'x', a.x, a.N, a.K, SIZE[a.x.type || 'f32']);
  weights(op, 'w', a.w, a.N, a.K);
  native().f8Pack({ x: at(a.x), ldx: a.x.ld || 0, type, N: a.N, K: a.K, w: at(a.w), ldw: a.w.ld || 0, s: at(a.w.s), lds: a.w.s.ld || 0 });
}

/** a = { x: { buf, off?, ld?, type? }, t?: likewise, tw?: view, out?: { buf, off?, ld? }, scale?, eps?, mode?: 'rms' | 'ln', w?: view, wOne?, b?: view,
 *        M, D, y: codes }: the stream's update and its norm */
export function f8Norm(g, a) {
  const op = 'f8_norm', type = pick(op, 'type', F8_TYPE, a.x.type, 'f32'), tt = a.t ? pick(op, 'type', F8_TYPE, a.t.type, 'f32') : 0;
  const size = SIZE[a.x.type || 'f32'];
  rows(op, 'x', a.x, a.M, a.D, size);
  if (a.t) rows(op, 't', a.t, a.M, a.D, SIZE[a.t.type || 'f32']);
  rows(op, 'out', a.out, a.M, a.D, size);
  for (const n of ['tw', 'w', 'b']) rows(op, n, a[n], 1, a.D, 4);
  acts(op, 'y', a.y, a.M, a.D);
  native().f8Norm({
    x: at(a.x), ldx: a.x.ld || 0, type, t: at(a.t), ldt: (a.t && a.t.ld) || 0, t_type: tt, tw: at(a.tw), x_out: at(a.out), ldo: (a.out && a.out.ld) || 0,
    scale: a.scale || 0, eps: a.eps || 0, mode: pick(op, 'mode', MODE, a.mode, 'rms'), w_one: a.wOne ? 1 : 0, w: at(a.w), b: at(a.b), M: a.M, D: a.D,
    y: at(a.y), ldy: a.y.ld || 0, s: at(a.y.s), lds: a.y.s.ld || 0,
  });
}

/** a = { x: { buf, off?, ld?, type?, up? }, glu?: 'none' | 'silu' | 'gelu', M, D, y: codes }: (gated) activations into codes */
export function f8Rows(g, a) {
  const op = 'f8_rows', type = pick(op, 'type', F8_TYPE, a.x.type, 'f32'), glu = pick(op, 'glu', GLU, a.glu, 'none');
  rows(op, 'x', a.x, a.M, glu ? (a.x.up || a.D) + a.D : a.D, SIZE[a.x.type || 'f32']);
  acts(op, 'y', a.y, a.M, a.D);
  native().f8Rows({ x: at(a.x), ldx: a.x.ld || 0, type, up: a.x.up || 0, glu, M: a.M, D: a.D, y: at(a.y), ldy: a.y.ld || 0, s: at(a.y.s), lds: a.y.s.ld || 0 });
}

/** a = { x: codes, w: codes, M, N, K, y: { buf, off?, ld?, type? } }  ->  2 M N K */
export function f8Gemm(g, a) {
  const op = 'f8_gemm', type = pick(op, 'type', F8_TYPE, a.y.type, 'f32');
  acts(op, 'x', a.x, a.M, a.K);
  weights(op, 'w', a.w, a.N, a.K);
  rows(op, 'y', a.y, a.M, a.N, SIZE[a.y.type || 'f32']);
  native().f8Gemm({
    x: at(a.x), ldx: a.x.ld || 0, xs: at(a.x.s), ldxs: a.x.s.ld || 0, w: at(a.w), ldw: a.w.ld || 0, ws: at(a.w.s), ldws: a.w.s.ld || 0,
    M: a.M, N: a.N, K: a.K, type, y: at(a.y), ldy: a.y.ld || 0,
  });
  return 2 * a.M * a.N * a.K;
}

/** a = { x: { buf, off?, ld?, ldh?, type? }, y?: { buf, off?, ld?, ldh? } (without: in place), rows, hq, hk?, dim, mode?: 'inter' | 'half', axisDim?: [..],
 *        freq?: 'own' | 'shared', pos: { buf, off?, ld? }, theta?, qw?: view, kw?: view, eps? } */
export function rope(g, a) {
  const op = 'rope', type = pick(op, 'type', F8_TYPE, a.x.type, 'f32'), size = SIZE[a.x.type || 'f32'], heads = a.hq + (a.hk || 0), y = a.y || a.x;
  const axes = a.axisDim || [a.dim];
  if (axes.length < 1 || axes.length > 4) throw new Error(`rope: ${axes.length} axes`);
  const ld = (v) => v.ld || heads * (v.ldh || a.dim), wide = (v) => (heads - 1) * (v.ldh || a.dim) + a.dim;
  rows(op, 'x', a.x, a.rows, wide(a.x), size, ld(a.x));
  rows(op, 'y', y, a.rows, wide(y), size, ld(y));
  rows(op, 'pos', a.pos, axes.length, a.rows, 4);
  for (const n of ['qw', 'kw']) rows(op, n, a[n], 1, a.dim, 4);
  native().rope({
    x: at(a.x), ldr: a.x.ld || 0, ldh: a.x.ldh || 0, y: at(y), y_ldr: y.ld || 0, y_ldh: y.ldh || 0, type, rows: a.rows, hq: a.hq, hk: a.hk || 0, dim: a.dim,
    mode: pick(op, 'mode', ROPE, a.mode, 'inter'), axes: axes.length, axis0: axes[0], axis1: axes[1] || 0, axis2: axes[2] || 0, axis3: axes[3] || 0,
    freq: pick(op, 'freq', FREQ, a.freq, 'own'), pos: at(a.pos), pos_ld: a.pos.ld || 0, theta: a.theta || 0, qw: at(a.qw), kw: at(a.kw), eps: a.eps || 0,
  });
}
