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

const at = (v) => (v && v.buf ? addr(v.buf) + (v.off || 0) : 0), ld = (v) => (v && v.ld) || 0;   // a view that is not there: 0, which the call refuses by name
const kind = (v) => (v && v.type) || 'f32', scales = (v) => v && v.s;
function pick(op, what, table, v, dflt) {
  const e = table[v === undefined ? dflt : v];
  if (e === undefined) throw new Error(`${op}: ${what} ${v}`);
  return e;
}
/** `rows` rows of `width` elements of `size` bytes fit the view */
function rows(op, name, v, n, width, size, apart) {
  if (v && v.buf && n > 0) within(op, name, v.buf, (v.off || 0) + ((n - 1) * (apart || v.ld || width) + width) * size);
}
/** codes of n rows of d channels with scales (activations: K / 128 rows of n) */
function acts(op, name, v, n, d) {
  const K = f8Width(d);
  rows(op, name, v, n, K, 1);
  rows(op, name + '.s', scales(v), n > 0 ? K / 128 : 0, n, 4);
}
function weights(op, name, v, n, d) {
  const K = f8Width(d);
  rows(op, name, v, n, K, 1);
  rows(op, name + '.s', scales(v), Math.ceil(n / 128), K / 128, 4);
}

/** a = { x: { buf, off?, ld?, type? }, N, K, w: codes }: a weight into codes */
export function f8Pack(g, a) {
  const op = 'f8_pack', type = pick(op, 'type', F8_TYPE, kind(a.x));
  rows(op, 'x', a.x, a.N, a.K, SIZE[kind(a.x)]);
  weights(op, 'w', a.w, a.N, a.K);
  native().f8Pack({ x: at(a.x), ldx: ld(a.x), type, N: a.N, K: a.K, w: at(a.w), ldw: ld(a.w), s: at(scales(a.w)), lds: ld(scales(a.w)) });
}

/** a = { x: { buf, off?, ld?, type? }, t?: likewise, tw?: view, out?: { buf, off?, ld? }, scale?, eps?, mode?: 'rms' | 'ln', w?: view, wOne?, b?: view,
 *        M, D, y: codes }: the stream's update and its norm */
export function f8Norm(g, a) {
  const op = 'f8_norm', type = pick(op, 'type', F8_TYPE, kind(a.x)), tt = a.t ? pick(op, 'type', F8_TYPE, kind(a.t)) : 0;
  const size = SIZE[kind(a.x)];
  rows(op, 'x', a.x, a.M, a.D, size);
  if (a.t) rows(op, 't', a.t, a.M, a.D, SIZE[kind(a.t)]);
  rows(op, 'out', a.out, a.M, a.D, size);
  for (const n of ['tw', 'w', 'b']) rows(op, n, a[n], 1, a.D, 4);
  acts(op, 'y', a.y, a.M, a.D);
  native().f8Norm({
    x: at(a.x), ldx: ld(a.x), type, t: at(a.t), ldt: ld(a.t), t_type: tt, tw: at(a.tw), x_out: at(a.out), ldo: ld(a.out),
    scale: a.scale || 0, eps: a.eps || 0, mode: pick(op, 'mode', MODE, a.mode, 'rms'), w_one: a.wOne ? 1 : 0, w: at(a.w), b: at(a.b), M: a.M, D: a.D,
    y: at(a.y), ldy: ld(a.y), s: at(scales(a.y)), lds: ld(scales(a.y)),
  });
}

/** a = { x: { buf, off?, ld?, type?, up? }, glu?: 'none' | 'silu' | 'gelu', M, D, y: codes }: (gated) activations into codes */
export function f8Rows(g, a) {
  const op = 'f8_rows', type = pick(op, 'type', F8_TYPE, kind(a.x)), glu = pick(op, 'glu', GLU, a.glu, 'none');
  rows(op, 'x', a.x, a.M, glu ? ((a.x && a.x.up) || a.D) + a.D : a.D, SIZE[kind(a.x)]);
  acts(op, 'y', a.y, a.M, a.D);
  native().f8Rows({ x: at(a.x), ldx: ld(a.x), type, up: (a.x && a.x.up) || 0, glu, M: a.M, D: a.D, y: at(a.y), ldy: ld(a.y), s: at(scales(a.y)), lds: ld(scales(a.y)) });
}

/** a = { x: codes, w: codes, M, N, K, y: { buf, off?, ld?, type? } }  ->  2 M N K */
export function f8Gemm(g, a) {
  const op = 'f8_gemm', type = pick(op, 'type', F8_TYPE, kind(a.y));
  acts(op, 'x', a.x, a.M, a.K);
  weights(op, 'w', a.w, a.N, a.K);
  rows(op, 'y', a.y, a.M, a.N, SIZE[kind(a.y)]);
  native().f8Gemm({
    x: at(a.x), ldx: ld(a.x), xs: at(scales(a.x)), ldxs: ld(scales(a.x)), w: at(a.w), ldw: ld(a.w), ws: at(scales(a.w)), ldws: ld(scales(a.w)),
    M: a.M, N: a.N, K: a.K, type, y: at(a.y), ldy: ld(a.y),
  });
  return 2 * a.M * a.N * a.K;
}

/** a = { x: { buf, off?, ld?, ldh?, type? }, y?: { buf, off?, ld?, ldh? } (without: in place), rows, hq, hk?, dim, mode?: 'inter' | 'half', axisDim?: [..],
 *        freq?: 'own' | 'shared', pos: { buf, off?, ld? }, theta?, qw?: view, kw?: view, eps? } */
export function rope(g, a) {
  const op = 'rope', x = a.x || {}, y = a.y || x, type = pick(op, 'type', F8_TYPE, kind(x)), size = SIZE[kind(x)], heads = a.hq + (a.hk || 0);
  const axes = a.axisDim || [a.dim];
  if (axes.length < 1 || axes.length > 4) throw new Error(`rope: ${axes.length} axes`);
  const apart = (v) => v.ld || heads * (v.ldh || a.dim), wide = (v) => (heads - 1) * (v.ldh || a.dim) + a.dim;
  rows(op, 'x', x, a.rows, wide(x), size, apart(x));
  rows(op, 'y', y, a.rows, wide(y), size, apart(y));
  rows(op, 'pos', a.pos, axes.length, a.rows, 4);
  for (const n of ['qw', 'kw']) rows(op, n, a[n], 1, a.dim, 4);
  native().rope({
    x: at(x), ldr: ld(x), ldh: x.ldh || 0, y: at(y), y_ldr: ld(y), y_ldh: y.ldh || 0, type, rows: a.rows, hq: a.hq, hk: a.hk || 0, dim: a.dim,
    mode: pick(op, 'mode', ROPE, a.mode, 'inter'), axes: axes.length, axis0: axes[0], axis1: axes[1] || 0, axis2: axes[2] || 0, axis3: axes[3] || 0,
    freq: pick(op, 'freq', FREQ, a.freq, 'own'), pos: at(a.pos), pos_ld: ld(a.pos), theta: a.theta || 0, qw: at(a.qw), kw: at(a.kw), eps: a.eps || 0,
  });
}
