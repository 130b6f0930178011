// kv.mjs - keys and values in 4-bit pages, their attention and their pages, and a beam search's step, on the MI355X library
// (include/p0pc0rn.h has each call's rules). Buffers are Gpu.buffer handles, views {buf, off}: `off` in bytes.
//
// A cache: { pages: view, n (pages), bytes? (from page to page), page (tokens: 32 .. 1024), heads, dim (64 | 128 | 256 | 512),
//            table: { buf, ld? }, cols, len: { buf } }
'use strict';
import { native } from '../native.mjs';
import { addr, within } from './lops.mjs';

export const KV_TYPE = { f32: 0, f16: 1, bf16: 2 };
const SIZE = { f32: 4, f16: 2, bf16: 2 };

/** bytes of a page of `page` tokens; 0 where there is no such page */
export const kvPageBytes = (page, heads, dim) => native().kvPageBytes(page, heads, dim);

const at = (v) => (v && v.buf ? addr(v.buf) + (v.off || 0) : 0);
const need = (op, name, v, bytes) => { if (v && v.buf) within(op, name, v.buf, (v.off || 0) + bytes); };
function typeOf(op, t) {
  const e = KV_TYPE[t || 'f32'];
  if (e === undefined) throw new Error(`${op}: type ${t}`);
  return e;
}
/** a cache descriptor's fields, its buffers checked for B sequences and `layers` layers */
function cache(op, c, B, layers = 1, layerBytes = 0) {
  const bytes = c.bytes || kvPageBytes(c.page, c.heads, c.dim), ld = (c.table && c.table.ld) || c.cols;
  need(op, 'pages', c.pages, (layers - 1) * (layerBytes || c.n * bytes) + c.n * bytes);
  need(op, 'table', c.table, B > 0 ? ((B - 1) * ld + c.cols) * 4 : 0);
  need(op, 'len', c.len, B * 4);
  return {
    kv_pages: at(c.pages), kv_n_pages: c.n, kv_page_bytes: c.bytes || 0, kv_page: c.page, kv_heads: c.heads, kv_dim: c.dim,
    kv_table: at(c.table), kv_table_ld: (c.table && c.table.ld) || 0, kv_cols: c.cols, kv_len: at(c.len),
  };
}
/** the extent of rows [B][M][heads][dim] at strides ldb, ldm, ldh (0: one after the other) */
function extent(B, M, heads, dim, v) {
  const ldh = v.ldh || dim, ldm = v.ldm || heads * ldh, ldb = v.ldb || M * ldm;
  return B > 0 && M > 0 ? (B - 1) * ldb + (M - 1) * ldm + (heads - 1) * ldh + dim : 0;
}
function rows(op, call, a) {
  const type = typeOf(op, a.type), n = extent(a.B, a.M, a.kv.heads, a.kv.dim, a) * SIZE[a.type || 'f32'];
  need(op, 'k', a.k, n);
  need(op, 'v', a.v, n);
  need(op, 'rows', a.rows, a.B * 4);
  need(op, 'at', a.at, a.B * 4);
  call({
    ...cache(op, a.kv, a.B), B: a.B, M: a.M, rows: at(a.rows), at: at(a.at), type, k: at(a.k), v: at(a.v),
    ldb: a.ldb || 0, ldm: a.ldm || 0, ldh: a.ldh || 0,
  });
}
/** a = { kv, B, M, rows?: view, at?: view, type: 'f32' | 'f16' | 'bf16', k: view, v: view, ldb?, ldm?, ldh? (elements) } */
export function kvPut(g, a) { rows('kv_put', (o) => native().kvPut(o), a); }
export function kvGet(g, a) { rows('kv_get', (o) => native().kvGet(o), a); }

/** a = { kv, B, M, rows?: view, heads, type, q: { buf, off?, ldb?, ldm?, ldh? }, y: likewise, scale?, window?, sinks?, maxLen? } */
export function kvAttn(g, a) {
  const op = 'kv_attn', type = typeOf(op, a.type), size = SIZE[a.type || 'f32'];
  need(op, 'q', a.q, extent(a.B, a.M, a.heads, a.kv.dim, a.q) * size);
  need(op, 'y', a.y, extent(a.B, a.M, a.heads, a.kv.dim, a.y) * size);
  need(op, 'rows', a.rows, a.B * 4);
  native().kvAttn({
    ...cache(op, a.kv, a.B), B: a.B, M: a.M, rows: at(a.rows), heads: a.heads, type,
    q: at(a.q), q_ldb: a.q.ldb || 0, q_ldm: a.q.ldm || 0, q_ldh: a.q.ldh || 0,
    y: at(a.y), y_ldb: a.y.ldb || 0, y_ldm: a.y.ldm || 0, y_ldh: a.y.ldh || 0,
    scale: a.scale || 0, window: a.window || 0, sinks: a.sinks || 0, max_len: a.maxLen || 0,
  });
}

/** a = { kv, B, Bo?, src?: view, keep?: view, grow?: view | number, window?, sinks?, layers?, layerBytes?,
 *        out: { table: { buf, ld? }, len: view, ref?: view, status: view } } */
export function kvUpdate(g, a) {
  const op = 'kv_update', Bo = a.Bo || a.B, o = a.out, ld = o.table.ld || a.kv.cols;
  need(op, 'table_out', o.table, Bo > 0 ? ((Bo - 1) * ld + a.kv.cols) * 4 : 0);
  need(op, 'len_out', o.len, Bo * 4);
  need(op, 'ref', o.ref, a.kv.n * 4);
  need(op, 'status', o.status, 16);
  for (const n of ['src', 'keep', 'grow']) if (a[n] && a[n].buf) need(op, n, a[n], Bo * 4);
  native().kvUpdate({
    ...cache(op, a.kv, a.B, a.layers || 1, a.layerBytes), B: a.B, Bo, src: at(a.src), keep: at(a.keep), grow: at(a.grow),
    grow_n: typeof a.grow === 'number' ? a.grow : 0, window: a.window || 0, sinks: a.sinks || 0, layers: a.layers || 0,
    layer_bytes: a.layerBytes || 0, table_out: at(o.table), out_ld: o.table.ld || 0, len_out: at(o.len), ref: at(o.ref), status: at(o.status),
  });
}
/** a = { kv, B, layers?, layerBytes?, out: { table: { buf, ld? }, status: view } } */
export function kvCompact(g, a) {
  const op = 'kv_compact', o = a.out, ld = o.table.ld || a.kv.cols;
  need(op, 'table_out', o.table, a.B > 0 ? ((a.B - 1) * ld + a.kv.cols) * 4 : 0);
  need(op, 'status', o.status, 8);
  native().kvCompact({
    ...cache(op, a.kv, a.B, a.layers || 1, a.layerBytes), B: a.B, layers: a.layers || 0, layer_bytes: a.layerBytes || 0,
    table_out: at(o.table), out_ld: o.table.ld || 0, status: at(o.status),
  });
}

/** a = { logits: { buf, off?, ld? }, n, W, V, k, score: view, done?: view, eos?, out: { token, parent, score, done? : views },
 *        hist?: { buf, off?, n, ld?, out: view } } */
export function beam(g, a) {
  const op = 'beam', o = a.out, h = a.hist, R = a.n * a.W, k = a.n * a.k;
  need(op, 'logits', a.logits, R > 0 ? ((R - 1) * (a.logits.ld || a.V) + a.V) * 4 : 0);
  need(op, 'score', a.score, R * 4);
  need(op, 'done', a.done, R * 4);
  for (const n of ['token', 'parent', 'score', 'done']) need(op, n, o[n], k * 4);
  if (h) {
    const ld = h.ld || h.n + 1;
    need(op, 'hist', h, R > 0 ? ((R - 1) * ld + h.n) * 4 : 0);
    need(op, 'hist_out', h.out, k > 0 ? ((k - 1) * ld + h.n + 1) * 4 : 0);
  }
  native().beam({
    logits: at(a.logits), ld: a.logits.ld || 0, n: a.n, W: a.W, V: a.V, k: a.k, score: at(a.score), done: at(a.done),
    eos: a.eos === undefined ? -1 : a.eos, token: at(o.token), parent: at(o.parent), score_out: at(o.score), done_out: at(o.done),
    hist: at(h), hist_out: h ? at(h.out) : 0, hist_n: h ? h.n : 0, hist_ld: (h && h.ld) || 0,
  });
}
