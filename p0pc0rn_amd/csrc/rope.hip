// rope.hip - the rotation of query and key heads by positions on one to four axes, after an optional norm of each head.
//
// Pair i of a head, (u, v) -> (u cos - v sin, v cos + u sin), has angle pos theta^-e: the same for every head of a row. A workgroup
// takes a few rows, works their cosines and sines out once (in LDS), and streams the rows' heads through. An angle of a far position
// is many turns: it is held in 64 bits, in turns; the fraction of a turn goes on in two 32-bit parts (in one, cosines are off by 3.3e-8 in the mean square, in two
// by 1.9e-8, at the same time: once a row, not once a head).
//
// Bound: HBM (32760 rows of 40 heads of 128 bf16 channels on three axes: 123 us for 671 MB, 5.4 TB/s; a copy of as many bytes 125), launch and
// round trips at few rows (1 row of 10 heads of 256 fp32 channels, normalised: 5.4-5.7 us, of the kernel 4.4). Halves whose pairs are no multiple
// of 8 take up to twice as long as whole ones, for runs that begin off any 32 bytes and single stores at their ends (us, 8000 rows of 10 bf16 heads: 126
// of 128 channels turn 21.2, all 10.6; 100 of 100 15.3, 96 of 96 9.7).
#include "f8_common.hpp"

#include <cmath>

namespace p0 {

constexpr int kRopeThreads = 256, kRopePairs = 256, kRopeTable = 2048;   // pairs of a head at most; angles of a workgroup's rows
struct RopeP {
  const void* x;
  void* y;
  const int32_t* pos;
  const float* qw;
  const float* kw;
  int64_t ldr, ldh, yldr, yldh, pos_ld, rows;
  double pow[4][8];           // an axis's frequency, in turns a position: pow[0] of its first pair's axis times the bits of the pair's number
  int heads, hq, dim, R;      // R: channels that turn
  int first[4];               // an axis's first pair
  int axes, shared, inter;
  int rb, hb, hblocks;        // rows, heads of a workgroup, workgroups a row block
  int ls, nl;                 // 1 << ls lanes take a head; halves: the first nl of them what turns
  float eps;
};

__device__ __forceinline__ float2 rope_turn(const RopeP& p, int64_t row, int i) {
  if (i >= p.R / 2) return float2{1.0f, 0.0f};
  int a = 0;
  for (int k = 1; k < p.axes; ++k) a = i >= p.first[k] ? k : a;
  // theta^-e / 2 pi: pair j of its axis (of all, where the axes share one range) has the frequency of pair 1 to the power of j, by j's bits
  const int j = p.shared ? i : i - p.first[a];
  double f = 0.15915494309189535;
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const double t = f * p.pow[a][b];
    f = j >> b & 1 ? t : f;
  }
  const double turns = (double)p.pos[a * p.pos_ld + row] * f;
  // half turns in two parts: the sine and cosine of the 32-bit one, turned on by what it rounds off (up to 2^-26 of a half turn: its square counts for nothing)
  const double half = 2.0 * (turns - rint(turns));
  const float at = (float)half, rest = (float)(half - (double)at) * 3.14159265f;
  float s, c;
  sincospif(at, &s, &c);
  return float2{__builtin_fmaf(-s, rest, c), __builtin_fmaf(c, rest, s)};
}

// A lane has the same up to 8 pairs (halves: 8 first channels and their 8 partners) or 4 (neighbours: a run of 8 channels) of its head throughout; channels
// that do not turn go to further lanes, 16 each (halves), or with their neighbours. Runs of 8 are whole 16-byte accesses at any alignment (9 rows of 24
// heads of 512 fp32 channels, of which 384 turn by halves: 4.7 us, where single channels took 6.1).
// WHOLE: every lane has all of its pairs, so no counts are looked at: 32760 rows of 40 heads of 128 bf16 channels, by halves and normalised, 132 us, with them 203.
template <int TYPE, bool HALF, bool WHOLE>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(const RopeP p) {
  __shared__ __attribute__((aligned(16))) float2 turn[kRopeTable + 8];   // (a last lane may read past its pairs)
  const int64_t group = f8_group(), blk = group / p.hblocks, row0 = blk * p.rb;
  const int h0 = (int)(group - blk * p.hblocks) * p.hb, pairs = p.dim / 2;
  if (row0 >= p.rows) return;
  const int rows = (int)(p.rows - row0 < p.rb ? p.rows - row0 : p.rb), hb = p.heads - h0 < p.hb ? p.heads - h0 : p.hb;
  for (int k = threadIdx.x; k < rows * pairs; k += kRopeThreads) {
    const int r = k / pairs;
    turn[k] = rope_turn(p, row0 + r, k - r * pairs);
  }
  __syncthreads();
  const int lane = threadIdx.x & ((1 << p.ls) - 1), items = rows * hb;
  const uint32_t magic = (1u << 20) / (uint32_t)hb + 1;   // it / hb = it * magic >> 20: exact while it * hb < 2^20
  // the lane's channels: nu from cu on and, halves, nv from cv on
  constexpr int V = HALF ? 8 : 4;
  const bool turns = WHOLE || !HALF || lane < p.nl;
  const int i0 = lane * V, rest = p.R + (lane - p.nl) * 16, cu = HALF ? (turns ? i0 : rest) : 2 * i0, cv = turns ? p.R / 2 + i0 : rest + 8;
  const int end = (HALF && turns ? p.R / 2 : p.dim) - cu, nu = WHOLE ? (end > 0 ? 8 : 0) : min(8, end),
            nv = !HALF ? 0 : WHOLE ? nu : min(8, (turns ? p.R : p.dim) - cv);
  for (int it = threadIdx.x >> p.ls; it < items; it += kRopeThreads >> p.ls) {
    const int r = (int)((uint32_t)it * magic >> 20), h = h0 + it - r * hb;
    const int64_t from = (row0 + r) * p.ldr + h * p.ldh, to = (row0 + r) * p.yldr + h * p.yldh;
    const float* w = h < p.hq ? p.qw : p.kw;
    float a[8], b[8];
    const int n8 = WHOLE ? 8 : nu, v8 = WHOLE ? 8 : nv, ru = WHOLE ? 8 : p.dim - cu, rv = WHOLE ? 8 : p.dim - cv;
    {
      F8Raw<TYPE> u, v;
      if (nu > 0) f8_fetch8<TYPE>(p.x, from + cu, cu, ru, u);
      if (nv > 0) f8_fetch8<TYPE>(p.x, from + cv, cv, rv, v);
      if (nu > 0) f8_take8<TYPE>(u, p.x, from + cu, n8, cu, ru, a);
      if (nv > 0) f8_take8<TYPE>(v, p.x, from + cv, v8, cv, rv, b);
    }
    if (w) {
      float ss = 0.0f, g[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += (nu > 0 ? a[j] * a[j] : 0.0f) + (nv > 0 ? b[j] * b[j] : 0.0f);
      for (int o = 1 << p.ls >> 1; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
      const float rstd = 1.0f / sqrtf(ss / (float)p.dim + p.eps);
      if (nu > 0) {
        f8_load8<P0_F32>(w, cu, n8, cu, ru, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] *= rstd * g[j];
      }
      if (nv > 0) {
        f8_load8<P0_F32>(w, cv, v8, cv, rv, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] *= rstd * g[j];
      }
    }
    if (nu > 0 && turns) {
      const float2* t = turn + r * pairs + i0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float u = HALF ? a[j] : a[2 * j], v = HALF ? b[j] : a[2 * j + 1], x = u * t[j].x - v * t[j].y, y = v * t[j].x + u * t[j].y;
        if constexpr (HALF) { a[j] = x; b[j] = y; }
        else if (i0 + j < p.R / 2) { a[2 * j] = x; a[2 * j + 1] = y; }   // (an infinity beside a channel that does not turn stays off it)
      }
    }
    if (nu > 0) f8_store8<TYPE>(p.y, to + cu, n8 == 8, n8, a);
    if (nv > 0) f8_store8<TYPE>(p.y, to + cv, v8 == 8, v8, b);
  }
}

static int rope_call(const p0_rope_args_t* a) {
  const char* op = "rope";
  if (!a) { set_error("%s: no arguments", op); return P0_EINVAL; }
  if (!f8_type(a->type)) { set_error("%s: type %d", op, (int)a->type); return P0_EINVAL; }
  if (a->mode != P0_ROPE_INTER && a->mode != P0_ROPE_HALF) { set_error("%s: mode %d", op, (int)a->mode); return P0_EINVAL; }
  if (a->freq != 0 && a->freq != 1) { set_error("%s: freq %d", op, (int)a->freq); return P0_EINVAL; }
  if (a->rows < 0 || a->rows > kF8MaxRows) { set_error("%s: rows %lld", op, (long long)a->rows); return P0_EINVAL; }
  if (a->dim < 2 || a->dim > 2 * kRopePairs || a->dim % 2) { set_error("%s: heads of %d channels", op, (int)a->dim); return P0_EINVAL; }
  const int64_t heads = (int64_t)a->hq + a->hk;
  if (a->hq < 0 || a->hk < 0 || heads < 1 || heads > 65535) { set_error("%s: %d and %d heads", op, (int)a->hq, (int)a->hk); return P0_EINVAL; }
  RopeP p{};
  int size_of[4];
  p.axes = a->axes ? a->axes : 1;
  if (p.axes < 1 || p.axes > 4) { set_error("%s: %d axes", op, (int)a->axes); return P0_EINVAL; }
  for (int k = 0; k < p.axes; ++k) {
    const int d = a->axis_dim[k] || p.axes > 1 ? a->axis_dim[k] : a->dim;
    if (d < 2 || d % 2 || d > a->dim - p.R) { set_error("%s: axis %d of %d channels (heads of %d)", op, k, d, (int)a->dim); return P0_EINVAL; }
    p.first[k] = p.R / 2;
    size_of[k] = d;
    p.R += d;
  }
  const double theta = a->theta != 0.0 ? a->theta : 10000.0;
  if (!(theta >= 1.0 && theta < 1e300)) { set_error("%s: theta %g", op, a->theta); return P0_EINVAL; }
  if (a->rows == 0) { if (int r = refuse_in_chain(op)) return r; return require_open(op); }
  const int size = f8_size(a->type);
  const int64_t wide = 1ll << 40;
  p.ldh = a->ldh ? a->ldh : a->dim;
  p.yldh = a->y_ldh ? a->y_ldh : a->dim;
  if (p.ldh < a->dim || p.yldh < a->dim || p.ldh > wide || p.yldh > wide) {
    set_error("%s: heads %lld and %lld apart", op, (long long)p.ldh, (long long)p.yldh); return P0_EINVAL;
  }
  const int64_t xw = (heads - 1) * p.ldh + a->dim, yw = (heads - 1) * p.yldh + a->dim;
  p.ldr = a->ldr ? a->ldr : heads * p.ldh;
  p.yldr = a->y_ldr ? a->y_ldr : heads * p.yldh;
  p.pos_ld = a->pos_ld ? a->pos_ld : a->rows;
  const Span x = f8_span(a->x, a->rows, xw, p.ldr, size), y = f8_span(a->y, a->rows, yw, p.yldr, size),
             pos = f8_span(a->pos, p.axes, a->rows, p.pos_ld, 4), qw{a->qw, 1, a->dim * 4, a->dim * 4}, kw{a->kw, 1, a->dim * 4, a->dim * 4};
  if (int r = f8_check(op, "x", x, size)) return r;
  if (int r = f8_check(op, "y", y, size)) return r;
  if (int r = f8_check(op, "pos", pos, 4)) return r;
  if (((uintptr_t)a->qw | (uintptr_t)a->kw) % 4) { set_error("%s: qw and kw must be 4-byte aligned", op); return P0_EINVAL; }
  const bool same = a->x == a->y && p.ldr == p.yldr && p.ldh == p.yldh;
  if ((overlap(x, y) && !same) || overlap(pos, y) || overlap(qw, y) || overlap(kw, y)) { set_error("%s: y overlaps an input", op); return P0_EINVAL; }
  if (int r = refuse_in_chain(op)) return r;
  if (int r = require_open(op)) return r;
  p.x = a->x; p.y = a->y; p.pos = a->pos; p.qw = a->qw; p.kw = a->kw; p.rows = a->rows;
  p.heads = (int)heads; p.hq = a->hq; p.dim = a->dim; p.shared = a->freq; p.inter = a->mode == P0_ROPE_INTER;
  p.eps = a->eps != 0.0f ? a->eps : 1e-6f;
  for (int k = 0; k < p.axes; ++k) {
    long double f = powl((long double)theta, -2.0L / (a->freq ? p.R : size_of[k]));   // squares of squares: in more bits than are kept
    for (int b = 0; b < 8; ++b, f *= f) p.pow[k][b] = (double)f;
  }
  const bool half = !p.inter, whole = half ? p.R == a->dim && a->dim % 16 == 0 : a->dim % 8 == 0;   // every lane has 8 pairs, or 4
  p.nl = (p.R / 2 + 7) / 8;
  const int lanes = half ? p.nl + (a->dim - p.R + 15) / 16 : (a->dim + 7) / 8;   // at most 64
  while (1 << p.ls < lanes) ++p.ls;
  const int side = kRopeThreads >> p.ls, pairs = a->dim / 2;
  // A workgroup's work is four rounds of its groups of lanes where that leaves work for every CU: several rows, or a part of a row's
  // heads; one round where it does not (us, one / four: 32760 rows of 40 heads of 128 bf16 channels 171 / 124, 4608 of 48 33.6 / 28.8, 8000 of 10 of 80
  // 9.7 / 9.6; 1021 rows of 10 heads of 256 fp32 channels 8.4 / 11.4, 16 rows 5.1 / 9.3)
  const int rounds = a->rows * heads >= (int64_t)side * 4 * 1024 ? 4 : 1;
  p.hb = (int)(heads < side * rounds ? heads : side * rounds);
  p.rb = side * rounds / p.hb;
  if (p.rb > kRopeTable / pairs) p.rb = kRopeTable / pairs;
  p.hblocks = (int)((heads + p.hb - 1) / p.hb);
  dim3 grid;
  if (!f8_grid((a->rows + p.rb - 1) / p.rb * p.hblocks, kRopeThreads, &grid)) { set_error("%s: %lld rows of %lld heads", op, (long long)a->rows, (long long)heads); return P0_EINVAL; }
#define P0_ROPE(T) if (a->type == T) hipLaunchKernelGGL((half ? (whole ? rope_kernel<T, true, true> : rope_kernel<T, true, false>) : whole ? rope_kernel<T, false, true> : rope_kernel<T, false, false>), grid, dim3(kRopeThreads), 0, ctx().cur, p)
  P0_ROPE(P0_F32);
  P0_ROPE(P0_F16);
  P0_ROPE(P0_BF16);
#undef P0_ROPE
  P0_LAUNCHED(op);
  return P0_OK;
}

}  // namespace p0

extern "C" int p0_rope(const p0_rope_args_t* a) { return p0::rope_call(a); }
