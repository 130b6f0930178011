// kv_attn.hip - attention of each sequence's newest rows over a cache of mxfp4 pages (kv_common.hpp has the layout).
//
// One pass over the keys and values with the running maximum and sum of the softmax. A wave owns 16 query rows of one key head
// (row = m * group + q: the heads that share keys fill the matrix instructions' columns) and takes every n-th run of 32
// tokens; waves with the same rows meet in LDS, workgroups with the same rows in the split-K workspace, where the last to
// arrive adds the others' sums in their order.
#include "kv_common.hpp"

#include <cmath>

namespace p0 {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

struct AttnP {
  KvP kv;
  const int32_t* rows;
  const void* q;
  void* y;
  int64_t q_ldb, q_ldm, q_ldh, y_ldb, y_ldm, y_ldh;
  int64_t window;
  int M, heads, group, R;   // R = M * group query rows of a key head
  int sinks;
  int type, q_vec, y_vec;
  float scale2;             // scale * log2(e)
  int tiles, streams;       // row tiles of a workgroup, waves that share a row tile
  int nsplit;               // workgroups that share their rows
  float* part;
  unsigned* cnt;
};

constexpr float kNone = -3.0e38f;    // the running maximum before any token
constexpr float kLift = 14.0f;       // probabilities are held times 2^14: fp16's normal range reaches 2^-28 of the largest

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

// the maximum / sum over the four lane groups of 16 lanes (lane ^ 16, lane ^ 32)
__device__ __forceinline__ float groups_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ float load_one(const void* q, int64_t i, int type) {
  if (type == P0_KV_F32) return ((const float*)q)[i];
  if (type == P0_KV_F16) return (float)((const _Float16*)q)[i];
  return __uint_as_float((uint32_t)((const uint16_t*)q)[i] << 16);
}
__device__ __forceinline__ uint16_t to_bf16(float v) {   // nearest even; NaN stays NaN
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)(u >> 16 | 0x40);
  return (uint16_t)((u + 0x7FFFu + (u >> 16 & 1)) >> 16);
}
__device__ __forceinline__ void load8(const void* q, int64_t i, int type, int vec, float (&v)[8]) {
  if (vec) {
    if (type == P0_KV_F32) {
      const float4_t a = *(const float4_t*)((const float*)q + i), b = *(const float4_t*)((const float*)q + i + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    } else {
      const uint4_t a = *(const uint4_t*)((const uint16_t*)q + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = a[j];
        if (type == P0_KV_F16) {
          const half2_t h = __builtin_bit_cast(half2_t, w);
          v[2 * j] = (float)h.x; v[2 * j + 1] = (float)h.y;
        } else {
          v[2 * j] = __uint_as_float(w << 16); v[2 * j + 1] = __uint_as_float(w & 0xFFFF0000u);
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = load_one(q, i + j, type);
  }
}
__device__ __forceinline__ void store8(void* y, int64_t i, int type, int vec, const float (&v)[8]) {
  if (type == P0_KV_F32) {
    float* o = (float*)y + i;
    if (vec) {
      *(float4_t*)o = float4_t{v[0], v[1], v[2], v[3]};
      *(float4_t*)(o + 4) = float4_t{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = v[j];
    }
    return;
  }
  uint16_t h[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    h[j] = type == P0_KV_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[j]) : to_bf16(v[j]);
  uint16_t* o = (uint16_t*)y + i;
  if (vec) {
    uint4_t w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
    *(uint4_t*)o = w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = h[j];
  }
}

// the f32 whose exponent field is byte `n` of w. The conversions read that field alone: what the shift leaves in the sign
// and the mantissa does not count
template <int N> __device__ __forceinline__ float exponent_of(uint32_t w) {
  return __uint_as_float(N == 0 ? w << 23 : N == 1 ? w << 15 : N == 2 ? w << 7 : w >> 1);
}
__device__ __forceinline__ half8_t operand(const half2_t (&v)[4]) {
  return half8_t{v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
}
// eight codes of one block
__device__ __forceinline__ half8_t widen(uint32_t w, float e) {
  const half2_t v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, e, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, e, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, e, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, e, 3)};
  return operand(v);
}

// a run's keys / values as a lane loads them
template <int D> struct KeyRegs {
  static constexpr int U = D == 64 ? 1 : D / 128;          // 16-byte pieces a tile of 16 tokens
  uint4_t code[D == 64 ? 1 : 2 * U];
  uint32_t exp[(2 * U + 3) / 4];                           // [tt][u] bytes
  __device__ __forceinline__ void load(const uint8_t* run, int lane) {
#pragma unroll
    for (int i = 0; i < (D == 64 ? 1 : 2 * U); ++i) code[i] = *(const uint4_t*)(run + i * 1024 + lane * 16);
    const uint8_t* e = run + 16 * D;
    if constexpr (D == 64) exp[0] = *(const uint16_t*)(e + ((lane >> 5) * 16 + (lane & 15)) * 2);
    else if constexpr (D == 128) exp[0] = *(const uint16_t*)(e + lane * 2);
    else if constexpr (D == 256) exp[0] = *(const uint32_t*)(e + lane * 4);
    else { const uint2_t w = *(const uint2_t*)(e + lane * 8); exp[0] = w.x; exp[1] = w.y; }
  }
};
template <int D> struct ValueRegs {
  uint4_t code[D / 64];      // [block / 2]: {block even: 8 tokens, block odd: 8 tokens}
  uint4_t exp[D / 64];
  __device__ __forceinline__ void load(const uint8_t* run, int lane) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) code[i] = *(const uint4_t*)(run + 17 * D + i * 1024 + lane * 16);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) exp[i] = *(const uint4_t*)(run + 33 * D + ((lane >> 4) * (D / 64) + i) * 16);
  }
  // tokens from `left` on (of this run's 32) count as 0, whatever their bytes hold
  __device__ __forceinline__ void cut(int left, int lane) {
    const int g = lane >> 4;
    uint32_t keep[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = left - (16 * h + 4 * g);
      keep[h] = n <= 0 ? 0u : n >= 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1;
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) { exp[i].x &= keep[0]; exp[i].y &= keep[1]; exp[i].z &= keep[0]; exp[i].w &= keep[1]; }
  }
};

// the tokens a tile of rows can see: runs [0, ns) and [lo, hi)
struct Span {
  int ns, lo, n;      // n runs in all
  int p0, p1;         // positions of the tile's first and last row
  __device__ __forceinline__ int run(int i) const { return i < ns ? i : lo + (i - ns); }
};
__device__ __forceinline__ Span span_of(const AttnP& p, int len, int p0, int p1) {
  Span s;
  s.p0 = p0;
  s.p1 = p1;
  const int hi = (p1 + kKvRun) / kKvRun;
  int64_t first = p.window ? (int64_t)p0 - p.window + 1 : 0;
  s.lo = first > 0 ? (int)(first / kKvRun) : 0;
  const int ns = (int)(((int64_t)p.sinks + kKvRun - 1) / kKvRun);
  s.ns = ns < s.lo ? ns : s.lo;
  s.n = s.ns + (hi > s.lo ? hi - s.lo : 0);
  return s;
}

// PARTS: fp16 values that a query's or a probability's f32 is taken as
template <int D, int QPARTS, int PPARTS>
__global__ __launch_bounds__(D == 512 ? 256 : 512) void kv_attn_kernel(const AttnP p) {
  constexpr int NW = D == 512 ? 4 : 8;
  constexpr int STEPS = D / 32, BLOCKS = D / 32;
  __shared__ __attribute__((aligned(16))) float s_o[NW / 2][16 * D];
  __shared__ float s_m[NW][16], s_l[NW][16];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int rg = blockIdx.y, h = blockIdx.z % p.kv.heads, b = blockIdx.z / p.kv.heads, split = blockIdx.x;
  const int tile = wave % p.tiles, stream = wave / p.tiles;
  const bool works = stream < p.streams;

  const int len = kv_len(p.kv, b), nrows = kv_rows(p.rows, b, p.M);
  // the tile's rows, and their positions; rows past the sequence's own see nothing
  const int row0 = (rg * p.tiles + tile) * 16, row = row0 + col, m = row / p.group;
  const int pos = row < p.R && m < nrows ? len - nrows + m : -1;
  const int mlast = min((row0 + 15) / p.group, nrows - 1), mfirst = row0 / p.group;
  const bool whole = min(row0 + 15, p.R - 1) / p.group < nrows;   // every row of the tile that is one is the sequence's
  Span sp{};
  if (row0 < p.R && mfirst <= mlast) sp = span_of(p, len, len - nrows + mfirst, len - nrows + mlast);
  // workgroups that have runs of any of their tiles: the last tile of the group sees the most
  int nmax = 0;
  for (int t = 0; t < p.tiles; ++t) {
    const int r0 = (rg * p.tiles + t) * 16, ml = min((r0 + 15) / p.group, nrows - 1), mf = r0 / p.group;
    if (r0 < p.R && mf <= ml) nmax = max(nmax, span_of(p, len, len - nrows + mf, len - nrows + ml).n);
  }
  const int active = max(1, min(p.nsplit, (nmax + p.streams - 1) / p.streams));
  if (split >= active) return;

  float4_t o[2 * BLOCKS];
#pragma unroll
  for (int i = 0; i < 2 * BLOCKS; ++i) o[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float mrun = kNone, lrun = 0.0f;
  const int first = split * p.streams + stream, stride = active * p.streams;

  if (works && first < sp.n) {
    // the queries, each row under a power of two that brings its largest value to [1, 2)
    half8_t qh[STEPS], ql[QPARTS == 2 ? STEPS : 1];
    float qs;
    {
      const bool in = pos >= 0;
      const int64_t base = in ? (int64_t)b * p.q_ldb + (int64_t)m * p.q_ldm + (int64_t)(h * p.group + row % p.group) * p.q_ldh : 0;
      auto channel = [&](int s) { return D == 64 ? g * 16 + 8 * s : (s >> 2) * 128 + g * 32 + 8 * (s & 3); };
      auto get = [&](int s, float (&v)[8]) {
        if (in) load8(p.q, base + channel(s), p.type, p.q_vec, v);
        else
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = 0.0f;
      };
      float most = 0.0f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        float v[8];
        get(s, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(v[j]));
      }
      most = groups_max(most);
      int e = (int)(__float_as_uint(most) >> 23) - 127;
      e = most == 0.0f || e == 128 ? 0 : e < -120 ? -120 : e > 126 ? 126 : e;
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
      qs = ldexpf(p.scale2, e);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        float v[8];
        get(s, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = v[j] * down;
          qh[s][j] = (_Float16)x;
          if constexpr (QPARTS == 2) ql[s][j] = (_Float16)(x - (float)qh[s][j]);
        }
      }
    }
    const int run_bytes = 34 * D, rlog = p.kv.page_log - 5, rmask = (1 << rlog) - 1;
    const uint8_t* head = p.kv.pages + ((int64_t)h << rlog) * run_bytes;
    auto page_of = [&](int i) {   // of run i of the tile's; past the last: any
      const int r = i < sp.n ? sp.run(i) : 0;
      return __builtin_amdgcn_readfirstlane(kv_page(p.kv, b, r >> rlog));
    };
    auto run_at = [&](int i, int pg) {
      const int r = i < sp.n ? sp.run(i) : 0;
      return head + (int64_t)(pg < 0 ? 0 : pg) * p.kv.page_bytes + (int64_t)(r & rmask) * run_bytes;
    };
    KeyRegs<D> kr;
    ValueRegs<D> vr;
    int pg = page_of(first), pg_next = page_of(first + stride);
    kr.load(run_at(first, pg), lane);
    vr.load(run_at(first, pg), lane);
    for (int i = first; i < sp.n; i += stride) {
      const int t0 = sp.run(i) * kKvRun;
      const bool dead = pg < 0;
      // ---- scores: lane (g, col) gets tokens 16 tt + 4 g + r of row col
      float4_t s[2];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        s[tt] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          uint32_t w;
          float e;
          if constexpr (D == 64) {
            w = kr.code[0][tt * 2 + st];
            e = tt == 0 ? exponent_of<0>(kr.exp[0]) : exponent_of<1>(kr.exp[0]);
          } else {
            constexpr int U = D / 128;
            const int u = st >> 2, x = tt * U + u;
            w = kr.code[x][st & 3];
            const uint32_t ew = kr.exp[x >> 2];
            e = (x & 3) == 0 ? exponent_of<0>(ew) : (x & 3) == 1 ? exponent_of<1>(ew) : (x & 3) == 2 ? exponent_of<2>(ew) : exponent_of<3>(ew);
          }
          const half8_t a = widen(w, e);
          s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[st], s[tt], 0, 0, 0);
          if constexpr (QPARTS == 2) s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[st], s[tt], 0, 0, 0);
        }
      }
      const int pg_after = page_of(i + 2 * stride);
      if (i + stride < sp.n) kr.load(run_at(i + stride, pg_next), lane);
      // ---- what the rows do not see
      const bool all = !dead && t0 + kKvRun - 1 <= sp.p0 && whole &&
                       (!p.window || t0 > (int64_t)sp.p1 - p.window || t0 + kKvRun <= p.sinks);
      if (!all) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int t = t0 + 16 * tt + 4 * g + r;
            const bool sees = !dead && t <= pos && (!p.window || t > pos - p.window || t < p.sinks);
            s[tt][r] = sees ? s[tt][r] : -INFINITY;
          }
        if (dead || t0 + kKvRun > len) vr.cut(dead ? 0 : len - t0, lane);
      }
      // ---- running maximum and sum
      float top = kNone;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[tt][r]);
      top = fmaxf(groups_max(top) * qs, mrun);
      if (__any(top > mrun)) {
        const float f = exp2_fast(mrun - top);
        lrun *= f;
#pragma unroll
        for (int k = 0; k < 2 * BLOCKS; ++k) o[k] *= f;
        mrun = top;
      }
      const float shift = kLift - mrun;
      half8_t ph, pl;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = exp2_fast(fmaf(s[tt][r], qs, shift));
          lrun += x;
          ph[tt * 4 + r] = (_Float16)x;
          if constexpr (PPARTS == 2) pl[tt * 4 + r] = (_Float16)(x - (float)ph[tt * 4 + r]);
        }
      // ---- outputs: lane (g, col) gets channels 32 bl + 8 g + 2 r + u of row col
#pragma unroll
      for (int bl = 0; bl < BLOCKS; ++bl) {
        const uint4_t cw = vr.code[bl >> 1], ew = vr.exp[bl >> 1];
        const uint32_t c0 = bl & 1 ? cw.z : cw.x, c1 = bl & 1 ? cw.w : cw.y, e0 = bl & 1 ? ew.z : ew.x, e1 = bl & 1 ? ew.w : ew.y;
        const half2_t v[8] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c0, exponent_of<0>(e0), 0),
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c0, exponent_of<1>(e0), 1),
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c0, exponent_of<2>(e0), 2),
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c0, exponent_of<3>(e0), 3),
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c1, exponent_of<0>(e1), 0),
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c1, exponent_of<1>(e1), 1),
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c1, exponent_of<2>(e1), 2),
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c1, exponent_of<3>(e1), 3)};
        const half8_t a0 = {v[0].x, v[1].x, v[2].x, v[3].x, v[4].x, v[5].x, v[6].x, v[7].x};
        const half8_t a1 = {v[0].y, v[1].y, v[2].y, v[3].y, v[4].y, v[5].y, v[6].y, v[7].y};
        o[2 * bl] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, ph, o[2 * bl], 0, 0, 0);
        o[2 * bl + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, ph, o[2 * bl + 1], 0, 0, 0);
        if constexpr (PPARTS == 2) {
          o[2 * bl] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, pl, o[2 * bl], 0, 0, 0);
          o[2 * bl + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, pl, o[2 * bl + 1], 0, 0, 0);
        }
      }
      if (i + stride < sp.n) vr.load(run_at(i + stride, pg_next), lane);
      pg = pg_next;
      pg_next = pg_after;
    }
    lrun = groups_sum(lrun);
  }

  // ---- waves with the same rows
  if (g == 0) { s_m[wave][col] = mrun; s_l[wave][col] = lrun; }
  __syncthreads();
  float mall = kNone, lall = 0.0f;
  for (int w = 0; w < p.streams; ++w) mall = fmaxf(mall, s_m[w * p.tiles + tile][col]);
  for (int w = 0; w < p.streams; ++w) lall += s_l[w * p.tiles + tile][col] * exp2_fast(s_m[w * p.tiles + tile][col] - mall);
  {
    const float f = exp2_fast(mrun - mall);
#pragma unroll
    for (int k = 0; k < 2 * BLOCKS; ++k) o[k] *= f;
  }
  for (int half = p.streams >> 1; half > 0; half >>= 1) {
    if (works && stream >= half && stream < 2 * half) {
      float* d = s_o[(stream - half) * p.tiles + tile] + lane * 4;
#pragma unroll
      for (int k = 0; k < 2 * BLOCKS; ++k) *(float4_t*)(d + k * 256) = o[k];
    }
    __syncthreads();
    if (stream < half) {
      const float* d = s_o[stream * p.tiles + tile] + lane * 4;
#pragma unroll
      for (int k = 0; k < 2 * BLOCKS; ++k) o[k] += *(const float4_t*)(d + k * 256);
    }
    __syncthreads();
  }
  const bool writes = stream == 0 && row < p.R;
  auto out_at = [&](int r) {
    return (int64_t)b * p.y_ldb + (int64_t)(r / p.group) * p.y_ldm + (int64_t)(h * p.group + r % p.group) * p.y_ldh;
  };
  if (active == 1) {
    if (writes) {
      const float inv = lall > 0.0f || lall != lall ? 1.0f / lall : 0.0f;
      const int64_t at = out_at(row);
#pragma unroll
      for (int bl = 0; bl < BLOCKS; ++bl) {
        float v[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) { v[2 * r] = o[2 * bl][r] * inv; v[2 * r + 1] = o[2 * bl + 1][r] * inv; }
        store8(p.y, at + 32 * bl + 8 * g, p.type, p.y_vec, v);
      }
    }
    return;
  }
  // ---- workgroups with the same rows: sums to the workspace (uncached: a store is in memory once acknowledged), the last to
  // arrive adds them in split order
  const int item = (b * p.kv.heads + h) * gridDim.y + rg, wgrows = min(p.tiles * 16, p.R - rg * p.tiles * 16);
  const int64_t step = wgrows * D + ((2 * wgrows + 3) & ~3);   // sums [wgrows][D], maxima, sums of probabilities
  float* part = p.part + (int64_t)item * p.nsplit * (p.tiles * 16) * (D + 4);
  float* mine = part + split * step;
  if (writes) {
    float* d = mine + (tile * 16 + col) * D + 8 * g;
#pragma unroll
    for (int bl = 0; bl < BLOCKS; ++bl) {
      float4_t lo, hi;
#pragma unroll
      for (int r = 0; r < 2; ++r) { lo[2 * r] = o[2 * bl][r]; lo[2 * r + 1] = o[2 * bl + 1][r]; hi[2 * r] = o[2 * bl][2 + r]; hi[2 * r + 1] = o[2 * bl + 1][2 + r]; }
      *(float4_t*)(d + 32 * bl) = lo;
      *(float4_t*)(d + 32 * bl + 4) = hi;
    }
    if (g == 0) {
      mine[wgrows * D + tile * 16 + col] = mall;
      mine[wgrows * D + wgrows + tile * 16 + col] = lall;
    }
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) {
    unsigned* c = p.cnt + item;
    s_last = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(active - 1);
    if (s_last) __hip_atomic_exchange(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // leave it at zero
  }
  __syncthreads();
  if (!s_last) return;
  for (int t = tid; t < wgrows * (D / 8); t += blockDim.x) {
    const int r = t / (D / 8), c = t % (D / 8) * 8;
    float mm = kNone, ll = 0.0f;
    for (int s = 0; s < active; ++s) mm = fmaxf(mm, __builtin_nontemporal_load(part + s * step + wgrows * D + r));
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < active; ++s) {
      const float* x = part + s * step;
      const float f = exp2_fast(__builtin_nontemporal_load(x + wgrows * D + r) - mm);
      ll += f * __builtin_nontemporal_load(x + wgrows * D + wgrows + r);
      const float4_t a = __builtin_nontemporal_load((const float4_t*)(x + r * D + c)), bb = __builtin_nontemporal_load((const float4_t*)(x + r * D + c + 4));
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] = fmaf(a[j], f, v[j]); v[4 + j] = fmaf(bb[j], f, v[4 + j]); }
    }
    const float inv = ll > 0.0f || ll != ll ? 1.0f / ll : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= inv;
    store8(p.y, out_at(rg * p.tiles * 16 + r) + c, p.type, p.y_vec, v);
  }
}

template <int D>
static void launch_attn(const AttnP& p, dim3 grid, hipStream_t s) {
  auto k = p.type == P0_KV_F32 ? kv_attn_kernel<D, 2, 2> : kv_attn_kernel<D, 1, 2>;
  hipLaunchKernelGGL(k, grid, dim3(D == 512 ? 256 : 512), 0, s, p);
}

}  // namespace p0

using namespace p0;

extern "C" int p0_kv_attn(const p0_kv_attn_args_t* a) {
  if (!a) { set_error("kv_attn: no arguments"); return P0_EINVAL; }
  AttnP p{};
  if (int r = kv_check("kv_attn", a->kv, a->B, &p.kv)) return r;
  if (a->M < 0 || a->M > (1 << 24)) { set_error("kv_attn: M %lld", (long long)a->M); return P0_EINVAL; }
  if (a->heads < 1 || a->heads > 4096 || a->heads % a->kv.heads) {
    set_error("kv_attn: %lld heads over %d key heads", (long long)a->heads, (int)a->kv.heads); return P0_EINVAL;
  }
  if (a->type < P0_KV_F32 || a->type > P0_KV_BF16) { set_error("kv_attn: type %d", (int)a->type); return P0_EINVAL; }
  if (a->window < 0 || a->sinks < 0 || a->max_len < 0) {
    set_error("kv_attn: window %lld, sinks %lld, max_len %lld", (long long)a->window, (long long)a->sinks, (long long)a->max_len);
    return P0_EINVAL;
  }
  if (!(a->scale >= 0.0f) || std::isinf(a->scale)) { set_error("kv_attn: scale %g", (double)a->scale); return P0_EINVAL; }
  if (!a->q || !a->y) { set_error("kv_attn: missing q or y buffer"); return P0_EINVAL; }
  const int size = a->type == P0_KV_F32 ? 4 : 2, D = a->kv.dim;
  if ((uintptr_t)a->q % size || (uintptr_t)a->y % size) { set_error("kv_attn: q or y is not aligned to its type"); return P0_EINVAL; }
  if (int r = refuse_in_chain("kv_attn")) return r;
  if (int r = require_open("kv_attn")) return r;
  if (a->B == 0 || a->M == 0) return P0_OK;
  p.rows = a->rows;
  p.q = a->q;
  p.y = a->y;
  p.q_ldh = a->q_ldh ? a->q_ldh : D;
  p.q_ldm = a->q_ldm ? a->q_ldm : a->heads * p.q_ldh;
  p.q_ldb = a->q_ldb ? a->q_ldb : a->M * p.q_ldm;
  p.y_ldh = a->y_ldh ? a->y_ldh : D;
  p.y_ldm = a->y_ldm ? a->y_ldm : a->heads * p.y_ldh;
  p.y_ldb = a->y_ldb ? a->y_ldb : a->M * p.y_ldm;
  const auto vec = [&](const void* q, int64_t x, int64_t y, int64_t z) {   // 16-byte accesses: 8 channels at a multiple of 8
    return (((uintptr_t)q | (uintptr_t)(x * size) | (uintptr_t)(y * size) | (uintptr_t)(z * size)) & 15) == 0;
  };
  p.q_vec = vec(a->q, p.q_ldh, p.q_ldm, p.q_ldb);
  p.y_vec = vec(a->y, p.y_ldh, p.y_ldm, p.y_ldb);
  p.type = a->type;
  p.M = (int)a->M;
  p.heads = (int)a->heads;
  p.group = (int)(a->heads / a->kv.heads);
  if (a->M * p.group > (1 << 28)) { set_error("kv_attn: M %lld of %d heads a key head", (long long)a->M, p.group); return P0_EINVAL; }
  p.R = p.M * p.group;
  const int64_t most = (int64_t)p.kv.cols << p.kv.page_log;
  p.window = a->window >= most + a->M ? 0 : a->window;   // a window as long as the sequence hides nothing
  p.sinks = (int)(a->sinks < most ? a->sinks : most);
  const float scale = a->scale != 0.0f ? a->scale : 1.0f / sqrtf((float)D);
  p.scale2 = scale * 1.44269504088896340736f;
  // a workgroup's waves: row tiles first, then streams over the runs
  const int NW = D == 512 ? 4 : 8, alltiles = (p.R + 15) / 16;
  p.tiles = alltiles < NW ? alltiles : NW;
  p.streams = 1;
  while (2 * p.streams * p.tiles <= NW) p.streams *= 2;
  const int groups = (alltiles + p.tiles - 1) / p.tiles;
  const int64_t items = a->B * p.kv.heads * groups;
  if (a->B * p.kv.heads > 65535 || groups > 65535) { set_error("kv_attn: %lld sequences of %d rows", (long long)a->B, p.R); return P0_EINVAL; }
  const int64_t longest = a->max_len && a->max_len < most ? a->max_len : most;
  const int64_t runs = (p.window && p.window + a->M + p.sinks + 2 * kKvRun < longest ? p.window + a->M + p.sinks + 2 * kKvRun : longest) / kKvRun + 1;
  int64_t split = 512 / items;
  if (split > runs / (2 * p.streams)) split = runs / (2 * p.streams);
  const int64_t room = (int64_t)ctx().part_floats / (items * p.tiles * 16 * (D + 4));
  if (split > room) split = room;
  p.nsplit = split < 1 ? 1 : (int)split;
  p.part = ctx().part;
  p.cnt = ctx().kv_counters;
  if (p.nsplit > 1 && items > kKvCounters) p.nsplit = 1;
  const dim3 grid((unsigned)p.nsplit, (unsigned)groups, (unsigned)(a->B * p.kv.heads));
  switch (D) {
    case 64: launch_attn<64>(p, grid, ctx().cur); break;
    case 128: launch_attn<128>(p, grid, ctx().cur); break;
    case 256: launch_attn<256>(p, grid, ctx().cur); break;
    default: launch_attn<512>(p, grid, ctx().cur); break;
  }
  P0_LAUNCHED("kv_attn");
  return P0_OK;
}
