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
  int window;               // 0 or at most 2^31 - 1 tokens: longer ones hide nothing
  int M, group, R;          // R = M * group query rows of a key head
  int sinks;
  int q_vec, y_vec;
  float scale2;             // scale * log2(e)
  int tiles, streams;       // row tiles of a workgroup, waves that share a row tile
  int groups, items;        // row groups of a key head; (sequence, key head, row group) triples
  int shared;               // 1: long items are dealt to several workgroups, 0: a workgroup an item
  int join;                 // 1: kv_join_kernel adds an item's parts, 0: the last workgroup to arrive does
  int64_t slot;             // floats of a part
  int32_t* dealt;           // [items][2]: the first workgroup and the parts of each, for kv_join_kernel
  float* part;              // a part a workgroup
  unsigned* cnt;            // per item
};

// A row's running maximum m is one of its scores, before their factor qs, and a probability 2^((s - m) qs + kLift): the largest
// score's is exactly 1 (lifted) however large the scores are. (2^(s qs - (m qs - kLift)), a rounded product under the fma's exact
// one, saves a subtraction a score, 1% of a call; past 2^24 it leaves whole powers of two, and infinities among them)
constexpr float kNone = -3.0e38f;    // before any token
constexpr float kLift = 14.0f;       // probabilities are held times 2^14: fp16's normal range reaches 2^-28 of the largest

// Parts go from workgroup to workgroup of one launch in device-scope accesses of 8 bytes: the workspace is uncached, so a store is
// in memory once acknowledged, but parts are not padded to cache lines, and a plain load could be served by a line that this
// CU's L1 took in for another item before this item's words in it were written
__device__ __forceinline__ float2 part_load(const float* a) {
  return __builtin_bit_cast(float2, __hip_atomic_load((const uint64_t*)a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ void part_store(float* a, float x, float y) {
  __hip_atomic_store((uint64_t*)a, __builtin_bit_cast(uint64_t, float2{x, y}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

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

__device__ __forceinline__ uint16_t to_bf16(float v) {   // nearest even; NaN stays NaN
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)(u >> 16 | 0x40);
  return (uint16_t)((u + 0x7FFFu + (u >> 16 & 1)) >> 16);
}
// eight channels from element i on; vec: 16-byte aligned
template <int TYPE> __device__ __forceinline__ void load8(const void* q, int64_t i, int vec, float (&v)[8]) {
  if constexpr (TYPE == P0_KV_F32) {
    const float* x = (const float*)q + i;
    if (vec) {
      const float4_t a = *(const float4_t*)x, b = *(const float4_t*)(x + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = x[j];
    }
  } else {
    const uint16_t* x = (const uint16_t*)q + i;
    uint32_t w[4];
    if (vec) {
      const uint4_t a = *(const uint4_t*)x;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = a[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = x[2 * j] | (uint32_t)x[2 * j + 1] << 16;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (TYPE == P0_KV_F16) {
        const half2_t h = __builtin_bit_cast(half2_t, w[j]);
        v[2 * j] = (float)h.x;
        v[2 * j + 1] = (float)h.y;
      } else {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
  }
}
template <int TYPE> __device__ __forceinline__ void store8(void* y, int64_t i, int vec, const float (&v)[8]) {
  if constexpr (TYPE == P0_KV_F32) {
    float* o = (float*)y + i;
    if (vec) {
      *(float4_t*)o = float4_t{v[0], v[1], v[2], v[3]};
      *(float4_t*)(o + 4) = float4_t{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = v[j];
    }
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (TYPE == P0_KV_F16) w[j] = __builtin_bit_cast(uint32_t, half2_t{(_Float16)v[2 * j], (_Float16)v[2 * j + 1]});
      else w[j] = to_bf16(v[2 * j]) | (uint32_t)to_bf16(v[2 * j + 1]) << 16;
    }
    uint16_t* o = (uint16_t*)y + i;
    if (vec) {
      *(uint4_t*)o = uint4_t{w[0], w[1], w[2], w[3]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[2 * j] = (uint16_t)w[j];
        o[2 * j + 1] = (uint16_t)(w[j] >> 16);
      }
    }
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

// a run's keys / values as a lane loads them; of 512 channels a wave has half (0 or 1)
template <int D> struct KeyRegs {
  static constexpr int U = D == 64 ? 1 : D == 512 ? 2 : D / 128;   // 16-byte pieces a tile of 16 tokens
  uint4_t code[D == 64 ? 1 : 2 * U];
  uint32_t exp[1];                                                 // [tt][u] bytes
  __device__ __forceinline__ void load(const uint8_t* run, int lane, int half) {
#pragma unroll
    for (int i = 0; i < (D == 64 ? 1 : 2 * U); ++i)
      code[i] = *(const uint4_t*)(run + (D == 512 ? (i / U) * 4 + 2 * half + i % U : i) * 1024 + lane * 16);
    const uint8_t* e = run + 16 * D;
    if constexpr (D == 64) exp[0] = *(const uint16_t*)(e + ((lane >> 5) * 16 + (lane & 15)) * 2);
    else if constexpr (D == 128) exp[0] = *(const uint16_t*)(e + lane * 2);
    else if constexpr (D == 256) exp[0] = *(const uint32_t*)(e + lane * 4);
    else exp[0] = *(const uint16_t*)(e + lane * 8 + 2 * half) | (uint32_t)*(const uint16_t*)(e + lane * 8 + 4 + 2 * half) << 16;
  }
  // 16 tokens' operand of a step of 32 channels
  __device__ __forceinline__ half8_t operand(int tt, int st) const {
    const int x = D == 64 ? tt : tt * U + (st >> 2);
    const float e = x == 0 ? exponent_of<0>(exp[0]) : x == 1 ? exponent_of<1>(exp[0]) : x == 2 ? exponent_of<2>(exp[0]) : exponent_of<3>(exp[0]);
    return widen(D == 64 ? code[0][tt * 2 + st] : code[x % (2 * U)][st & 3], e);
  }
};
// 32 tokens' operands of the even and the odd channels of a block: 8 code bytes (c0, c1), 8 exponents (e0, e1)
__device__ __forceinline__ void value_operands(uint32_t c0, uint32_t c1, uint32_t e0, uint32_t e1, half8_t (&a)[2]) {
  const half2_t v[8] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c0, exponent_of<0>(e0), 0),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c0, exponent_of<1>(e0), 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c0, exponent_of<2>(e0), 2),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c0, exponent_of<3>(e0), 3),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c1, exponent_of<0>(e1), 0),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c1, exponent_of<1>(e1), 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c1, exponent_of<2>(e1), 2),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c1, exponent_of<3>(e1), 3)};
  a[0] = half8_t{v[0].x, v[1].x, v[2].x, v[3].x, v[4].x, v[5].x, v[6].x, v[7].x};
  a[1] = half8_t{v[0].y, v[1].y, v[2].y, v[3].y, v[4].y, v[5].y, v[6].y, v[7].y};
}
// a mask of the first n of four bytes
__device__ __forceinline__ uint32_t keep_bytes(int n) { return n <= 0 ? 0u : n >= 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1; }
template <int D> struct ValueRegs {
  static constexpr int N = D == 512 ? 4 : D / 64;
  uint4_t code[N];           // [block / 2]: {block even: 8 tokens, block odd: 8 tokens}
  uint4_t exp[N];
  __device__ __forceinline__ void load(const uint8_t* run, int lane, int half) {
    const uint8_t *c = run + 17 * D + (N * half * 64 + lane) * 16, *e = run + 33 * D + ((lane >> 4) * (D / 64) + N * half) * 16;
#pragma unroll
    for (int i = 0; i < N; ++i) code[i] = *(const uint4_t*)(c + i * 1024);
#pragma unroll
    for (int i = 0; i < N; ++i) exp[i] = *(const uint4_t*)(e + i * 16);
  }
  __device__ __forceinline__ void operands(int bl, half8_t (&a)[2]) const {
    const uint4_t cw = code[bl >> 1], ew = exp[bl >> 1];
    value_operands(bl & 1 ? cw.z : cw.x, bl & 1 ? cw.w : cw.y, bl & 1 ? ew.z : ew.x, bl & 1 ? ew.w : ew.y, a);
  }
  // tokens from `left` on (of this run's 32) count as 0, whatever their bytes hold
  __device__ __forceinline__ void cut(int left, int lane) {
    const uint32_t keep[2] = {keep_bytes(left - 4 * (lane >> 4)), keep_bytes(left - 16 - 4 * (lane >> 4))};
#pragma unroll
    for (int i = 0; i < N; ++i) { exp[i].x &= keep[0]; exp[i].y &= keep[1]; exp[i].z &= keep[0]; exp[i].w &= keep[1]; }
  }
};

// the tokens that an item's rows can see: runs [0, ns) and [lo, ..), n in all
struct Span {
  int ns, lo, n;
  int p0, p1;         // positions of the item's first and last row
  __device__ __forceinline__ int run(int i) const { return i < ns ? i : lo + (i - ns); }
};
struct Item {
  int b, h, rg, len, nrows;
};
__device__ __forceinline__ Span span_of(const AttnP& p, int rg, int len, int nrows) {
  Span s{};
  const int row0 = rg * p.tiles * 16, m0 = row0 / p.group, m1 = min((min(row0 + p.tiles * 16, p.R) - 1) / p.group, nrows - 1);
  s.p0 = len - nrows + m0;
  s.p1 = len - nrows + m1;
  if (m0 > m1 || s.p1 < 0) return s;
  const int64_t first = p.window ? (int64_t)s.p0 - p.window + 1 : 0;
  s.lo = first > 0 ? (int)(first / kKvRun) : 0;
  const int ns = (int)(((int64_t)p.sinks + kKvRun - 1) / kKvRun), hi = (s.p1 + kKvRun) / kKvRun;
  s.ns = ns < s.lo ? ns : s.lo;
  s.n = s.ns + (hi > s.lo ? hi - s.lo : 0);
  return s;
}
// item i: sequence, then row group, then key head (so that an XCD, which gets every eighth workgroup, keeps to few heads)
template <bool UNIFORM> __device__ __forceinline__ Item item_of(const AttnP& p, int i) {
  Item it;
  const int pair = i / p.kv.heads;
  it.h = i - pair * p.kv.heads;
  it.b = p.groups == 1 ? pair : pair / p.groups;
  it.rg = pair - it.b * p.groups;
  if constexpr (UNIFORM) {
    it.len = kv_len_uniform(p.kv, it.b);
    const int n = p.rows ? kv_scalar(p.rows, it.b) : p.M;
    it.nrows = n < 0 ? 0 : n < p.M ? n : p.M;
  } else {
    it.len = kv_len(p.kv, it.b);
    it.nrows = kv_rows(p.rows, it.b, p.M);
  }
  return it;
}

// Long items in parts, a workgroup a part: each item in as many equal parts as bring none over a common share, the least share
// that leaves no more parts than workgroups, so that all of them run at once and end together however ragged the lengths are.
// (Equal shares of all runs in a row, parts of two items to a workgroup where one ends, took 57 us where this takes 37: 64
// sequences of up to 8192 tokens.) A key head's items are alike, so a lane looks at (sequence, row group) pairs; every wave works
// the deal out for itself, without LDS and barriers.
constexpr int kMostItems = 512;   // 2 items <= workgroups <= 1024
constexpr int kMostPairs = 512;   // that are dealt so; more fill the chip an item each
__device__ __forceinline__ int wave_sum(int v) {
  const auto a = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
  v = (int)(a[0] + a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
  v = (int)(b[0] + b[1]);
  v += __builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, true);
  v += __builtin_amdgcn_mov_dpp(v, 0x124, 0xF, 0xF, true);
  v += __builtin_amdgcn_mov_dpp(v, 0x122, 0xF, 0xF, true);
  return v + __builtin_amdgcn_mov_dpp(v, 0x121, 0xF, 0xF, true);
}
struct Part {
  int item, part, parts;   // item -1: this workgroup has none
};
// zeros(item): an item whose rows see nothing, one workgroup's
template <class F> __device__ __forceinline__ Part part_of(const AttnP& p, int wg, int wgs, F zeros) {
  const int lane = threadIdx.x & 63, H = p.kv.heads, pairs = p.items / H;
  int n[kMostPairs / 64], total = 0, some = 0;   // runs of this lane's pairs; of all; pairs with runs
#pragma unroll
  for (int k = 0; k < kMostPairs / 64; ++k) {
    n[k] = 0;
    if (k * 64 >= pairs) continue;
    const int i = k * 64 + lane;
    if (i < pairs) {
      const Item it = item_of<false>(p, i * H);
      n[k] = span_of(p, it.rg, it.len, it.nrows).n;
    }
    total += wave_sum(n[k]);
    some += __popcll(__ballot(n[k] > 0));
    for (uint64_t none = __ballot(i < pairs && n[k] == 0); none; none &= none - 1) {
      const int z = (k * 64 + __ffsll((unsigned long long)none) - 1) * H;
      for (int h = (wg + wgs - z % wgs) % wgs; h < H; h += wgs) zeros(z + h);
    }
  }
  total = __builtin_amdgcn_readfirstlane(total);
  // an item's last part wastes half a share on average: first as if so, then as if a whole one, which always fits
  Part r{-1, 0, 1};
  for (int t = 1; t <= 2; ++t) {
    const int room = max(1, wgs - some * H * t / 2);
    int share = ((int64_t)total * H + room - 1) / room;
    share = (max(share, 1) + p.streams - 1) / p.streams * p.streams;
    int first = 0;   // parts before
    r.item = -1;
#pragma unroll
    for (int k = 0; k < kMostPairs / 64; ++k) {
      if (k * 64 >= pairs) continue;
      const int c = (n[k] + share - 1) / share;
      int x = c;
#pragma unroll
      for (int s = 1; s < 64; s <<= 1) {
        const int y = __shfl_up(x, s, 64);
        if (lane >= s) x += y;
      }
      const int under = first + (x - c) * H;
      const uint64_t here = __ballot(c > 0 && under <= wg && wg < under + c * H);
      if (here) {
        const int l = __ffsll((unsigned long long)here) - 1, in = wg - __builtin_amdgcn_readlane(under, l);
        r.parts = __builtin_amdgcn_readlane(c, l);
        r.item = (k * 64 + l) * H + in / r.parts;
        r.part = in % r.parts;
      }
      first += __builtin_amdgcn_readlane(x, 63) * H;
    }
    if (first <= wgs) break;
  }
  return r;
}

// the place of eight channels of a row in y
__device__ __forceinline__ int64_t out_at(const AttnP& p, const Item& it, int r) {
  return (int64_t)it.b * p.y_ldb + (int64_t)(r / p.group) * p.y_ldm + (int64_t)(it.h * p.group + r % p.group) * p.y_ldh;
}

// fp16 values that a query's or a probability's f32 is taken as. A probability of one part is off by up to 2^-12 of itself. In f16
// that shows (one row of 16 heads over 700 tokens, relative L2: 2.14e-4 in two parts, the rounding of the output, 2.69e-4 in one), in
// bf16 it does not (1.54e-3 either way; 3% of the outputs round to the neighbour), and it spares a third of the products (2 x 1024
// rows of 16 heads over 4096 tokens: f16 130 us, 110 in one part; bf16 113, 134 in two)
template <int TYPE> constexpr int kQParts = TYPE == P0_KV_F32 ? 2 : 1;
template <int TYPE> constexpr int kPParts = TYPE == P0_KV_BF16 ? 1 : 2;

// Queries as fp16 operands: f16 as it is. Else a row is taken under the power of two that brings its largest value to [2^14, 2^15),
// the top of fp16's range, as keys may be 0 where the query is large and large where it is small. bf16's 8 bits are whole down to
// 2^-17, that is 2^-31 of the largest, and off by 2^-39 of it at the most below. f32's second part is the rest times 2^12, with an
// accumulator of its own: 22 bits down to 2^-29 of the largest, off by 2^-51 of it below.
constexpr int kQTop = 14;
constexpr float kQRest = 4096.0f;
// the exponent of that power of two for a row whose largest magnitude is `most`. 0 for rows of nothing, and of an infinity
template <int TYPE> __device__ __forceinline__ int query_exponent(float most) {
  if constexpr (TYPE == P0_KV_F16) return 0;
  const int e = (int)(__float_as_uint(most) >> 23) - 127 - kQTop;
  return most == 0.0f || most == INFINITY ? 0 : e < -127 ? -127 : e;
}
// the factor of such a row's scores: neither 0 nor infinite, so that it leaves the scores of -infinity of what is not seen, and those of 0
__device__ __forceinline__ float score_factor(float scale2, int e) { return fminf(fmaxf(ldexpf(scale2, e), 0x1p-126f), 0x1.fffffep127f); }
template <int TYPE> __device__ __forceinline__ void query_operand(const float (&v)[8], int e, half8_t& hi, half8_t& lo) {
  const float down = __uint_as_float((uint32_t)(127 - e) << 23);   // e is -127 .. 113
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = TYPE == P0_KV_F16 ? v[j] : v[j] * down;
    hi[j] = (_Float16)x;
    if constexpr (kQParts<TYPE> == 2) lo[j] = (_Float16)((x - (float)hi[j]) * kQRest);
  }
}

// a part's maximum with its factor, as a row's parts are joined by it; *f: what makes up for the product's rounding
__device__ __forceinline__ float part_maximum(float m, float qs, float* f) {
  const float r = m * qs;
  *f = fabsf(r) < 0x1p20f ? exp2_fast(fmaf(m, qs, -r)) : 1.0f;
  return m == kNone ? kNone : r;
}

// A workgroup of kv_attn_kernel: waves of 16 rows each, W of them or, at 512 channels, W pairs (the registers of one wave a
// SIMD would hold them all, but a wave alone issues at half the rate): each of a pair has half of the channels' products and
// outputs, and they exchange their halves of the scores through LDS
// Bound: latency. The registers leave two waves a SIMD at 256 and 512 channels, and a run is a chain of loads, conversions,
// products, maximum and exponentials. Of the cycles of 64 sequences of up to 8192 tokens (256 channels, 4 heads a key head, 136 MB
// in 36 us, 3.8 TB/s of the 6.3 that a read reaches) the VALU is busy in 42%, most of it turning 4-bit codes into fp16 operands,
// the MFMA in 17%, LDS in 4%; of 5 rows of 8 heads of 512 channels over 131071 tokens (67 us and a join of 9.5) 40, 15 and 5%. Of a
// short sequence it is the chain from the page table to the first scores, then two or three runs a wave one after the other (one row over 517
// tokens: 12.5 us)
template <int D> constexpr int kRowSplit = D == 512 ? 2 : 1;
template <int D, int W> constexpr int kRowThreads = 64 * W * kRowSplit<D>;
template <int D> constexpr int kRowGroups = D == 64 ? 4 : D == 128 ? 3 : D == 256 ? 2 : 1;   // of them on a CU: what the registers allow

// 1 / (sum of probabilities), 0 where a row has seen nothing
__device__ __forceinline__ float inverse(float l) { return l > 0.0f || l != l ? 1.0f / l : 0.0f; }

template <int D, int TYPE, int W>
__global__ __launch_bounds__((kRowThreads<D, W>), D == 512 || W == 8 ? 2 : kRowGroups<D>) void kv_attn_kernel(const AttnP p) {
  constexpr int NW = W, SPLIT = kRowSplit<D>, STEPS = D / 32 / SPLIT, BLOCKS = D / 32 / SPLIT;
  constexpr int QPARTS = kQParts<TYPE>, PPARTS = kPParts<TYPE>;
  constexpr int TASKS = (D == 512 ? W : 2) * 16 * (D / 8), ROUNDS = (TASKS + kRowThreads<D, W> - 1) / kRowThreads<D, W>;
  // the queries as operands [part][tile][step][lane], then the halves of the scores [round % 2][wave][tile][lane], then the waves' sums
  __shared__ __attribute__((aligned(16))) float s_o[NW * SPLIT][16 * D / SPLIT];
  __shared__ float s_m[NW][16], s_l[NW][16], s_qs[NW * 16];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15, wg = blockIdx.x;
  const int half = wave % SPLIT, tile = wave / SPLIT % p.tiles, stream = wave / SPLIT / p.tiles;
  const bool works = stream < p.streams;

  int item = wg, part = 0, parts = 1;
  if (p.shared) {
    const Part r = part_of(p, wg, gridDim.x, [&](int i) {   // rows that see nothing
      if (tid == 0) p.dealt[2 * i + 1] = 0;
      const Item it = item_of<true>(p, i);
      const int rows = min(p.tiles * 16, p.R - it.rg * p.tiles * 16);
      const float zero[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma nounroll
      for (int t = tid; t < rows * (D / 8); t += blockDim.x)
        store8<TYPE>(p.y, out_at(p, it, it.rg * p.tiles * 16 + t / (D / 8)) + t % (D / 8) * 8, p.y_vec, zero);
    });
    if (r.item < 0) return;
    item = r.item;
    part = r.part;
    parts = r.parts;
    if (part == 0 && tid == 0) {
      p.dealt[2 * item] = wg;
      p.dealt[2 * item + 1] = parts;
    }
  }
  const Item it = item_of<true>(p, item);
  const Span sp = span_of(p, it.rg, it.len, it.nrows);
  const int each = ((sp.n + parts - 1) / parts + p.streams - 1) / p.streams * p.streams, off = part * each, end = min(sp.n, off + each);
  const int row0 = (it.rg * p.tiles + tile) * 16, row = row0 + col, m = row / p.group;
  const int pos = row < p.R && m < it.nrows ? it.len - it.nrows + m : -1;
  const bool whole = min(row0 + 15, p.R - 1) / p.group < it.nrows;   // every row of the tile that is one is the sequence's
  const int wgrow0 = it.rg * p.tiles * 16, wgrows = min(p.tiles * 16, p.R - wgrow0);
  const int first = off + stream;
  const bool active = works && first < end && row0 < p.R;

  // ---- the loads of the queries, of the first run's page and of the run: two waits on memory, not four
  float v[ROUNDS][8];
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int t = tid + k * kRowThreads<D, W>, r = t / (D / 8), c = t % (D / 8) * 8, mm = (wgrow0 + r) / p.group;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[k][j] = 0.0f;
    if (r < wgrows && mm < it.nrows)
      load8<TYPE>(p.q, (int64_t)it.b * p.q_ldb + (int64_t)mm * p.q_ldm + (int64_t)(it.h * p.group + wgrow0 + r - mm * p.group) * p.q_ldh + c,
                  p.q_vec, v[k]);
  }
  const int run_bytes = 34 * D, rlog = p.kv.page_log - 5, rmask = (1 << rlog) - 1;
  const uint8_t* head = p.kv.pages + ((int64_t)it.h << rlog) * run_bytes;
  // of run i of the span; past the last of these: the first again, so that the loads of the next run need no branch (with one
  // the compiler waits for all of them at the loop's head, the values that are wanted last among them)
  auto clamped = [&](int i) { return sp.run(i < end ? i : off); };
  auto page_of = [&](int i) { return kv_page_uniform(p.kv, it.b, __builtin_amdgcn_readfirstlane(clamped(i) >> rlog)); };
  auto run_at = [&](int i, int pg) {
    return head + (int64_t)(pg < 0 ? 0 : pg) * p.kv.page_bytes + (int64_t)(clamped(i) & rmask) * run_bytes;
  };
  KeyRegs<D> kr;
  ValueRegs<D> vr;
  int pg = -1, pg_next = -1;
  if (active) {
    pg = page_of(first);
    pg_next = page_of(first + p.streams);
    kr.load(run_at(first, pg), lane, half);
    vr.load(run_at(first, pg), lane, half);
  }
  // ---- the queries as operands, each row under its power of two: D / 8 lanes a row
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int t = tid + k * kRowThreads<D, W>, r = t / (D / 8), c = t % (D / 8) * 8;
    float most = 0.0f;
    if constexpr (TYPE != P0_KV_F16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(v[k][j]));
#pragma unroll
      for (int s = 1; s < D / 8; s <<= 1) most = fmaxf(most, __shfl_xor(most, s, 64));
    }
    const int e = query_exponent<TYPE>(most);
    half8_t hi, lo;
    query_operand<TYPE>(v[k], e, hi, lo);
    if (r < p.tiles * 16) {
      const int st = D == 64 ? c >> 3 & 1 : (c >> 7) * 4 + (c >> 3 & 3), gg = D == 64 ? c >> 4 : c >> 5 & 3;
      // (a row's lanes are one bank apart in `st` and `gg`: the column is turned by them)
      half8_t* sq = (half8_t*)&s_o[0][0] + ((r >> 4) * (D / 32) + st) * 64 + gg * 16 + ((r ^ (4 * st + gg)) & 15);
      *sq = hi;
      if constexpr (QPARTS == 2) sq[p.tiles * (D / 32) * 64] = lo;
      if (c == 0) s_qs[r] = score_factor(p.scale2, e);
    }
  }
  __syncthreads();

  float4_t o[2 * BLOCKS];
#pragma unroll
  for (int i = 0; i < 2 * BLOCKS; ++i) o[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float mrun = kNone, lrun = 0.0f;
  half8_t qh[STEPS], ql[QPARTS == 2 ? STEPS : 1];
  const half8_t* sq = (const half8_t*)&s_o[0][0] + ((works ? tile : 0) * (D / 32) + half * STEPS) * 64 + g * 16;
#pragma unroll
  for (int st = 0; st < STEPS; ++st) {
    const int c = st * 64 + ((col ^ (4 * (half * STEPS + st) + g)) & 15);
    qh[st] = sq[c];
    if constexpr (QPARTS == 2) ql[st] = sq[p.tiles * (D / 32) * 64 + c];
  }
  const float qs = s_qs[(works ? tile : 0) * 16 + col];
  if constexpr (SPLIT == 2) __syncthreads();   // the scores' halves go where the queries were
  if (SPLIT == 2 || active) {
#pragma nounroll
    for (int i = first, par = 0; i - stream < end; i += p.streams, par ^= 1) {   // the same rounds for every stream
      const bool has = active && i < end;
      if (SPLIT == 1 && !has) break;
      const int t0 = sp.run(has ? i : off) * kKvRun;
      const bool dead = pg < 0;
      // ---- scores: lane (g, col) gets tokens 16 tt + 4 g + r of row col. A chain of products per tile and part
      float4_t s[2], sl[2];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) s[tt] = sl[tt] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
      if (SPLIT == 1 || has) {
#pragma unroll
        for (int st = 0; st < STEPS; ++st)
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) {
            const half8_t a = kr.operand(tt, st);
            s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[st], s[tt], 0, 0, 0);
            if constexpr (QPARTS == 2) sl[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[st], sl[tt], 0, 0, 0);
          }
      }
      if constexpr (QPARTS == 2) {
        s[0] += sl[0] * (1.0f / kQRest);
        s[1] += sl[1] * (1.0f / kQRest);
      }
      const int pg_after = page_of(i + 2 * p.streams);
      if constexpr (SPLIT == 2) {
        float4_t* x = (float4_t*)&s_o[0][0] + par * NW * SPLIT * 128;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) x[(wave * 2 + tt) * 64 + lane] = s[tt];
        if (has) kr.load(run_at(i + p.streams, pg_next), lane, half);
        __syncthreads();
        if (!has) continue;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) s[tt] += x[((wave ^ 1) * 2 + tt) * 64 + lane];
      } else {
        kr.load(run_at(i + p.streams, pg_next), lane, half);
      }
      // ---- what the rows do not see
      const bool all = !dead && t0 + kKvRun - 1 <= sp.p0 && whole &&
                       (!p.window || t0 > sp.p1 - p.window || t0 + kKvRun <= p.sinks);
      if (!all) {
        const int last = dead ? -1 : pos, since = p.window ? pos - p.window + 1 : 0;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int t = t0 + 16 * tt + 4 * g + r;
            s[tt][r] = (t <= last) & ((t >= since) | (t < p.sinks)) ? s[tt][r] : -INFINITY;
          }
        if (dead || t0 + kKvRun > it.len) vr.cut(dead ? 0 : it.len - t0, lane);
      }
      // ---- running maximum and sum
      float top = kNone;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[tt][r]);
      top = fmaxf(groups_max(top), mrun);
      if (__any(top > mrun)) {
        const float f = exp2_fast((mrun - top) * qs);
        lrun *= f;
#pragma unroll
        for (int k = 0; k < 2 * BLOCKS; ++k) o[k] *= f;
        mrun = top;
      }
      half8_t ph, pl;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = exp2_fast(fmaf(s[tt][r] - mrun, qs, kLift));
          lrun += x;
          ph[tt * 4 + r] = (_Float16)x;
          if constexpr (PPARTS == 2) pl[tt * 4 + r] = (_Float16)(x - (float)ph[tt * 4 + r]);
        }
      // ---- outputs: lane (g, col) gets channels 32 bl + 8 g + 2 r + u of row col
#pragma unroll
      for (int bl = 0; bl < BLOCKS; ++bl) {
        half8_t a[2];
        vr.operands(bl, a);
#pragma unroll
        for (int u = 0; u < 2; ++u) o[2 * bl + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[u], ph, o[2 * bl + u], 0, 0, 0);
        if constexpr (PPARTS == 2) {
#pragma unroll
          for (int u = 0; u < 2; ++u) o[2 * bl + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[u], pl, o[2 * bl + u], 0, 0, 0);
        }
      }
      vr.load(run_at(i + p.streams, pg_next), lane, half);
      pg = pg_next;
      pg_next = pg_after;
    }
    lrun = groups_sum(lrun);
  }

  // ---- waves with the same rows, through LDS: a thread adds eight channels of a row over the streams
  __syncthreads();   // the queries there have been read
  if (g == 0 && half == 0) { s_m[wave / SPLIT][col] = mrun; s_l[wave / SPLIT][col] = lrun; }
  if (works) {
#pragma unroll
    for (int k = 0; k < 2 * BLOCKS; ++k) *(float4_t*)(s_o[wave] + k * 256 + lane * 4) = o[k];
  }
  __syncthreads();
  float* mine = p.part + (int64_t)wg * p.slot;
#pragma nounroll
  for (int t = tid; t < p.tiles * (D / 32) * 64; t += kRowThreads<D, W>) {
    const int tl = t / (D / 32 * 64), bl = t / 64 % (D / 32), c = t & 15, gg = t >> 4 & 3, r = tl * 16 + c;
    if (r >= wgrows) continue;
    const float rqs = s_qs[r];
    float mall = kNone, lall = 0.0f, f[NW], made_up = 1.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {   // past the last stream: the first again, at no weight
      f[w] = w < p.streams ? s_m[w * p.tiles + tl][c] : kNone;
      mall = fmaxf(mall, f[w]);
    }
    const float mpart = parts == 1 ? 0.0f : part_maximum(mall, rqs, &made_up);
    float4_t x = {0.0f, 0.0f, 0.0f, 0.0f}, z = x;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const int sw = (w < p.streams ? w : 0) * p.tiles + tl;
      f[w] = w < p.streams ? exp2_fast((f[w] - mall) * rqs) * made_up : 0.0f;
      lall = w < p.streams ? fmaf(s_l[sw][c], f[w], lall) : lall;
      const float* d = s_o[sw * SPLIT + bl / BLOCKS] + bl % BLOCKS * 512 + (t & 63) * 4;
      const float4_t a = *(const float4_t*)d, b = *(const float4_t*)(d + 256);
      if (w < p.streams) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = fmaf(a[j], f[w], x[j]);
          z[j] = fmaf(b[j], f[w], z[j]);
        }
      }
    }
    if (parts == 1) {
      const float inv = inverse(lall);
      const float y[8] = {x[0] * inv, z[0] * inv, x[1] * inv, z[1] * inv, x[2] * inv, z[2] * inv, x[3] * inv, z[3] * inv};
      store8<TYPE>(p.y, out_at(p, it, wgrow0 + r) + 32 * bl + 8 * gg, p.y_vec, y);
    } else {
      float* d = mine + r * D + 32 * bl + 8 * gg;
      if (p.join) {   // for the next launch
        *(float4_t*)d = float4_t{x[0], z[0], x[1], z[1]};
        *(float4_t*)(d + 4) = float4_t{x[2], z[2], x[3], z[3]};
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) part_store(d + 2 * j, x[j], z[j]);
      }
      if (bl == 0 && gg == 0) part_store(mine + wgrows * D + 2 * r, mpart, lall);
    }
  }
  if (parts > 1 && !p.join) {
    // ---- workgroups with the same rows: parts in the workspace, the last to arrive adds them in order, four in flight
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      unsigned* c = p.cnt + item;
      s_last = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(parts - 1);
      if (s_last) __hip_atomic_exchange(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // leave it at zero
    }
    __syncthreads();
    if (s_last) {
      const float* all = p.part + (int64_t)(wg - part) * p.slot;
#pragma nounroll
      for (int t = tid; t < wgrows * (D / 8); t += kRowThreads<D, W>) {
        const int r = t / (D / 8), c = t % (D / 8) * 8;
        float mm = kNone, ll = 0.0f, y[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma nounroll
        for (int w0 = 0; w0 < parts; w0 += 4) {   // past the last part: the last again, at no weight
          float2 ml[4], a[4][4];   // maximum and sum; eight channels
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float* x = all + min(w0 + u, parts - 1) * p.slot;
            ml[u] = part_load(x + wgrows * D + 2 * r);
#pragma unroll
            for (int j = 0; j < 4; ++j) a[u][j] = part_load(x + r * D + c + 2 * j);
          }
          const float was = mm;
#pragma unroll
          for (int u = 0; u < 4; ++u) mm = fmaxf(mm, ml[u].x);
          const float f0 = exp2_fast(was - mm);
          ll *= f0;
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] *= f0;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (w0 + u >= parts) continue;
            const float f = exp2_fast(ml[u].x - mm);
            ll = fmaf(f, ml[u].y, ll);
#pragma unroll
            for (int j = 0; j < 4; ++j) { y[2 * j] = fmaf(a[u][j].x, f, y[2 * j]); y[2 * j + 1] = fmaf(a[u][j].y, f, y[2 * j + 1]); }
          }
        }
        const float inv = inverse(ll);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] *= inv;
        store8<TYPE>(p.y, out_at(p, it, wgrow0 + r) + c, p.y_vec, y);
      }
    }
  }
}

// ---- many rows of at most 128 channels: the runs are converted once for a workgroup, into LDS as operands, and each of eight
// waves reads them for its 16 rows. Two buffers of two runs: while the waves work on one, each converts its share of the next
// (whose bytes it loaded two rounds before) into the other; one barrier a round.
// Bound: latency between the barriers, at 16 KB of operands from LDS a wave and run. 2 x 1024 bf16 rows of 16 heads of 128 channels
// under a window of 4096, 96 us and a join of 7: VALU busy in 34% of the cycles, LDS in 19, MFMA in 14; two workgroups a CU hide each
// other's barriers (one of 16 waves: 114 us where two of 8 take 95). 8 x 1024 rows of 16 heads over 4096 tokens: bf16 355 us, 678 TFLOP/s, f16 424, f32 497. Wider heads leave too few waves for that, and run
// faster where each wave converts for itself (256 channels, 2 x 1024 rows over 4096: 467 us here, 237 there).
template <int D> struct TileShape {
  static constexpr int TILES = 8, RUNS = 2, kWaves = TILES, kThreads = 64 * kWaves;
  // 8 bytes a lane of a run's codes at a time: two steps of a tile's keys (64 channels: a tile's both), a block of values
  static constexpr int KU = D == 64 ? 2 : 4 * (D / 128), VU = D / 32;
  static constexpr int UNITS = RUNS * (KU + VU), PER = UNITS / kWaves;  // pieces a round, of them a wave's
  static constexpr int FRAGS = 4 * (D / 32);                            // a run's operands (64 lanes of 16 bytes): half keys, half values
  static constexpr int DEPTH = 2;                                       // rounds whose bytes are on their way
};
template <int D, int TYPE>
__global__ __launch_bounds__(TileShape<D>::kThreads, 4) void kv_attn_tiles_kernel(const AttnP p) {
  using S = TileShape<D>;
  constexpr int RUNS = S::RUNS, PER = S::PER, DEPTH = S::DEPTH, STEPS = D / 32, BLOCKS = D / 32;
  constexpr int QPARTS = kQParts<TYPE>, PPARTS = kPParts<TYPE>;
  extern __shared__ __attribute__((aligned(16))) uint8_t s_raw[];
  half8_t* buf = (half8_t*)s_raw;   // [2][RUNS][FRAGS][64]
  __shared__ int s_dead[2][RUNS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15, wg = blockIdx.x;

  int item = wg, part = 0, parts = 1;
  if (p.shared) {
    const Part r = part_of(p, wg, gridDim.x, [&](int i) {   // rows that see nothing
      if (tid == 0) p.dealt[2 * i + 1] = 0;
      const Item it = item_of<true>(p, i);
      const int rows = min(p.tiles * 16, p.R - it.rg * p.tiles * 16);
      const float zero[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma nounroll
      for (int t = tid; t < rows * (D / 8); t += blockDim.x)
        store8<TYPE>(p.y, out_at(p, it, it.rg * p.tiles * 16 + t / (D / 8)) + t % (D / 8) * 8, p.y_vec, zero);
    });
    if (r.item < 0) return;
    item = r.item;
    part = r.part;
    parts = r.parts;
    if (part == 0 && tid == 0) {
      p.dealt[2 * item] = wg;
      p.dealt[2 * item + 1] = parts;
    }
  }
  const Item it = item_of<true>(p, item);
  const Span sp = span_of(p, it.rg, it.len, it.nrows);
  const int each = ((sp.n + parts - 1) / parts + RUNS - 1) / RUNS * RUNS, off = part * each, end = min(sp.n, off + each);
  const int wgrow0 = it.rg * p.tiles * 16, wgrows = min(p.tiles * 16, p.R - wgrow0);
  const int row0 = wgrow0 + wave * 16;
  // this wave's rows: positions of the first and the last that are the sequence's
  const int m0 = row0 / p.group, m1 = min((min(row0 + 16, p.R) - 1) / p.group, it.nrows - 1);
  const bool active = row0 < p.R && m0 <= m1;
  const int pos0 = it.len - it.nrows + m0, pos1 = it.len - it.nrows + m1;
  const bool whole = (min(row0 + 16, p.R) - 1) / p.group < it.nrows;

  const int run_bytes = 34 * D, rlog = p.kv.page_log - 5, rmask = (1 << rlog) - 1;
  const uint8_t* head = p.kv.pages + ((int64_t)it.h << rlog) * run_bytes;
  // this wave's pieces of a round: codes and exponents, and what is cut off them
  struct Bytes {
    uint2_t code[PER], exps[PER];
    int left[PER];
  } ahead[DEPTH];
  // the pages of this wave's pieces of the round to be fetched next: a round ahead of the loads that need them
  int pages[PER];
  auto look = [&](int j) {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int rr = (wave + n * S::kWaves) / (S::KU + S::VU);
      pages[n] = kv_page_uniform(p.kv, it.b, sp.run(j + rr < end ? j + rr : off) >> rlog);
    }
  };
  auto fetch = [&](Bytes& y, int j) {   // the round that begins with run j of the span
    auto& [code, exps, left] = y;
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int u = wave + n * S::kWaves, rr = u / (S::KU + S::VU), x = u % (S::KU + S::VU);
      const int r = sp.run(j + rr < end ? j + rr : off), pg = pages[n];
      const uint8_t* run = head + (int64_t)(pg < 0 ? 0 : pg) * p.kv.page_bytes + (int64_t)(r & rmask) * run_bytes;
      left[n] = j + rr >= end || pg < 0 ? 0 : it.len - r * kKvRun;   // tokens of the run that are there
      if (x < S::KU) {
        code[n] = *(const uint2_t*)(run + (x >> 1) * 1024 + lane * 16 + (x & 1) * 8);
        if constexpr (D == 64) exps[n].x = run[16 * D + ((lane >> 5) * 16 + (lane & 15)) * 2 + x];
        else exps[n].x = run[16 * D + (lane * 2 + (x >> 1) / (D / 128)) * (D / 128) + (x >> 1) % (D / 128)];
      } else {
        code[n] = *(const uint2_t*)(run + 17 * D + ((x - S::KU) >> 1) * 1024 + lane * 16 + ((x - S::KU) & 1) * 8);
        exps[n] = *(const uint2_t*)(run + 33 * D + ((lane >> 4) * (D / 32) + x - S::KU) * 8);
      }
    }
  };
  auto convert = [&](Bytes& y, int to) {
    auto& [code, exps, left] = y;
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int u = wave + n * S::kWaves, rr = u / (S::KU + S::VU), x = u % (S::KU + S::VU);
      half8_t* d = buf + (to * RUNS + rr) * S::FRAGS * 64 + lane;
      if (x < S::KU) {
        const float e = exponent_of<0>(exps[n].x);
        d[x * 2 * 64] = widen(code[n].x, e);
        d[(x * 2 + 1) * 64] = widen(code[n].y, e);
        if (x == 0 && lane == 0) s_dead[to][rr] = left[n] <= 0;
      } else {
        if (left[n] < kKvRun) {
          exps[n].x &= keep_bytes(left[n] - 4 * g);
          exps[n].y &= keep_bytes(left[n] - 16 - 4 * g);
        }
        half8_t a[2];
        value_operands(code[n].x, code[n].y, exps[n].x, exps[n].y, a);
        d[(2 * STEPS + 2 * (x - S::KU)) * 64] = a[0];
        d[(2 * STEPS + 2 * (x - S::KU) + 1) * 64] = a[1];
      }
    }
  };
  // (past the last round: of the first again, so that the loads need no branch and no wait before their time)
  auto round_at = [&](int j) { return j < end ? j : off; };
#pragma unroll
  for (int k = 0; k < DEPTH; ++k) {
    look(round_at(off + k * RUNS));
    fetch(ahead[k], round_at(off + k * RUNS));
  }
  look(round_at(off + DEPTH * RUNS));

  // ---- the queries: lane (g, col) has 8 channels a step of row col
  const int row = row0 + col, m = row / p.group;
  const bool in = row < p.R && m < it.nrows;
  const int pos = in ? it.len - it.nrows + m : -1;
  half8_t qh[STEPS], ql[QPARTS == 2 ? STEPS : 1];
  float qs;
  {
    const int64_t base = in ? (int64_t)it.b * p.q_ldb + (int64_t)m * p.q_ldm + (int64_t)(it.h * p.group + row - m * p.group) * p.q_ldh : 0;
    auto query = [&](int st, float (&v)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
      if (in) load8<TYPE>(p.q, base + (D == 64 ? g * 16 + 8 * st : (st >> 2) * 128 + g * 32 + 8 * (st & 3)), p.q_vec, v);
    };
    float most = 0.0f;
    if constexpr (TYPE != P0_KV_F16) {
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        float v[8];
        query(st, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(v[j]));
      }
      most = groups_max(most);
    }
    const int e = query_exponent<TYPE>(most);
    qs = score_factor(p.scale2, e);
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      float v[8];
      query(st, v);
      query_operand<TYPE>(v, e, qh[st], ql[QPARTS == 2 ? st : 0]);
    }
  }

  float4_t o[2 * BLOCKS];
  float mrun = kNone, lrun = 0.0f;
#pragma unroll
  for (int i = 0; i < 2 * BLOCKS; ++i) o[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  convert(ahead[0], 0);
  fetch(ahead[0], round_at(off + DEPTH * RUNS));
  look(round_at(off + (1 + DEPTH) * RUNS));
  __syncthreads();
  int j = off, cur = 0;
  auto round = [&](Bytes& next) {   // false: it was the last
    convert(next, cur ^ 1);
    fetch(next, round_at(j + (1 + DEPTH) * RUNS));
    look(round_at(j + (2 + DEPTH) * RUNS));
#pragma unroll
    for (int rr = 0; rr < RUNS; ++rr) {
      const int i = j + rr, t0 = sp.run(i < end ? i : off) * kKvRun;
      const bool dead = i >= end || __builtin_amdgcn_readfirstlane(s_dead[cur][rr]);
      // runs that none of this wave's rows sees are left out (all waves take part in the barriers)
      const bool seen = active && !dead && t0 <= pos1 && (!p.window || t0 + kKvRun > pos0 - p.window + 1 || t0 < p.sinks);
      if (seen) {
        const half8_t* kf = buf + (cur * RUNS + rr) * S::FRAGS * 64 + lane;
        const half8_t* vf = kf + 2 * STEPS * 64;
        float4_t s[2], sl[2];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) s[tt] = sl[tt] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < STEPS; ++st)
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) {
            const half8_t a = kf[(tt * STEPS + st) * 64];
            s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[st], s[tt], 0, 0, 0);
            if constexpr (QPARTS == 2) sl[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[st], sl[tt], 0, 0, 0);
          }
        if constexpr (QPARTS == 2) {
          s[0] += sl[0] * (1.0f / kQRest);
          s[1] += sl[1] * (1.0f / kQRest);
        }
        const bool all = t0 + kKvRun - 1 <= pos0 && whole && (!p.window || t0 > pos1 - p.window || t0 + kKvRun <= p.sinks);
        if (!all) {
          const int since = p.window ? pos - p.window + 1 : 0;
#pragma unroll
          for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int t = t0 + 16 * tt + 4 * g + r;
              s[tt][r] = (t <= pos) & ((t >= since) | (t < p.sinks)) ? s[tt][r] : -INFINITY;
            }
        }
        float top = kNone;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) top = fmaxf(top, s[tt][r]);
        top = fmaxf(groups_max(top), mrun);
        if (__any(top > mrun)) {
          const float f = exp2_fast((mrun - top) * qs);
          lrun *= f;
#pragma unroll
          for (int k = 0; k < 2 * BLOCKS; ++k) o[k] *= f;
          mrun = top;
        }
        half8_t ph, pl;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = exp2_fast(fmaf(s[tt][r] - mrun, qs, kLift));
            lrun += x;
            ph[tt * 4 + r] = (_Float16)x;
            if constexpr (PPARTS == 2) pl[tt * 4 + r] = (_Float16)(x - (float)ph[tt * 4 + r]);
          }
#pragma unroll
        for (int k = 0; k < 2 * BLOCKS; ++k) {
          const half8_t a = vf[k * 64];
          o[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph, o[k], 0, 0, 0);
          if constexpr (PPARTS == 2) o[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, o[k], 0, 0, 0);
        }
      }
    }
    __syncthreads();
    cur ^= 1;
    j += RUNS;
    return j < end;
  };
#pragma nounroll
  while (off < end) {
    if (!round(ahead[1])) break;
    if (!round(ahead[0])) break;
  }

  lrun = groups_sum(lrun);
  const int r = wave * 16 + col;
  if (r >= wgrows) return;
  float made_up;
  const float mpart = part_maximum(mrun, qs, &made_up), inv = parts == 1 ? inverse(lrun) : made_up;
  float* mine = p.part + (int64_t)wg * p.slot;
  const int64_t at = out_at(p, it, wgrow0 + r);
#pragma unroll
  for (int k = 0; k < BLOCKS; ++k) {
    const float4_t a = o[2 * k], b = o[2 * k + 1];
    const float y[8] = {a[0] * inv, b[0] * inv, a[1] * inv, b[1] * inv, a[2] * inv, b[2] * inv, a[3] * inv, b[3] * inv};
    if (parts == 1) store8<TYPE>(p.y, at + 32 * k + 8 * g, p.y_vec, y);
    else store8<P0_KV_F32>(mine, (int64_t)r * D + 32 * k + 8 * g, 1, y);
  }
  if (parts > 1 && g == 0) {
    mine[wgrows * D + 2 * r] = mpart;
    mine[wgrows * D + 2 * r + 1] = lrun * made_up;
  }
}

// The parts of an item in a launch of their own: LANES threads for eight channels of a row, each its share of the parts, then LDS.
// Bound: memory latency, a few round trips (256 parts of 40 rows of 512 channels, 21 MB from the caches: 9 us)
template <int D, int TYPE, int LANES>
__global__ __launch_bounds__(256) void kv_join_kernel(const AttnP p) {
  constexpr int TASKS = 256 / LANES;
  __shared__ __attribute__((aligned(16))) float s_v[LANES > 1 ? 256 : 1][12];   // a thread's maximum, sum, eight channels
  const int tid = threadIdx.x, item = blockIdx.y, t = blockIdx.x * TASKS + tid % TASKS, part0 = tid / TASKS;
  const int wg0 = p.dealt[2 * item], parts = p.dealt[2 * item + 1];
  if (parts <= 1) return;
  const Item it = item_of<true>(p, item);
  const int wgrow0 = it.rg * p.tiles * 16, wgrows = min(p.tiles * 16, p.R - wgrow0);
  const int r = t / (D / 8), c = t % (D / 8) * 8;
  const bool in = r < wgrows;
  const float* x = p.part + (int64_t)wg0 * p.slot;
  float mm = kNone, ll = 0.0f, v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (in) {
#pragma nounroll
    for (int w0 = part0; w0 < parts; w0 += 4 * LANES) {   // four in flight; past the last: the last again, at no weight
      float pm[4], pl[4];
      float4_t a[4], b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float* y = x + min(w0 + u * LANES, parts - 1) * p.slot;
        pm[u] = y[wgrows * D + 2 * r];
        pl[u] = y[wgrows * D + 2 * r + 1];
        a[u] = *(const float4_t*)(y + r * D + c);
        b[u] = *(const float4_t*)(y + r * D + c + 4);
      }
      const float was = mm;
#pragma unroll
      for (int u = 0; u < 4; ++u) mm = fmaxf(mm, pm[u]);
      const float f0 = exp2_fast(was - mm);
      ll *= f0;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= f0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (w0 + u * LANES >= parts) continue;
        const float f = exp2_fast(pm[u] - mm);
        ll = fmaf(f, pl[u], ll);
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = fmaf(a[u][j], f, v[j]); v[4 + j] = fmaf(b[u][j], f, v[4 + j]); }
      }
    }
  }
  if constexpr (LANES > 1) {
    float* mine = s_v[tid];
    mine[8] = mm;
    mine[9] = ll;
    *(float4_t*)mine = float4_t{v[0], v[1], v[2], v[3]};
    *(float4_t*)(mine + 4) = float4_t{v[4], v[5], v[6], v[7]};
    __syncthreads();
    if (part0) return;
#pragma unroll 4
    for (int w = 1; w < LANES; ++w) mm = fmaxf(mm, s_v[w * TASKS + tid][8]);
    const float f0 = exp2_fast(mine[8] - mm);
    ll *= f0;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= f0;
#pragma unroll 4
    for (int w = 1; w < LANES; ++w) {
      const float* y = s_v[w * TASKS + tid];
      const float f = exp2_fast(y[8] - mm);
      const float4_t a = *(const float4_t*)y, b = *(const float4_t*)(y + 4);
      ll = fmaf(f, y[9], ll);
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] = fmaf(a[j], f, v[j]); v[4 + j] = fmaf(b[j], f, v[4 + j]); }
    }
  }
  if (!in) return;
  const float inv = inverse(ll);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= inv;
  store8<TYPE>(p.y, out_at(p, it, wgrow0 + r) + c, p.y_vec, v);
}

template <int D> constexpr int kTileLds = 2 * TileShape<D>::RUNS * TileShape<D>::FRAGS * 64 * 16;
enum Form { kRows4, kRows8, kTiles };
template <int D, int TYPE>
static void launch_typed(const AttnP& p, Form form, int wgs, hipStream_t s) {
  if constexpr (D <= 128) {
    if (form == kTiles) hipLaunchKernelGGL((kv_attn_tiles_kernel<D, TYPE>), dim3((unsigned)wgs), dim3(TileShape<D>::kThreads), kTileLds<D>, s, p);
  }
  if constexpr (D < 512) {
    if (form == kRows8) hipLaunchKernelGGL((kv_attn_kernel<D, TYPE, 8>), dim3((unsigned)wgs), dim3(kRowThreads<D, 8>), 0, s, p);
  }
  if (form == kRows4) hipLaunchKernelGGL((kv_attn_kernel<D, TYPE, 4>), dim3((unsigned)wgs), dim3(kRowThreads<D, 4>), 0, s, p);
  if (p.join) {   // an item's parts: about wgs / items
    const int tasks = (p.R < p.tiles * 16 ? p.R : p.tiles * 16) * (D / 8);
    if (wgs > 8 * p.items) hipLaunchKernelGGL((kv_join_kernel<D, TYPE, 32>), dim3((tasks + 7) / 8, p.items), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((kv_join_kernel<D, TYPE, 1>), dim3((tasks + 255) / 256, p.items), dim3(256), 0, s, p);
  }
}
template <int D> static hipError_t allow_lds() {
  for (const void* k : {(const void*)kv_attn_tiles_kernel<D, P0_KV_F32>, (const void*)kv_attn_tiles_kernel<D, P0_KV_F16>,
                        (const void*)kv_attn_tiles_kernel<D, P0_KV_BF16>})
    if (hipError_t e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, kTileLds<D>); e != hipSuccess) return e;
  return hipSuccess;
}
int kv_attn_init() {
  P0_HIP(allow_lds<64>(), "p0_open: kv_attn");
  P0_HIP(allow_lds<128>(), "p0_open: kv_attn");
  return P0_OK;
}
template <int D>
static void launch_attn(const AttnP& p, int type, Form form, int wgs, hipStream_t s) {
  if (type == P0_KV_F32) launch_typed<D, P0_KV_F32>(p, form, wgs, s);
  else if (type == P0_KV_F16) launch_typed<D, P0_KV_F16>(p, form, wgs, s);
  else launch_typed<D, P0_KV_BF16>(p, form, wgs, s);
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
  p.M = (int)a->M;
  p.group = (int)(a->heads / a->kv.heads);
  if (a->M * p.group > (1 << 28)) { set_error("kv_attn: M %lld of %d heads a key head", (long long)a->M, p.group); return P0_EINVAL; }
  p.R = p.M * p.group;
  const int64_t most = (int64_t)p.kv.cols << p.kv.page_log;
  p.window = a->window >= most ? 0 : (int)a->window;   // a window as long as the sequence hides nothing
  p.sinks = (int)(a->sinks < most ? a->sinks : most);
  const float scale = a->scale != 0.0f ? a->scale : 1.0f / sqrtf((float)D);
  p.scale2 = scale * 1.44269504088896340736f;
  const int alltiles = (p.R + 15) / 16;
  const int64_t longest = a->max_len && a->max_len < most ? a->max_len : most, seen = p.window + a->M + p.sinks + 2 * kKvRun;
  const int64_t runs = (p.window && seen < longest ? seen : longest) / kKvRun + 1;
  // Rows share converted runs where the chip's workgroups get enough runs each to outweigh a longer start and a barrier a round,
  // fewer of 16-bit queries, whose products are cheaper beside the conversion. (us, shared / each wave for itself, 128 channels,
  // 4 key heads of 4 heads over 4096 tokens: f16 32 x 32 rows 88 / 95, 2 x 1024 130 / 142, 4 x 128 54 / 58; over 2048, 8 key
  // heads, 2 x 128 rows, 42 / 39; bf16 2 x 1024 113 / 127, 4 x 128 52 / 55; f32 2 x 1024 152 / 159, 32 x 64 160 / 168, 4 x 128
  // 65 / 61; 64 channels, f16, 8 x 256 92 / 104, 4 x 64 37 / 33.)
  const int64_t work = a->B * p.kv.heads * ((p.R + 16 * TileShape<64>::TILES - 1) / (16 * TileShape<64>::TILES)) * runs;
  Form form = D <= 128 && p.R >= 128 && work >= (a->type == P0_KV_F32 ? 48 : 12) * 512 ? kTiles : kRows4;
  if (form == kTiles) {
    p.tiles = TileShape<64>::TILES;
    p.streams = 2;
  } else {   // a workgroup's waves: row tiles first, then streams over the runs
    p.tiles = alltiles < 2 ? alltiles : D == 512 ? (alltiles < 4 ? alltiles : 4) : 2;
    p.streams = 4 / p.tiles;
  }
  p.groups = (alltiles + p.tiles - 1) / p.tiles;
  const int64_t items = a->B * p.kv.heads * p.groups;
  if (items > 0x7FFFFFFF) { set_error("kv_attn: %lld sequences of %d rows", (long long)a->B, p.R); return P0_EINVAL; }
  p.items = (int)items;
  const int64_t rows = p.R < p.tiles * 16 ? p.R : p.tiles * 16;
  p.slot = rows * (D + 4);
  p.dealt = (int32_t*)ctx().part;
  p.part = ctx().part + 2 * kMostItems;
  p.cnt = ctx().kv_counters;
  int64_t wgs = 256 * (form == kTiles ? 2 : D == 64 ? kRowGroups<64> : D == 128 ? kRowGroups<128> : D == 256 ? kRowGroups<256> : kRowGroups<512>);
  const int64_t room = ((int64_t)ctx().part_floats - 2 * kMostItems) / p.slot, need = items * ((runs + 4 * p.streams - 1) / (4 * p.streams));
  wgs = wgs < room ? wgs : room;
  wgs = wgs < need ? wgs : need;
  // Few items in parts, where the runs that a part saves outweigh the join. (us, in parts / not: one row of 4 heads a key head,
  // 256 channels, 800 tokens 16.2 / 14.9, 1200 16.5 / 18.5, 2500 18.0 / 29.0; 512 channels, one row of 8 heads, 600 tokens
  // 20.3 / 21.5, five rows, 150 tokens 29.9 / 25.0, 300 33.4 / 37.3.)
  // (The deal counts the runs of all pairs in 32 bits: where the table holds more, whatever max_len says, there are no parts.)
  const int64_t pairs = items / p.kv.heads;
  p.shared = pairs <= kMostPairs && pairs * (most / kKvRun + 1) <= 0x7FFFFFFF && 2 * items <= wgs && runs > (D == 512 ? 3 * p.streams + 4 : 9 * p.streams);
  if (!p.shared) {
    wgs = items;
    if (form == kRows4 && D < 512 && items <= 256 && runs > p.streams) {   // CUs to spare: eight waves an item (one row over 517 tokens 12.5 us, 14.3 in four)
      form = kRows8;
      p.streams = 8 / p.tiles;
    }
  }
  p.join = p.shared && (form == kTiles || wgs > 16 * items);
  switch (D) {
    case 64: launch_attn<64>(p, a->type, form, (int)wgs, ctx().cur); break;
    case 128: launch_attn<128>(p, a->type, form, (int)wgs, ctx().cur); break;
    case 256: launch_attn<256>(p, a->type, form, (int)wgs, ctx().cur); break;
    default: launch_attn<512>(p, a->type, form, (int)wgs, ctx().cur); break;
  }
  P0_LAUNCHED("kv_attn");
  return P0_OK;
}
