// kv.hip - rows into and out of a cache of mxfp4 pages (kv_common.hpp has the layout).
#include "kv_common.hpp"

namespace p0 {

int64_t kv_page_bytes(const p0_kv_t& kv) {
  return kv.page_bytes ? kv.page_bytes : p0_kv_page_bytes(kv.page, kv.heads, kv.dim);
}

int kv_check(const char* op, const p0_kv_t& kv, int64_t B, KvP* out) {
  const int64_t bytes = p0_kv_page_bytes(kv.page, kv.heads, kv.dim);
  if (!bytes) {
    set_error("%s: no pages of %d tokens, %d heads of %d", op, (int)kv.page, (int)kv.heads, (int)kv.dim);
    return P0_EINVAL;
  }
  if (kv.n_pages < 1 || kv.n_pages > (1 << 30)) { set_error("%s: %lld pages", op, (long long)kv.n_pages); return P0_EINVAL; }
  if (kv.page_bytes && (kv.page_bytes < bytes || kv.page_bytes % 16 || kv.page_bytes > (1ll << 62) / kv.n_pages)) {
    set_error("%s: page_bytes %lld (a page is %lld)", op, (long long)kv.page_bytes, (long long)bytes); return P0_EINVAL;
  }
  if (!kv.pages || !kv.table || !kv.len) { set_error("%s: missing pages, table or len buffer", op); return P0_EINVAL; }
  if ((uintptr_t)kv.pages % 16) { set_error("%s: pages must be 16-byte aligned", op); return P0_EINVAL; }
  if (kv.cols < 1 || kv.cols > ((1ll << 31) - 64) / kv.page || (kv.table_ld && kv.table_ld < kv.cols)) {
    set_error("%s: table of %lld columns, stride %lld", op, (long long)kv.cols, (long long)kv.table_ld); return P0_EINVAL;
  }
  if (B < 0 || B > 65535) { set_error("%s: B %lld", op, (long long)B); return P0_EINVAL; }
  out->pages = (uint8_t*)kv.pages;
  out->table = kv.table;
  out->len = kv.len;
  out->page_bytes = kv.page_bytes ? kv.page_bytes : bytes;
  out->table_ld = kv.table_ld ? kv.table_ld : kv.cols;
  out->n_pages = (int)kv.n_pages;
  out->cols = (int)kv.cols;
  out->page_log = __builtin_ctz(kv.page);
  out->heads = kv.heads;
  return P0_OK;
}

struct RowsP {
  KvP kv;
  const int32_t* rows;
  const int32_t* at;
  uint8_t* k;
  uint8_t* v;
  int64_t ldb, ldm, ldh;
  int M, type, vec;
};

// A workgroup takes the rows of one sequence and head that lie in one run of 32 tokens: rows [m0, m1), token t0 + m - m0 of the run;
// of them those in [lo, hi) are tokens that are there, in run `run` (null: no page).
struct Segment {
  int b, h, m0, m1, t0, lo, hi;
  uint8_t* run;
};
__device__ __forceinline__ Segment segment_of(const RowsP& p, int D) {
  Segment s;
  s.h = blockIdx.y % p.kv.heads;
  s.b = blockIdx.y / p.kv.heads;
  const int len = kv_len_uniform(p.kv, s.b), given = p.rows ? kv_scalar(p.rows, s.b) : p.M, n = given < 0 ? 0 : given < p.M ? given : p.M;
  const int64_t pos0 = p.at ? (int64_t)kv_scalar(p.at, s.b) : (int64_t)len - n, q = (pos0 >> 5) + blockIdx.x;
  const int64_t m0 = q * kKvRun - pos0, m1 = m0 + kKvRun;
  s.m0 = (int)(m0 > 0 ? m0 : 0);
  s.m1 = (int)(m1 < p.M ? m1 : p.M);
  s.t0 = (int)(pos0 + s.m0 - q * kKvRun);
  const bool there = q >= 0 && q * kKvRun < len;
  s.lo = s.m0;
  s.hi = !there ? s.m0 : (int)(n < len - pos0 ? n : len - pos0);
  s.hi = s.hi < s.m1 ? s.hi : s.m1;
  s.run = nullptr;
  if (there && s.lo < s.hi) {
    const int pg = kv_page_uniform(p.kv, s.b, (int)(q >> (p.kv.page_log - 5))), runs = 1 << (p.kv.page_log - 5);
    if (pg >= 0) s.run = p.kv.pages + pg * p.kv.page_bytes + ((int64_t)s.h * runs + (int)(q & (runs - 1))) * (34 * D);
  }
  return s;
}

// E consecutive elements of a row; vec: aligned to all of them, or to 16 bytes
template <int E> __device__ __forceinline__ void row_load(const uint8_t* x, int64_t i, int type, int vec, float (&f)[E]) {
  if (type == P0_KV_F32) {
    const float* a = (const float*)x + i;
    if (vec) {
      if constexpr (E == 2) { const float2 v = *(const float2*)a; f[0] = v.x; f[1] = v.y; }
      else
#pragma unroll
        for (int j = 0; j < E; j += 4) { const float4 v = *(const float4*)(a + j); f[j] = v.x; f[j + 1] = v.y; f[j + 2] = v.z; f[j + 3] = v.w; }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) f[j] = a[j];
    }
    return;
  }
  const uint16_t* a = (const uint16_t*)x + i;
  uint32_t w[E / 2];
  if (vec) {
    if constexpr (E == 2) w[0] = *(const uint32_t*)a;
    else if constexpr (E == 4) { const uint2 v = *(const uint2*)a; w[0] = v.x; w[1] = v.y; }
    else
#pragma unroll
      for (int j = 0; j < E / 2; j += 4) { const uint4 v = *(const uint4*)(a + 2 * j); w[j] = v.x; w[j + 1] = v.y; w[j + 2] = v.z; w[j + 3] = v.w; }
  } else {
#pragma unroll
    for (int j = 0; j < E / 2; ++j) w[j] = a[2 * j] | (uint32_t)a[2 * j + 1] << 16;
  }
#pragma unroll
  for (int j = 0; j < E / 2; ++j) {
    f[2 * j] = type == P0_KV_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)w[j]) : __uint_as_float(w[j] << 16);
    f[2 * j + 1] = type == P0_KV_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)(w[j] >> 16)) : __uint_as_float(w[j] & 0xFFFF0000u);
  }
}
template <int E> __device__ __forceinline__ void row_store(uint8_t* x, int64_t i, int type, int vec, const float (&f)[E]) {   // exact in every type
  if (type == P0_KV_F32) {
    float* a = (float*)x + i;
    if (vec) {
      if constexpr (E == 2) *(float2*)a = float2{f[0], f[1]};
      else
#pragma unroll
        for (int j = 0; j < E; j += 4) *(float4*)(a + j) = float4{f[j], f[j + 1], f[j + 2], f[j + 3]};
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) a[j] = f[j];
    }
    return;
  }
  uint32_t w[E / 2];
#pragma unroll
  for (int j = 0; j < E / 2; ++j)
    w[j] = type == P0_KV_F16 ? __builtin_bit_cast(uint16_t, (_Float16)f[2 * j]) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * j + 1]) << 16
                             : __float_as_uint(f[2 * j]) >> 16 | (__float_as_uint(f[2 * j + 1]) & 0xFFFF0000u);
  uint16_t* a = (uint16_t*)x + i;
  if (vec) {
    if constexpr (E == 2) *(uint32_t*)a = w[0];
    else if constexpr (E == 4) *(uint2*)a = uint2{w[0], w[1]};
    else
#pragma unroll
      for (int j = 0; j < E / 2; j += 4) *(uint4*)(a + 2 * j) = uint4{w[j], w[j + 1], w[j + 2], w[j + 3]};
  } else {
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      a[2 * j] = (uint16_t)w[j];
      a[2 * j + 1] = (uint16_t)(w[j] >> 16);
    }
  }
}

// the exponent byte of a block whose largest magnitude is `most`: the least e with most <= 6 * 2^e, that is the exponent
// field less 2, one more where the mantissa is over 1.5
__device__ __forceinline__ int block_exp(float most) {
  const int e = (int)((__float_as_uint(most) + 0x3FFFFFu) >> 23) - 2;
  return e < kKvMinExp ? kKvMinExp : e > kKvMaxExp ? kKvMaxExp : e;
}

// A wave takes one row at a time: lanes 0-31 its key, 32-63 its value, D / 32 consecutive channels each. A whole run is put
// together in LDS and leaves in 16-byte stores (a token's value codes are single bytes 16 apart: 19.5 us for 16336 rows of 256
// f16 channels without, 10.4 with); of a part of one each byte is stored by itself, as its other tokens stay.
// Bound: launch and three memory round trips at one row (3.2 us). At many neither HBM nor a unit is full (16336 rows: 21.2 MB read and
// written in 10.4 us, 2.0 TB/s; VALU busy in 33% of the cycles, LDS in 19, three quarters of that bank conflicts of single bytes):
// two rounds of loads one after the other, then the run's way through LDS, in workgroups of one run.
constexpr int kRunThreads = 256, kRunWaves = kRunThreads / 64;
template <int D>
__global__ __launch_bounds__(kRunThreads) void kv_put_kernel(const RowsP p) {
  constexpr int E = D / 32, L = 32 / E, AHEAD = D == 512 ? 2 : 4;   // channels a lane, lanes a block, rows on their way
  __shared__ __attribute__((aligned(16))) uint8_t image[34 * D];
  const Segment s = segment_of(p, D);
  if (!s.run) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (lane & 31) * E;
  const bool value = lane >= 32, all = s.hi - s.lo == kKvRun;
  const uint8_t* x = value ? p.v : p.k;
  uint8_t* to = all ? image : s.run;
  for (int m0 = s.lo + wave; m0 < s.hi; m0 += AHEAD * kRunWaves) {
    float f[AHEAD][E];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {   // past the last row: the last again
      const int m = min(m0 + u * kRunWaves, s.hi - 1);
      row_load<E>(x, s.b * p.ldb + m * p.ldm + s.h * p.ldh + c, p.type, p.vec, f[u]);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int m = m0 + u * kRunWaves, t = s.t0 + m - s.m0;
      if (m >= s.hi) break;
      float most = 0.0f;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        bad = bad || !(fabsf(f[u][i]) < INFINITY);
        most = fmaxf(most, fabsf(f[u][i]));
      }
#pragma unroll
      for (int w = 1; w < L; w <<= 1) most = fmaxf(most, __shfl_xor(most, w, 64));
      const bool nan = __any(bad);
      const int e = block_exp(most);
      const float scale = __uint_as_float((uint32_t)e << 23);
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const uint32_t w = nan ? 0u : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, f[u][i], f[u][i + 1], scale, 0);
        to[value ? kv_v_code<D>(t, c + i) : kv_k_code<D>(t, c + i)] = (uint8_t)w;
      }
      if ((lane & (L - 1)) == 0) to[value ? kv_v_exp<D>(t, c) : kv_k_exp<D>(t, c)] = (uint8_t)(nan ? (value ? kKvMinExp : kKvNan) : e);
    }
  }
  if (!all) return;
  __syncthreads();
  for (int i = threadIdx.x; i < 34 * D / 16; i += kRunThreads) ((uint4*)s.run)[i] = ((const uint4*)image)[i];
}

// The way back: several rows of a run from a copy of it in LDS, few straight from the page. Bound as above (16336 rows of 256
// f16 channels 8.5 to 9.4 us, 2.3 to 2.5 TB/s; LDS busy in 21% of the cycles, four fifths of that conflicts)
template <int D>
__global__ __launch_bounds__(kRunThreads) void kv_get_kernel(const RowsP p) {
  constexpr int E = D / 32;
  __shared__ __attribute__((aligned(16))) uint8_t image[34 * D];
  const Segment s = segment_of(p, D);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (lane & 31) * E;
  const bool value = lane >= 32, many = s.run && s.hi - s.lo >= 8;
  uint8_t* x = value ? p.v : p.k;
  const uint8_t* from = many ? image : s.run;
  if (many) {
    for (int i = threadIdx.x; i < 34 * D / 16; i += kRunThreads) ((uint4*)image)[i] = ((const uint4*)s.run)[i];
    __syncthreads();
  }
  for (int m = s.m0 + wave; m < s.m1; m += kRunWaves) {
    const int t = s.t0 + m - s.m0;
    float f[E];
    if (s.run && m < s.hi) {
      const float e = __uint_as_float((uint32_t)from[value ? kv_v_exp<D>(t, c) : kv_k_exp<D>(t, c)] << 23);
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(from[value ? kv_v_code<D>(t, c + i) : kv_k_code<D>(t, c + i)], e, 0);
        f[i] = v[0];
        f[i + 1] = v[1];
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = 0.0f;
    }
    row_store<E>(x, s.b * p.ldb + m * p.ldm + s.h * p.ldh + c, p.type, p.vec, f);
  }
}

static int rows_call(const char* op, const p0_kv_rows_args_t* a, bool put) {
  if (!a) { set_error("%s: no arguments", op); return P0_EINVAL; }
  RowsP p{};
  if (int r = kv_check(op, a->kv, a->B, &p.kv)) return r;
  if (a->M < 0 || a->M > (1 << 24)) { set_error("%s: M %lld", op, (long long)a->M); return P0_EINVAL; }
  if (a->type < P0_KV_F32 || a->type > P0_KV_BF16) { set_error("%s: type %d", op, (int)a->type); return P0_EINVAL; }
  if (!a->k || !a->v) { set_error("%s: missing k or v buffer", op); return P0_EINVAL; }
  const int size = a->type == P0_KV_F32 ? 4 : 2;
  if ((uintptr_t)a->k % size || (uintptr_t)a->v % size) { set_error("%s: k or v is not aligned to its type", op); return P0_EINVAL; }
  if (a->B * a->kv.heads > 65535) { set_error("%s: %lld sequences of %d heads", op, (long long)a->B, (int)a->kv.heads); return P0_EINVAL; }
  if (int r = refuse_in_chain(op)) return r;
  if (int r = require_open(op)) return r;
  if (a->B == 0 || a->M == 0) return P0_OK;
  p.rows = a->rows;
  p.at = a->at;
  p.k = (uint8_t*)a->k;
  p.v = (uint8_t*)a->v;
  p.ldh = a->ldh ? a->ldh : a->kv.dim;
  p.ldm = a->ldm ? a->ldm : a->kv.heads * p.ldh;
  p.ldb = a->ldb ? a->ldb : a->M * p.ldm;
  p.M = (int)a->M;
  p.type = a->type;
  const int D = a->kv.dim, unit = D / 32 * size < 16 ? D / 32 * size : 16;   // a lane's channels
  p.vec = (((uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)(p.ldh * size) | (uintptr_t)(p.ldm * size) | (uintptr_t)(p.ldb * size)) & (unit - 1)) == 0;
  const int64_t y = a->B * a->kv.heads;
  auto k = put ? (D == 64 ? kv_put_kernel<64> : D == 128 ? kv_put_kernel<128> : D == 256 ? kv_put_kernel<256> : kv_put_kernel<512>)
               : (D == 64 ? kv_get_kernel<64> : D == 128 ? kv_get_kernel<128> : D == 256 ? kv_get_kernel<256> : kv_get_kernel<512>);
  // M rows from any token on lie in at most this many runs
  hipLaunchKernelGGL(k, dim3((unsigned)((a->M + kKvRun - 2) / kKvRun + 1), (unsigned)y), dim3(kRunThreads), 0, ctx().cur, p);
  P0_LAUNCHED(op);
  return P0_OK;
}

}  // namespace p0

using namespace p0;

extern "C" int64_t p0_kv_page_bytes(int32_t page, int32_t heads, int32_t dim) {
  if (page < 32 || page > 1024 || (page & (page - 1)) || heads < 1 || heads > 1024) return 0;
  if (dim != 64 && dim != 128 && dim != 256 && dim != 512) return 0;
  return (int64_t)heads * (page / kKvRun) * 34 * dim;
}
extern "C" int p0_kv_put(const p0_kv_rows_args_t* a) { return rows_call("kv_put", a, true); }
extern "C" int p0_kv_get(const p0_kv_rows_args_t* a) { return rows_call("kv_get", a, false); }
