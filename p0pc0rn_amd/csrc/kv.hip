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
  if (kv.page_bytes && (kv.page_bytes < bytes || kv.page_bytes % 16)) {
    set_error("%s: page_bytes %lld (a page is %lld)", op, (long long)kv.page_bytes, (long long)bytes); return P0_EINVAL;
  }
  if (!kv.pages || !kv.table || !kv.len) { set_error("%s: missing pages, table or len buffer", op); return P0_EINVAL; }
  if ((uintptr_t)kv.pages % 16) { set_error("%s: pages must be 16-byte aligned", op); return P0_EINVAL; }
  if (kv.cols < 1 || kv.cols * kv.page > (1ll << 31) - 64 || (kv.table_ld && kv.table_ld < kv.cols)) {
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
  int M, type;
};

// the run and token of row m of sequence b, head h; null where there is none
__device__ __forceinline__ uint8_t* kv_run(const RowsP& p, int D, int64_t b, int m, int h, int* t) {
  const int len = kv_len(p.kv, b), n = kv_rows(p.rows, b, p.M);
  if (m >= n) return nullptr;
  const int64_t pos = (p.at ? (int64_t)p.at[b] : (int64_t)len - n) + m;
  if (pos < 0 || pos >= len) return nullptr;
  const int pg = kv_page(p.kv, b, (int)(pos >> p.kv.page_log));
  if (pg < 0) return nullptr;
  const int in = (int)(pos & ((1 << p.kv.page_log) - 1)), runs = 1 << (p.kv.page_log - 5);
  *t = in & 31;
  return p.kv.pages + pg * p.kv.page_bytes + ((int64_t)h * runs + (in >> 5)) * (34 * D);
}

__device__ __forceinline__ float row_load(const uint8_t* x, int64_t i, int type) {
  if (type == P0_KV_F32) return ((const float*)x)[i];
  if (type == P0_KV_F16) return (float)((const _Float16*)x)[i];
  return __uint_as_float((uint32_t)((const uint16_t*)x)[i] << 16);
}
__device__ __forceinline__ void row_store(uint8_t* x, int64_t i, int type, float v) {   // every value is exact in every type
  if (type == P0_KV_F32) ((float*)x)[i] = v;
  else if (type == P0_KV_F16) ((_Float16*)x)[i] = (_Float16)v;
  else ((uint16_t*)x)[i] = (uint16_t)(__float_as_uint(v) >> 16);
}

// the exponent byte of a block whose largest magnitude is `most`: the least e with most <= 6 * 2^e, that is the exponent
// field less 2, one more where the mantissa is over 1.5
__device__ __forceinline__ int block_exp(float most) {
  const int e = (int)((__float_as_uint(most) + 0x3FFFFFu) >> 23) - 2;
  return e < kKvMinExp ? kKvMinExp : e > kKvMaxExp ? kKvMaxExp : e;
}

// A wave takes one row of one head: lanes 0-31 the key, 32-63 the value, D / 32 consecutive channels each.
template <int D>
__global__ __launch_bounds__(256) void kv_put_kernel(const RowsP p, int64_t n) {
  constexpr int E = D / 32, L = 32 / E;   // channels a lane, lanes a block
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= n) return;
  const int h = (int)(row % p.kv.heads), m = (int)(row / p.kv.heads % p.M);
  const int64_t b = row / p.kv.heads / p.M;
  int t;
  uint8_t* run = kv_run(p, D, b, m, h, &t);
  if (!run) return;
  const bool value = lane >= 32;
  const int c = (lane & 31) * E;
  const uint8_t* x = value ? p.v : p.k;
  float f[E], most = 0.0f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    f[i] = row_load(x, b * p.ldb + m * p.ldm + h * p.ldh + c + i, p.type);
    bad = bad || !(fabsf(f[i]) < INFINITY);
    most = fmaxf(most, fabsf(f[i]));
  }
#pragma unroll
  for (int s = 1; s < L; s <<= 1) most = fmaxf(most, __shfl_xor(most, s, 64));
  const bool nan = __any(bad);
  const int e = block_exp(most);
  const float scale = __uint_as_float((uint32_t)e << 23);
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    const uint32_t w = nan ? 0u : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, f[i], f[i + 1], scale, 0);
    run[value ? kv_v_code<D>(t, c + i) : kv_k_code<D>(t, c + i)] = (uint8_t)w;
  }
  if ((lane & (L - 1)) == 0) run[value ? kv_v_exp<D>(t, c) : kv_k_exp<D>(t, c)] = nan ? (value ? kKvMinExp : kKvNan) : e;
}

template <int D>
__global__ __launch_bounds__(256) void kv_get_kernel(const RowsP p, int64_t n) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= n) return;
  const int h = (int)(row % p.kv.heads), m = (int)(row / p.kv.heads % p.M);
  const int64_t b = row / p.kv.heads / p.M;
  int t = 0;
  const uint8_t* run = kv_run(p, D, b, m, h, &t);
  const bool value = lane >= 32;
  const int c = (lane & 31) * E;
  uint8_t* x = value ? p.v : p.k;
  const float e = run ? __uint_as_float((uint32_t)run[value ? kv_v_exp<D>(t, c) : kv_k_exp<D>(t, c)] << 23) : 0.0f;
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    const uint32_t w = run ? run[value ? kv_v_code<D>(t, c + i) : kv_k_code<D>(t, c + i)] : 0u;
    const auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, e, 0);
    const int64_t at = b * p.ldb + m * p.ldm + h * p.ldh + c + i;
    row_store(x, at, p.type, run ? v[0] : 0.0f);
    row_store(x, at + 1, p.type, run ? v[1] : 0.0f);
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
  const int64_t n = a->B * a->M * a->kv.heads, blocks = (n + 3) / 4;
  if (blocks > 0x7FFFFFFF) { set_error("%s: %lld rows", op, (long long)n); return P0_EINVAL; }
  const int D = a->kv.dim;
  auto k = put ? (D == 64 ? kv_put_kernel<64> : D == 128 ? kv_put_kernel<128> : D == 256 ? kv_put_kernel<256> : kv_put_kernel<512>)
               : (D == 64 ? kv_get_kernel<64> : D == 128 ? kv_get_kernel<128> : D == 256 ? kv_get_kernel<256> : kv_get_kernel<512>);
  hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(256), 0, ctx().cur, p, n);
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
