// f8_gemm.hip - the product of e4m3 activations and weights with a scale per block of 128 (include/p0pc0rn.h):
//   y[m][n] = sum_kb xs[kb][m] ws[n / 128][kb] sum_{k in kb} x[m][k] w[n][k]
//
// The weight's rows are the matrix instruction's rows, the activations' its columns: a lane then holds 4 consecutive outputs of one
// activation row, whose scale is one value of the lane. A block's sum comes out of the matrix instructions in fp32, and one fma a
// value adds it, times the block's two scales, to the running sum.
//
// Two arithmetics. v_mfma_f32_16x16x128_f8f6f4 takes a whole block of k, at twice the fp16 rate, but adds the products of each 8
// consecutive k in the alignment of their largest, cutting them off 13 bits below its leading one (measured, as for the older
// 16x16x32 fp8 instruction; the sums of 8 then meet in fp32): a result is off by 2e-5 to 1e-4 of itself, nothing beside the rounding to
// 16 bits, but over fp32's. So fp32 results are taken on v_mfma_f32_16x16x32_f16, which keeps products and sums in fp32 (every e4m3
// value is an fp16 value), at half the rate; so are few rows in every type, where the weights' bytes bound the call.
//
// Both operands' k may come in any order that is the same for both: lane group g (16 lanes) holds bytes [16 g, 16 g + 16) and
// [64 + 16 g, 80 + 16 g) of a block.
#include "dma.hpp"
#include "f8_common.hpp"

namespace p0 {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct F8GemmP {
  const uint8_t* x;
  const float* xs;
  const uint8_t* w;
  const float* ws;
  void* y;
  int64_t ldx, ldxs, ldw, ldws, ldy;
  int M, N, blocks;    // blocks of 128 k
  int nt;              // tiles of N
  int yvec;            // 4 consecutive outputs from a multiple of 4 on are aligned together
};

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));

// a lane's 32 codes of a block -> 32 fp16 values, exactly
__device__ __forceinline__ void to_half(const uint4& c0, const uint4& c1, half8v (&h)[4]) {
  const uint32_t w[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const half2v lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[2 * i + j], 1.0f, false);
      const half2v hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[2 * i + j], 1.0f, true);
      h[i][4 * j] = lo.x; h[i][4 * j + 1] = lo.y; h[i][4 * j + 2] = hi.x; h[i][4 * j + 3] = hi.y;
    }
}
__device__ __forceinline__ f32x4 mfma_half(const half8v (&a)[4], const half8v (&b)[4]) {
  f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], b[i], d, 0, 0, 0);
  return d;
}
__device__ __forceinline__ f32x4 mfma_block(const uint4& w0, const uint4& w1, const uint4& x0, const uint4& x1) {
  const i32x8 a = {(int)w0.x, (int)w0.y, (int)w0.z, (int)w0.w, (int)w1.x, (int)w1.y, (int)w1.z, (int)w1.w};
  const i32x8 b = {(int)x0.x, (int)x0.y, (int)x0.z, (int)x0.w, (int)x1.x, (int)x1.y, (int)x1.z, (int)x1.w};
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0, 0, 0, 0);   // e4m3 both, no block scales of its own
}

// outputs n .. n + 3 of row m
template <int TYPE> __device__ __forceinline__ void store4(const F8GemmP& p, int m, int n, const f32x4& v) {
  const int64_t o = (int64_t)m * p.ldy + n;
  if constexpr (TYPE == P0_F32) {
    float* y = (float*)p.y + o;
    if (p.yvec && n + 4 <= p.N) *(float4*)y = float4{v[0], v[1], v[2], v[3]};
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) y[i] = v[i];
  } else {
    uint16_t* y = (uint16_t*)p.y + o;
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = f8_half<TYPE>(v[i]);
    if (p.yvec && n + 4 <= p.N) *(uint2*)y = uint2{h[0] | h[1] << 16, h[2] | h[3] << 16};
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) y[i] = (uint16_t)h[i];
  }
}

// Few rows: a workgroup takes 16 outputs of 16 rows, its waves the blocks of k in turn; their sums meet in LDS.
constexpr int kThinWaves = 4;
template <int TYPE>
__global__ __launch_bounds__(64 * kThinWaves) void f8_thin_kernel(const F8GemmP p) {
  __shared__ f32x4 part[kThinWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
  const int mt = blockIdx.x / (unsigned)p.nt, n0 = (blockIdx.x - mt * p.nt) * 16, m0 = mt * 16;
  const int n = min(n0 + (lane & 15), p.N - 1), m = min(m0 + (lane & 15), p.M - 1);   // rows past the last: it again
  const uint8_t* w = p.w + n * p.ldw + g * 16;
  const uint8_t* x = p.x + m * p.ldx + g * 16;
  const float* ws = p.ws + (int64_t)(n0 >> 7) * p.ldws;
  const float* xs = p.xs + m;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int U = 4;
  for (int kb = wave; kb < p.blocks; kb += U * kThinWaves) {
    uint4 a[U][2], b[U][2];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {   // past the last block: it again, times 0
      const int k = min(kb + u * kThinWaves, p.blocks - 1);
      a[u][0] = *(const uint4*)(w + (int64_t)k * 128);
      a[u][1] = *(const uint4*)(w + (int64_t)k * 128 + 64);
      b[u][0] = *(const uint4*)(x + (int64_t)k * 128);
      b[u][1] = *(const uint4*)(x + (int64_t)k * 128 + 64);
      s[u] = xs[k * p.ldxs] * ws[k];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kb + u * kThinWaves >= p.blocks) break;
      half8v ah[4], bh[4];
      to_half(a[u][0], a[u][1], ah);
      to_half(b[u][0], b[u][1], bh);
      const f32x4 d = mfma_half(ah, bh);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(d[i], s[u], acc[i]);
    }
  }
  part[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int k = 1; k < kThinWaves; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += part[k][lane][i];
  if (m0 + (lane & 15) < p.M) store4<TYPE>(p, m0 + (lane & 15), n0 + 4 * g, acc);
}

static int gemm_f8_call(const p0_f8_gemm_args_t* a) {
  const char* op = "f8_gemm";
  if (!a) { set_error("%s: no arguments", op); return P0_EINVAL; }
  if (!f8_type(a->type)) { set_error("%s: type %d", op, (int)a->type); return P0_EINVAL; }
  if (a->M < 0 || a->M > (1 << 30)) { set_error("%s: M %lld", op, (long long)a->M); return P0_EINVAL; }
  if (a->N < 0 || a->N > (1 << 30)) { set_error("%s: N %lld", op, (long long)a->N); return P0_EINVAL; }
  if (a->K < 128 || a->K % 128 || a->K > (1 << 20)) { set_error("%s: K %lld must be a multiple of 128", op, (long long)a->K); return P0_EINVAL; }
  if (a->M == 0 || a->N == 0) { if (int r = refuse_in_chain(op)) return r; return require_open(op); }
  const int size = f8_size(a->type);
  const int64_t M = a->M, N = a->N, K = a->K, blocks = K / 128, nb = f8_blocks(N);
  const int64_t ldx = a->ldx ? a->ldx : K, ldw = a->ldw ? a->ldw : K, ldxs = a->ldxs ? a->ldxs : M, ldws = a->ldws ? a->ldws : blocks,
                ldy = a->ldy ? a->ldy : N;
  if (ldx > (1 << 22) || ldw > (1 << 22)) { set_error("%s: rows %lld and %lld B apart", op, (long long)ldx, (long long)ldw); return P0_EINVAL; }
  const Span x = f8_span(a->x, M, K, ldx, 1), w = f8_span(a->w, N, K, ldw, 1), xs = f8_span(a->xs, blocks, M, ldxs, 4),
             ws = f8_span(a->ws, nb, blocks, ldws, 4), y = f8_span(a->y, M, N, ldy, size);
  if (int r = f8_check(op, "x", x, 16)) return r;
  if (int r = f8_check(op, "w", w, 16)) return r;
  if (int r = f8_check(op, "xs", xs, 4)) return r;
  if (int r = f8_check(op, "ws", ws, 4)) return r;
  if (int r = f8_check(op, "y", y, size)) return r;
  if (overlap(x, y) || overlap(w, y) || overlap(xs, y) || overlap(ws, y)) { set_error("%s: y overlaps an input", op); return P0_EINVAL; }
  const int64_t tiles = (N + 15) / 16 * ((M + 15) / 16);
  if (tiles >= (1ll << 31)) { set_error("%s: %lld x %lld outputs", op, (long long)M, (long long)N); return P0_EINVAL; }
  if (int r = refuse_in_chain(op)) return r;
  if (int r = require_open(op)) return r;
  F8GemmP p{(const uint8_t*)a->x, a->xs, (const uint8_t*)a->w, a->ws, a->y, ldx, ldxs, ldw, ldws, ldy, (int)M, (int)N, (int)blocks};
  p.nt = (int)((N + 15) / 16);
  p.yvec = ((uintptr_t)a->y | (uintptr_t)(ldy * size)) % (4 * size) == 0;
  auto k = a->type == P0_F32 ? f8_thin_kernel<P0_F32> : a->type == P0_F16 ? f8_thin_kernel<P0_F16> : f8_thin_kernel<P0_BF16>;
  hipLaunchKernelGGL(k, dim3((unsigned)tiles), dim3(64 * kThinWaves), 0, ctx().cur, p);
  P0_LAUNCHED(op);
  return P0_OK;
}

}  // namespace p0

extern "C" int p0_f8_gemm(const p0_f8_gemm_args_t* a) { return p0::gemm_f8_call(a); }
