// f8_rows.hip - values into e4m3 codes with a scale per block of 128: weights (f8_pack), the residual stream's update and norm
// (f8_norm), activations and gated ones (f8_rows).
//
// A lane holds 8 consecutive channels, 16 lanes a block: its largest magnitude is 4 lane moves away. All three read their
// input once into registers and write codes from there.
#include "f8_common.hpp"

namespace p0 {

// ------------------------------------------------------------------------------------------------ weights
struct PackP {
  const void* x;
  uint8_t* w;
  float* s;
  int64_t ldx, ldw, lds;
  int64_t N, K;
  int blocks;   // of 128 channels in a row
};
// A workgroup takes a block of 128 x 128, a thread 8 rows of 8 channels: 8 loads of 16 bytes on their way at once.
// Bound: HBM (18432 x 9216 bf16 values: 94.4 us for 510 MB, 5.4 TB/s; a copy of as many bytes 95); launch and round trips for small ones (1536 x
// 2048 f16 values, 192 workgroups: 4.9 us).
template <int TYPE>
__global__ __launch_bounds__(256) void f8_pack_kernel(const PackP p) {
  __shared__ float red[4];
  const int64_t blk = f8_group(), nb = blk / p.blocks;
  if (nb * 128 >= p.N) return;
  const int kb = (int)(blk - nb * p.blocks), c = kb * 128 + (threadIdx.x & 15) * 8, lane = threadIdx.x & 63;
  const int64_t n0 = nb * 128 + (threadIdx.x >> 4);
  const int n = (int)(p.K - c < 8 ? (p.K - c < 0 ? 0 : p.K - c) : 8);
  F8Raw<TYPE> raw[8];
  float f[8][8], most = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t r = n0 + 16 * j;
    if (r < p.N && n > 0) f8_fetch8<TYPE>(p.x, r * p.ldx + c, c, n, raw[j]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t r = n0 + 16 * j;
    if (r < p.N && n > 0) f8_take8<TYPE>(raw[j], p.x, r * p.ldx + c, n, c, n, f[j]);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) f[j][i] = 0.0f;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) most = fmaxf(most, f8_most_finite(f[j]));
  most = f8_max16(most);
  most = fmaxf(most, __shfl_xor(most, 16, 64));
  most = fmaxf(most, __shfl_xor(most, 32, 64));
  if (lane == 0) red[threadIdx.x >> 6] = most;
  __syncthreads();
  most = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float s = f8_scale(most), inv = f8_inverse(s);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t r = n0 + 16 * j;
    if (r < p.N) *(uint2*)(p.w + r * p.ldw + c) = f8_codes(f[j], inv);
  }
  if (threadIdx.x == 0) p.s[nb * p.lds + kb] = s;
}

// ------------------------------------------------------------------------------------------------ activations
// g u sigmoid(z), z = g (silu), or 2 sqrt(2 / pi) (g + 0.044715 g^3) (gelu: 0.5 g (1 + tanh(z / 2))), within 8 units of 2^-24. An error of z is one of exp(-z) z times
// as large, so what its products and constants round off is kept (c) and put back: without, 9 units at z = -20 and 21 at -80 (silu), 46 at g = -5 and 129 at -8 (gelu).
// A sigmoid below the least normal value (z < -87.3) is 0. A NaN gate is one in g.
template <int TYPE> __device__ __forceinline__ float gated(int glu, float g, float u) {
#pragma clang fp contract(off)
  constexpr float Ln = 0.69314718056f;
  float t, c;   // |z| log2 e = t + c
  if (glu == P0_GLU_SILU) {
    constexpr float L = 1.4426950409f, Ll = 1.925963e-8f;   // log2 e = L + Ll
    const float z = fminf(fabsf(g), 200.0f);
    t = z * L;
    c = __builtin_fmaf(z, Ll, __builtin_fmaf(z, L, -t));
  } else {
    constexpr float L = 2.3022082f, Ll = 1.2948402e-8f, K = 0.044715f, Kl = 1.5461444e-9f;   // 2 sqrt(2 / pi) log2 e = L + Ll, 0.044715 = K + Kl
    const float x = fminf(fabsf(g), 16.0f), xx = x * x, p = __builtin_fmaf(xx, K, 1.0f), z = x * p;   // times 2 sqrt(2 / pi): |z|
    float pe = __builtin_fmaf(xx, Kl, __builtin_fmaf(xx, K, 1.0f - p));
    if constexpr (TYPE == P0_F32) pe = __builtin_fmaf(__builtin_fmaf(x, x, -xx), K, pe);   // squares of 16-bit values are exact
    t = z * L;
    c = __builtin_fmaf(__builtin_fmaf(x, pe, __builtin_fmaf(x, p, -z)), L, __builtin_fmaf(z, Ll, __builtin_fmaf(z, L, -t)));
  }
  const float e = __builtin_amdgcn_exp2f(-t), E = __builtin_fmaf(e, c * -Ln, e), d = 1.0f + E;   // exp(-|z|)
  const float r = __builtin_amdgcn_rcpf(d), q = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
  return g * (g < 0.0f ? E : 1.0f) * q * u;
}
struct RowsF8P {
  const void* x;
  uint8_t* y;
  float* s;
  int64_t ldx, up, ldy, lds;
  int64_t M, D;
  int strips, ls;   // 1 << ls lanes side by side take a strip of 8 << ls channels of a row
  int glu;
};
// A workgroup takes a strip of 256 >> ls rows.
// Bound: HBM (4608 rows of 9216 f16 channels: 24 us for 128 MB, 5.3 TB/s), gated ones nearly as much the arithmetic: silu 42-43 us, gelu 46-48 for 214 MB, 4.5-5 TB/s (a copy of as
// many bytes 41). Few rows are a launch (5 of 8192 fp32 channels, gated: 4.9 us).
// Two rows a thread took 4% longer, four 13%: the other waves cover a wave's loads better than its own.
template <int TYPE, bool GLU>
__global__ __launch_bounds__(256) void f8_rows_kernel(const RowsF8P p) {
  const int64_t blk = f8_group(), rblk = blk / p.strips;
  const int side = 256 >> p.ls, c = (((int)(blk - rblk * p.strips) << p.ls) + (threadIdx.x & ((1 << p.ls) - 1))) * 8;
  const int64_t m = rblk * side + (threadIdx.x >> p.ls);
  if (c >= (int)((p.D + 127) / 128 * 128) || m >= p.M) return;   // whole blocks of lanes
  const int n = (int)(p.D - c < 8 ? (p.D - c < 0 ? 0 : p.D - c) : 8);
  float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (n > 0) {
    F8Raw<TYPE> gate, up;
    f8_fetch8<TYPE>(p.x, m * p.ldx + c, c, n, gate);
    if constexpr (GLU) f8_fetch8<TYPE>(p.x, m * p.ldx + p.up + c, c, n, up);
    f8_take8<TYPE>(gate, p.x, m * p.ldx + c, n, c, n, f);
    if constexpr (GLU) {
      float u[8];
      f8_take8<TYPE>(up, p.x, m * p.ldx + p.up + c, n, c, n, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = gated<TYPE>(p.glu, f[j], u[j]);
    }
  }
  const float s = f8_scale(f8_block_most(f));
  *(uint2*)(p.y + m * p.ldy + c) = f8_codes(f, f8_inverse(s));
  if ((threadIdx.x & 15) == 0) p.s[(int64_t)(c >> 7) * p.lds + m] = s;
}

// ------------------------------------------------------------------------------------------------ the stream's norm
struct NormP {
  const void* x;
  const void* t;
  void* xo;          // null: the sum is not stored
  const float* tw;
  const float* w;
  const float* b;
  uint8_t* y;
  float* s;
  int64_t ldx, ldt, ldo, ldy, lds;
  int64_t M;
  int D, mode, one;
  float scale, eps;
};
__device__ __forceinline__ float sum64(float v) {
  v += f8_dpp<0x128>(v);
  v += f8_dpp<0x124>(v);
  v += f8_dpp<0x122>(v);
  v += f8_dpp<0x121>(v);
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
// A workgroup takes a row, its up to 16 waves 512 channels each of NC steps, a lane 8 of them. The row stays in registers; each sum is one
// exchange through LDS.
// VEC: every run of 8 channels is there whole or not at all.
// Bound: HBM at many rows (32760 rows of 2560 bf16 channels, modulated: 117-120 us for 590 MB, 4.9-5.0 TB/s; a copy of as many bytes 114),
// launch and round trips at few (1 row of 2048 fp32 channels: 2.9 us, 5.5 with the host's part). Rows whose last run of 8 is not whole take a third more: every
// wave carries the counts and the moves of the odd end (us, 644 rows of 14425 bf16 channels 21.0, of 14424 15.4; 908 of 13303 with the norm of t 33.7, of 13304
// 25.6; in single channels 644 of 14425 took 84). A wave with a row of its own, four in a workgroup, took 136 and 3.7: five loads a lane at a time and their
// registers leave fewer waves to cover them.
template <int XT, int TT, int NC, bool VEC>
__global__ __launch_bounds__(1024) void f8_norm_kernel(const NormP p) {
  __shared__ float red[3][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, W = blockDim.x >> 6;
  const int64_t m = f8_group();
  if (m >= p.M) return;
  const int c0 = (wave * 64 + lane) * 8;
  auto total = [&](float v, int slot) {
    v = sum64(v);
    if (W == 1) return v;
    if (lane == 0) red[slot][wave] = v;
    __syncthreads();
    v = red[slot][0];
    for (int i = 1; i < W; ++i) v += red[slot][i];
    return v;
  };
  auto count = [&](int c) { return VEC ? 8 : p.D - c < 8 ? p.D - c : 8; };   // of the 8 channels from c < D on
  auto fill = [&](float (&v)[8], float x) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = x;
  };
  float f[NC][8];
  F8Raw<XT> xr[NC];
  F8Raw<TT> tr[NC];
  const float over = 1.0f / (float)p.D;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = c0 + i * 512 * W;
    if (c < p.D) f8_fetch8<XT>(p.x, m * p.ldx + c, c, count(c), xr[i]);
    if (p.t && c < p.D) f8_fetch8<TT>(p.t, m * p.ldt + c, c, count(c), tr[i]);
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = c0 + i * 512 * W;
    fill(f[i], 0.0f);
    if (c < p.D) f8_take8<XT>(xr[i], p.x, m * p.ldx + c, count(c), c, count(c), f[i]);
  }
  if (p.t) {
    float t[NC][8], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = c0 + i * 512 * W;
      fill(t[i], 0.0f);
      if (c < p.D) f8_take8<TT>(tr[i], p.t, m * p.ldt + c, count(c), c, count(c), t[i]);
    }
    if (p.tw) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(t[i][j], t[i][j], ss);
      const float r = 1.0f / sqrtf(total(ss, 0) * over + p.eps);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = c0 + i * 512 * W;
        if (c >= p.D) continue;
        float g[8];
        f8_load8<P0_F32>(p.tw, c, count(c), c, count(c), g);
#pragma unroll
        for (int j = 0; j < 8; ++j) t[i][j] *= r * g[j];
      }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i][j] += t[i][j];
  }
  float sum = 0.0f, sq = 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[i][j] = f8_rounded<XT>(f[i][j] * p.scale);
      sum += f[i][j];
    }
    const int c = c0 + i * 512 * W;
    if (p.xo && c < p.D) f8_store8<XT>(p.xo, m * p.ldo + c, VEC || count(c) == 8, count(c), f[i]);
  }
  const float mean = p.mode == 0 ? total(sum, 1) * over : 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = c0 + i * 512 * W;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[i][j] = (VEC ? c : c + j) < p.D ? f[i][j] - mean : 0.0f;
      sq = __builtin_fmaf(f[i][j], f[i][j], sq);
    }
  }
  const float rstd = 1.0f / sqrtf(total(sq, 2) * over + p.eps);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = c0 + i * 512 * W;
    if (c >= (p.D + 127) / 128 * 128) break;   // whole blocks of lanes
    if (c < p.D) {
      float g[8], b[8];
      if (p.w) f8_load8<P0_F32>(p.w, c, count(c), c, count(c), g);
      else fill(g, p.one ? 0.0f : 1.0f);
      if (p.b) f8_load8<P0_F32>(p.b, c, count(c), c, count(c), b);
      else fill(b, 0.0f);
      const float one = p.one ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i][j] = VEC || c + j < p.D ? f[i][j] * rstd * (g[j] + one) + b[j] : 0.0f;
    }
    const float s = f8_scale(f8_block_most(f[i]));
    *(uint2*)(p.y + m * p.ldy + c) = f8_codes(f[i], f8_inverse(s));
    if ((lane & 15) == 0) p.s[(int64_t)(c >> 7) * p.lds + m] = s;
  }
}

// ------------------------------------------------------------------------------------------------ the calls
static int refuse(const char* op) {
  if (int r = refuse_in_chain(op)) return r;
  return require_open(op);
}
static int rows_count(const char* op, const char* name, int64_t M) {
  if (M < 0 || M > kF8MaxRows) { set_error("%s: %s %lld", op, name, (long long)M); return P0_EINVAL; }
  return P0_OK;
}

static int pack_call(const p0_f8_pack_args_t* a) {
  const char* op = "f8_pack";
  if (!a) { set_error("%s: no arguments", op); return P0_EINVAL; }
  if (!f8_type(a->type)) { set_error("%s: type %d", op, (int)a->type); return P0_EINVAL; }
  if (int r = rows_count(op, "N", a->N)) return r;
  if (a->K < 1 || a->K > (1 << 20)) { set_error("%s: K %lld", op, (long long)a->K); return P0_EINVAL; }
  if (a->N == 0) return refuse(op);
  const int size = f8_size(a->type);
  const int64_t blocks = f8_blocks(a->K), K8 = blocks * 128, ldx = a->ldx ? a->ldx : a->K, ldw = a->ldw ? a->ldw : K8,
                lds = a->lds ? a->lds : blocks;
  const Span x = f8_span(a->x, a->N, a->K, ldx, size), w = f8_span(a->w, a->N, K8, ldw, 1), s = f8_span(a->s, f8_blocks(a->N), blocks, lds, 4);
  if (int r = f8_check(op, "x", x, size)) return r;
  if (int r = f8_check(op, "w", w, 16)) return r;
  if (int r = f8_check(op, "s", s, 4)) return r;
  if (overlap(x, w) || overlap(x, s) || overlap(w, s)) { set_error("%s: outputs overlap", op); return P0_EINVAL; }
  dim3 grid;
  if (!f8_grid(f8_blocks(a->N) * blocks, 256, &grid)) { set_error("%s: %lld x %lld values", op, (long long)a->N, (long long)a->K); return P0_EINVAL; }
  if (int r = refuse(op)) return r;
  PackP p{a->x, (uint8_t*)a->w, a->s, ldx, ldw, lds, a->N, a->K, (int)blocks};
  auto k = a->type == P0_F32 ? f8_pack_kernel<P0_F32> : a->type == P0_F16 ? f8_pack_kernel<P0_F16> : f8_pack_kernel<P0_BF16>;
  hipLaunchKernelGGL(k, grid, dim3(256), 0, ctx().cur, p);
  P0_LAUNCHED(op);
  return P0_OK;
}

static auto rows_kernel(int type, bool glu) {
  return type == P0_F32 ? (glu ? f8_rows_kernel<P0_F32, true> : f8_rows_kernel<P0_F32, false>)
       : type == P0_F16 ? (glu ? f8_rows_kernel<P0_F16, true> : f8_rows_kernel<P0_F16, false>)
                        : (glu ? f8_rows_kernel<P0_BF16, true> : f8_rows_kernel<P0_BF16, false>);
}

static int rows_f8_call(const p0_f8_rows_args_t* a) {
  const char* op = "f8_rows";
  if (!a) { set_error("%s: no arguments", op); return P0_EINVAL; }
  if (!f8_type(a->type)) { set_error("%s: type %d", op, (int)a->type); return P0_EINVAL; }
  if (a->glu < P0_GLU_NONE || a->glu > P0_GLU_GELU) { set_error("%s: glu %d", op, (int)a->glu); return P0_EINVAL; }
  if (int r = rows_count(op, "M", a->M)) return r;
  if (a->D < 1 || a->D > (1 << 20)) { set_error("%s: D %lld", op, (long long)a->D); return P0_EINVAL; }
  const bool glu = a->glu != P0_GLU_NONE;
  const int size = f8_size(a->type);
  const int64_t up = !glu ? 0 : a->up ? a->up : a->D;
  if (up < 0 || up > (1ll << 31)) { set_error("%s: up %lld", op, (long long)a->up); return P0_EINVAL; }
  if (a->M == 0) return refuse(op);
  const int64_t blocks = f8_blocks(a->D), K8 = blocks * 128, ldx = a->ldx ? a->ldx : up + a->D, ldy = a->ldy ? a->ldy : K8,
                lds = a->lds ? a->lds : a->M;
  const Span x = f8_span(a->x, a->M, up + a->D, ldx, size), y = f8_span(a->y, a->M, K8, ldy, 1), s = f8_span(a->s, blocks, a->M, lds, 4);
  if (int r = f8_check(op, "x", x, size)) return r;
  if (int r = f8_check(op, "y", y, 16)) return r;
  if (int r = f8_check(op, "s", s, 4)) return r;
  if (overlap(x, y) || overlap(x, s) || overlap(y, s)) { set_error("%s: outputs overlap", op); return P0_EINVAL; }
  if (int r = refuse(op)) return r;
  RowsF8P p{a->x, (uint8_t*)a->y, a->s, ldx, up, ldy, lds, a->M, a->D, 0, 7, a->glu};
  // strips of up to 128 lanes that leave no more than an eighth idle (us, strips of 16 lanes / of 128, f16: 20000 rows of 520 channels 8.9 / 9.6, gated by
  // silu 14.1 / 17.9; 4608 of 9216 26.9 / 26.3, gated 41.2 / 42.7)
  const int64_t chunks = K8 / 8;
  while (p.ls > 4 && ((chunks + (1 << p.ls) - 1) >> p.ls << p.ls) - chunks > chunks / 8) --p.ls;
  p.strips = (int)((chunks + (1 << p.ls) - 1) >> p.ls);
  dim3 grid;
  if (!f8_grid((a->M + (256 >> p.ls) - 1) / (256 >> p.ls) * p.strips, 256, &grid)) { set_error("%s: %lld rows of %lld", op, (long long)a->M, (long long)a->D); return P0_EINVAL; }
  hipLaunchKernelGGL(rows_kernel(a->type, glu), grid, dim3(256), 0, ctx().cur, p);
  P0_LAUNCHED(op);
  return P0_OK;
}

typedef void (*NormKernel)(NormP);
template <int XT, int TT> static NormKernel norm_kernel(bool vec, int NC) {
  if (!vec) return NC == 1 ? f8_norm_kernel<XT, TT, 1, false> : NC == 2 ? f8_norm_kernel<XT, TT, 2, false> : f8_norm_kernel<XT, TT, 4, false>;
  return NC == 1 ? f8_norm_kernel<XT, TT, 1, true> : NC == 2 ? f8_norm_kernel<XT, TT, 2, true> : f8_norm_kernel<XT, TT, 4, true>;
}

static int norm_call(const p0_f8_norm_args_t* a) {
  const char* op = "f8_norm";
  if (!a) { set_error("%s: no arguments", op); return P0_EINVAL; }
  if (!f8_type(a->type) || (a->t && !f8_type(a->t_type))) { set_error("%s: type %d, t_type %d", op, (int)a->type, (int)a->t_type); return P0_EINVAL; }
  if (a->mode != 0 && a->mode != 1) { set_error("%s: mode %d", op, (int)a->mode); return P0_EINVAL; }
  if (int r = rows_count(op, "M", a->M)) return r;
  if (a->D < 1 || a->D > 32768) { set_error("%s: D %lld (1 .. 32768)", op, (long long)a->D); return P0_EINVAL; }
  if (a->tw && !a->t) { set_error("%s: tw needs t", op); return P0_EINVAL; }
  if (a->M == 0) return refuse(op);
  const int xsize = f8_size(a->type), tsize = a->t ? f8_size(a->t_type) : 4;
  const int64_t M = a->M, D = a->D, blocks = f8_blocks(D), K8 = blocks * 128, ldx = a->ldx ? a->ldx : D, ldt = a->ldt ? a->ldt : D,
                ldo = a->x_out ? (a->ldo ? a->ldo : D) : ldx, ldy = a->ldy ? a->ldy : K8, lds = a->lds ? a->lds : M;
  const float scale = a->scale != 0.0f ? a->scale : 1.0f;
  void* xo = a->x_out ? a->x_out : a->t || scale != 1.0f ? a->x : nullptr;
  const Span x = f8_span(a->x, M, D, ldx, xsize), t = f8_span(a->t, M, D, ldt, tsize), o = f8_span(xo, M, D, ldo, xsize),
             y = f8_span(a->y, M, K8, ldy, 1), s = f8_span(a->s, blocks, M, lds, 4), tw{a->tw, 1, D * 4, D * 4}, w{a->w, 1, D * 4, D * 4},
             b{a->b, 1, D * 4, D * 4};
  if (int r = f8_check(op, "x", x, xsize)) return r;
  if (a->t) { if (int r = f8_check(op, "t", t, tsize)) return r; }
  if (xo) { if (int r = f8_check(op, "x_out", o, xsize)) return r; }
  if (int r = f8_check(op, "y", y, 16)) return r;
  if (int r = f8_check(op, "s", s, 4)) return r;
  if (((uintptr_t)a->tw | (uintptr_t)a->w | (uintptr_t)a->b) % 4) { set_error("%s: tw, w and b must be 4-byte aligned", op); return P0_EINVAL; }
  const bool same = xo == a->x && ldo == ldx;
  const Span* in[] = {&x, &t, &tw, &w, &b};
  for (const Span* i : in)
    if (overlap(*i, y) || overlap(*i, s) || (overlap(*i, o) && !(i == &x && same))) { set_error("%s: outputs overlap", op); return P0_EINVAL; }
  if (overlap(y, s) || overlap(o, y) || overlap(o, s)) { set_error("%s: outputs overlap", op); return P0_EINVAL; }
  if (int r = refuse(op)) return r;
  NormP p{};
  p.x = a->x; p.t = a->t; p.xo = xo; p.tw = a->tw; p.w = a->w; p.b = a->b; p.y = (uint8_t*)a->y; p.s = a->s;
  p.ldx = ldx; p.ldt = ldt; p.ldo = ldo; p.ldy = ldy; p.lds = lds; p.M = M; p.D = (int)D;
  const bool vec = D % 8 == 0;
  p.mode = a->mode; p.one = a->w_one ? 1 : 0; p.scale = scale; p.eps = a->eps != 0.0f ? a->eps : 1e-6f;
  // Waves of one step, but for two where rows are longer than 16 waves' one, and for 16-bit rows that fill the chip several times over (us,
  // one step / two: 32760 rows of 2560 bf16 channels 128 / 112, 4608 of 4096 28.9 / 27.4; 1021 of 1536 5.0 / 5.8; 4608 of 2048 fp32 channels
  // 23.8 / 25.6), and four for the longest
  const int steps = (int)((K8 + 511) / 512);
  const bool two = steps > 16 || (xsize == 2 && steps > 1 && M * steps >= 16384);
  const int NC = steps > 32 ? 4 : two ? 2 : 1, W = (steps + NC - 1) / NC;
  const int tt = a->t ? a->t_type : a->type;
  NormKernel k = nullptr;
#define P0_NORM(XT, TT) if (a->type == XT && tt == TT) k = norm_kernel<XT, TT>(vec, NC)
  P0_NORM(P0_F32, P0_F32); P0_NORM(P0_F32, P0_F16); P0_NORM(P0_F32, P0_BF16);
  P0_NORM(P0_F16, P0_F32); P0_NORM(P0_F16, P0_F16); P0_NORM(P0_F16, P0_BF16);
  P0_NORM(P0_BF16, P0_F32); P0_NORM(P0_BF16, P0_F16); P0_NORM(P0_BF16, P0_BF16);
#undef P0_NORM
  dim3 grid;
  if (!f8_grid(M, 64 * W, &grid)) { set_error("%s: M %lld", op, (long long)M); return P0_EINVAL; }
  hipLaunchKernelGGL(k, grid, dim3(64 * W), 0, ctx().cur, p);
  P0_LAUNCHED(op);
  return P0_OK;
}

}  // namespace p0

using namespace p0;

extern "C" int p0_f8_pack(const p0_f8_pack_args_t* a) { return pack_call(a); }
extern "C" int p0_f8_norm(const p0_f8_norm_args_t* a) { return norm_call(a); }
extern "C" int p0_f8_rows(const p0_f8_rows_args_t* a) { return rows_f8_call(a); }
