// f8_common.hpp - what the 8-bit operators and the rotation share (f8_rows.hip, f8_gemm.hip, rope.hip): e4m3 codes with a scale
// per block of 128 (include/p0pc0rn.h has the format), loads and stores of 8 values of a type, checks of arguments.
#pragma once
#include "common.hpp"

namespace p0 {

constexpr int kF8Block = 128;
constexpr int64_t kF8MaxRows = (1ll << 31) - 1;

// ---- arguments: `rows` rows of `width` bytes, `ld` bytes apart
struct Span {
  const void* at;
  int64_t rows, width, ld;
};
// of elements; a stride that no buffer has (negative, past 2^56) becomes one that f8_check refuses
inline Span f8_span(const void* at, int64_t rows, int64_t width, int64_t ld, int size) {
  return Span{at, rows, width * size, ld < 0 || ld > (1ll << 56) ? -size : ld * size};
}
// rows of one stride may lie in each other's gaps; of two strides the whole extents have to be apart
inline bool overlap(const Span& a, const Span& b) {
  if (!a.at || !b.at || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
  const auto end = [](const Span& w) { return (__int128)(uintptr_t)w.at + (__int128)(w.rows - 1) * w.ld + w.width; };
  if ((__int128)(uintptr_t)a.at >= end(b) || (__int128)(uintptr_t)b.at >= end(a)) return false;
  if ((a.rows > 1 && b.rows > 1 && a.ld != b.ld) || (a.rows == 1 && b.rows == 1)) return true;
  const __int128 step = a.rows > 1 ? a.ld : b.ld, d = (__int128)(uintptr_t)b.at - (__int128)(uintptr_t)a.at, in = (d % step + step) % step;
  return in < (__int128)a.width || in + (__int128)b.width > step;
}
// a matrix argument: there, aligned, its rows apart and its extent within 2^62 bytes
inline int f8_check(const char* op, const char* name, const Span& s, int align) {
  if (!s.at) { set_error("%s: missing %s buffer", op, name); return P0_EINVAL; }
  if ((uintptr_t)s.at % align || s.ld % align) { set_error("%s: %s must be %d-byte aligned, its rows too", op, name, align); return P0_EINVAL; }
  if (s.ld < s.width || (__int128)s.rows * s.ld > ((__int128)1 << 62)) {
    set_error("%s: %s has rows of %lld B, %lld B apart", op, name, (long long)s.width, (long long)s.ld); return P0_EINVAL;
  }
  return P0_OK;
}
// a launch of n workgroups: at most 2^32 threads lie along x, the rest goes along y (f8_group gives a workgroup's number; the last ones may
// be past n)
inline bool f8_grid(int64_t n, int threads, dim3* g) {
  const int64_t x = (1ll << 31) / threads, y = (n + x - 1) / x;
  if (y > 65535) return false;
  *g = dim3((unsigned)(y > 1 ? x : n), (unsigned)y);
  return true;
}
__device__ __forceinline__ int64_t f8_group() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }
inline bool f8_type(int t) { return t >= P0_F32 && t <= P0_BF16; }
inline int f8_size(int t) { return t == P0_F32 ? 4 : 2; }
inline int64_t f8_blocks(int64_t n) { return (n + kF8Block - 1) / kF8Block; }

// ---- values
template <int TYPE> __device__ __forceinline__ float f8_value(uint32_t h) {   // a 16-bit value's low half
  return TYPE == P0_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __uint_as_float(h << 16);
}
// 16 bytes at any element's address: one access, as global memory takes them unaligned
struct __attribute__((packed, aligned(2))) F8Any16 { uint32_t w[4]; };
__device__ __forceinline__ uint4 f8_load16(const void* a) {
  const F8Any16 v = *(const F8Any16*)a;
  return uint4{v.w[0], v.w[1], v.w[2], v.w[3]};
}
struct __attribute__((packed, aligned(2))) F8Any8 { uint32_t w[2]; };
__device__ __forceinline__ void f8_store8(void* a, const uint2& v) { *(F8Any8*)a = F8Any8{{v.x, v.y}}; }
__device__ __forceinline__ void f8_store16(void* a, const uint4& v) { *(F8Any16*)a = F8Any16{{v.x, v.y, v.z, v.w}}; }
// n of 8 consecutive elements (n >= 1) from element i on, of a row that has `before` elements ahead of it and n or more (`room`) from it on; the others
// are 0. f8_fetch8 asks for them, f8_take8 makes them values: of several, all are asked for first. One or two 16-byte accesses: of the row's last 8
// elements, moved down, where there are fewer than 8 from i on (one by one only in rows shorter than 8). What is read beside the n is not used: it may
// change meanwhile.
template <int TYPE> struct F8Raw { uint32_t w[TYPE == P0_F32 ? 8 : 4]; };
template <int TYPE> __device__ __forceinline__ void f8_fetch8(const void* x, int64_t i, int before, int room, F8Raw<TYPE>& f) {
  constexpr int W = TYPE == P0_F32 ? 8 : 4;
  const int back = room < 8 ? 8 - room : 0;
  if (back == 0 || back <= before) {
    const char* a = (const char*)x + (i - back) * (TYPE == P0_F32 ? 4 : 2);
#pragma unroll
    for (int k = 0; k < W / 4; ++k) {
      const uint4 u = f8_load16(a + 16 * k);
      f.w[4 * k] = u.x; f.w[4 * k + 1] = u.y; f.w[4 * k + 2] = u.z; f.w[4 * k + 3] = u.w;
    }
  }
}
template <int TYPE> __device__ __forceinline__ void f8_take8(const F8Raw<TYPE>& raw, const void* x, int64_t i, int n, int before, int room, float (&f)[8]) {
  constexpr int W = TYPE == P0_F32 ? 8 : 4;
  uint32_t w[W];
#pragma unroll
  for (int k = 0; k < W; ++k) w[k] = raw.w[k];
  const int back = room < 8 ? 8 - room : 0;
  if (back > before) {
    if constexpr (TYPE == P0_F32) {
#pragma unroll
      for (int k = 0; k < W; ++k) w[k] = ((const uint32_t*)x)[i + min(k, n - 1)];
    } else {
      const uint16_t* a = (const uint16_t*)x + i;
#pragma unroll
      for (int k = 0; k < W; ++k) w[k] = a[min(2 * k, n - 1)] | (uint32_t)a[min(2 * k + 1, n - 1)] << 16;
    }
  } else if (back) {   // down by `back` elements
#pragma unroll
    for (int b = W / 2; b > 0; b /= 2) {
      const bool on = back & (TYPE == P0_F32 ? b : 2 * b);
#pragma unroll
      for (int k = 0; k < W; ++k) w[k] = on ? (k + b < W ? w[k + b] : 0u) : w[k];
    }
    if constexpr (TYPE != P0_F32) {
      const bool on = back & 1;
#pragma unroll
      for (int k = 0; k < W; ++k) w[k] = on ? w[k] >> 16 | (k + 1 < W ? w[k + 1] << 16 : 0u) : w[k];
    }
  }
#pragma unroll
  for (int k = 0; k < W; ++k) {
    if constexpr (TYPE == P0_F32) f[k] = __uint_as_float(w[k]);
    else {
      f[2 * k] = f8_value<TYPE>(w[k] & 0xFFFFu);
      f[2 * k + 1] = TYPE == P0_F16 ? f8_value<TYPE>(w[k] >> 16) : __uint_as_float(w[k] & 0xFFFF0000u);
    }
  }
  if (n < 8) {
#pragma unroll
    for (int k = 1; k < 8; ++k) f[k] = k < n ? f[k] : 0.0f;
  }
}
template <int TYPE> __device__ __forceinline__ void f8_load8(const void* x, int64_t i, int n, int before, int room, float (&f)[8]) {
  F8Raw<TYPE> raw;
  f8_fetch8<TYPE>(x, i, before, room, raw);
  f8_take8<TYPE>(raw, x, i, n, before, room, f);
}
// to the nearest value of a 16-bit type, ties to the even one
template <int TYPE> __device__ __forceinline__ uint32_t f8_half(float v) {
  if constexpr (TYPE == P0_F16) return __builtin_bit_cast(uint16_t, (_Float16)v);
  else return __builtin_bit_cast(uint16_t, (__bf16)v);
}
template <int TYPE> __device__ __forceinline__ float f8_rounded(float v) {
  if constexpr (TYPE == P0_F32) return v;
  else return f8_value<TYPE>(f8_half<TYPE>(v));
}
template <int TYPE> __device__ __forceinline__ void f8_store8(void* x, int64_t i, bool all, int n, const float (&f)[8]) {
  if constexpr (TYPE == P0_F32) {
    float* a = (float*)x + i;
    if (all) {
      f8_store16(a, uint4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])});
      f8_store16(a + 4, uint4{__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])});
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) a[j] = f[j];
    }
  } else {
    uint16_t* a = (uint16_t*)x + i;
    if (all) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = f8_half<TYPE>(f[2 * j]) | f8_half<TYPE>(f[2 * j + 1]) << 16;
      f8_store16(a, uint4{w[0], w[1], w[2], w[3]});
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) a[j] = (uint16_t)f8_half<TYPE>(f[j]);
    }
  }
}

// ---- codes
template <int CTRL> __device__ __forceinline__ float f8_dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float f8_max16(float v) {   // of the lane's 16: rotations within a row of lanes
  v = fmaxf(v, f8_dpp<0x128>(v));
  v = fmaxf(v, f8_dpp<0x124>(v));
  v = fmaxf(v, f8_dpp<0x122>(v));
  return fmaxf(v, f8_dpp<0x121>(v));
}
// the largest magnitude of 8 values (NaN does not count), and the largest finite one
__device__ __forceinline__ float f8_most(const float (&f)[8]) {
  float most = fabsf(f[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) most = fmaxf(most, fabsf(f[j]));
  return most;
}
__device__ __forceinline__ float f8_most_finite(const float (&f)[8]) {
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(f[j]) < INFINITY ? fabsf(f[j]) : 0.0f);
  return most;
}
// the largest finite magnitude of a block, 8 values a lane of 16. A block of NaN alone has none (0), one with an infinity is looked through again
__device__ __forceinline__ float f8_block_most(const float (&f)[8]) {
  const float most = f8_max16(f8_most(f));
  return most < INFINITY ? most : f8_max16(f8_most_finite(f));
}
// max(most / 448, 2^-126) and 1 / s, each rounded to nearest: a reciprocal within a unit, and one correction that makes it and a quotient right
// to the last bit (every mantissa tried; quotients below 2^-126 do not count). The divisions in full are 25 instructions of some 100 for 8 values
__device__ __forceinline__ float f8_scale(float most) {
  constexpr float c = 1.0f / 448.0f;
  const float q = most * c;
  return fmaxf(__builtin_fmaf(__builtin_fmaf(-448.0f, q, most), c, q), 0x1p-126f);
}
__device__ __forceinline__ float f8_inverse(float s) {
  const float r = __builtin_amdgcn_rcpf(s);
  return __builtin_fmaf(__builtin_fmaf(-s, r, 1.0f), r, r);
}
// x * inv rounded to e4m3, ties to the even code; |x * inv| of a finite x is below 448.001 and so never past the largest
__device__ __forceinline__ uint2 f8_codes(const float (&f)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * j] * inv, f[4 * j + 1] * inv, 0, false);
    w[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * j + 2] * inv, f[4 * j + 3] * inv, r, true);
  }
  return uint2{w[0], w[1]};
}

}  // namespace p0
