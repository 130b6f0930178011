// f8_gemm.hip - the product of e4m3 activations and weights with a scale per block of 128 (include/p0pc0rn.h):
//   y[m][n] = sum_kb xs[kb][m] ws[n / 128][kb] sum_{k in kb} x[m][k] w[n][k]
//
// The weight's rows are the matrix instruction's rows, the activations' its columns: a lane then holds 4 consecutive outputs of one
// activation row, whose scale is one value of the lane. A block's sum comes out of the matrix instructions in fp32, and one fma a
// value adds it, times the block's two scales, to the running sum.
//
// Two arithmetics. v_mfma_f32_16x16x128_f8f6f4 takes a whole block of k, at twice the fp16 rate, but adds the products of each 8
// consecutive k in the alignment of their largest, cutting them off 13 bits below its leading one (measured, as for the older
// 16x16x32 fp8 instruction; the sums of 8 then meet in fp32): a result is off by up to 7 * 2^-13 of the largest product of each 8, summed
// over all 8s (measured: a product loses at most 0.94 * 2^-13 of it). Of random operands that is 2e-5 to 2e-4 of the products' magnitudes, which the
// rounding to 16 bits hides (f16 results' error against 64 bits in the 2-norm 2.07e-4 -> 2.08e-4); of operands that cancel it is not. So fp32 results are
// taken on v_mfma_f32_16x16x32_f16, which keeps products and sums in fp32 (every e4m3 value is an fp16 value), at half the rate; so are few rows
// in every type, where the weights' bytes bound the call.
//
// Both operands' k may come in any order that is the same for both: lane group g (16 lanes) holds bytes [16 g, 16 g + 16) and
// [64 + 16 g, 80 + 16 g) of a block.
#include "dma.hpp"
#include "f8_choice.hpp"
#include "f8_common.hpp"

#include <type_traits>
#include <utility>

namespace p0 {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Consecutive workgroups go to the 8 XCDs in turn: of n in a line XCD i has the i-th of 8 runs
__device__ __forceinline__ int f8_run(int b, int n) {
  const int xcd = b & 7;
  return xcd * (n >> 3) + min(xcd, n & 7) + (b >> 3);
}

struct F8GemmP {
  const uint8_t* x;
  const float* xs;
  const uint8_t* w;
  const float* ws;
  void* y;
  int64_t ldx, ldxs, ldw, ldws, ldy;
  int M, N, blocks;    // blocks of 128 k
  int turned, run;     // few rows: rows lie along the grid's x; run: the grid is a line, workgroups of `run` along y for each along x
};

// a lane's 32 codes of a block: 16 bytes from two places
__device__ __forceinline__ i32x8 codes32(const i32x4& lo, const i32x4& hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));

// a lane's 32 codes of a block -> 32 fp16 values, exactly
__device__ __forceinline__ void to_half(const i32x8& w, half8v (&h)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const half2v lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[2 * i + j], 1.0f, false);
      const half2v hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[2 * i + j], 1.0f, true);
      h[i][4 * j] = lo.x; h[i][4 * j + 1] = lo.y; h[i][4 * j + 2] = hi.x; h[i][4 * j + 3] = hi.y;
    }
}
__device__ __forceinline__ f32x4 mfma_half(const half8v (&a)[4], const half8v (&b)[4]) {
  f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], b[i], d, 0, 0, 0);
  return d;
}
__device__ __forceinline__ f32x4 mfma_block(const i32x8& a, const i32x8& b) {
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0, 0, 0, 0);   // e4m3 both, no block scales of its own
}

// outputs n .. n + 3 of row m
template <int TYPE> __device__ __forceinline__ void store4(const F8GemmP& p, int m, int n, const f32x4& v) {
  const int64_t o = (int64_t)m * p.ldy + n;
  if constexpr (TYPE == P0_F32) {
    float* y = (float*)p.y + o;
    if (n + 4 <= p.N) f8_store16(y, uint4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) y[i] = v[i];
  } else {
    uint16_t* y = (uint16_t*)p.y + o;
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = f8_half<TYPE>(v[i]);
    if (n + 4 <= p.N) f8_store8(y, uint2{h[0] | h[1] << 16, h[2] | h[3] << 16});
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) y[i] = (uint16_t)h[i];
  }
}

// A row's 16-byte chunk c of a block lies in LDS at position c ^ key(row): a fragment's read takes chunk g (and g ^ 4) of rows 0 .. 15 for the lane
// groups g = 0 .. 3, and LDS serves lanes 0-3, 12-15 of one group with 4-11 of the next; under key = r & 6 those 16 lie in 16 different (row
// parity, position) pairs, so no bank conflicts (the counter reads 0; a key that suits 16 lanes of one group each, (r ^ r / 8) & 7, read 48%).
__device__ __forceinline__ int f8_key(int r) { return r & 6; }

// Few rows: a workgroup takes 16 NT outputs (weight rows) of 8 XD rows, its W waves the blocks of k in turn; their sums meet in LDS. A wave
// keeps S of its turns' blocks in LDS of its own, filled by loads that go straight there, 8 whole rows of 128 codes each: no barrier before the end.
// Lanes that load their own fragments from global memory ask 64 times an instruction, 16 rows side by side, where these ask 16 times: 16 rows, 2048 x 8192
// 9.4 us that way, 6.0 this.
// PAIR: 8 outputs of up to 8 rows, two blocks of k at a time: the matrix instruction's rows 8 - 15 are the same weights' next block, its columns 8 - 15 the
// same rows', and of its four quarters the two that pair a block with itself are kept.
// Bound: the weight's bytes, and below some 30 MB of them launch and round trips: 1 row, 16384 outputs x 2048 k 7.4 us (33.6 MB, 4.5 TB/s), 9216 x 14720 24.8 us
// (5.5 TB/s); 5 rows, 2048 x 8192 5.1 us (16.9 MB, 3.3 TB/s).
template <int W_, int NT_, int XD_, bool PAIR_, int S_>
struct F8Few {
  static constexpr int W = W_, NT = NT_, XD = XD_, S = S_, MT = (XD + 1) / 2;
  static constexpr bool PAIR = PAIR_;
  static constexpr int BN = PAIR ? 8 : 16 * NT, BM = 8 * XD, Step = PAIR ? 2 : 1;   // outputs and rows of a workgroup, blocks of a wave's turn
  static constexpr int XL = PAIR ? 2 : XD, Loads = 2 * NT + XL + Step;              // loads of x rows, all of a turn's
  static constexpr int Codes = (2 * NT + XL) * 1024, Stage = Codes + 256 * Step, Mine = S * Stage + 512, Lds = W * Mine;
  static_assert(!PAIR || (NT == 1 && XD == 1), "one tile of pairs");
  static_assert(NT * MT * 1024 <= Mine && BM <= 64, "tile");
};

template <int TYPE, class T>
__global__ __launch_bounds__(64 * T::W) void f8_few_kernel(const F8GemmP p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  constexpr int NT = T::NT, MT = T::MT, W = T::W, S = T::S, Step = T::Step;
  constexpr bool Exact = TYPE == P0_F32 || T::BM <= 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, l16 = lane & 15;
  int bx = blockIdx.x, by = blockIdx.y;
  if (p.run) {
    const int at = f8_run(bx, gridDim.x);
    bx = at / p.run;
    by = at - bx * p.run;
  }
  const int n0 = (p.turned ? by : bx) * T::BN, m0 = (p.turned ? bx : by) * T::BM;
  const int own = T::PAIR ? l16 >> 3 : 0;
  uint8_t* mine = lds + wave * T::Mine;
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)mine;
  const i32x4 rw = resource(p.w + (int64_t)n0 * p.ldw), rx = resource(p.x + (int64_t)m0 * p.ldx), rws = resource(p.ws + (int64_t)(n0 >> 7) * p.ldws);
  const int last = p.blocks - 1, r8 = lane >> 3, c8 = ((lane & 7) ^ f8_key(r8)) * 16;
  int wo[2 * NT], xo[T::XL];   // rows past the last: it again
#pragma unroll
  for (int i = 0; i < 2 * NT; ++i) wo[i] = min(T::PAIR ? r8 : 8 * i + r8, p.N - 1 - n0) * (int)p.ldw + c8;
#pragma unroll
  for (int i = 0; i < T::XL; ++i) xo[i] = min(T::PAIR ? r8 : 8 * i + r8, p.M - 1 - m0) * (int)p.ldx + c8;
  const int so = min(lane % T::BM, p.M - 1 - m0) * 4;
  const int turns = (p.blocks - wave * Step + W * Step - 1) / (W * Step);   // this wave's
  auto load = [&](int t, int st) {   // turn t's blocks into the stage at LDS offset st; past the last block: it again
    const int kb = (t * W + wave) * Step;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) dma16(base + st + i * 1024, wo[i], rw, (T::PAIR ? min(kb + i, last) : kb) * 128);
#pragma unroll
    for (int i = 0; i < T::XL; ++i) dma16(base + st + (2 * NT + i) * 1024, xo[i], rx, (T::PAIR ? min(kb + i, last) : kb) * 128);
#pragma unroll
    for (int i = 0; i < Step; ++i) dma4(base + st + T::Codes + i * 256, so, resource(p.xs + m0 + (int64_t)min(kb + i, last) * p.ldxs), 0);
  };
  // the weight's scales of 64 / Step turns, and of the next
  auto load_ws = [&](int t) {
    const int u = t + lane / Step;
    dma4(base + S * T::Stage + (t / (64 / Step) & 1) * 256, min((u * W + wave) * Step + lane % Step, last) * 4, rws, 0);
  };
  const int chunk = (g ^ f8_key(l16)) << 4;
  f32x4 acc[MT][NT];
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (turns > 0) load_ws(0);
#pragma unroll
  for (int t = 0; t < S; ++t)
    if (t < turns) load(t, t * T::Stage);
  int at = 0;
  for (int t = 0; t < turns; ++t) {
    if (t % (64 / Step) == 0 && t + 64 / Step < turns) load_ws(t + 64 / Step);   // (one load more than counted: the wait is for more, not less)
    if (t + S <= turns) wait_dma<(S - 1) * T::Loads>();
    else wait_dma<0>();
    const uint8_t* st = mine + at;
    auto frag = [&](int row) { return codes32(*(const i32x4*)(st + row * 128 + chunk), *(const i32x4*)(st + row * 128 + (chunk ^ 64))); };
    i32x8 a[NT], b[MT];
    float s[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) a[i] = frag(16 * i + l16);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int row = T::XL == 1 ? l16 & 7 : 16 * j + l16;
      b[j] = frag(16 * NT + row);
      s[j] = *(const float*)(st + T::Codes + own * 256 + (T::PAIR ? l16 & 7 : row) * 4);
    }
    const float sw = *(const float*)(mine + S * T::Stage + (t / (64 / Step) & 1) * 256 + (t % (64 / Step) * Step + own) * 4);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + S < turns) load(t + S, at);
    at = at + T::Stage == S * T::Stage ? 0 : at + T::Stage;
    const bool in = !T::PAIR || (t * W + wave) * Step + own <= last;   // past the last block: times 0
    half8v ah[Exact ? NT : 1][4];
    if constexpr (Exact) {
#pragma unroll
      for (int i = 0; i < NT; ++i) to_half(a[i], ah[i]);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      half8v bh[4];
      if constexpr (Exact) to_half(b[j], bh);
      const float f = in ? s[j] * sw : 0.0f;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        f32x4 d;
        if constexpr (Exact) d = mfma_half(ah[i], bh);
        else d = mfma_block(a[i], b[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][i][e] = __builtin_fmaf(d[e], f, acc[j][i][e]);
      }
    }
  }
  wait_dma<0>();
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int i = 0; i < NT; ++i) ((f32x4*)mine)[(j * NT + i) * 64 + lane] = acc[j][i];
  __syncthreads();
#pragma unroll
  for (int c = 0; c < NT * MT; c += W) {
    const int cell = c + wave;
    if (cell >= NT * MT) return;
    auto part = [&](int k) { return ((const f32x4*)(lds + k * T::Mine))[cell * 64 + lane]; };
    f32x4 v = part(0);
#pragma unroll
    for (int k = 1; k < W; ++k) v += part(k);
    const int n = n0 + cell % NT * 16 + 4 * g, m = m0 + cell / NT * 16 + l16;
    if constexpr (T::PAIR) {   // the other block's sums: 32 lanes of outputs and 8 columns further on
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += __shfl(v[e], lane + 40, 64);
      if (g >= 2 || l16 >= 8) return;
    }
    if (l16 < T::BM && m < p.M && n < p.N) store4<TYPE>(p, m, n, v);
  }
}

// The sums of a wave's 16 AM rows from row m on, of 16 AN outputs from output n on
template <int TYPE, int AM, int AN>
__device__ __forceinline__ void tile_out(const F8GemmP& p, const f32x4 (&acc)[AM][AN], int m, int n, int lane) {
  const int l16 = lane & 15, g = lane >> 4;
  const bool whole = m + 16 * AM <= p.M && n + 16 * AN <= p.N;
#pragma unroll
  for (int j = 0; j < AM; ++j) {
    const int mr = m + 16 * j + l16;
    if (whole && TYPE != P0_F32) {
      // two cells' outputs change places between neighbouring groups of 16 lanes: 8 consecutive ones a lane, 64 bytes a row and store
#pragma unroll
      for (int i = 0; i < AN; i += 2) {
        uint32_t a[2], b[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const auto x = __builtin_amdgcn_permlane16_swap(f8_half<TYPE>(acc[j][i][2 * h]) | f8_half<TYPE>(acc[j][i][2 * h + 1]) << 16,
                                                          f8_half<TYPE>(acc[j][i + 1][2 * h]) | f8_half<TYPE>(acc[j][i + 1][2 * h + 1]) << 16, false, false);
          a[h] = x[0];
          b[h] = x[1];
        }
        f8_store16((uint16_t*)p.y + (int64_t)mr * p.ldy + n + 16 * (i + (g & 1)) + 8 * (g >> 1), uint4{a[0], a[1], b[0], b[1]});
      }
    } else if (mr < p.M) {
#pragma unroll
      for (int i = 0; i < AN; ++i)
        if (n + 16 * i + 4 * g < p.N) store4<TYPE>(p, mr, n + 16 * i + 4 * g, acc[j][i]);
    }
    __builtin_amdgcn_sched_barrier(0);   // one row of cells at a time: the registers of more are not there
  }
}

// Many rows: a workgroup takes BN outputs (weight rows) of BM activation rows, its WN x WM waves 16 AN x 16 AM of them each. A stage in LDS is
// a block of k of every row: BN + BM rows of 128 codes and BM scales, S stages in all, filled by loads that go straight to LDS,
// S - 1 steps ahead and dealt out over a step; chunks lie as above.
// Bound: the matrix instructions at the clock that they leave. 4608 rows, 9216 outputs x 9216 k, fp16 results: 350-372 us box to box, 2.1-2.2 PFLOP/s (a
// library's product with a scale per row 327; of 8192 each way 2.36). On random codes the 16 x 16 x 128 instruction by itself reaches 3.75 PFLOP/s, with an fma a
// value beside it 3.38, on zeros 4.88: the clock goes down under them. Tried on the widest tile, us: 32 x 32 x 64 instructions the same; two groups of waves
// half a step apart the same; the next stage's lines into L2 ahead 9% more; workgroups that stay and take tile after tile 359; the tiles' blocks of
// k dealt out evenly 402 (neighbours no longer share lines in L2); bands of 2 or 8 row tiles slower.
// One barrier a step, ahead of the step's last matrix instructions: every wave then holds the rest of its step in registers, the
// next step's first fragments are read while those run, and the stage just left is free for loads.
template <int WN_, int WM_, int AN_, int AM_, int S_>
struct F8Tile {
  static constexpr int WN = WN_, WM = WM_, AN = AN_, AM = AM_, S = S_;
  static constexpr int Waves = WN * WM, Threads = 64 * Waves, BN = 16 * AN * WN, BM = 16 * AM * WM;
  static constexpr int Rows = BN + BM, Loads = Rows / 8 / Waves;   // loads of 8 rows, per wave
  static constexpr int Codes = Rows * 128, Stage = Codes + 4 * (BM < 64 ? 64 : BM), Ring = S * Stage;
  static constexpr int Lds = Ring + 512 * Waves;   // behind the stages: a wave's weight scales, of 64 steps and of the next 64
  static constexpr bool Slices = AN * AM < 32;   // the widest tile is for outputs that fill the chip without
  static_assert(Rows % (8 * Waves) == 0 && 128 % (16 * AN) == 0 && BM <= 64 * Waves, "tile");
};

struct F8TileP {
  F8GemmP g;
  int nbx, nby;   // tiles of N, of M
  int nks, spk;   // slices of K, blocks of one
  float* part;    // the slices' sums: [tile][slice][wave][cell][lane]
  unsigned* cnt;
};

template <int TYPE, class T>
__global__ __launch_bounds__(T::Threads, 2) void f8_tile_kernel(const F8TileP a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int s_last;
  constexpr bool Exact = TYPE == P0_F32;
  const F8GemmP& p = a.g;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wv % T::WN, wm = wv / T::WN, l16 = lane & 15, g = lane >> 4;
  // each XCD takes a contiguous run of tiles, which goes down a band of 4 row tiles, then on to the next column tile
  constexpr int kBand = 4;
  const int t = f8_run(blockIdx.x, a.nbx * a.nby * a.nks);
  const int per = a.nbx * a.nks * kBand, band = t / per, brows = min(kBand, a.nby - band * kBand), in = t - band * per;
  const int mb = band * kBand + in % brows, cs = in / brows, ks = cs % a.nks, nb = cs / a.nks;
  const int m0 = mb * T::BM, n0 = nb * T::BN;
  const int kb0 = ks * a.spk, nk = min(p.blocks, kb0 + a.spk);

  const uint32_t lbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  const i32x4 rw = resource(p.w + (int64_t)n0 * p.ldw), rx = resource(p.x + (int64_t)m0 * p.ldx);
  // load i of a wave fills rows (i Waves + wv) 8 .. + 7 of the stage: weights first; rows past the last are it again
  int off[T::Loads];
#pragma unroll
  for (int i = 0; i < T::Loads; ++i) {
    const int r = (i * T::Waves + wv) * 8 + (lane >> 3), c = ((lane & 7) ^ f8_key(r)) * 16;
    const bool isw = (i * T::Waves + wv) * 8 < T::BN;
    off[i] = isw ? min(r, p.N - 1 - n0) * (int)p.ldw + c : min(r - T::BN, p.M - 1 - m0) * (int)p.ldx + c;
  }
  const int soff = min(tid % T::BM, p.M - 1 - m0) * 4;   // scales: wave wv takes those of rows 64 wv on (mod BM)
  // block kb into the stage at LDS offset `st`; past the last block it is that again, never read: every step's loads count alike
  auto load = [&](int kb, int st, int i) {
    const bool isw = (i * T::Waves + wv) * 8 < T::BN;
    dma16(lbase + st + (i * T::Waves + wv) * 1024, off[i], isw ? rw : rx, min(kb, nk - 1) * 128);
  };
  auto load_scales = [&](int kb, int st) {
    dma4(lbase + st + T::Codes + (wv * 64 % T::BM) * 4, soff, resource(p.xs + m0 + (int64_t)min(kb, nk - 1) * p.ldxs), 0);
  };

  f32x4 acc[T::AM][T::AN];
#pragma unroll
  for (int j = 0; j < T::AM; ++j)
#pragma unroll
    for (int i = 0; i < T::AN; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // fragments: row 16 i + l16 of the wave's, chunks g and g + 4
  const int chunk = (g ^ f8_key(l16)) << 4, wrow = (wn * 16 * T::AN + l16) * 128, xrow = (T::BN + wm * 16 * T::AM + l16) * 128;
  const int w0 = wrow + chunk, w1 = wrow + (chunk ^ 64), x0 = xrow + chunk, x1 = xrow + (chunk ^ 64);
  const int srow = T::Codes + (wm * 16 * T::AM + l16) * 4;
  // the weight's scales of this wave's rows: 64 steps' at a time, 64 steps ahead
  const i32x4 rws = resource(p.ws + (int64_t)(min(n0 + wn * 16 * T::AN, p.N - 1) >> 7) * p.ldws);
  const int wsat = T::Ring + wv * 512;
  auto load_ws = [&](int kb) { dma4(lbase + wsat + ((kb - kb0) & 64) * 4, min(kb + lane, nk - 1) * 4, rws, 0); };
  float w;
  auto read_ws = [&](int kb) { w = *(const float*)(lds + wsat + ((kb - kb0) & 127) * 4); };

  i32x8 wf[2], xf[T::AM];
  half8v xh[Exact ? T::AM : 1][4], wh[4];
  float sf[T::AM], s[T::AM];   // the activations' scales as read, times the weight's
  f32x4 d[4];                  // the last blocks' sums, on their way into acc
  auto read_w = [&](const uint8_t* st, int i) { wf[i & 1] = codes32(*(const i32x4*)(st + w0 + i * 2048), *(const i32x4*)(st + w1 + i * 2048)); };
  auto read_x = [&](const uint8_t* st, int j) {
    xf[j] = codes32(*(const i32x4*)(st + x0 + j * 2048), *(const i32x4*)(st + x1 + j * 2048));
    sf[j] = *(const float*)(st + srow + j * 64);
  };
#pragma unroll
  for (int q = 0; q < 4; ++q) d[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < T::AM; ++j) s[j] = 0.0f;

  // A step is AN AM cells of one block product each: its matrix instruction, and the fmas of the product two cells before, which is done
  // by then. The next weight fragment is read an AM ahead; the next step's first ones follow the barrier in the last AM cells.
  constexpr int Q = T::AN * T::AM, Each = (T::Loads + Q - T::AM - 2) / (Q - T::AM - 1);   // loads a cell before the barrier; the last: scales
  static_assert((T::AM == 2 || T::AM == 4) && T::AN % 2 == 0, "cells");
  auto fold = [&](int q) {
    f32x4& v = acc[q % T::AM][q / T::AM];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(d[q & 3][e], s[q % T::AM], v[e]);
    asm volatile("" : "+v"(v));   // here and below: keeps the cell's order
  };
  auto step = [&](int kb, const uint8_t* st, const uint8_t* st_next, int st_load) {
    if (((kb - kb0) & 63) == 0 && kb + 64 < nk) load_ws(kb + 64);   // (one load more than the count below knows of: that waits for more, not less)
    if constexpr (Exact) {
#pragma unroll
      for (int j = 0; j < T::AM; ++j) to_half(xf[j], xh[j]);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = q / T::AM, j = q % T::AM;
      if (q == Q - T::AM) {
        // this wave's loads of the next stage have come (those of later ones need not have), and its reads of this one
        wait_dma<(T::S - 2) * (T::Loads + 1)>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        read_w(st_next, 0);
      }
      if constexpr (Exact) {
        if (j == 0) to_half(wf[i & 1], wh);
        d[q & 3] = mfma_half(wh, xh[j]);
      } else {
        __builtin_amdgcn_s_setprio(1);   // ahead of the other wave's fmas: 2% of the widest tile's time
        d[q & 3] = mfma_block(wf[i & 1], xf[j]);
        __builtin_amdgcn_s_setprio(0);
      }
      asm volatile("" : "+v"(d[q & 3]));
      if (i == T::AN - 1) {
        read_x(st_next, j);
      } else {
        if (j == 0) read_w(st, i + 1);
#pragma unroll
        for (int l = q * Each; l < (q + 1) * Each && l < T::Loads; ++l) load(kb + T::S - 1, st_load, l);
        if (q == Q - T::AM - 1) load_scales(kb + T::S - 1, st_load);
      }
      fold((q + Q - 2) % Q);
      if (q == 1) {
#pragma unroll
        for (int k = 0; k < T::AM; ++k) s[k] = sf[k] * w;
      }
      if (q == Q - 1) read_ws(kb + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  load_ws(kb0);
#pragma unroll
  for (int kb = 0; kb < T::S - 1; ++kb) {
#pragma unroll
    for (int l = 0; l < T::Loads; ++l) load(kb0 + kb, kb * T::Stage, l);
    load_scales(kb0 + kb, kb * T::Stage);
  }
  wait_dma<(T::S - 2) * (T::Loads + 1)>();   // the first stage has come
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int j = 0; j < T::AM; ++j) read_x(lds, j);
  read_w(lds, 0);
  read_ws(kb0);
  int at = 0, to = (T::S - 1) * T::Stage;
  for (int kb = kb0; kb < nk; ++kb) {
    const int next = at + T::Stage == T::Ring ? 0 : at + T::Stage;
    step(kb, lds + at, lds + next, to);
    to = at;
    at = next;
  }
  fold(Q - 2);
  fold(Q - 1);
  wait_dma<0>();   // loads that nothing reads must not land in another workgroup's LDS

  if (T::Slices && a.nks > 1) {
    // The slices' sums meet in the workspace: it is uncached, a store is in memory once acknowledged and device-scope loads read memory,
    // so the arrival count needs no fence. The last workgroup to arrive adds the slices in order and leaves the count at zero.
    typedef unsigned long long u64;
    const int64_t tile = (int64_t)nb * a.nby + mb, slice = (int64_t)T::BM * T::BN / 2;   // in pairs of values
    u64* mine = (u64*)a.part + (tile * a.nks + ks) * slice + wv * (Q * 128) + lane;
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4& v = acc[q % T::AM][q / T::AM];
        __hip_atomic_store(mine + (q * 2 + h) * 64, (u64)__float_as_uint(v[2 * h]) | (u64)__float_as_uint(v[2 * h + 1]) << 32, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
      }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) {
      const unsigned prev = __hip_atomic_fetch_add(a.cnt + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const int last_in = prev == (unsigned)(a.nks - 1);
      if (last_in) __hip_atomic_exchange(a.cnt + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_last = last_in;
    }
    __syncthreads();
    if (!s_last) return;
    const u64* all = (const u64*)a.part + tile * a.nks * slice + wv * (Q * 128) + lane;
    constexpr int QB = Q < 8 ? Q : 8;   // cells whose words are on their way together
#pragma unroll
    for (int q0 = 0; q0 < Q; q0 += QB) {
      f32x4 v[QB];
#pragma unroll
      for (int q = 0; q < QB; ++q) v[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      auto add = [&](auto count, int k0) {   // `count` slices' words on their way together
        constexpr int KB = decltype(count)::value;
        u64 w[KB][QB][2];
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
          for (int q = 0; q < QB; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              w[k][q][h] = __hip_atomic_load(all + (k0 + k) * slice + ((q0 + q) * 2 + h) * 64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
          for (int q = 0; q < QB; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              v[q][2 * h] += __uint_as_float((uint32_t)w[k][q][h]);
              v[q][2 * h + 1] += __uint_as_float((uint32_t)(w[k][q][h] >> 32));
            }
      };
      int k = 0;
      for (; k + 4 <= a.nks; k += 4) add(std::integral_constant<int, 4>{}, k);
      for (; k + 2 <= a.nks; k += 2) add(std::integral_constant<int, 2>{}, k);
      if (k < a.nks) add(std::integral_constant<int, 1>{}, k);
#pragma unroll
      for (int q = 0; q < QB; ++q) acc[(q0 + q) % T::AM][(q0 + q) / T::AM] = v[q];
    }
  }

  tile_out<TYPE, T::AM, T::AN>(p, acc, m0 + wm * 16 * T::AM, n0 + wn * 16 * T::AN, lane);
}

using FewPairs = F8Few<8, 1, 1, true, 2>;    // 8 outputs of 8 rows, 8 waves of two blocks a turn
using FewPairs4 = F8Few<4, 1, 1, true, 2>;   // the same, 4 waves
using Few8 = F8Few<4, 1, 1, false, 2>;       // 16 outputs of 8 rows, 4 waves
using Few16 = F8Few<8, 1, 2, false, 2>;      // 16 of 16, 8 waves
using Few16b = F8Few<4, 1, 2, false, 2>;     // the same, 4 waves
using Few32 = F8Few<8, 1, 4, false, 2>;      // 16 of 32, 8 waves
using Few32w = F8Few<8, 2, 4, false, 1>;     // 32 of 32, 8 waves
using Few32x = F8Few<8, 4, 4, false, 1>;     // 64 of 32, 8 waves
using Few64 = F8Few<8, 4, 8, false, 1>;      // 64 of 64, 8 waves
using TileSmall = F8Tile<2, 2, 2, 2, 9>;   // 64 outputs of 64 rows, 4 waves of 32 x 32
using TileLow = F8Tile<4, 1, 2, 4, 6>;     // 128 of 64, 4 waves of 32 x 64
using TileHalf = F8Tile<2, 4, 4, 2, 4>;    // 128 of 128, 8 waves of 64 x 32
using TileLong = F8Tile<2, 4, 4, 4, 3>;    // 128 of 256, 8 waves of 64 x 64
using TileWide = F8Tile<2, 4, 8, 4, 2>;    // 256 of 256, 8 waves of 128 x 64

template <class T> static auto f8_few_of(int type) {
  return type == P0_F32 ? f8_few_kernel<P0_F32, T> : type == P0_F16 ? f8_few_kernel<P0_F16, T> : f8_few_kernel<P0_BF16, T>;
}
template <class T> static void f8_few_launch(const F8GemmP& g, int type, hipStream_t s) {
  F8GemmP p = g;
  unsigned nx = (unsigned)((p.N + T::BN - 1) / T::BN), ny = (unsigned)((p.M + T::BM - 1) / T::BM);
  if (ny > 1) {
    // The operand with more rows goes along x: consecutive workgroups go to the 8 XCDs in turn, so each L2 holds an eighth of it (us, weights along x /
    // rows: 1021 rows, 130 outputs x 8192 k 12.3 / 7.9). Where x is no multiple of 8 the XCDs take runs of a line of all workgroups, so that none has more than
    // another (1737 rows, 563 x 3968 in 28 x 9 tiles 11.6, x filled up to 32 19.4)
    p.turned = p.M > p.N;
    if (p.turned) std::swap(nx, ny);
    if (nx % 8) {
      p.run = (int)ny;
      nx *= ny;
      ny = 1;
    }
  }
  hipLaunchKernelGGL(f8_few_of<T>(type), dim3(nx, ny), dim3(64 * T::W), T::Lds, s, p);
}
template <class T> static int f8_few_init() {
  for (int type : {P0_F32, P0_F16, P0_BF16})
    P0_HIP(hipFuncSetAttribute((const void*)f8_few_of<T>(type), hipFuncAttributeMaxDynamicSharedMemorySize, T::Lds), "p0_open: f8_gemm");
  return P0_OK;
}
template <class T> static auto f8_tile_of(int type) {   // fp32 results hold more in registers: not in the widest tile's
  constexpr int F = T::AN * T::AM < 32 ? P0_F32 : P0_BF16;
  return type == P0_F32 ? f8_tile_kernel<F, T> : type == P0_F16 ? f8_tile_kernel<P0_F16, T> : f8_tile_kernel<P0_BF16, T>;
}
template <class T> static void f8_tile_launch(const F8GemmP& g, int type, int nks, hipStream_t s) {
  F8TileP a{g, (g.N + T::BN - 1) / T::BN, (g.M + T::BM - 1) / T::BM};
  a.spk = (g.blocks + nks - 1) / nks;
  a.nks = (g.blocks + a.spk - 1) / a.spk;
  a.part = ctx().part;
  a.cnt = ctx().kv_counters;   // one per tile where there are slices: at most half as many as CUs
  hipLaunchKernelGGL(f8_tile_of<T>(type), dim3((unsigned)(a.nbx * a.nby * a.nks)), dim3(T::Threads), T::Lds, s, a);
}
template <class T> static int f8_tile_init() {
  for (int type : {P0_F32, P0_F16, P0_BF16})
    P0_HIP(hipFuncSetAttribute((const void*)f8_tile_of<T>(type), hipFuncAttributeMaxDynamicSharedMemorySize, T::Lds), "p0_open: f8_gemm");
  return P0_OK;
}
int f8_gemm_init() {
  if (int r = f8_few_init<FewPairs>()) return r;
  if (int r = f8_few_init<FewPairs4>()) return r;
  if (int r = f8_few_init<Few8>()) return r;
  if (int r = f8_few_init<Few16>()) return r;
  if (int r = f8_few_init<Few16b>()) return r;
  if (int r = f8_few_init<Few32>()) return r;
  if (int r = f8_few_init<Few32w>()) return r;
  if (int r = f8_few_init<Few32x>()) return r;
  if (int r = f8_few_init<Few64>()) return r;
  if (int r = f8_tile_init<TileSmall>()) return r;
  if (int r = f8_tile_init<TileLow>()) return r;
  if (int r = f8_tile_init<TileHalf>()) return r;
  if (int r = f8_tile_init<TileLong>()) return r;
  return f8_tile_init<TileWide>();
}

// false: more outputs than a launch takes
static bool f8_launch(const F8GemmP& p, int type, hipStream_t s) {
  const F8Choice c = f8_choice(p.M, p.N, p.blocks, type == P0_F32, ctx().cu_count, ctx().part_floats);
  switch (c.form) {
    case kF8TileSmall: f8_tile_launch<TileSmall>(p, type, c.slices, s); break;
    case kF8TileLow: f8_tile_launch<TileLow>(p, type, c.slices, s); break;
    case kF8TileHalf: f8_tile_launch<TileHalf>(p, type, c.slices, s); break;
    case kF8TileLong: f8_tile_launch<TileLong>(p, type, c.slices, s); break;
    case kF8TileWide: f8_tile_launch<TileWide>(p, type, 1, s); break;
    case kF8Few32: f8_few_launch<Few32>(p, type, s); break;
    case kF8Few32w: f8_few_launch<Few32w>(p, type, s); break;
    case kF8Few32x: f8_few_launch<Few32x>(p, type, s); break;
    case kF8Few64: f8_few_launch<Few64>(p, type, s); break;
    case kF8Few8: f8_few_launch<Few8>(p, type, s); break;
    case kF8Pairs4: f8_few_launch<FewPairs4>(p, type, s); break;
    case kF8Pairs: f8_few_launch<FewPairs>(p, type, s); break;
    case kF8Few16b: f8_few_launch<Few16b>(p, type, s); break;
    case kF8Few16: f8_few_launch<Few16>(p, type, s); break;
    default: return false;
  }
  return true;
}

static int gemm_f8_call(const p0_f8_gemm_args_t* a) {
  const char* op = "f8_gemm";
  if (!a) { set_error("%s: no arguments", op); return P0_EINVAL; }
  if (!f8_type(a->type)) { set_error("%s: type %d", op, (int)a->type); return P0_EINVAL; }
  if (a->M < 0 || a->M > (1 << 30)) { set_error("%s: M %lld", op, (long long)a->M); return P0_EINVAL; }
  if (a->N < 0 || a->N > (1 << 26)) { set_error("%s: N %lld", op, (long long)a->N); return P0_EINVAL; }
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
  if (int r = refuse_in_chain(op)) return r;
  if (int r = require_open(op)) return r;
  F8GemmP p{(const uint8_t*)a->x, a->xs, (const uint8_t*)a->w, a->ws, a->y, ldx, ldxs, ldw, ldws, ldy, (int)M, (int)N, (int)blocks, 0, 0};
  if (!f8_launch(p, a->type, ctx().cur)) { set_error("%s: %lld x %lld outputs", op, (long long)M, (long long)N); return P0_EINVAL; }
  P0_LAUNCHED(op);
  return P0_OK;
}

}  // namespace p0

extern "C" int p0_f8_gemm(const p0_f8_gemm_args_t* a) { return p0::gemm_f8_call(a); }
