// beam.hip - a beam search's step: the best continuations of each search's beams, from the head's logits.
//
// One pass over the logits: a workgroup takes 8192 of a row, holds them in registers, and leaves their maximum, the sum of
// their exponentials against it and their k best as 64-bit keys (the value's order, then the lower token). The last workgroup of a
// search to arrive joins them: the rows' sums of exponentials, each row's k best, then the k best of all beams.
// A row's best need no sort: with the lanes in k groups, the least of the groups' best is at or below k values, so what lies
// under it is out, and what is left is ranked by counting (of 8192 logits some 50 for k up to 8). Where many are left, the lanes'
// best are sorted for a closer bound: of a wave's lanes no more than k have anything at or above the k-th best of them. (For k over
// 8 the first bound leaves some 370 of 8192, more than is ranked, so nearly every workgroup takes the second.)
// Bound: HBM at many rows and k up to 8 (32 searches of 8 beams, 262144 logits: 268 MB), the VALU for k over 8 (k = 32: 135 us and a join
// of 26, busy in 71% of the cycles), launch and the join's round trips at few.
#include "common.hpp"

namespace p0 {

constexpr int kBmThreads = 256, kBmValues = 32, kBmChunk = kBmThreads * kBmValues, kBmMostK = 32;

struct BeamP {
  const float* logits;
  int64_t ld;
  int V, W, k, chunks, eos;
  const float* score;
  const int32_t* done;
  int32_t *token, *parent;
  float* score_out;
  int32_t* done_out;
  const int32_t* hist;
  int32_t* hist_out;
  int64_t hist_n, hist_ld;
  // in the workspace (uncached), written and read with device-scope accesses: a store is in memory once acknowledged, and a join
  // in the same launch gets no line that its CU's L1 took in before another workgroup's words of it were written
  uint64_t* keys;      // [rows][chunks][k]
  uint64_t* sums;      // [rows][chunks]: maximum (low word), sum of exponentials
  unsigned* cnt;       // per search
};

// floats in their order as unsigned: the larger float has the larger code
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t o) { return __uint_as_float(o ^ (o >> 31 ? 0x80000000u : 0xFFFFFFFFu)); }
__device__ __forceinline__ uint64_t key_of(float v, int token) { return (uint64_t)order_of(v) << 32 | (uint32_t)~token; }

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
  return (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), m, 64) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)v, m, 64);
}
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int l) {
  return (uint64_t)(uint32_t)__shfl((int)(v >> 32), l, 64) << 32 | (uint32_t)__shfl((int)(uint32_t)v, l, 64);
}
// lanes 8 .. 1 apart by rotations of a row of 16 (whose values then have that period), 16 and 32 apart by swaps of rows and halves
template <int S, class F> __device__ __forceinline__ float with_lane(float v, F f) {
  if constexpr (S == 32) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  } else if constexpr (S == 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  } else {
    return f(v, __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), 0x120 + S, 0xF, 0xF, true)));
  }
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ float added(float a, float b) { return a + b; }
template <class F> __device__ __forceinline__ float wave_all(float v, F f) {
  return with_lane<1>(with_lane<2>(with_lane<4>(with_lane<8>(with_lane<16>(with_lane<32>(v, f), f), f), f), f), f);
}
// the least of the largest of KM groups of lanes (the lanes with the same lane % KM): at most as large as KM of their values
template <int KM> __device__ __forceinline__ float least_of_groups(float v) {
  if constexpr (KM == 8) {
    v = with_lane<8>(with_lane<16>(with_lane<32>(v, larger), larger), larger);
    return with_lane<1>(with_lane<2>(with_lane<4>(v, smaller), smaller), smaller);
  } else {
    v = with_lane<32>(v, larger);
    return with_lane<1>(with_lane<2>(with_lane<4>(with_lane<8>(with_lane<16>(v, smaller), smaller), smaller), smaller), smaller);
  }
}
// the wave's values, largest in lane 0: a bitonic sort over its lanes
__device__ __forceinline__ uint64_t wave_sort(uint64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int n = 2; n <= 64; n <<= 1)
#pragma unroll
    for (int s = n >> 1; s > 0; s >>= 1) {
      const uint64_t o = shfl_xor64(v, s);
      const bool larger = ((lane & s) == 0) == ((lane & n) == 0 || n == 64);
      v = (o > v) == larger ? o : v;
    }
  return v;
}

constexpr int kBmWaves = kBmThreads / 64, kBmBatch = 16;
struct Cand {
  uint64_t hi, lo;   // (score, beam), (logit, token)
};
__device__ __forceinline__ bool above(const Cand& a, const Cand& b) { return a.hi > b.hi || (a.hi == b.hi && a.lo > b.lo); }
// KM: the most k. A chunk's list holds what the sorted bound leaves at the most
template <int KM> struct PartLds {
  uint64_t list[kBmWaves * KM * kBmValues];
};
template <int KM, int WAVES> struct JoinLds {
  uint64_t list[WAVES][kBmBatch * KM], top[WAVES][KM];
  Cand cand[WAVES * KM + KM];   // a round's rows and the best of the rounds before
  Cand best[KM];
  int row[KM], tok[KM];
};
constexpr float kLog2e = 1.44269504088896340736f;
__device__ __forceinline__ uint64_t ws_load(const uint64_t* a) { return __hip_atomic_load(a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void ws_store(uint64_t* a, uint64_t v) { __hip_atomic_store(a, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// a wave's LDS writes before its lanes' reads of them. (The LDS takes a wave's accesses in order; the fence keeps the compiler to it)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
typedef float float4a4 __attribute__((ext_vector_type(4), aligned(4)));   // a 16-byte load at 4-byte alignment

// a row's k best of its chunks' keys and its sum of exponentials: lane r < k gets the r-th candidate of beam w
template <int KM, int WAVES>
__device__ __forceinline__ Cand row_best(const BeamP& p, JoinLds<KM, WAVES>& l, int64_t row, int w) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = p.k;
  // what the row has left, all on its way before the first wait; an ended beam's too
  const uint64_t* keys = p.keys + row * p.chunks * k;
  const int total = p.chunks * k;
  uint64_t q[kBmBatch], top = 0;
  // 15 keys a lane at a time beside the best of the batches before. A chunk's keys descend, so the lanes turn from one 64 to the
  // next: each gets keys of many ranks, and the k-th best of the lanes' best leaves few (32 of 262144 logits: 33 us the call, 92
  // where a lane kept to a rank)
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kBmBatch - 1; ++u) {
      const int i = i0 + u * 64 + (lane + 13 * u) % 64;
      q[u] = i < total ? ws_load(keys + i) : 0;
    }
  };
  load(0);
  const float score = p.score[row];
  const bool ended = p.done && p.done[row];
  float most = -INFINITY, sum = 0.0f;
  for (int c = lane; c < p.chunks; c += 64) {
    const uint64_t ms = ws_load(p.sums + row * p.chunks + c);
    const float m = __uint_as_float((uint32_t)ms), e = __uint_as_float((uint32_t)(ms >> 32)), both = fmaxf(most, m);
    sum = both == -INFINITY ? 0.0f : sum * exp2f((most - both) * kLog2e) + e * exp2f((m - both) * kLog2e);
    most = both;
  }
  if (ended) {
    const float s = lane == 0 && score == score ? score : -INFINITY;
    return lane < k ? Cand{(uint64_t)order_of(s + 0.0f) << 32 | (uint32_t)~w, (uint64_t)(kBmMostK - lane) << 32 | (uint32_t)~p.eos} : Cand{0, 0};
  }
  const float own = most;
  most = wave_all(most, larger);
  sum = wave_all(own == -INFINITY ? 0.0f : sum * exp2f((own - most) * kLog2e), added);
  const float lse = most + logf(sum);
#pragma nounroll
  for (int i0 = 0; i0 < total; i0 += 64 * (kBmBatch - 1)) {
    if (i0) load(i0);
    uint64_t best = top;
#pragma unroll
    for (int u = 0; u < kBmBatch - 1; ++u) best = q[u] > best ? q[u] : best;
    q[kBmBatch - 1] = top;
    uint64_t least = shfl64(wave_sort(best), k - 1);
    if (least == 0) least = 1;
    int n = 0;
#pragma unroll
    for (int u = 0; u < kBmBatch; ++u) {
      const uint64_t in = __ballot(q[u] >= least);
      if (q[u] >= least) l.list[wave][n + __popcll(in & ((1ull << lane) - 1))] = q[u];
      n += __popcll(in);
    }
    l.top[wave][lane % KM] = 0;
    wave_sync();
    for (int i = lane; i < n; i += 64) {
      const uint64_t key = l.list[wave][i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += l.list[wave][j] > key;
      if (rank < k) l.top[wave][rank] = key;
    }
    wave_sync();
    top = lane < k ? l.top[wave][lane] : 0;
    wave_sync();
  }
  float s = score + (of_order((uint32_t)(top >> 32)) - lse);
  if (s != s) s = -INFINITY;
  return lane < k ? Cand{(uint64_t)order_of(s + 0.0f) << 32 | (uint32_t)~w, top} : Cand{0, 0};
}
// a search's k best, written out: a workgroup, a wave a row at a time
template <int KM, int WAVES>
__device__ __forceinline__ void search_best(const BeamP& p, JoinLds<KM, WAVES>& l, int64_t g) {
  static_assert((WAVES + 1) * KM <= 64 * WAVES, "a candidate a thread");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = p.k;
  if (tid < k) l.best[tid] = Cand{0, 0};
#pragma nounroll
  for (int w0 = 0; w0 < p.W; w0 += WAVES) {
    const int w = w0 + wave;
    Cand mine{0, 0};
    if (w < p.W) mine = row_best(p, l, g * p.W + w, w);
    if (lane < k) l.cand[wave * k + lane] = mine;
    if (tid < k) l.cand[WAVES * k + tid] = l.best[tid];
    __syncthreads();
    const int n = (WAVES + 1) * k;
    if (tid < n) {
      const Cand c = l.cand[tid];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += above(l.cand[j], c);
      if (rank < k && c.hi) l.best[rank] = c;
    }
    __syncthreads();
  }
  if (tid < k) {
    const Cand c = l.best[tid];
    const int w = (int)~(uint32_t)c.hi, token = (int)~(uint32_t)c.lo, row = (int)(g * p.W + w);
    p.token[g * k + tid] = token;
    p.parent[g * k + tid] = row;
    p.score_out[g * k + tid] = of_order((uint32_t)(c.hi >> 32));
    if (p.done_out) p.done_out[g * k + tid] = (p.done && p.done[row]) || (p.eos >= 0 && token == p.eos);
    l.row[tid] = row;
    l.tok[tid] = token;
  }
  if (!p.hist) return;
  __syncthreads();
  for (int r = wave; r < k; r += WAVES)
    for (int64_t c = lane; c <= p.hist_n; c += 64)
      p.hist_out[(g * k + r) * p.hist_ld + c] = c < p.hist_n ? p.hist[l.row[r] * p.hist_ld + c] : l.tok[r];
}

// The pass over the logits: 43 us for 256 rows of 262144 (6.2 TB/s, HBM); at few rows one memory round trip and the ranking.
// JOIN: the last of a search's workgroups to arrive joins them. It saves a launch where its four waves have a row each and few
// workgroups wait for their own stores before they count themselves in; else a join of eight waves a search is sooner. (us, one
// launch / two: a search of 4 beams of 262144 logits 13.9 / 14.5, of 8 20.1 / 16.3; 4 searches of 4 18.0 / 16.2, 32 of 8 118 / 61.)
template <int KM, bool JOIN>
__global__ __launch_bounds__(kBmThreads) void beam_kernel(const BeamP p) {
  __shared__ union {
    PartLds<KM> part;
    JoinLds<JOIN ? KM : 1, kBmWaves> join;
  } lds;
  __shared__ float s_f[kBmWaves], s_b[kBmWaves];
  __shared__ uint64_t s_t[kBmWaves];
  __shared__ int s_n, s_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.y;
  const int c0 = blockIdx.x * kBmChunk;
  const float* x = p.logits + row * p.ld;
  float v[kBmValues];   // of token c0 + (i / 4) * 1024 + tid * 4 + i % 4
  if (c0 + kBmChunk <= p.V) {
#pragma unroll
    for (int i = 0; i < kBmValues / 4; ++i) {
      const float4a4 q = *(const float4a4*)(x + c0 + i * 1024 + tid * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = q[j];
    }
  } else {   // a row's end: four that are there, turned to where they belong
    float few[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) few[j] = x[j < p.V ? j : 0];
#pragma unroll
    for (int i = 0; i < kBmValues / 4; ++i) {
      const int c = c0 + i * 1024 + tid * 4, at = min(c, max(p.V - 4, 0)), d = c - at;
      float4a4 q = {few[0], few[1], few[2], 0.0f};
      if (p.V >= 4) q = *(const float4a4*)(x + at);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y = q[j];
#pragma unroll
        for (int n = 1; n < 4 - j; ++n) y = d == n ? q[j + n] : y;
        v[4 * i + j] = c + j < p.V ? y : -INFINITY;
      }
    }
  }
  if (tid == 0) s_n = 0;
  // the lane's best: the first of its largest (its tokens ascend). NaN is -infinity: the maximum drops it
  float bv = -INFINITY;
  int bi = 0;
#pragma unroll
  for (int i = 0; i < kBmValues; ++i) {
    v[i] = fmaxf(v[i], -INFINITY);
    bi = v[i] > bv ? i : bi;
    bv = fmaxf(v[i], bv);
  }
  const auto token = [&](int i) { return c0 + (i >> 2) * 1024 + tid * 4 + (i & 3); };
  const uint64_t best = token(bi) < p.V ? key_of(bv + 0.0f, token(bi)) : 0;
  float most = wave_all(bv, larger), bound = least_of_groups<KM>(bv);
  if (lane == 0) { s_f[wave] = most; s_b[wave] = bound; }
  __syncthreads();
  most = fmaxf(fmaxf(s_f[0], s_f[1]), fmaxf(s_f[2], s_f[3]));
  bound = fmaxf(fmaxf(s_b[0], s_b[1]), fmaxf(s_b[2], s_b[3]));
  // at or above `least` there are at least k keys: those of the bound's value and larger ones
  uint64_t least = (uint64_t)order_of(bound + 0.0f) << 32;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kBmValues; ++i) sum += __builtin_amdgcn_exp2f((v[i] - most) * kLog2e);
  if (most == -INFINITY) sum = 0.0f;
  sum = wave_all(sum, added);
  // the keys at or above `least`, in any order; past `most_n` they are counted only
  auto collect = [&](int most_n) {
    const float lv = of_order((uint32_t)(least >> 32));
#pragma unroll
    for (int i = 0; i < kBmValues; ++i) {
      if (!(v[i] >= lv)) continue;
      const uint64_t key = key_of(v[i] + 0.0f, token(i));
      if (key >= least && token(i) < p.V) {
        const int at = atomicAdd(&s_n, 1);
        if (at < most_n) lds.part.list[at] = key;
      }
    }
    __syncthreads();
    return s_n;
  };
  constexpr int kSmall = 256;
  int n = collect(kSmall);
  if (n > kSmall) {
    const uint64_t kth = shfl64(wave_sort(best), p.k - 1);
    __syncthreads();   // s_n has been read
    if (lane == 0) s_t[wave] = kth;
    if (tid == 0) s_n = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kBmWaves; ++w) least = w == 0 || s_t[w] > least ? s_t[w] : least;
    if (least == 0) least = (uint64_t)order_of(-INFINITY) << 32;   // fewer lanes than k have a token: all of theirs
    n = collect(kBmWaves * KM * kBmValues);
  }
  if (lane == 0) s_f[wave] = sum;
  uint64_t* out = p.keys + (row * p.chunks + blockIdx.x) * p.k;
  for (int i = tid; i < n; i += kBmThreads) {
    const uint64_t key = lds.part.list[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += lds.part.list[j] > key;
    if (rank < p.k) ws_store(out + rank, key);
  }
  if (tid >= n && tid < p.k) ws_store(out + tid, 0);   // a chunk of fewer than k
  __syncthreads();
  if (tid == 0)
    ws_store(p.sums + row * p.chunks + blockIdx.x, (uint64_t)__float_as_uint((s_f[0] + s_f[1]) + (s_f[2] + s_f[3])) << 32 | __float_as_uint(most));
  if constexpr (!JOIN) return;
  const int64_t g = row / p.W;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (tid == 0) {
    unsigned* c = p.cnt + g;
    s_last = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(p.W * p.chunks - 1);
    if (s_last) __hip_atomic_exchange(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // leave it at zero
  }
  __syncthreads();
  if constexpr (JOIN)
    if (s_last) search_best(p, lds.join, g);
}
constexpr int kBmJoinWaves = 8;
// bound: memory latency, one round trip a row, then the ranks from LDS (32 searches of 8 beams of 32 chunks: 10.6 us)
template <int KM>
__global__ __launch_bounds__(64 * kBmJoinWaves) void beam_join_kernel(const BeamP p) {
  __shared__ JoinLds<KM, kBmJoinWaves> lds;
  search_best(p, lds, blockIdx.x);
}
template <int KM>
static void launch_beam(const BeamP& p, int64_t n, hipStream_t s) {
  const dim3 grid((unsigned)p.chunks, (unsigned)(n * p.W));
  if (p.W <= kBmWaves && n * p.W * p.chunks <= 256) {
    hipLaunchKernelGGL((beam_kernel<KM, true>), grid, dim3(kBmThreads), 0, s, p);
    return;
  }
  hipLaunchKernelGGL((beam_kernel<KM, false>), grid, dim3(kBmThreads), 0, s, p);
  hipLaunchKernelGGL(beam_join_kernel<KM>, dim3((unsigned)n), dim3(64 * kBmJoinWaves), 0, s, p);
}

}  // namespace p0

using namespace p0;

extern "C" int p0_beam(const p0_beam_args_t* a) {
  if (!a) { set_error("beam: no arguments"); return P0_EINVAL; }
  if (a->n < 0 || a->n > 65535 || a->W < 1 || a->W > 65535 || a->n * a->W > 65535) {
    set_error("beam: %lld searches of %lld beams", (long long)a->n, (long long)a->W); return P0_EINVAL;
  }
  if (a->V < 1 || a->V > (1 << 30) || (a->ld && a->ld < a->V)) { set_error("beam: V %lld, ld %lld", (long long)a->V, (long long)a->ld); return P0_EINVAL; }
  if (a->k < 1 || a->k > kBmMostK || a->k > a->V) { set_error("beam: k %lld (1..%d, at most V)", (long long)a->k, kBmMostK); return P0_EINVAL; }
  if (!a->logits || !a->score || !a->token || !a->parent || !a->score_out) {
    set_error("beam: missing logits, score, token, parent or score_out buffer"); return P0_EINVAL;
  }
  if ((a->hist != nullptr) != (a->hist_out != nullptr)) { set_error("beam: hist and hist_out go together"); return P0_EINVAL; }
  if (a->hist && (a->hist_n < 0 || a->hist_n > (1 << 24) || (a->hist_ld && a->hist_ld <= a->hist_n))) {
    set_error("beam: hist of %lld tokens, stride %lld", (long long)a->hist_n, (long long)a->hist_ld); return P0_EINVAL;
  }
  if (a->hist) {
    const int64_t ld = a->hist_ld ? a->hist_ld : a->hist_n + 1;
    if (overlap({a->hist, a->n * a->W, a->hist_n, ld}, {a->hist_out, a->n * a->k, a->hist_n + 1, ld})) {
      set_error("beam: hist and hist_out overlap"); return P0_EINVAL;
    }
  }
  if (a->done && a->eos < 0) { set_error("beam: done needs an eos token"); return P0_EINVAL; }
  BeamP p{};
  const int64_t rows = a->n * a->W, chunks = (a->V + kBmChunk - 1) / kBmChunk;
  const int64_t bytes = rows * chunks * (a->k * 8 + 8);
  if (bytes > (int64_t)(64 << 20)) {
    set_error("beam: %lld rows of %lld logits need %lld B of workspace", (long long)rows, (long long)a->V, (long long)bytes); return P0_EINVAL;
  }
  if (int r = refuse_in_chain("beam")) return r;
  if (int r = require_open("beam")) return r;
  if (a->n == 0) return P0_OK;
  p.logits = a->logits;
  p.ld = a->ld ? a->ld : a->V;
  p.V = (int)a->V;
  p.W = (int)a->W;
  p.k = (int)a->k;
  p.chunks = (int)chunks;
  p.eos = a->eos;
  p.score = a->score;
  p.done = a->done;
  p.token = a->token;
  p.parent = a->parent;
  p.score_out = a->score_out;
  p.done_out = a->done_out;
  p.hist = a->hist;
  p.hist_out = a->hist_out;
  p.hist_n = a->hist_n;
  p.hist_ld = a->hist_ld ? a->hist_ld : a->hist_n + 1;
  p.keys = (uint64_t*)ctx().part;
  p.sums = p.keys + rows * chunks * a->k;
  p.cnt = ctx().kv_counters;
  if (a->k <= 8) launch_beam<8>(p, a->n, ctx().cur);
  else launch_beam<32>(p, a->n, ctx().cur);
  P0_LAUNCHED("beam");
  return P0_OK;
}
