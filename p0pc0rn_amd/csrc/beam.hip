// beam.hip - a beam search's step: the best continuations of each search's beams, from the head's logits.
//
// One pass over the logits: a workgroup takes 8192 of a row, holds them in registers, and leaves their maximum, the sum of
// their exponentials against it and their k best as 64-bit keys (the value's order, then the lower token). A second launch
// joins a search's: the rows' sums of exponentials, each row's k best, then the k best of all beams.
// A row's best need no full sort: at least k lanes of a wave have a maximum at or above the k-th of their sorted maxima, so
// what lies below that is out, and what is left (a little over k values as a rule) is ranked by counting.
#include "common.hpp"

namespace p0 {

constexpr int kBmThreads = 256, kBmValues = 32, kBmChunk = kBmThreads * kBmValues, kBmMostK = 32;

struct BeamP {
  const float* logits;
  int64_t ld;
  int V, W, k, chunks, vec, eos;
  const float* score;
  const int32_t* done;
  int32_t *token, *parent;
  float* score_out;
  int32_t* done_out;
  const int32_t* hist;
  int32_t* hist_out;
  int64_t hist_n, hist_ld;
  uint64_t* keys;      // [rows][chunks][k]
  float* sums;         // [rows][chunks][2]: maximum, sum of exponentials
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

__global__ __launch_bounds__(kBmThreads) void beam_part_kernel(const BeamP p) {
  __shared__ float s_f[4];
  __shared__ uint64_t s_t[4];
  __shared__ uint64_t s_list[4 * kBmMostK * kBmValues];
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.y;
  const int c0 = blockIdx.x * kBmChunk;
  const float* x = p.logits + row * p.ld;
  float v[kBmValues];
#pragma unroll
  for (int i = 0; i < kBmValues / 4; ++i) {
    const int c = c0 + i * 1024 + tid * 4;
    if (p.vec && c + 4 <= p.V) {
      const float4 q = *(const float4*)(x + c);
      v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = c + j < p.V ? x[c + j] : -INFINITY;
    }
  }
  if (tid == 0) s_n = 0;
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < kBmValues; ++i) {
    v[i] = v[i] == v[i] ? v[i] + 0.0f : -INFINITY;   // -0 is 0
    most = fmaxf(most, v[i]);
  }
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) most = fmaxf(most, __shfl_xor(most, s, 64));
  if (lane == 0) s_f[wave] = most;
  // the lane's best: the first of its largest (its tokens ascend)
  uint64_t best = 0;
#pragma unroll
  for (int i = 0; i < kBmValues; ++i) {
    const int c = c0 + (i >> 2) * 1024 + tid * 4 + (i & 3);
    const uint64_t key = c < p.V ? key_of(v[i], c) : 0;
    best = key > best ? key : best;
  }
  const uint64_t sorted = wave_sort(best);
  const uint64_t kth = shfl64(sorted, p.k - 1);
  if (lane == 0) s_t[wave] = kth;
  __syncthreads();
  most = fmaxf(fmaxf(s_f[0], s_f[1]), fmaxf(s_f[2], s_f[3]));
  uint64_t least = s_t[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) least = s_t[w] > least ? s_t[w] : least;
  if (least == 0) least = 1;   // no key is 0: what lies past the row
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kBmValues; ++i) sum += most == -INFINITY ? 0.0f : exp2f((v[i] - most) * 1.44269504088896340736f);
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) sum += __shfl_xor(sum, s, 64);
#pragma unroll
  for (int i = 0; i < kBmValues; ++i) {
    const int c = c0 + (i >> 2) * 1024 + tid * 4 + (i & 3);
    const uint64_t key = c < p.V ? key_of(v[i], c) : 0;
    if (key >= least) s_list[atomicAdd(&s_n, 1)] = key;
  }
  __syncthreads();   // s_f and the list
  if (lane == 0) s_f[wave] = sum;
  const int n = s_n;
  uint64_t* out = p.keys + (row * p.chunks + blockIdx.x) * p.k;
  for (int i = tid; i < n; i += kBmThreads) {
    const uint64_t key = s_list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s_list[j] > key;
    if (rank < p.k) out[rank] = key;
  }
  if (tid >= n && tid < p.k) out[tid] = 0;   // a chunk of fewer than k
  __syncthreads();
  if (tid == 0) {
    p.sums[(row * p.chunks + blockIdx.x) * 2] = most;
    p.sums[(row * p.chunks + blockIdx.x) * 2 + 1] = (s_f[0] + s_f[1]) + (s_f[2] + s_f[3]);
  }
}

struct Cand {
  uint64_t hi, lo;   // (score, beam), (logit, token)
};
__device__ __forceinline__ bool above(const Cand& a, const Cand& b) { return a.hi > b.hi || (a.hi == b.hi && a.lo > b.lo); }

// a workgroup a search: a wave a row at a time
constexpr int kBmJoinThreads = 512, kBmJoinWaves = kBmJoinThreads / 64, kBmBatch = 16;
__global__ __launch_bounds__(kBmJoinThreads) void beam_join_kernel(const BeamP p) {
  __shared__ uint64_t s_list[kBmJoinWaves][kBmBatch * kBmMostK];
  __shared__ Cand s_cand[kBmJoinWaves * kBmMostK + kBmMostK];   // a round's rows and the best of the rounds before
  __shared__ Cand s_best[kBmMostK];
  __shared__ int s_row[kBmMostK], s_tok[kBmMostK];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = p.k;
  const int64_t g = blockIdx.x;
  for (int i = tid; i < k; i += kBmJoinThreads) s_best[i] = Cand{0, 0};
  for (int w0 = 0; w0 < p.W; w0 += kBmJoinWaves) {
    const int w = w0 + wave;
    Cand mine{0, 0};   // lane r < k: the row's r-th
    if (w < p.W) {
      const int64_t row = g * p.W + w;
      const float score = p.score[row];
      if (p.done && p.done[row]) {
        if (lane < k) {
          const float s = lane == 0 && score == score ? score : -INFINITY;
          mine = Cand{(uint64_t)order_of(s + 0.0f) << 32 | (uint32_t)~w, (uint64_t)(kBmMostK - lane) << 32 | (uint32_t)~p.eos};
        }
      } else {
        // the row's sum of exponentials
        float most = -INFINITY;
        for (int c = lane; c < p.chunks; c += 64) most = fmaxf(most, p.sums[(row * p.chunks + c) * 2]);
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) most = fmaxf(most, __shfl_xor(most, s, 64));
        float sum = 0.0f;
        for (int c = lane; c < p.chunks; c += 64) {
          const float m = p.sums[(row * p.chunks + c) * 2], e = p.sums[(row * p.chunks + c) * 2 + 1];
          sum += m == -INFINITY ? 0.0f : e * exp2f((m - most) * 1.44269504088896340736f);
        }
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) sum += __shfl_xor(sum, s, 64);
        const float lse = most + logf(sum);
        // its k best, 15 keys a lane at a time beside those of the batches before
        const uint64_t* keys = p.keys + row * p.chunks * k;
        const int total = p.chunks * k;
        uint64_t top = 0;
        for (int i0 = 0; i0 < total; i0 += 64 * (kBmBatch - 1)) {
          uint64_t q[kBmBatch], best = top;
#pragma unroll
          for (int u = 0; u < kBmBatch - 1; ++u) {
            const int i = i0 + u * 64 + lane;
            q[u] = i < total ? keys[i] : 0;
            best = q[u] > best ? q[u] : best;
          }
          q[kBmBatch - 1] = top;
          uint64_t least = shfl64(wave_sort(best), k - 1);
          if (least == 0) least = 1;
          int n = 0;
#pragma unroll
          for (int u = 0; u < kBmBatch; ++u) {
            const uint64_t in = __ballot(q[u] >= least);
            if (q[u] >= least) s_list[wave][n + __popcll(in & ((1ull << lane) - 1))] = q[u];
            n += __popcll(in);
          }
          __builtin_amdgcn_wave_barrier();
          top = 0;
          uint64_t next = 0;
          for (int i = lane; i < n + 63 - (n + 63) % 64; i += 64) {   // every lane the same number of times
            const uint64_t key = i < n ? s_list[wave][i] : 0;
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += s_list[wave][j] > key;
            const bool in = i < n && rank < k;
            // lane `rank` takes it
            uint64_t m = __ballot(in);
            while (m) {
              const int l = __ffsll((unsigned long long)m) - 1;
              const uint64_t v = shfl64(key, l);
              if (lane == __shfl(rank, l, 64)) next = v;
              m &= m - 1;
            }
          }
          top = next;
          __builtin_amdgcn_wave_barrier();
        }
        if (lane < k) {
          float s = score + (of_order((uint32_t)(top >> 32)) - lse);
          if (s != s) s = -INFINITY;
          mine = Cand{(uint64_t)order_of(s + 0.0f) << 32 | (uint32_t)~w, top};
        }
      }
    }
    if (lane < k) s_cand[wave * k + lane] = mine;
    if (tid < k) s_cand[kBmJoinWaves * k + tid] = s_best[tid];
    __syncthreads();
    const int n = (kBmJoinWaves + 1) * k;
    for (int i = tid; i < n; i += kBmJoinThreads) {
      const Cand c = s_cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += above(s_cand[j], c);
      if (rank < k && c.hi) s_best[rank] = c;
    }
    __syncthreads();
  }
  if (tid < k) {
    const Cand c = s_best[tid];
    const int w = (int)~(uint32_t)c.hi, token = (int)~(uint32_t)c.lo, row = (int)(g * p.W + w);
    p.token[g * k + tid] = token;
    p.parent[g * k + tid] = row;
    p.score_out[g * k + tid] = of_order((uint32_t)(c.hi >> 32));
    if (p.done_out) p.done_out[g * k + tid] = (p.done && p.done[row]) || (p.eos >= 0 && token == p.eos);
    s_row[tid] = row;
    s_tok[tid] = token;
  }
  if (!p.hist) return;
  __syncthreads();
  for (int64_t i = tid; i < k * (p.hist_n + 1); i += kBmJoinThreads) {
    const int r = (int)(i / (p.hist_n + 1)), c = (int)(i % (p.hist_n + 1));
    p.hist_out[(g * k + r) * p.hist_ld + c] = c < p.hist_n ? p.hist[s_row[r] * p.hist_ld + c] : s_tok[r];
  }
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
    const uintptr_t in = (uintptr_t)a->hist, out = (uintptr_t)a->hist_out;
    if (in < out + a->n * a->k * ld * 4 && out < in + a->n * a->W * ld * 4) { set_error("beam: hist and hist_out overlap"); return P0_EINVAL; }
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
  p.vec = (uintptr_t)a->logits % 16 == 0 && p.ld % 4 == 0;
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
  p.sums = (float*)(p.keys + rows * chunks * a->k);
  hipLaunchKernelGGL(beam_part_kernel, dim3((unsigned)chunks, (unsigned)rows), dim3(kBmThreads), 0, ctx().cur, p);
  hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)a->n), dim3(kBmJoinThreads), 0, ctx().cur, p);
  P0_LAUNCHED("beam");
  return P0_OK;
}
