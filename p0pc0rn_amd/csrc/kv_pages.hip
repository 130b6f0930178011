// kv_pages.hip - the pages of a cache: the sequences of the next step from those of the last (kv_update), and the live pages
// to the pool's front (kv_compact). Tables, lengths and counts are device memory and no call waits for the device; the
// copies of pages that both end with are one more launch over a list that the table work leaves in the workspace.
//
// Bound: a table of a few thousand entries is launch and memory latency, so it is one workgroup's from end to end, counts and
// free list in LDS; larger ones are a launch a phase over the whole chip, counts in the workspace (uncached: what one launch
// leaves, the next finds in memory). Every count is an integer and every place a rank in ascending order, so results do not
// depend on the order of the atomics.
#include "kv_common.hpp"

namespace p0 {

constexpr int kPgThreads = 1024;
constexpr int kPgMaxPages = 1 << 21;
// What a single workgroup takes. (us, one workgroup / over the chip, the copies' launch included: kv_update of 8 sequences of 513
// tokens in pages of 64 7.4 / 17.2, of 128 of 3000 16.2 / 20.3, of 192 of 3500, 10700 pages, 22.3 / 21.7; kv_compact of 2200 pages
// 9.9 / 16.1, of 8200 23.7 / 23.6, of 11000 29.6 / 26.8.)
constexpr int kPgSmallRows = 1024, kPgSmallEntries = 1 << 15, kPgSmallPages = 8192;

// the workspace: a few words, per sequence, per page
struct PgWs {
  int32_t* head;      // [0] pages wanted, [1] free pages, [2] sequences that cannot grow, [3] copies
  int32_t *src, *kept, *grown, *open, *first_free, *copy_to;   // per sequence
  int32_t *from, *to;                                          // the copies
  int32_t *ref, *writers, *leader, *list;                      // per page
};

struct UpdP {
  KvP kv;
  const int32_t *src, *keep, *grow;
  int64_t window;
  int grow_n, sinks, B, Bo;
  int32_t* table_out;
  int64_t out_ld;
  int32_t *len_out, *ref, *status;
  PgWs ws;
};

struct Seq {
  int src, kept, grown;   // source (-1: none), tokens it keeps, tokens it then has
};
__device__ __forceinline__ Seq seq_of(const UpdP& p, int b) {
  Seq s;
  s.src = p.src ? p.src[b] : b;
  if (s.src < 0 || s.src >= p.B) s.src = -1;
  const int len = s.src < 0 ? 0 : kv_len(p.kv, s.src);
  const int keep = p.keep ? p.keep[b] : len;
  s.kept = keep < 0 ? 0 : keep < len ? keep : len;
  const int g = p.grow ? p.grow[b] : p.grow_n;
  const int64_t n = (int64_t)s.kept + (g > 0 ? g : 0);
  s.grown = n < 0x7FFFFFFF ? (int)n : 0x7FFFFFFF;
  return s;
}
__device__ __forceinline__ int pages_of(const KvP& kv, int64_t tokens) { return (int)((tokens + (1ll << kv.page_log) - 1) >> kv.page_log); }
// the page that column j keeps, -1 for none
__device__ __forceinline__ int kept_page(const UpdP& p, const Seq& s, int j) {
  if (s.src < 0 || j >= pages_of(p.kv, s.kept)) return -1;
  const int64_t t0 = (int64_t)j << p.kv.page_log, t1 = t0 + (1ll << p.kv.page_log);
  if (p.window && t1 <= s.kept - p.window + 1 && t0 >= p.sinks) return -1;
  return kv_page(p.kv, s.src, j);
}
// the column that new tokens begin in, where it is begun already; -1 for none
__device__ __forceinline__ int open_column(const KvP& kv, const Seq& s) {
  return s.grown > s.kept && (s.kept & ((1 << kv.page_log) - 1)) ? s.kept >> kv.page_log : -1;
}
__device__ __forceinline__ bool too_long(const KvP& kv, const Seq& s) { return s.grown > ((int64_t)kv.cols << kv.page_log); }
// whether it cannot grow: past the columns, or on in a column begun already whose page is none (open < 0). A free page there would
// show its old bytes as the column's earlier tokens
__device__ __forceinline__ bool stuck(const KvP& kv, const Seq& s, int open) {
  return too_long(kv, s) || (open < 0 && open_column(kv, s) >= 0);
}
__device__ __forceinline__ int wanted_by(const KvP& kv, const Seq& s, int open, bool copy) {
  return s.grown > s.kept && !stuck(kv, s, open) ? pages_of(kv, s.grown) - pages_of(kv, s.kept) + (copy ? 1 : 0) : 0;
}

// the exclusive prefix of one value a thread over the workgroup, in thread order; *all: the sum
__device__ __forceinline__ int block_prefix(int v, int* all) {
  __shared__ int s_sum[kPgThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int y = __shfl_up(x, s, 64);
    if (lane >= s) x += y;
  }
  __syncthreads();   // the sums of the call before have been read
  if (lane == 63) s_sum[wave] = x;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kPgThreads / 64; ++w) {
    const int n = s_sum[w];
    before += w < wave ? n : 0;
    total += n;
  }
  *all = total;
  return before + x - v;
}

// ---- kv_update in one workgroup: latency, a chain of LDS and memory round trips (8 sequences 5.0 us, 64 of 3000 tokens 9.4).
// LDS: counts of each page, the free list, the sequences
__global__ __launch_bounds__(kPgThreads) void kv_update_small_kernel(const UpdP p) {
  extern __shared__ int lds[];
  int* ref = lds;
  int* list = ref + p.kv.n_pages;
  int* s_src = list + p.kv.n_pages;
  int* s_kept = s_src + p.Bo;
  int* s_grown = s_kept + p.Bo;
  int* s_open = s_grown + p.Bo;
  int* s_first = s_open + p.Bo;
  int* s_copy = s_first + p.Bo;
  __shared__ int s_stuck, s_copies;
  const int tid = threadIdx.x, P = p.kv.n_pages, cols = p.kv.cols;
  for (int i = tid; i < P; i += kPgThreads) ref[i] = 0;
  if (tid == 0) s_stuck = s_copies = 0;
  Seq mine{-1, 0, 0};
  if (tid < p.Bo) {
    mine = seq_of(p, tid);
    s_src[tid] = mine.src;
    s_kept[tid] = mine.kept;
    s_grown[tid] = mine.grown;
    s_open[tid] = -1;
    s_copy[tid] = -1;
  }
  __syncthreads();
  for (int e = tid; e < p.Bo * cols; e += kPgThreads) {
    const int b = (unsigned)e / (unsigned)cols, j = e - b * cols;
    const Seq s{s_src[b], s_kept[b], s_grown[b]};
    const int pg = kept_page(p, s, j);
    p.table_out[b * p.out_ld + j] = pg;
    if (pg >= 0) {
      atomicAdd(&ref[pg], 1);
      if (j == open_column(p.kv, s)) s_open[b] = pg;
    }
  }
  __syncthreads();
  int want = 0, copy = 0;
  if (tid < p.Bo) {
    const int open = s_open[tid];
    if (open >= 0 && ref[open] > 1) {
      int writers = 0, leader = p.Bo;
      for (int b = 0; b < p.Bo; ++b)
        if (s_open[b] == open) {
          ++writers;
          leader = min(leader, b);
        }
      copy = !(writers == ref[open] && leader == tid);
    }
    want = wanted_by(p.kv, mine, open, copy);
    if (stuck(p.kv, mine, open)) atomicAdd(&s_stuck, 1);
  }
  int total, nfree = 0;
  const int before = block_prefix(want, &total);
  if (tid < p.Bo) s_first[tid] = before;
  for (int i0 = 0; i0 < P; i0 += 4 * kPgThreads) {   // four pages a thread
    int n = 0, all;
#pragma unroll
    for (int u = 0; u < 4; ++u) n += i0 + 4 * tid + u < P && ref[i0 + 4 * tid + u] == 0;
    int r = nfree + block_prefix(n, &all);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + 4 * tid + u < P && ref[i0 + 4 * tid + u] == 0) list[r++] = i0 + 4 * tid + u;
    nfree += all;
  }
  __syncthreads();
  const bool fail = total > nfree || s_stuck > 0;
  if (!fail) {
    if (copy) {
      s_copy[tid] = atomicAdd(&s_copies, 1);
      atomicSub(&ref[s_open[tid]], 1);
    }
    __syncthreads();
    for (int b = tid >> 6; b < p.Bo; b += kPgThreads / 64) {   // a wave a sequence, a lane a page
      const Seq s{s_src[b], s_kept[b], s_grown[b]};
      const int n = (b + 1 < p.Bo ? s_first[b + 1] : total) - s_first[b], c0 = pages_of(p.kv, s.grown) - n;
      for (int i = tid & 63; i < n; i += 64) {
        const int pg = list[s_first[b] + i];
        p.table_out[b * p.out_ld + c0 + i] = pg;
        ref[pg] = 1;
        if (i == 0 && s_copy[b] >= 0) {
          p.ws.from[s_copy[b]] = s_open[b];
          p.ws.to[s_copy[b]] = pg;
        }
      }
    }
  } else {
    for (int e = tid; e < p.Bo * cols; e += kPgThreads) {
      const int b = (unsigned)e / (unsigned)cols, j = e - b * cols;
      p.table_out[b * p.out_ld + j] = b < p.B && j < pages_of(p.kv, kv_len(p.kv, b)) ? kv_page(p.kv, b, j) : -1;
    }
  }
  __syncthreads();
  if (tid < p.Bo) p.len_out[tid] = !fail ? mine.grown : tid < p.B ? kv_len(p.kv, tid) : 0;
  if (p.ref && !fail)
    for (int i = tid; i < P; i += kPgThreads) p.ref[i] = ref[i];
  if (tid == 0) {
    p.status[0] = total > nfree ? total - nfree : 0;
    p.status[1] = fail ? nfree : nfree - total;
    p.status[2] = s_copies;
    p.status[3] = s_stuck;
    p.ws.head[3] = s_copies;
  }
}

// ---- kv_update over the chip, a launch a phase: 17 us for any few, each launch 2 to 3 us of latency
__global__ __launch_bounds__(256) void kv_clear_kernel(int32_t* a, int32_t* b, int32_t* c, int64_t n, int32_t* head) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) {
    a[i] = 0;
    if (b) b[i] = 0;
    if (c) c[i] = 0x7FFFFFFF;
  }
  if (i < 4) head[i] = 0;
}
__global__ __launch_bounds__(256) void kv_keep_kernel(const UpdP p) {   // grid: columns / 256, sequences
  const int b = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  const Seq s = seq_of(p, b);
  const int oc = open_column(p.kv, s);
  if (j == 0) {
    p.ws.src[b] = s.src;
    p.ws.kept[b] = s.kept;
    p.ws.grown[b] = s.grown;
    p.ws.copy_to[b] = -1;
    if (oc < 0) p.ws.open[b] = -1;
  }
  if (j >= p.kv.cols) return;
  const int pg = kept_page(p, s, j);
  p.table_out[b * p.out_ld + j] = pg;
  if (pg >= 0) atomicAdd(&p.ws.ref[pg], 1);
  if (j == oc) {
    p.ws.open[b] = pg;
    if (pg >= 0) {
      atomicAdd(&p.ws.writers[pg], 1);
      atomicMin(&p.ws.leader[pg], b);
    }
  }
}
__device__ __forceinline__ bool copies(const UpdP& p, int b, int open) {
  return open >= 0 && p.ws.ref[open] > 1 && !(p.ws.writers[open] == p.ws.ref[open] && p.ws.leader[open] == b);
}
__global__ __launch_bounds__(kPgThreads) void kv_decide_kernel(const UpdP p) {   // one workgroup
  int base = 0;
  for (int b0 = 0; b0 < p.Bo; b0 += kPgThreads) {
    const int b = b0 + threadIdx.x;
    int want = 0, all;
    if (b < p.Bo) {
      const Seq s{p.ws.src[b], p.ws.kept[b], p.ws.grown[b]};
      const int open = p.ws.open[b];
      const bool copy = copies(p, b, open);
      if (copy) p.ws.copy_to[b] = atomicAdd(&p.ws.head[3], 1);
      want = wanted_by(p.kv, s, open, copy);
      if (stuck(p.kv, s, open)) atomicAdd(&p.ws.head[2], 1);
    }
    const int at = base + block_prefix(want, &all);
    if (b < p.Bo) p.ws.first_free[b] = at;
    base += all;
  }
  if (threadIdx.x == 0) p.ws.head[0] = base;
}
// Ranks of the pages with a count of 0 (what = 0) in ascending order: list[rank] = page. A workgroup ranks `seg` pages and
// counts those before them itself: no launch in between, and P^2 / (2 seg) reads from the caches.
__global__ __launch_bounds__(kPgThreads) void kv_free_kernel(const int32_t* ref, int32_t* list, int64_t P, int64_t seg, int32_t* nfree) {
  const int64_t lo = blockIdx.x * seg, hi = lo + seg < P ? lo + seg : P;
  int n = 0, base;
  for (int64_t i = threadIdx.x; i < lo; i += kPgThreads) n += ref[i] == 0;
  block_prefix(n, &base);
  for (int64_t i0 = lo; i0 < hi; i0 += kPgThreads) {
    const int64_t i = i0 + threadIdx.x;
    const bool f = i < hi && ref[i] == 0;
    int all;
    const int r = base + block_prefix(f, &all);
    if (f) list[r] = (int)i;
    base += all;
  }
  if (hi == P && threadIdx.x == 0) *nfree = base;
}
__global__ __launch_bounds__(256) void kv_assign_kernel(const UpdP p) {   // grid: max(columns, pages / sequences) / 256, sequences
  const int b = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  const int total = p.ws.head[0], nfree = p.ws.head[1], held_up = p.ws.head[2];
  const bool fail = total > nfree || held_up > 0;
  if (j < p.kv.cols) {
    if (fail) {
      p.table_out[b * p.out_ld + j] = b < p.B && j < pages_of(p.kv, kv_len(p.kv, b)) ? kv_page(p.kv, b, j) : -1;
    } else {
      const Seq s{p.ws.src[b], p.ws.kept[b], p.ws.grown[b]};
      const int n = (b + 1 < p.Bo ? p.ws.first_free[b + 1] : total) - p.ws.first_free[b], c1 = pages_of(p.kv, s.grown);
      if (j >= c1 - n && j < c1) {
        const int pg = p.ws.list[p.ws.first_free[b] + j - (c1 - n)];
        p.table_out[b * p.out_ld + j] = pg;
        if (j == c1 - n && p.ws.copy_to[b] >= 0) {
          p.ws.from[p.ws.copy_to[b]] = p.ws.open[b];
          p.ws.to[p.ws.copy_to[b]] = pg;
        }
      }
    }
  }
  if (j == 0) p.len_out[b] = !fail ? p.ws.grown[b] : b < p.B ? kv_len(p.kv, b) : 0;
  if (j == 0 && b == 0) {
    p.status[0] = total > nfree ? total - nfree : 0;
    p.status[1] = fail ? nfree : nfree - total;
    p.status[2] = fail ? 0 : p.ws.head[3];
    p.status[3] = held_up;
  }
}
// the counts of the new tables: a kept page's holders less those that took a copy of it, 1 for one taken from the free list
__global__ __launch_bounds__(256) void kv_count_kernel(const UpdP p) {
  const int total = p.ws.head[0], nfree = p.ws.head[1];
  if (total > nfree || p.ws.head[2] > 0) return;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.kv.n_pages) return;
  const int n = p.ws.ref[i], w = p.ws.writers[i];
  if (n > 0) p.ref[i] = n > 1 && w > 0 ? n - (w == n ? w - 1 : w) : n;
  else p.ref[i] = total > 0 && i <= p.ws.list[total - 1];   // the free list is ascending: its first `total` have been taken
}

// ---- pages to other places: a workgroup takes 16 KiB pieces of the listed pages, layer by layer. Bound: HBM, read and write
// (285 MB in 67 us, 4.3 TB/s; a large copy reaches 4.5 to 5.1)
constexpr int kPgPiece = 16384;   // four 16-byte loads of each of 256 threads
__global__ __launch_bounds__(256) void kv_move_kernel(uint8_t* pages, int64_t page_bytes, int64_t bytes, int64_t layer_bytes, int layers,
                                                      const int32_t* count, const int32_t* from, const int32_t* to,
                                                      const int32_t* wanted, const int32_t* nfree, const int32_t* held_up) {
  if (wanted && (*wanted > *nfree || *held_up > 0)) return;
  const int pieces = (int)((bytes + kPgPiece - 1) / kPgPiece);
  const int64_t n = (int64_t)*count * layers * pieces;
  for (int64_t u = blockIdx.x; u < n; u += gridDim.x) {
    const int i = (int)(u / ((int64_t)layers * pieces)), r = (int)(u - (int64_t)i * layers * pieces), layer = r / pieces, piece = r % pieces;
    const int64_t at = layer * layer_bytes + (int64_t)piece * kPgPiece;
    const uint4* a = (const uint4*)(pages + at + from[i] * page_bytes);
    uint4* d = (uint4*)(pages + at + to[i] * page_bytes);
    const int words = (int)((bytes - (int64_t)piece * kPgPiece < kPgPiece ? bytes - (int64_t)piece * kPgPiece : kPgPiece) / 16);
    const int t = threadIdx.x, last = words - 1;   // past the piece's end: its last 16 bytes again
    const uint4 v0 = a[min(t, last)], v1 = a[min(t + 256, last)], v2 = a[min(t + 512, last)], v3 = a[min(t + 768, last)];
    d[min(t, last)] = v0;
    d[min(t + 256, last)] = v1;
    d[min(t + 512, last)] = v2;
    d[min(t + 768, last)] = v3;
  }
}

// ---- kv_compact
struct CmpP {
  KvP kv;
  int B;
  int32_t* table_out;
  int64_t out_ld;
  int32_t* status;
  PgWs ws;
};
__device__ __forceinline__ int live_page(const CmpP& p, int b, int j) {
  return j < pages_of(p.kv, kv_len(p.kv, b)) ? kv_page(p.kv, b, j) : -1;
}
// in one workgroup (latency; 96 pages 4.8 us, 4096 pages of 64 sequences 11): a bit per page and the live pages before each 32 in LDS, then the free pages below the count, by rank
__global__ __launch_bounds__(kPgThreads) void kv_compact_small_kernel(const CmpP p) {
  extern __shared__ int lds[];
  const int tid = threadIdx.x, P = p.kv.n_pages, words = (P + 31) / 32, cols = p.kv.cols;
  unsigned* bits = (unsigned*)lds;
  int* before = lds + words;
  int* hole = before + words;
  for (int i = tid; i < words; i += kPgThreads) bits[i] = 0;
  __syncthreads();
  for (int e = tid; e < p.B * cols; e += kPgThreads) {
    const int b = (unsigned)e / (unsigned)cols, pg = live_page(p, b, e - b * cols);
    if (pg >= 0) atomicOr(&bits[pg >> 5], 1u << (pg & 31));
  }
  __syncthreads();
  int n = 0;
  for (int i0 = 0; i0 < words; i0 += kPgThreads) {
    int all;
    const int i = i0 + tid, r = n + block_prefix(i < words ? __popc(bits[i]) : 0, &all);
    if (i < words) before[i] = r;
    n += all;
  }
  __syncthreads();
  auto rank = [&](int pg) { return before[pg >> 5] + __popc(bits[pg >> 5] & ((1u << (pg & 31)) - 1)); };   // live pages before pg
  for (int i = tid; i < words; i += kPgThreads) {
    const int top = n - 32 * i;
    unsigned m = ~bits[i] & (top >= 32 ? 0xFFFFFFFFu : top <= 0 ? 0u : (1u << top) - 1);
    for (int r = 32 * i - before[i]; m; m &= m - 1) hole[r++] = 32 * i + __ffs(m) - 1;
  }
  const int low = n < P ? rank(n) : n;   // live pages that stay
  __syncthreads();
  for (int i = tid; i < words; i += kPgThreads) {
    const int top = n - 32 * i;
    unsigned m = bits[i] & (top >= 32 ? 0u : top <= 0 ? 0xFFFFFFFFu : ~((1u << top) - 1));
    for (int r = (top > 0 && top < 32 ? low : before[i]) - low; m; m &= m - 1, ++r) {
      p.ws.from[r] = 32 * i + __ffs(m) - 1;
      p.ws.to[r] = hole[r];
    }
  }
  for (int e = tid; e < p.B * cols; e += kPgThreads) {
    const int b = (unsigned)e / (unsigned)cols, j = e - b * cols, pg = live_page(p, b, j);
    p.table_out[b * p.out_ld + j] = pg < n ? pg : hole[rank(pg) - low];
  }
  if (tid == 0) {
    p.status[0] = n;
    p.status[1] = p.ws.head[3] = n - low;
  }
}
__global__ __launch_bounds__(256) void kv_mark_kernel(const CmpP p) {
  const int b = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  const int pg = j < p.kv.cols ? live_page(p, b, j) : -1;
  if (pg >= 0) p.ws.ref[pg] = 1;
}
// after kv_free_kernel's list of the free pages: the r-th of them is a hole if it lies below the count n of live pages; the
// r-th live page at or above n has r = (live pages before it) - (live pages below n)
__global__ __launch_bounds__(kPgThreads) void kv_holes_kernel(const CmpP p, int64_t seg) {
  const int64_t P = p.kv.n_pages, lo = blockIdx.x * seg, hi = lo + seg < P ? lo + seg : P;
  const int n = (int)P - p.ws.head[1];
  int before = 0, under = 0, base, low;
  for (int64_t i = threadIdx.x; i < lo || i < n; i += kPgThreads) {
    const int live = p.ws.ref[i] != 0;
    before += i < lo ? live : 0;
    under += i < n ? live : 0;
  }
  block_prefix(before, &base);
  block_prefix(under, &low);
  for (int64_t i0 = lo; i0 < hi; i0 += kPgThreads) {
    const int64_t i = i0 + threadIdx.x;
    const bool live = i < hi && p.ws.ref[i] != 0;
    int all;
    const int r = base + block_prefix(live, &all) - low;
    if (live) p.ws.leader[i] = i < n ? (int)i : p.ws.list[r];
    if (live && i >= n) {
      p.ws.from[r] = (int)i;
      p.ws.to[r] = p.ws.list[r];
    }
    base += all;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.status[0] = n;
    p.status[1] = p.ws.head[3] = n - low;
  }
}
__global__ __launch_bounds__(256) void kv_retable_kernel(const CmpP p) {
  const int b = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  if (j >= p.kv.cols) return;
  const int pg = live_page(p, b, j);
  p.table_out[b * p.out_ld + j] = pg < 0 ? -1 : p.ws.leader[pg];
}

static PgWs workspace(int64_t rows, int64_t pages) {
  PgWs w;
  int32_t* at = (int32_t*)ctx().part;
  const auto take = [&](int64_t n) { int32_t* q = at; at += (n + 31) / 32 * 32; return q; };
  w.head = take(32);
  for (int32_t** q : {&w.src, &w.kept, &w.grown, &w.open, &w.first_free, &w.copy_to}) *q = take(rows);
  for (int32_t** q : {&w.from, &w.to, &w.ref, &w.writers, &w.leader, &w.list}) *q = take(pages);
  return w;
}
static_assert((32 + 6ll * (65535 + 32) + 6ll * kPgMaxPages) * 4 <= (64ll << 20), "the per-page arrays fit the workspace");

static int layers_check(const char* op, const p0_kv_t& kv, int64_t rows, int64_t layers, int64_t layer_bytes, int64_t out_ld, const void* table_out,
                        const void* status) {
  if (rows * kv.cols > (1 << 30)) { set_error("%s: %lld sequences of %lld columns", op, (long long)rows, (long long)kv.cols); return P0_EINVAL; }
  if (kv.n_pages > kPgMaxPages) { set_error("%s: %lld pages (at most %d)", op, (long long)kv.n_pages, kPgMaxPages); return P0_EINVAL; }
  if (layers < 0 || layers > 65536 || layer_bytes < 0 || layer_bytes % 16 ||
      (layer_bytes && layers > 1 && layer_bytes < kv.n_pages * kv_page_bytes(kv))) {
    set_error("%s: %lld layers, %lld B apart", op, (long long)layers, (long long)layer_bytes); return P0_EINVAL;
  }
  if (!table_out || !status) { set_error("%s: missing table_out or status buffer", op); return P0_EINVAL; }
  if (out_ld && out_ld < kv.cols) { set_error("%s: out_ld %lld of %lld columns", op, (long long)out_ld, (long long)kv.cols); return P0_EINVAL; }
  return P0_OK;
}
static void launch_moves(const p0_kv_t& kv, int64_t layers, int64_t layer_bytes, const PgWs& w, bool update, int64_t most) {
  const int64_t page = kv_page_bytes(kv), bytes = p0_kv_page_bytes(kv.page, kv.heads, kv.dim);
  layers = layers ? layers : 1;
  const int64_t units = most * layers * ((bytes + kPgPiece - 1) / kPgPiece);
  hipLaunchKernelGGL(kv_move_kernel, dim3((unsigned)(units < 2048 ? units : 2048)), dim3(256), 0, ctx().cur, (uint8_t*)kv.pages, page, bytes,
                     layer_bytes ? layer_bytes : kv.n_pages * page, (int)layers, w.head + 3, w.from, w.to, update ? w.head : nullptr,
                     w.head + 1, w.head + 2);
}
int kv_pages_init() {
  P0_HIP(hipFuncSetAttribute((const void*)kv_update_small_kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                             (2 * kPgSmallPages + 6 * kPgSmallRows) * 4), "p0_open: kv_update");
  P0_HIP(hipFuncSetAttribute((const void*)kv_compact_small_kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                             (2 * kPgSmallPages / 32 + 2 + kPgSmallPages) * 4), "p0_open: kv_compact");
  return P0_OK;
}

}  // namespace p0

using namespace p0;

extern "C" int p0_kv_update(const p0_kv_update_args_t* a) {
  if (!a) { set_error("kv_update: no arguments"); return P0_EINVAL; }
  UpdP p{};
  if (int r = kv_check("kv_update", a->kv, a->B, &p.kv)) return r;
  const int64_t Bo = a->Bo ? a->Bo : a->B;
  if (Bo < 0 || Bo > 65535) { set_error("kv_update: Bo %lld", (long long)Bo); return P0_EINVAL; }
  if (Bo != a->B && !a->src) { set_error("kv_update: %lld sequences of %lld need src", (long long)Bo, (long long)a->B); return P0_EINVAL; }
  if (a->window < 0 || a->sinks < 0) { set_error("kv_update: window %lld, sinks %lld", (long long)a->window, (long long)a->sinks); return P0_EINVAL; }
  if (int r = layers_check("kv_update", a->kv, a->B > Bo ? a->B : Bo, a->layers, a->layer_bytes, a->out_ld, a->table_out, a->status)) return r;
  if (!a->len_out) { set_error("kv_update: missing len_out buffer"); return P0_EINVAL; }
  const int64_t cols = a->kv.cols, ld = a->out_ld ? a->out_ld : cols;
  const Words table{a->kv.table, a->B, cols, p.kv.table_ld}, len{a->kv.len, 1, a->B, 0}, status{a->status, 1, 4, 0},
      table_out{a->table_out, Bo, cols, ld}, len_out{a->len_out, 1, Bo, 0}, ref{a->ref, 1, a->kv.n_pages, 0};
  bool over = overlap(table_out, table) || overlap(table_out, len) || overlap(len_out, table) || overlap(len_out, len);
  for (const int32_t* q : {a->src, a->keep, a->grow}) over = over || overlap(table_out, {q, 1, Bo, 0});
  if (over) { set_error("kv_update: table_out or len_out overlaps what is read"); return P0_EINVAL; }
  for (const Words& w : {ref, status})
    if (overlap(w, table) || overlap(w, len)) { set_error("kv_update: ref or status overlaps what is read"); return P0_EINVAL; }
  if (overlap(table_out, len_out) || overlap(table_out, ref) || overlap(table_out, status) || overlap(len_out, ref) || overlap(len_out, status) ||
      overlap(ref, status)) {
    set_error("kv_update: two of table_out, len_out, ref and status overlap"); return P0_EINVAL;
  }
  if (int r = refuse_in_chain("kv_update")) return r;
  if (int r = require_open("kv_update")) return r;
  p.src = a->src;
  p.keep = a->keep;
  p.grow = a->grow;
  p.grow_n = (int)(a->grow_n < 0 ? 0 : a->grow_n < 0x7FFFFFFF ? a->grow_n : 0x7FFFFFFF);
  const int64_t most = cols * a->kv.page;
  p.window = a->window > most ? 0 : a->window;
  p.sinks = (int)(a->sinks < most ? a->sinks : most);
  p.B = (int)a->B;
  p.Bo = (int)Bo;
  p.table_out = a->table_out;
  p.out_ld = ld;
  p.len_out = a->len_out;
  p.ref = a->ref;
  p.status = a->status;
  p.ws = workspace(Bo, a->kv.n_pages);
  const int64_t P = a->kv.n_pages;
  hipStream_t s = ctx().cur;
  const bool small = P <= kPgSmallPages && Bo <= kPgSmallRows && Bo * cols <= kPgSmallEntries;
  if (small) {
    hipLaunchKernelGGL(kv_update_small_kernel, dim3(1), dim3(kPgThreads), (size_t)(2 * P + 6 * Bo) * 4, s, p);
  } else {
    const unsigned pg = (unsigned)((P + 255) / 256), cg = (unsigned)((cols + 255) / 256);
    const int64_t seg = P / 64 < kPgThreads ? kPgThreads : (P / 64 + kPgThreads - 1) / kPgThreads * kPgThreads;
    hipLaunchKernelGGL(kv_clear_kernel, dim3(pg), dim3(256), 0, s, p.ws.ref, p.ws.writers, p.ws.leader, P, p.ws.head);
    if (Bo) hipLaunchKernelGGL(kv_keep_kernel, dim3(cg, (unsigned)Bo), dim3(256), 0, s, p);
    hipLaunchKernelGGL(kv_decide_kernel, dim3(1), dim3(kPgThreads), 0, s, p);
    hipLaunchKernelGGL(kv_free_kernel, dim3((unsigned)((P + seg - 1) / seg)), dim3(kPgThreads), 0, s, p.ws.ref, p.ws.list, P, seg, p.ws.head + 1);
    if (Bo) hipLaunchKernelGGL(kv_assign_kernel, dim3(cg, (unsigned)Bo), dim3(256), 0, s, p);
    if (p.ref) hipLaunchKernelGGL(kv_count_kernel, dim3(pg), dim3(256), 0, s, p);
  }
  if (Bo) launch_moves(a->kv, a->layers, a->layer_bytes, p.ws, !small, Bo);
  P0_LAUNCHED("kv_update");
  return P0_OK;
}

extern "C" int p0_kv_compact(const p0_kv_compact_args_t* a) {
  if (!a) { set_error("kv_compact: no arguments"); return P0_EINVAL; }
  CmpP p{};
  if (int r = kv_check("kv_compact", a->kv, a->B, &p.kv)) return r;
  if (int r = layers_check("kv_compact", a->kv, a->B, a->layers, a->layer_bytes, a->out_ld, a->table_out, a->status)) return r;
  const int64_t cols = a->kv.cols, ld = a->out_ld ? a->out_ld : cols, P = a->kv.n_pages;
  const Words table{a->kv.table, a->B, cols, p.kv.table_ld}, len{a->kv.len, 1, a->B, 0}, table_out{a->table_out, a->B, cols, ld},
      status{a->status, 1, 2, 0};
  if (overlap(table_out, table)) { set_error("kv_compact: table_out overlaps what is read"); return P0_EINVAL; }
  if (overlap(table_out, len) || overlap(status, table) || overlap(status, len) || overlap(status, table_out)) {
    set_error("kv_compact: table_out or status overlaps what is read"); return P0_EINVAL;
  }
  if (int r = refuse_in_chain("kv_compact")) return r;
  if (int r = require_open("kv_compact")) return r;
  p.B = (int)a->B;
  p.table_out = a->table_out;
  p.out_ld = ld;
  p.status = a->status;
  p.ws = workspace(a->B, P);
  hipStream_t s = ctx().cur;
  if (P <= kPgSmallPages && a->B * cols <= kPgSmallEntries) {
    hipLaunchKernelGGL(kv_compact_small_kernel, dim3(1), dim3(kPgThreads), (size_t)(2 * ((P + 31) / 32) + P) * 4, s, p);
  } else {
    const unsigned cg = (unsigned)((cols + 255) / 256);
    const int64_t seg = P / 64 < kPgThreads ? kPgThreads : (P / 64 + kPgThreads - 1) / kPgThreads * kPgThreads;
    const unsigned sg = (unsigned)((P + seg - 1) / seg);
    hipLaunchKernelGGL(kv_clear_kernel, dim3((unsigned)((P + 255) / 256)), dim3(256), 0, s, p.ws.ref, (int32_t*)nullptr, (int32_t*)nullptr, P, p.ws.head);
    if (a->B) hipLaunchKernelGGL(kv_mark_kernel, dim3(cg, (unsigned)a->B), dim3(256), 0, s, p);
    hipLaunchKernelGGL(kv_free_kernel, dim3(sg), dim3(kPgThreads), 0, s, p.ws.ref, p.ws.list, P, seg, p.ws.head + 1);
    hipLaunchKernelGGL(kv_holes_kernel, dim3(sg), dim3(kPgThreads), 0, s, p, seg);
    if (a->B) hipLaunchKernelGGL(kv_retable_kernel, dim3(cg, (unsigned)a->B), dim3(256), 0, s, p);
  }
  const int64_t entries = a->B * cols;
  if (entries) launch_moves(a->kv, a->layers, a->layer_bytes, p.ws, false, entries < P / 2 + 1 ? entries : P / 2 + 1);
  P0_LAUNCHED("kv_compact");
  return P0_OK;
}
