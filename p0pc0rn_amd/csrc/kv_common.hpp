// kv_common.hpp - where a cache page keeps its bytes, and the checks of a cache descriptor that every kv_* call makes.
//
// A run holds 32 tokens of one head: key codes [16 D], key exponents [D], value codes [16 D], value exponents [D]. The orders
// are those of v_mfma_f32_16x16x32_f16's operands, so that the attention's lane loads its own 16 bytes and converts them with
// v_cvt_scalef32_pk_f16_fp4 (two values and their exponent an instruction) straight into an operand:
//  * scores S^T = K Q^T (A = 16 tokens x 32 channels): lane (g = lane / 16, t = lane % 16) holds token 16 tt + t. Of the
//    channels it takes 32 consecutive ones per 128, u * 128 + g * 32 .. (one block, one exponent), 8 per step; the order of a
//    contraction is free. Key codes [tt][u][g][t][16 B], key exponents [g][t][tt][u]. D = 64: a lane has 16 channels of both
//    tokens t and 16 + t: codes [g][t][tt][8 B], exponents [block][t][tt].
//  * outputs O^T = V^T P^T (A = 16 channels x 32 tokens): the tokens of lane group g are those whose scores the lane got from
//    the two key tiles, 4 g .. 4 g + 3 and 16 + 4 g .., so the probabilities never move between lanes. A lane's two tiles of
//    a block of 32 channels are channels 2 c and 2 c + 1 (c = lane % 16), the two codes of a byte. Value codes
//    [block / 2][g][c][block % 2][8 tokens], exponents [g][block][8 tokens].
#pragma once
#include "common.hpp"

namespace p0 {

constexpr int kKvRun = 32;                        // tokens of a run
constexpr int kKvMinExp = 127 - 23, kKvMaxExp = 127 + 13, kKvNan = 255;

// a cache as the kernels take it
struct KvP {
  uint8_t* pages;
  const int32_t* table;
  const int32_t* len;
  int64_t page_bytes, table_ld;
  int32_t n_pages, cols, page_log, heads;
};

// byte offsets inside a run: of the code byte with channels (c, c + 1), c even, and of the exponent of channel c's block
template <int D> __host__ __device__ constexpr int kv_k_code(int t, int c) {
  return D == 64 ? ((c >> 4) * 16 + (t & 15)) * 16 + (t >> 4) * 8 + ((c & 15) >> 1)
                 : ((t >> 4) * (D / 128) + (c >> 7)) * 1024 + (((c >> 5) & 3) * 16 + (t & 15)) * 16 + ((c & 31) >> 1);
}
template <int D> __host__ __device__ constexpr int kv_k_exp(int t, int c) {
  return 16 * D + (D == 64 ? ((c >> 5) * 16 + (t & 15)) * 2 + (t >> 4)
                           : ((((c >> 5) & 3) * 16 + (t & 15)) * 2 + (t >> 4)) * (D / 128) + (c >> 7));
}
__host__ __device__ constexpr int kv_slot(int t) { return (t >> 4) * 4 + (t & 3); }   // of the 8 tokens of group (t & 15) / 4
template <int D> __host__ __device__ constexpr int kv_v_code(int t, int c) {
  return 17 * D + (c >> 6) * 1024 + (((t & 15) >> 2) * 16 + ((c & 31) >> 1)) * 16 + ((c >> 5) & 1) * 8 + kv_slot(t);
}
template <int D> __host__ __device__ constexpr int kv_v_exp(int t, int c) {
  return 33 * D + (((t & 15) >> 2) * (D / 32) + (c >> 5)) * 8 + kv_slot(t);
}

// sequence b's tokens, and its page of column j (-1: none). Reads stay inside the table whatever it holds
__device__ __forceinline__ int kv_len(const KvP& p, int64_t b) {
  const int64_t most = (int64_t)p.cols << p.page_log;
  const int n = p.len[b];
  return n < 0 ? 0 : n < most ? n : (int)most;
}
__device__ __forceinline__ int kv_page(const KvP& p, int64_t b, int j) {
  const int pg = p.table[b * p.table_ld + j];
  return pg >= 0 && pg < p.n_pages ? pg : -1;
}
// the same where b and j are one for the wave: loads through the scalar cache, which no wait for vector loads holds up (the tables
// are not written by the kernels that use these)
typedef const __attribute__((address_space(4))) int32_t* KvConst;
__device__ __forceinline__ int kv_scalar(const int32_t* a, int64_t i) { return ((KvConst)(uintptr_t)a)[i]; }
__device__ __forceinline__ int kv_len_uniform(const KvP& p, int b) {
  const int64_t most = (int64_t)p.cols << p.page_log;
  const int n = kv_scalar(p.len, b);
  return n < 0 ? 0 : n < most ? n : (int)most;
}
__device__ __forceinline__ int kv_page_uniform(const KvP& p, int b, int j) {
  const int pg = kv_scalar(p.table, b * p.table_ld + j);
  return pg >= 0 && pg < p.n_pages ? pg : -1;
}
// rows of sequence b: [0, M]
__device__ __forceinline__ int kv_rows(const int32_t* rows, int64_t b, int M) {
  const int n = rows ? rows[b] : M;
  return n < 0 ? 0 : n < M ? n : M;
}

// P0_OK and the kernels' form of a descriptor, or P0_EINVAL and the message
int kv_check(const char* op, const p0_kv_t& kv, int64_t B, KvP* out);
int64_t kv_page_bytes(const p0_kv_t& kv);   // page_bytes, or its default

}  // namespace p0
