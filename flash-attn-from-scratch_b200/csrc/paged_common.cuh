// paged_common.cuh — what the attention kernels over a paged key/value cache share: their
// parameters, the split of all keys among the blocks of a launch, and the join of partial sums.
//
// Items and units.  An item is one (sequence, K/V head, tile of query rows); its keys are cut
// into units of kUnit keys (at least one, so that a sequence without keys gets its zeros).  The
// units of all items form one line, b-major, and block c of nc takes units
// [c U / nc, (c + 1) U / nc): every block has the same number of keys whatever the sequences'
// lengths, and only a block's first and last item can be shared with its neighbours.  Blocks
// that share an item each leave (m, l, o) of their keys in the workspace, and the last of them
// to arrive joins them in block order -- the same order, and the same bits, on every call.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fa_common.cuh"
#include "lk_sm100.cuh"

namespace lk {
namespace paged {

enum Site : int {
  kSitePage = 311,    // a page id outside the cache
  kSiteLength = 312,  // a length past the block table's room
};

constexpr int kCounters = 4096;  // ints at the workspace's start: one per block, zero between calls
constexpr float kLn2 = 0.69314718055994531f;

struct Params {
  const void* q;
  void* out;
  float* lse;
  const void *k, *v;
  const int *table, *lengths, *prefix_pages;
  int64_t q_sb, q_ss, q_sh, o_sb, o_ss, o_sh;        // (sequence, token, head)
  int64_t k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;        // (page, row, head)
  int64_t table_ld;
  int B, n, H, Hk, G, D;
  int rows;                                          // query rows of a (sequence, K/V head): n G
  int num_pages, page_size, table_cols;
  int prefix;                                        // keys before the sequences' own, common to all
  float scale_log2;
  int* counters;   // [kCounters]
  float* partial;  // slots of partial sums
};

// Keys of sequence b in its own pages.
__device__ __forceinline__ int own_length(const Params& p, int b) {
  int L = p.lengths[b];
  if (L < 0) L = 0;
  if ((int64_t)L > (int64_t)p.table_cols * p.page_size) {
    record_bad_index(kSiteLength);
    L = p.table_cols * p.page_size;
  }
  return L;
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return fa::pack2<kBf16>(lo, hi);
}

// exp2 of a difference of two log2-scaled maxima, 0 where the first is -inf (also beside -inf).
__device__ __forceinline__ float weight(float m, float top) { return m == -INFINITY ? 0.f : fa::ex2(m - top); }

// The line of units of a launch: its length, and where a block's share of it lies.
struct Line {
  int64_t units;  // U
  int nc;         // blocks
  __device__ __forceinline__ int64_t begin(int c) const { return (int64_t)c * units / nc; }
  // The block that has unit u: the largest c with c U / nc < u + 1.
  __device__ __forceinline__ int block_of(int64_t u) const { return (int)(((u + 1) * nc - 1) / units); }
};

}  // namespace paged
}  // namespace lk
