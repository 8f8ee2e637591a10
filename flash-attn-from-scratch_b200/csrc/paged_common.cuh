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

#include <utility>

#include "fa_common.cuh"
#include "lk_abi.h"
#include "lk_sm100.cuh"

namespace lk {
namespace paged {

enum Site : int {
  kSitePage = 311,    // a page id outside the cache
  kSiteLength = 312,  // a length past the block table's room
};

constexpr int kCounters = 4096;  // ints at the workspace's start: one per block, zero between calls
constexpr float kLn2 = 0.69314718055994531f;

// Where the shares of a shared prefix lie that the 256-row kernel left (paged_wide.cu): its
// items are (K/V head, pair of 128-row tiles of all the batch's query rows), each of `units`
// units.  With `lines` = pairs, the pairs of a K/V head are walked side by side by blocks of
// their own (block % lines), so that they read the same keys at the same time; with lines = 1
// all items form one line.
struct PrefixShares {
  float* slots;  // nullptr: no prefix pass
  int pairs, units, lines, nc;  // nc: blocks of a line
  int tile;      // query rows of a pair: 256, or 128 where there are no more
};
constexpr int kWideRows = 256;
// A share's slot: O as [rows][DP] in 32 bits, then (m, l) of each row.
template <int DP>
constexpr int64_t kSlotFloats = (int64_t)kWideRows * (DP + 2);

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
  PrefixShares pre;
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

// Finds the sequence whose units hold unit u of the line, by the whole block (kThreads of it):
// units_of(b) is a sequence's count per K/V head and per_seq the count of K/V heads.  Two passes
// over the lengths: their sum, which `first` turns into u, and a scan up to u.  Returns the
// sequence and u's offset among its units.  scratch: 8-byte aligned, kThreads / 32 + 2 values.
struct Found {
  int b;
  int64_t offset;
};
template <int kThreads, class UnitsOf, class First>
__device__ __forceinline__ Found locate(int B, int per_seq, long long* scratch, int64_t* total, UnitsOf units_of, First first) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = (int)threadIdx.x < B ? units_of((int)threadIdx.x) : 0;
  long long mine = head;
  for (int b = threadIdx.x + kThreads; b < B; b += kThreads) mine += units_of(b);
  for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(~0u, mine, o);
  if (lane == 0) scratch[warp] = mine;
  __syncthreads();
  long long all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all += scratch[w];
  *total = all * per_seq;
  const int64_t u = first(*total);
  long long base = 0;
  for (int b0 = 0; b0 < B; b0 += kThreads) {
    const int b = b0 + (int)threadIdx.x;
    const int n = b0 == 0 ? head : (b < B ? units_of(b) : 0);
    int scan = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(~0u, scan, o);
      if (lane >= o) scan += x;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = scan;
    __syncthreads();
    long long before = base, step = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scratch[w];
      step += scratch[w];
    }
    const long long lo = (before + scan - n) * per_seq, hi = (before + scan) * per_seq;
    if (n > 0 && lo <= u && u < hi) {
      scratch[kWarps] = b;
      scratch[kWarps + 1] = u - lo;
    }
    base += step;
    if (base * per_seq > u) break;
  }
  __syncthreads();
  const Found f{(int)scratch[kWarps], (int64_t)scratch[kWarps + 1]};
  __syncthreads();
  return f;
}

template <int DP>
__device__ __forceinline__ float* prefix_slot(const PrefixShares& s, int Hk, int line, int item, int block) {
  // (item, block) pairs walk a staircase, so item + block numbers them.
  const int64_t per_line = (int64_t)(s.lines > 1 ? Hk : Hk * s.pairs) + s.nc;
  return s.slots + (line * per_line + item + block) * kSlotFloats<DP>;
}

// Joins n shares (slot(x) is the x-th; slots of `rows` rows) of row r, columns d .. d + kPer, to the
// sums (mm, ll, v), kBatch loads at a time: a share after the other, the load latencies would add up.
template <int DP, int kPer, int kBatch, class Slot>
__device__ __forceinline__ void join_shares(int n, Slot slot, int rows, int r, int d, float& mm, float& ll, float (&v)[kPer]) {
  for (int x0 = 0; x0 < n; x0 += kBatch) {
    float2 ml[kBatch];
    float4 f[kBatch][kPer / 4];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float* s = slot(min(x0 + i, n - 1));
      ml[i] = __ldcg(reinterpret_cast<const float2*>(s + (int64_t)rows * DP + 2 * r));
#pragma unroll
      for (int e = 0; e < kPer / 4; ++e) f[i][e] = __ldcg(reinterpret_cast<const float4*>(s + (int64_t)r * DP + d + 4 * e));
      if (x0 + i >= n) ml[i].x = -INFINITY;
    }
    float top = mm;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) top = fmaxf(top, ml[i].x);
    const float a = weight(mm, top);
    mm = top;
    ll *= a;
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] *= a;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (ml[i].x == -INFINITY) continue;  // no key: its O may not have been written
      const float b = weight(ml[i].x, top);
      ll += b * ml[i].y;
#pragma unroll
      for (int e = 0; e < kPer / 4; ++e) {
        v[4 * e] += b * f[i][e].x, v[4 * e + 1] += b * f[i][e].y;
        v[4 * e + 2] += b * f[i][e].z, v[4 * e + 3] += b * f[i][e].w;
      }
    }
  }
}

// Adds the prefix's shares for query row `row` (of all the batch's rows of K/V head hk).
template <int DP, int kPer, int kBatch>
__device__ __forceinline__ void join_prefix(const PrefixShares& s, int Hk, int hk, int64_t row, int d, float& mm, float& ll,
                                            float (&v)[kPer]) {
  const int pair = (int)(row / s.tile), r = (int)(row - (int64_t)pair * s.tile);
  const int line = s.lines > 1 ? pair : 0, item = s.lines > 1 ? hk : hk * s.pairs + pair;
  Line l;
  l.units = (int64_t)s.units * (s.lines > 1 ? Hk : Hk * s.pairs);
  l.nc = s.nc;
  const int cf = l.block_of((int64_t)item * s.units), cl = l.block_of((int64_t)(item + 1) * s.units - 1);
  join_shares<DP, kPer, kBatch>(
      cl - cf + 1, [&](int x) { return prefix_slot<DP>(s, Hk, line, item, cf + x); }, kWideRows, r, d, mm, ll, v);
}

// Launches `kern`; `dependent`: as a programmatic dependent of the launch before it (it calls
// griddep_wait before it reads what that one writes).
template <class... P, class... A>
inline int launch_kernel(void (*kern)(P...), int grid, int threads, size_t smem, bool dependent, cudaStream_t s, A&&... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...));
}

// The 256-row kernel (paged_wide.cu).  prefix_pass: over the prefix's keys for all the batch's
// rows, leaving shares; otherwise over each sequence's own keys, joining the shares in p.pre.
int launch_wide(const Params& p, bool bf16, bool prefix_pass, int64_t max_units, cudaStream_t s);
// Rows of a page that one TMA box may hold (0: the 256-row kernel cannot read such pages).
int wide_box_rows(int page_size);

}  // namespace paged
}  // namespace lk
