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

#include <type_traits>
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

// 16 bytes global -> shared memory, or 16 zeros.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
}

// n / d for 0 <= n < 2^31 by a multiplication: with s = ceil(log2 d) and mul = ceil(2^(31 + s) / d),
// mul d - 2^(31 + s) < d <= 2^s, so n mul / 2^(31 + s) exceeds n / d by less than 1 / d.  A 64-bit
// division in its place is a hundred instructions, which a block that lives for microseconds
// fetches cold.
struct FastDiv {
  uint32_t d, mul;
  int shift;
  static FastDiv of(int64_t d) {
    FastDiv f{};
    f.d = (uint32_t)d;
    int s = 0;
    while ((1ll << s) < d) ++s;
    f.mul = (uint32_t)(((1ull << (31 + s)) + (uint64_t)d - 1) / (uint64_t)d);
    f.shift = 31 + s;
    return f;
  }
  __device__ __forceinline__ int div(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};

// Of the counters: the count of blocks of a line that the prefix pass used, or minus that of an item.
constexpr int kPrefixBlocks = 4095;
constexpr int kCounters = 4096;  // ints at the workspace's start: one per team or warp, zero between calls
constexpr float kLn2 = 0.69314718055994531f;

// Where the shares of a shared prefix lie that the 256-row kernel left (paged_wide.cu): its
// items are (K/V head, pair of 128-row tiles of all the batch's query rows), each of `units`
// units.  With `lines` = pairs, the pairs of a K/V head are walked side by side by blocks of
// their own (block % lines), so that they read the same keys at the same time; with lines = 1
// all items form one line.
struct PrefixShares {
  float* slots;  // nullptr: no prefix pass
  int pairs, units, lines, nc;  // nc: blocks of a line, at most (the pass may leave SMs to the sequences' own keys)
  int tile;      // query rows of a pair: 256, or 128 where there are no more
  int own_shift;  // log2 of the keys of a unit of the 16-row kernel, if that one takes the own keys: it may
                  // start beside the pass; 0: the 256-row kernel does, which has no room there
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
  FastDiv by_G, by_rows, by_page;                    // of G, rows and page_size
  int prefix;                                        // keys before the sequences' own, common to all
  int sms;
  float scale_log2;
  int* counters;   // [kCounters]
  float* partial;  // slots of partial sums
  PrefixShares pre;
  // With a prefix pass: where each query row's sums over its own keys go, O [B n H][DP] and then
  // (m, l) of each row, for the join with the prefix's shares; nullptr: `out` is final.
  float* row_share;
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

// The prefix pass is bound by the tensor pipe, the one over the sequences' own keys by memory and by
// the latency of its start and end, and that one may start as soon as SMs are free (it is a
// programmatic dependent).  A short prefix pass therefore yields: the SMs are shared out by the two
// passes' work, measured by what an SM does of each in a nanosecond.  (32 sequences of 1-512 keys
// behind 8192: 34 us, 53 without; 8 tokens of each of 16 sequences of 1-500 keys behind 2000: 40, 56
// without.)
//
// The constants' two sides, in us, as "sequences x tokens of own keys behind the prefix" (32/8 heads,
// D = 128, single tokens where none are given; the constant's own value gives the figure in front).

// An SM's time for a unit of 256 rows, of 128.  Also for D = 64, whose units hold half the work: with the
// own keys counted twice beside them 64 x 5 of 1-500 behind 2000 (16/4 heads) 42, 50; 128 of 100 behind
// 4096 27.6, 26.7.
constexpr float kUnitNs = 2250.f, kHalfUnitNs = 1300.f;
// Bytes that an SM reads in a nanosecond where memory is not shared by all.  At 30: 200 of 1-300 behind
// 512 67, 77; 16 x 4 of 1-500 behind 4000 34, 30.  At 120: 16 x 8 of 1-500 behind 2000 40, 49; 32 of
// 1-512 behind 8192 32, 36; 64 of 1-4096 behind 1024 135, 119.
constexpr float kSmBytesPerNs = 60.f;
// A launch of the pass, before and behind its units.  At 4000: 200 of 1-300 behind 512 67, 78.  At 36000:
// 256 of 1-1024 behind 2048 160, 174; 64 of 1-4096 behind 1024 135, 119.
constexpr float kStartNs = 12000.f;
// Keys that a sequence's own count for at least.  At 16: 128 of 1-20 behind 3000 33, 36; 81 of 1-10 behind
// 2000 30, 26.  At 256: 128 of 1-16 behind 8192 41, 58.
constexpr int kLeastKeys = 64;
// Units of a block up to which the prefix pass yields: longer ones slow the other pass more than the
// overlap gives (256 of 16-1024 behind 32768 yielding 282, 263).  At 4: 128 of 1-16 behind 8192 41, 47;
// 64 x 5 of 1-500 behind 2000 100, 92.  At 16, D = 64: 300 of 1-300 behind 8192 62, 65; 600 of 1-64
// behind 4096 59, 52.
constexpr int kYieldUnits = 8;
// Times the prefix pass's that the own keys' may take on the SMs left to it; a longer one takes all SMs,
// in the second wave of its blocks.  At 1: 32 of 1-2048 behind 8192 61, 66; 64 of 1-4096 behind 1024 at
// D = 64 49, 68.  At 10: 256 of 1-1024 behind 2048 160, 173; 64 of 1-4096 behind 1024 135, 119.
constexpr float kMuchLonger = 3.f;
// The share of the SMs that the own keys' blocks are laid out for at least (they run behind the pass if
// none are left).  At a third: 16 of none behind 16384 33, 37.  At 1/32, D = 64: the same 25, 29.
constexpr int kLeastShare = 8;
__device__ __forceinline__ bool brief(const PrefixShares& s, int line_units) { return line_units <= kYieldUnits * s.nc; }
// Whether the prefix pass leaves SMs to the 16-row kernel; both go by this and by own_bytes.
__device__ __forceinline__ bool yields(const PrefixShares& s, int line_units) { return s.own_shift > 0 && brief(s, line_units); }
// What the pass takes on nc blocks a line.
__device__ __forceinline__ float prefix_ns(const PrefixShares& s, int line_units, int nc) {
  return kStartNs + (float)((line_units + nc - 1) / nc) * (s.tile == kWideRows ? kUnitNs : kHalfUnitNs);
}
// Items of a sequence in the 16-row kernel.
constexpr int kRows = 16;  // query rows of one
__device__ __forceinline__ int own_items(const Params& p) { return p.Hk * ((p.rows + kRows - 1) / kRows); }
// Bytes of K and V that the 16-row kernel reads in `units` units, `items` of them a sequence at least.
__device__ __forceinline__ float own_bytes(const Params& p, int units, int items) {
  return fmaxf((float)units * (float)(1 << p.pre.own_shift), (float)p.B * items * kLeastKeys) * p.D * 4.f;
}
// Units of 2^shift keys (one at least, so that a sequence without keys gets its zeros).
__device__ __forceinline__ int units_of(int keys, int shift) { return max(1, (keys + (1 << shift) - 1) >> shift); }
// Blocks of a line that the prefix pass keeps beside `bytes` of the sequences' own keys.
__device__ __forceinline__ int yielding_blocks(const PrefixShares& s, int sms, int line_units, float bytes) {
  const float mine = (float)line_units * s.lines * (s.tile == kWideRows ? kUnitNs : kHalfUnitNs), its = bytes / kSmBytesPerNs;
  return max((s.nc + 1) / 2, min(s.nc, (int)(sms / s.lines * (mine / (mine + its)) + 0.5f)));
}

// The line of units of a launch and its even cut: the first `more` blocks have q + 1 units, the
// others q.
struct Line {
  int q, more, nc;
  __device__ __forceinline__ void cut(int units, int blocks) {
    nc = min(blocks, units);  // every block that takes part has a unit
    q = (int)((unsigned)units / (unsigned)nc);
    more = units - q * nc;
  }
  __device__ __forceinline__ int begin(int c) const { return c * q + min(c, more); }
  __device__ __forceinline__ int block_of(int u) const {
    const int longer = more * (q + 1);
    return u < longer ? (int)((unsigned)u / (unsigned)(q + 1)) : more + (int)((unsigned)(u - longer) / (unsigned)q);
  }
};

// Finds where a block's teams (kTeams of them, consecutive on the line from team `team0`) begin, by
// the whole block: units_of(b) is sequence b's count of units; the host sees to it that the line fits
// 31 bits.  Two passes over the lengths: their sum, by which the line is cut among most(sum) teams, and
// a scan up to the places looked for.  found[i] = (sequence, unit among the sequence's) for team i.
// scratch: kThreads / 32 values.
template <int kThreads, int kTeams, class UnitsOf, class Most>
__device__ __forceinline__ void locate(int B, int team0, int* scratch, int2* found, Line& line, UnitsOf units_of, Most most) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = (int)threadIdx.x < B ? units_of((int)threadIdx.x) : 0;
  int mine = head;
  for (int b = threadIdx.x + kThreads; b < B; b += kThreads) mine += units_of(b);
#pragma unroll
  for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(~0u, mine, o);
  if (lane == 0) scratch[warp] = mine;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all += scratch[w];
  line.cut(all, max(1, most(all)));
  const int last = line.begin(min(team0 + kTeams, line.nc) - 1);  // the last place looked for
  int base = 0;
  for (int b0 = 0; b0 < B && base <= last; b0 += kThreads) {
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
    int before = base, step = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int x = scratch[w];
      if (w < warp) before += x;
      step += x;
    }
    const int lo = before + scan - n;
#pragma unroll
    for (int i = 0; i < kTeams; ++i) {
      if (team0 + i >= line.nc) break;
      const int u = line.begin(team0 + i) - lo;
      if (u >= 0 && u < n) found[i] = make_int2(b, u);
    }
    base += step;
  }
  __syncthreads();
}

__device__ __forceinline__ int up_div(int a, int b) { return (int)((unsigned)(a + b - 1) / (unsigned)b); }

// Blocks of each item of the prefix pass if its items are cut one by one (nc becomes their count), 0 if
// their line is cut evenly among nc blocks.  A share costs about as much as kShareUnits units besides its
// own (Q, the first S, and the way of O through memory), and in the even cut most blocks have the end of
// one item and the begin of the next.  (32/8 heads: 16 sequences without own keys behind 16384 37 us against
// 47, 128 of 1-20 keys behind 3000 33 against 49.  A long prefix pass beside single tokens keeps the even
// cut, which leaves a few SMs more to them: 32 sequences behind 20000 keys 56 us against 58.  At 0 units
// 32 sequences of 1-512 keys behind 8192 take 38 us against 32, and 256 of 1-1024 behind 2048 155 against
// 160; at 3 nothing changes by 2%.)
constexpr int kShareUnits = 1;
__device__ __forceinline__ int blocks_per_item(int items, int units, int& nc) {
  if (items == 1 || items > nc) return 0;
  const int part = up_div(units, (int)((unsigned)nc / (unsigned)items));
  if (part > up_div(units * items, nc) + kShareUnits) return 0;
  const int used = up_div(units, part);
  nc = used * items;
  return used;
}

template <int DP>
__device__ __forceinline__ float* prefix_slot(const PrefixShares& s, int Hk, int line, int item, int block) {
  // (item, block) pairs walk a staircase, so item + block numbers them.
  const int64_t per_line = (int64_t)(s.lines > 1 ? Hk : Hk * s.pairs) + s.nc;
  return s.slots + (line * per_line + item + block) * kSlotFloats<DP>;
}

// Joins n shares (slot(x) is the x-th; slots of `rows` rows), columns d .. d + kPer of rows r[0 .. kR)
// (whose (m, l) is that of row r + ml_off), to the sums (mm, ll, v) of each.  kR kBatch loads are in flight at a time: a round trip to memory
// takes over a microsecond, so one share of one row after the other is what a join must not do.
template <int DP, int kPer, int kR, int kBatch, class Slot>
__device__ __forceinline__ void join_shares(int n, Slot slot, int rows, const int (&r)[kR], int ml_off, int d, float (&mm)[kR], float (&ll)[kR],
                                            float (&v)[kR][kPer]) {
  using V = typename std::conditional<kPer % 4 == 0, float4, float2>::type;
  constexpr int kW = sizeof(V) / 4;
#pragma unroll 1
  for (int x0 = 0; x0 < n; x0 += kBatch) {
    float2 ml[kBatch][kR];
    V f[kBatch][kR][kPer / kW];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float* s = slot(min(x0 + i, n - 1));
#pragma unroll
      for (int k = 0; k < kR; ++k) {
        ml[i][k] = __ldcg(reinterpret_cast<const float2*>(s + rows * DP + 2 * (r[k] + ml_off)));
#pragma unroll
        for (int e = 0; e < kPer / kW; ++e) f[i][k][e] = __ldcg(reinterpret_cast<const V*>(s + r[k] * DP + d + kW * e));
      }
    }
#pragma unroll
    for (int k = 0; k < kR; ++k) {
      float top = mm[k];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (x0 + i >= n) ml[i][k].x = -INFINITY;
        top = fmaxf(top, ml[i][k].x);
      }
      const float a = weight(mm[k], top);
      mm[k] = top;
      ll[k] *= a;
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[k][e] *= a;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (ml[i][k].x == -INFINITY) continue;  // no key: its O may not have been written
        const float b = weight(ml[i][k].x, top);
        ll[k] += b * ml[i][k].y;
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[k][e] += b * reinterpret_cast<const float*>(&f[i][k][e / kW])[e % kW];
      }
    }
  }
}

// Leaves the sums of columns d .. d + kPer of query row `row` (of B n H) for the join with the prefix.
template <int DP, int kPer>
__device__ __forceinline__ void leave_row(const Params& p, int row, int d, float mm, float ll, const float (&v)[kPer]) {
  using V = typename std::conditional<kPer % 4 == 0, float4, float2>::type;
  constexpr int kW = sizeof(V) / 4;
  float* dst = p.row_share + (int64_t)row * DP + d;
#pragma unroll
  for (int e = 0; e < kPer; e += kW) *reinterpret_cast<V*>(dst + e) = *reinterpret_cast<const V*>(&v[e]);
  if (d == 0) *reinterpret_cast<float2*>(p.row_share + (int64_t)p.B * p.n * p.H * DP + 2 * (int64_t)row) = make_float2(mm, ll);
}

// Adds the prefix's shares, of nc blocks a line (negative: of -nc blocks an item), for query row `row`
// (of all the batch's rows of K/V head hk).
template <int DP, int kPer, int kBatch>
__device__ __forceinline__ void join_prefix(const PrefixShares& s, int nc, int Hk, int hk, int row, int d, float (&mm)[1], float (&ll)[1],
                                            float (&v)[1][kPer]) {
  const int pair = s.tile == kWideRows ? row / kWideRows : row / (kWideRows / 2), r[1] = {row - pair * s.tile};
  const int line = s.lines > 1 ? pair : 0, item = s.lines > 1 ? hk : hk * s.pairs + pair;
  Line l;
  int cf, cl;
  if (nc < 0) {
    cf = item * -nc, cl = cf - nc - 1;
  } else {
    l.cut(s.units * (s.lines > 1 ? Hk : Hk * s.pairs), nc);
    cf = l.block_of(item * s.units), cl = l.block_of((item + 1) * s.units - 1);
  }
  join_shares<DP, kPer, 1, kBatch>(
      cl - cf + 1, [&](int x) { return prefix_slot<DP>(s, Hk, line, item, cf + x); }, kWideRows, r, 0, d, mm, ll, v);
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
// rows, leaving shares; otherwise over each sequence's own keys.
int launch_wide(const Params& p, bool bf16, bool prefix_pass, int64_t max_units, cudaStream_t s);
// Rows of a page that one TMA box may hold (0: the 256-row kernel cannot read such pages).
int wide_box_rows(int page_size);

}  // namespace paged
}  // namespace lk
