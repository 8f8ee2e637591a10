// paged_wide.cu — attention over a paged key/value cache for many query rows per K/V head, on
// the tensor cores: tcgen05 MMAs into tensor memory, K/V pages streamed by TMA.
//
// Two uses of one kernel.  The prefix pass: all the batch's queries of a K/V head against the
// keys that the sequences share, read once for 256 rows; it leaves (m, l, o) shares that the
// kernel over the sequences' own keys joins.  And sequences with more than 16 query rows per
// K/V head (pieces of prompts, many drafted tokens, one K/V head for many query heads).
//
// Bound: with 256 rows a block does 256 flops per byte of K/V, near the card's balance (~250), so
// both matter: the tensor pipe runs S = Q K^T and O += P V of two 128-row tiles in turn while
// eight softmax warps (a thread = a row) work on the other tile's exponentials, and TMA streams
// pages through a ring.  The roles and the tensor-memory layout are those of the flash-attention
// forward kernel (flash_attn.cu):
//   warps 0-3, 4-7  softmax of tile 0, 1; they also gather the rows of Q (any stride, any group
//                   size) into swizzled shared memory, and write or share the results
//   warp 8          TMA producer: K_0, V_0, K_1, V_1, ... of 128 keys, page by page: a box is the
//                   largest power of two of rows that divides the page (8 to 128), a lane each
//   warp 9          tensor memory and MMA issue
// A block walks its share of the line of units (paged_common.cuh; a unit is 128 keys) through as
// many items as that holds; the barriers' phases run on across items.
//
// With no more than 128 rows the second tile would idle and S -> softmax -> PV would be one
// serial chain; there tile 1 takes the same queries over every second key block (two halves of
// the keys, joined at the item's end: the two tiles' warps see the same lanes of tensor memory).
//
// Measured (B200, 32/8 heads, D = 128, bf16): 2.2 us for a unit of 256 rows x 128 keys, as the
// flash-attention forward takes (1100 TFLOP/s); 4 x 500 prompt tokens at up to 9000 keys 220 us (728
// TFLOP/s: a share costs 15-20 thousand cycles besides its units, for Q, the first S, and the way of O
// through memory where blocks share an item).  A launch of one unit takes 12 us, mostly instruction
// fetches and round trips to memory that nothing hides yet.
//
// The softmax loop takes all 168 registers and spills a little: a warp makes 3 loads (5 where D = 64) and one
// store of local memory a unit, measured by how those requests grow with the keys.  The probabilities are
// rounded to the inputs' type for the second product, as in the flash-attention forward; kept in two parts
// they would cost the tensor pipe half as much again.
//
// Keys behind a sequence's last one: whole boxes of them are not read (an out-of-range page
// coordinate gives zeros); in the box that holds the end the rows of V behind it are zeroed in
// shared memory before the MMA may see them (0 x NaN), and S is masked.
#include <cuda.h>

#include <atomic>

#include "lk_abi.h"
#include "paged_common.cuh"

namespace lk {
namespace paged {
namespace {

constexpr int kThreads = 320;
constexpr int kTileM = 128;
constexpr int kBlockN = 128;  // keys of a unit
constexpr float kJoinUnits = 1.f;  // what the join of a share costs, in units
constexpr float kLazy = 8.0f;  // log2 units that the maximum may grow by before O is rescaled

enum WideSite : int {
  kSiteEmpty = 321,
  kSiteQ = 322,
  kSiteKV = 323,
  kSiteP = 324,
  kSiteS = 325,
  kSiteO = 326,
  kSiteFix = 327,
  kSiteMeet = 328,
  kSiteTeardown = 329,
};

template <int D>
struct Cfg {
  static constexpr int kBoxes = D / 64;              // 128-byte columns of a row
  static constexpr int kTile = kTileM * D * 2;       // bytes of a tile of Q, K or V
  static constexpr int kFit = (232448 - 1024 - 1024 - 2 * kTile) / kTile;
  static constexpr int kStages = kFit > 8 ? 8 : kFit;  // 5 (D = 128), 8 (D = 64)
  static constexpr int kSmem = (2 + kStages) * kTile + 1024 + 1024;
  static constexpr int kOCol = 256;
};

struct WideParams {
  Params p;
  int prefix_pass;
  int rows;        // query rows of an item's (sequence, K/V head); prefix pass: of the K/V head
  int pairs;       // tiles of 256 (halves == 2: 128) rows
  int halves;      // 2: tile 1 holds tile 0's queries and takes the odd key blocks
  int box_rows;    // rows of a page in one TMA box
  int lines;       // prefix pass: lines of units (paged_common.cuh)
};

// An item's share of a block: blocks [j0, j1) of 128 keys of item (b, hk, pair).
struct Item {
  int b, hk, pair;
  int units;    // key blocks of the item
  int keys;     // keys that lie in the pages
  int visible;  // keys that its last row sees
};

// Where a softmax warp stands on its block's share.  Kept in shared memory: the softmax loop
// needs its registers for a row of S.
struct Walk {
  Item it;
  int j0, done, todo, c, line_id, item, unit;
  Line line;
};

__device__ __forceinline__ int visible_keys(const WideParams& w, int L, int pair) {
  if (w.prefix_pass) return L;
  const int last_row = min(w.rows, w.halves == 2 ? kTileM : (pair + 1) * 2 * kTileM) - 1;
  return max(0, L - w.p.n + w.p.by_G.div(last_row) + 1);
}
__device__ __forceinline__ int units_of_keys(int keys) { return max(1, (keys + kBlockN - 1) / kBlockN); }

__device__ __forceinline__ void enter(const WideParams& w, Item& it) {
  it.visible = visible_keys(w, it.keys, it.pair);
  it.units = units_of_keys(it.visible);
}
// The item behind `it` on the block's line.
__device__ __forceinline__ void next_item(const WideParams& w, Item& it) {
  if (w.prefix_pass) {
    if (w.lines > 1) {
      ++it.hk;
    } else if (++it.pair == w.pairs) {
      it.pair = 0;
      ++it.hk;
    }
    return;  // all items have the prefix's units
  }
  if (++it.pair == w.pairs) {
    it.pair = 0;
    if (++it.hk == w.p.Hk) {
      it.hk = 0;
      ++it.b;
      it.keys = it.b < w.p.B ? own_length(w.p, it.b) : 0;
    }
  }
  enter(w, it);
}

// Query row `row` of the item: its sequence, token and head.
struct Row {
  int b, i, head;
};
__device__ __forceinline__ Row query_row(const WideParams& w, const Item& it, int row) {
  Row r;
  r.b = it.b;
  if (w.prefix_pass) {
    r.b = w.p.by_rows.div(row);
    row -= r.b * w.p.rows;
  }
  r.i = w.p.by_G.div(row);
  r.head = it.hk * w.p.G + row - r.i * w.p.G;
  return r;
}

// Max of n fp32 values (bit patterns), four chains of three-input max.
template <int n>
__device__ __forceinline__ float row_max(const uint32_t (&sr)[n]) {
  float m[4] = {__uint_as_float(sr[0]), __uint_as_float(sr[1]), __uint_as_float(sr[2]), __uint_as_float(sr[3])};
#pragma unroll
  for (int c = 4; c < n - 4; c += 8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = max3(m[e], __uint_as_float(sr[c + 2 * e]), __uint_as_float(sr[c + 2 * e + 1]));
  }
  m[0] = max3(m[0], __uint_as_float(sr[n - 4]), __uint_as_float(sr[n - 3]));
  m[1] = max3(m[1], __uint_as_float(sr[n - 2]), __uint_as_float(sr[n - 1]));
  return fmaxf(max3(m[0], m[1], m[2]), m[3]);
}

// What a softmax warp hands on of an item.
template <int D>
struct HandOn {
  const WideParams* w;
  Item it;
  uint8_t* sQ;
  uint32_t tmem;
  float m_row, l_row;   // of this thread's row
  float w0, w1;         // weights of O_0 and O_1 in it
  bool any0, any1;      // whether O_0 and O_1 hold anything
  int row_begin;        // first query row of the tile
  int quad_rows;        // queries among the warp's 32 rows
  int cf, cl, me;       // blocks that share the item, first and last, and this one
  __device__ __forceinline__ float* slot_of(int x) const {  // of a sequence's own keys
    return w->p.partial + (int64_t)(2 * x + (x == cf ? 1 : 0)) * kSlotFloats<D>;
  }
};

// Hands on this warp's rows (with two halves, half of their columns): into `share`, or (nullptr)
// joined with the others' shares as the result.  What a row needs once (weights, addresses) its
// thread works out; values go through shared memory, from a row per thread to whole rows per warp.
template <int D, bool kBf16>
__device__ __forceinline__ void hand_on(const HandOn<D>& h, float* share, int lane, int warp) {
  using C = Cfg<D>;
  const WideParams& w = *h.w;
  const Params& p = w.p;
  const int t = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
  const bool halves = w.halves == 2, two = h.cl - h.cf == 1;
  const int quad_rows = h.quad_rows, c0 = halves ? t * (D / 2) : 0, c1 = halves ? c0 + D / 2 : D;
  const uint32_t o_tmem = h.tmem + ((uint32_t)(quad * 32) << 16) + C::kOCol;
  // Row `row` of the tile, columns col .. col + 3 of the D / 2 at hand in 32 bits, in this warp's own
  // rows of the tile's Q buffer (128-byte swizzle).
  auto stage_at = [&](int row, int col) {
    return reinterpret_cast<float4*>(h.sQ + t * C::kTile + (col >> 5) * (kTileM * 128) + row * 128 +
                                     ((((col >> 2) & 7) ^ (row & 7)) << 4));
  };
  // The slot's row of O of this warp's first row, and the slot's place of its (m, l) (with two halves
  // each tile's warps leave one, for their own columns).
  const int o_row = (halves ? 0 : t * kTileM) + quad * 32, ml_at = kWideRows * D + 2 * (t * kTileM + r);
  // Shares to read: none, the other of two, or all (this warp's own among them).
  const int others = share || w.prefix_pass || h.cf == h.cl ? 0 : (two ? 1 : h.cl - h.cf + 1);
  auto other = [&](int x) { return h.slot_of(two ? h.cf + h.cl - h.me : h.cf + x); };
  auto other_ml = [&](int x) { return __ldcg(reinterpret_cast<const float2*>(other(min(x, others - 1)) + ml_at)); };
  const bool with_own = others < 2;
  float mm = with_own ? h.m_row : -INFINITY, ll = with_own ? h.l_row : 0.f;
#pragma unroll 1
  for (int x0 = 0; x0 < others; x0 += 4) {  // four round trips to memory at a time
    float2 ml[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) ml[x] = other_ml(x0 + x);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (x0 + x >= others) break;
      const float top = fmaxf(mm, ml[x].x);
      ll = __fadd_rn(__fmul_rn(ll, weight(mm, top)), __fmul_rn(ml[x].y, weight(ml[x].x, top)));
      mm = top;
    }
  }
  const float inv = share || p.row_share ? 1.f : (ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll));
  const float own = !with_own ? 0.f : others ? weight(h.m_row, mm) * inv : inv;
  // No weight, no value: where the shares are all read from the workspace, O counts there.
  const float w0 = own == 0.f ? 0.f : h.w0, w1 = own == 0.f ? 0.f : h.w1;
  uint64_t to = 0;  // where this thread's row goes
  if (lane < quad_rows) {
    if (share) {
      *reinterpret_cast<float2*>(share + ml_at) = make_float2(mm, ll);
      to = reinterpret_cast<uint64_t>(share + (int64_t)(o_row + lane) * D);
    } else {
      const Row at = query_row(w, h.it, h.row_begin + r);
      const int64_t out_row = ((int64_t)at.b * p.n + at.i) * p.H + at.head;
      if (p.row_share) {
        to = reinterpret_cast<uint64_t>(p.row_share + out_row * D);
        if (c0 == 0)
          *reinterpret_cast<float2*>(p.row_share + (int64_t)p.B * p.n * p.H * D + 2 * out_row) = make_float2(mm, ll);
      } else {
        to = reinterpret_cast<uint64_t>(static_cast<uint16_t*>(p.out) + at.b * p.o_sb + at.i * p.o_ss + at.head * p.o_sh);
        if (p.lse && c0 == 0) p.lse[out_row] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * kLn2;
      }
    }
  }
#pragma unroll 1
  for (int cb = c0; cb < c1; cb += D / 2) {
#pragma unroll 1
    for (int x = 0; x < D / 64; ++x) {
      uint32_t ov[32];
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = 0.f;
      if (h.any0) {
        tmem_ld32(o_tmem + cb + x * 32, ov);
        tmem_wait_ld();
        if (w0 != 0.f) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = w0 * __uint_as_float(ov[i]);
        }
      }
      __syncwarp();
      if (h.any1) {
        tmem_ld32(o_tmem + D + cb + x * 32, ov);
        tmem_wait_ld();
        if (w1 != 0.f) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] += w1 * __uint_as_float(ov[i]);
        }
      }
      __syncwarp();
      // The weight goes to the sum, which is what another block would find in the share.
#pragma unroll
      for (int i = 0; i < 32; i += 4)
        *stage_at(r, x * 32 + i) = make_float4(own * v[i], own * v[i + 1], own * v[i + 2], own * v[i + 3]);
    }
    __syncwarp();
    constexpr int kLanes = D / 8, kRowsPer = 32 / kLanes, kG = 16 / kRowsPer;  // 4 columns a lane
    const int col = lane % kLanes * 4, sub = lane / kLanes;
#pragma unroll 1
    for (int x = 0; x < others; ++x) {
      const float f = weight(other_ml(x).x, mm) * inv;
      const float* src = other(x) + (int64_t)o_row * D + cb + col;
#pragma unroll 1
      for (int r0 = 0; r0 < quad_rows; r0 += kG * kRowsPer) {  // 16 rows in flight
        float4 g[kG];
#pragma unroll
        for (int k = 0; k < kG; ++k)
          g[k] = __ldcg(reinterpret_cast<const float4*>(src + min(r0 + k * kRowsPer + sub, quad_rows - 1) * D));
#pragma unroll
        for (int k = 0; k < kG; ++k) {
          const int rr = r0 + k * kRowsPer + sub;
          const float fr = __shfl_sync(~0u, f, rr & 31);
          if (rr >= quad_rows || fr == 0.f) continue;  // a share without a key may not hold O
          float4* at = stage_at(quad * 32 + rr, col);
          float4 a = *at;
          // Products rounded before the sum: of two shares it is then the same both ways round.
          a.x = __fadd_rn(a.x, __fmul_rn(fr, g[k].x)), a.y = __fadd_rn(a.y, __fmul_rn(fr, g[k].y));
          a.z = __fadd_rn(a.z, __fmul_rn(fr, g[k].z)), a.w = __fadd_rn(a.w, __fmul_rn(fr, g[k].w));
          *at = a;
        }
      }
      __syncwarp();
    }
    if (share || p.row_share) {
#pragma unroll 4
      for (int r0 = 0; r0 < 32; r0 += kRowsPer) {
        const int rr = r0 + sub;
        float* dst = reinterpret_cast<float*>(__shfl_sync(~0u, to, rr));
        if (rr < quad_rows) *reinterpret_cast<float4*>(dst + cb + col) = *stage_at(quad * 32 + rr, col);
      }
    } else {
      constexpr int kLanes8 = D / 16, kRows8 = 32 / kLanes8;  // 8 columns a lane
      const int col8 = lane % kLanes8 * 8;
#pragma unroll 4
      for (int r0 = 0; r0 < 32; r0 += kRows8) {
        const int rr = r0 + lane / kLanes8;
        uint16_t* dst = reinterpret_cast<uint16_t*>(__shfl_sync(~0u, to, rr));
        if (rr < quad_rows && cb + col8 < p.D) {
          const float4 a = *stage_at(quad * 32 + rr, col8), b = *stage_at(quad * 32 + rr, col8 + 4);
          *reinterpret_cast<uint4*>(dst + cb + col8) =
              make_uint4(pack2<kBf16>(a.x, a.y), pack2<kBf16>(a.z, a.w), pack2<kBf16>(b.x, b.y), pack2<kBf16>(b.z, b.w));
        }
      }
    }
    __syncwarp();
  }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1)
    paged_wide_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ WideParams w) {
  using C = Cfg<D>;
  constexpr int S = C::kStages;
  constexpr uint32_t kIdescS = make_idesc(1, kBf16 ? 1 : 0, kBf16 ? 1 : 0, 0, 0, kTileM, kBlockN);
  constexpr uint32_t kIdescO = make_idesc(1, kBf16 ? 1 : 0, kBf16 ? 1 : 0, 0, 1, kTileM, D);
  const Params& p = w.p;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                  // [2][kTile]
  uint8_t* sRing = smem + 2 * C::kTile;  // [S][kTile]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRing + S * C::kTile);
  uint64_t* q_full = bars;           // [2]  the softmax warps of tile t have written Q_t
  uint64_t* kv_full = q_full + 2;    // [S]
  uint64_t* kv_empty = kv_full + S;  // [S]
  uint64_t* s_full = kv_empty + S;   // [2]  S_t in TMEM, PV_t of the block before complete
  uint64_t* p_half = s_full + 2;     // [2]  keys 0-63 of P_t in TMEM, O_t rescaled
  uint64_t* p_full = p_half + 2;     // [2]  all of P_t
  uint64_t* o_full = p_full + 2;     // [2]  the item's last PV_t complete
  uint64_t* fix = o_full + 2;        // [1]  a V tile that needs zeros has landed
  uint64_t* meet_bar = fix + 1;      // [1]  the eight softmax warps meet
  uint64_t* drain = meet_bar + 1;    // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile Walk* walks = reinterpret_cast<volatile Walk*>(drain + 2);  // [8] of the softmax warps
  int* scratch = reinterpret_cast<int*>(sQ);  // before the pipeline starts

  const int warp = warp_id();
  const int lane = threadIdx.x & 31;
  griddep_launch_dependents();

  // ------------------------------------------------------------------ this block's share
  Line line;
  Item first;
  int c, line_id = 0;
  int j_first, u0, todo;
  if (w.prefix_pass) {
    c = blockIdx.x;
    if (w.lines > 1) {
      c = (int)((unsigned)blockIdx.x / (unsigned)w.lines);
      line_id = blockIdx.x - c * w.lines;
    }
    first.keys = p.prefix;
    first.visible = p.prefix;
    first.units = p.pre.units;
    const int items = p.Hk * (w.lines > 1 ? 1 : w.pairs), line_units = first.units * items;
    int nc = p.pre.nc;
    if (yields(p.pre, line_units)) {
      int units = 0;  // of one item of each sequence
      for (int b = threadIdx.x; b < p.B; b += kThreads) units += units_of(own_length(p, b), p.pre.own_shift);
#pragma unroll
      for (int o = 16; o; o >>= 1) units += __shfl_xor_sync(~0u, units, o);
      if (lane == 0) scratch[warp] = units;
      __syncthreads();
      units = 0;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) units += scratch[i];
      const int each = own_items(p);
      nc = yielding_blocks(p.pre, p.sms, line_units, own_bytes(p, units * each, each));
    }
    const int per_item = (brief(p.pre, line_units) || !p.pre.own_shift) ? blocks_per_item(items, first.units, nc) : 0;
    if (!per_item) {  // no more blocks than the longest share needs
      const int longest = up_div(line_units, nc);
      nc = up_div(line_units, longest);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.counters[kPrefixBlocks] = per_item ? -per_item : nc;
    if (c >= nc) return;
    int item;
    if (per_item) {
      line.cut(first.units, per_item);
      item = (int)((unsigned)c / (unsigned)per_item);
      j_first = line.begin(c - item * per_item);
      u0 = item * first.units + j_first;
      todo = line.begin(c - item * per_item + 1) - j_first;
    } else {
      line.cut(line_units, nc);
      u0 = line.begin(c), todo = line.begin(c + 1) - u0;
      item = (int)((unsigned)u0 / (unsigned)first.units);
      j_first = u0 - item * first.units;
    }
    first.b = 0;
    first.hk = item;
    first.pair = line_id;
    if (w.lines == 1 && w.pairs > 1) {
      first.hk = item / w.pairs;
      first.pair = item - first.hk * w.pairs;
    }
  } else {
    c = blockIdx.x;
    int2* found = reinterpret_cast<int2*>(scratch + kThreads / 32);
    // Units of one K/V head of a sequence.
    auto per_head = [&](int L) {
      int sum = 0;
#pragma unroll 1
      for (int x = 0; x < w.pairs; ++x) sum += units_of_keys(visible_keys(w, L, x));
      return sum;
    };
    // A share costs about a unit's time when it is joined, and the shares of an item are joined one
    // after the other: units / nc + nc / items is least at this nc.  (64 tokens of 32/8
    // heads at 2000 keys: 44 us, against 54 where a join counts two units and 58 where it counts a half; at
    // 8000 keys 81, 75 and 87.)
    const float items = (float)p.B * p.Hk * w.pairs;
    locate<kThreads, 1>(
        p.B, c, scratch, found, line, [&](int b) { return per_head(own_length(p, b)) * p.Hk; },
        [&](int units) { return min((int)gridDim.x, (int)(sqrtf(units * items * (1.f / kJoinUnits)) + 1.f)); });
    if (c >= line.nc) return;
    first.b = found->x;
    first.keys = own_length(p, first.b);
    const int each = per_head(first.keys);
    first.hk = (int)((unsigned)found->y / (unsigned)each);
    j_first = found->y - first.hk * each;
    first.pair = 0;
    enter(w, first);
    while (j_first >= first.units) {
      j_first -= first.units;
      ++first.pair;
      enter(w, first);
    }
    u0 = line.begin(c), todo = line.begin(c + 1) - u0;
    __syncthreads();  // the scratch is Q's
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 4);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_half[t], 4);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(fix, 1);
    mbar_init(meet_bar, 8);
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Key blocks of the item's share [j0, j1) that tile t takes: from `from` to `to` in steps of
  // `halves` (none where from >= to).
  const int step = w.halves;
  auto tile_rows_begin = [&](const Item& it, int t) {  // first row of tile t
    return step == 2 ? it.pair * kTileM : (it.pair * 2 + t) * kTileM;
  };
  auto tile_units = [&](const Item& it, int t) {  // key blocks that tile t's last row sees, at least one
    const int begin = tile_rows_begin(it, t);
    if (begin >= w.rows) return 0;
    if (w.prefix_pass) return it.units;
    return units_of_keys(max(0, it.keys - p.n + p.by_G.div(min(w.rows, begin + kTileM) - 1) + 1));
  };
  auto tile_range = [&](const Item& it, int t, int j0, int j1, int& from, int& to) {
    from = step == 2 ? j0 + ((j0 ^ t) & 1) : j0;
    to = min(j1, tile_units(it, t));
  };

  if (warp == 8) {
    // ---------------------------------------------------------------- TMA producer
    // Ring items in the order that the MMAs take them.  One tile after the other on a block:
    // K_0 V_0 K_1 V_1 ...; with two halves S of the next block goes before PV of this one:
    // K_0 K_1 V_0 K_2 V_1 ... K_last V_last-1 V_last (any other order leaves a load waiting for
    // a slot that is freed only when it is needed).
    bool ok = true;
    int issued = 0, fixes = 0;
    const int box = w.box_rows, boxes = kBlockN / box;
    Item it = first;
    int j = j_first;
    // Lane g has box g of a block: its page (-1: behind the last key) and the row in it.  Looked
    // up a block ahead, and not looked at before its turn: the load takes longer than an issue.
    auto look_up = [&](int& in) {
      const int t = j * kBlockN + lane * box;
      in = 0;
      if (lane >= boxes || t >= it.keys) return -1;
      const int col = p.by_page.div(t);
      in = t - col * p.page_size;
      return w.prefix_pass ? p.prefix_pages[col] : p.table[it.b * p.table_ld + col];
    };
    // K or V of a block: `page` and `in` are this lane's box, `have` the keys that it holds.
    auto copy = [&](bool is_v, int page, int in, int hk, int have) {
      const int slot = issued % S;
      if (!mbar_wait_warp(&kv_empty[slot], ((issued / S) & 1) ^ 1u, kSiteEmpty)) return false;
      // The box that holds the sequence's end is partly not its: V gets zeros there.
      const bool mend = is_v && have < kBlockN && have > 0 && have % box != 0;
      uint64_t* bar = mend ? fix : &kv_full[slot];
      uint8_t* dst = sRing + slot * C::kTile;
      if (lane == 0) mbar_arrive_expect_tx(bar, C::kTile);
      __syncwarp();
      if (lane < boxes) {
        const CUtensorMap* tm = is_v ? &tmV : &tmK;
#pragma unroll
        for (int x = 0; x < C::kBoxes; ++x)
          tma_load_4d(dst + x * (kTileM * 128) + lane * box * 128, tm, bar, 64 * x, in, hk, page);
      }
      ++issued;
      if (!mend) return true;
      const bool landed = __all_sync(0xffffffffu, mbar_wait_drain(fix, fixes & 1, kSiteFix));
      ++fixes;
      const int end = (have + box - 1) / box * box;
      for (int i = lane; i < (end - have) * C::kBoxes * 8; i += 32) {
        const int r = have + i / (C::kBoxes * 8), piece = i % (C::kBoxes * 8);
        *reinterpret_cast<uint4*>(dst + (piece >> 3) * (kTileM * 128) + r * 128 + (piece & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&kv_full[slot]);
      return landed;
    };
    int in_next, page_next = look_up(in_next);
    int v_page = 0, v_in = 0, v_have = 0;  // two halves: the block whose V is still to come
    for (int done = 0; done < todo && ok; ++done) {
      const int in = in_next, hk = it.hk, have = it.keys - j * kBlockN;
      const bool begins = done == 0 || j == 0, ends = j + 1 == it.units || done + 1 == todo;
      const bool held = lane < boxes && lane * box < have;
      int page = page_next;
      if (done + 1 < todo) {
        if (++j == it.units) {
          next_item(w, it);
          j = 0;
        }
        page_next = look_up(in_next);
      }
      if ((unsigned)page >= (unsigned)p.num_pages) {
        if (held) record_bad_index(kSitePage);
        page = p.num_pages;  // out of range: zeros
      }
      ok = copy(false, page, in, hk, have);
      if (step == 2) {
        if (ok && !begins) ok = copy(true, v_page, v_in, hk, v_have);
        v_page = page, v_in = in, v_have = have;
      }
      if (ok && (step == 1 || ends)) ok = copy(true, page, in, hk, have);
    }
    // Every copy issued must land before the block can exit.
    for (int i = (issued > S ? issued - S : 0); i < issued; ++i)
      mbar_wait_drain(&kv_full[i % S], (i / S) & 1, kSiteTeardown);
  } else if (warp == 9) {
    // ---------------------------------------------------------------- MMA issuer (whole warp)
    // Every instruction between a softmax warp's arrival and the MMAs that answer it is on the
    // chain of a tile's blocks, so the ring is walked by one running slot (items are taken in the
    // order that they were loaded) and the descriptors are advanced, not built.
    bool ok = true;
    const uint64_t q_desc[2] = {sdesc_sw128(smem_u32(sQ), 16, 1024),
                                step == 2 ? sdesc_sw128(smem_u32(sQ), 16, 1024)
                                          : sdesc_sw128(smem_u32(sQ + C::kTile), 16, 1024)};
    const uint64_t ring_k = sdesc_sw128(smem_u32(sRing), 16, 1024);
    const uint64_t ring_v = sdesc_sw128(smem_u32(sRing), kTileM * 128, 1024);
    int slot = -1;
    uint32_t par = 1;       // of the slot's phase in use
    uint32_t p_par = 0;     // bit t: parity of tile t's next P
    uint32_t q_par = 0;     // bit t: parity of tile t's next Q
    auto take = [&]() {     // the next ring item
      if (++slot == S) slot = 0;
      if (slot == 0) par ^= 1;
      return slot;
    };
    auto landed = [&](int at) {
      ok = mbar_wait_warp(&kv_full[at], par, kSiteKV);
      tc_fence_after();
      return ok;
    };
    auto issue_s = [&](int t, int at) {
      const uint64_t kd = sdesc_add(ring_k, at * C::kTile);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint32_t off = (ks >> 2) * (kTileM * 128) + (ks & 3) * 32;
        mma_f16_ss_warp(tmem + t * kBlockN, sdesc_add(q_desc[t], off), sdesc_add(kd, off), kIdescS, ks > 0);
      }
      tc_commit_warp(&s_full[t]);
    };
    auto issue_pv = [&](int t, uint64_t vd, int ks0, int ks1, bool add) {
#pragma unroll
      for (int ks = ks0; ks < ks1; ++ks)
        mma_f16_ts_warp(tmem + C::kOCol + t * D, tmem + t * kBlockN + ks * 8, sdesc_add(vd, ks * 16 * 128), kIdescO,
                        (add || ks > 0) ? 1u : 0u);
    };
    Item it = first;
    int j0 = j_first;
    for (int done = 0; done < todo && ok;) {
      const int seg = min(it.units - j0, todo - done), j1 = j0 + seg;
      int from[2], to[2];
      for (int t = 0; t < 2; ++t) tile_range(it, t, j0, j1, from[t], to[t]);
      // Q_t is in (its softmax warps write it once the item before is done with it).
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (ok && (step == 2 ? t == 0 : from[t] < to[t])) {
          ok = mbar_wait_warp(&q_full[t], (q_par >> t) & 1, kSiteQ);
          q_par ^= 1u << t;
        }
      tc_fence_after();
      // The first S of each tile.
      for (int i = 0; i < min(step, seg) && ok; ++i) {
        const int at = take();
        if (!landed(at)) break;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (from[t] == j0 + i && from[t] < to[t]) issue_s(t, at);
        tc_commit_warp(&kv_empty[at]);
      }
#pragma unroll 1
      for (int j = j0; j < j1 && ok; ++j) {
        // V_j, and K of the block that its tiles take next.
        const int v_at = take();
        if (!landed(v_at)) break;
        const uint64_t vd = sdesc_add(ring_v, v_at * C::kTile);
        const bool more = j + step < j1;
        int k_at = 0;
        bool k_in = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || j < from[t] || j >= to[t] || (step == 2 && ((j ^ t) & 1))) continue;
          const uint32_t pp = (p_par >> t) & 1;
          p_par ^= 1u << t;
          if (!(ok = mbar_wait_warp(&p_half[t], pp, kSiteP))) break;
          tc_fence_after();
          issue_pv(t, vd, 0, kBlockN / 32, j > from[t]);
          if (!(ok = mbar_wait_warp(&p_full[t], pp, kSiteP))) break;
          tc_fence_after();
          issue_pv(t, vd, kBlockN / 32, kBlockN / 16, j > from[t]);
          if (j + step < to[t]) {
            // Behind PV_t(j) in issue order: S_t overwrites P_t only once that has read it.
            if (!k_in) {
              k_at = take();
              k_in = true;
              if (!landed(k_at)) break;
            }
            issue_s(t, k_at);
          } else {
            tc_commit_warp(&o_full[t]);
          }
        }
        if (!ok) break;
        tc_commit_warp(&kv_empty[v_at]);
        if (more) {
          if (!k_in) {  // no tile takes it
            k_at = take();
            if (!landed(k_at)) break;
          }
          tc_commit_warp(&kv_empty[k_at]);
        }
      }
      done += seg;
      j0 = 0;
      if (done < todo) next_item(w, it);
    }
    tc_commit_warp(drain);
    mbar_wait_drain(drain, 0, kSiteTeardown);
  } else {
    // ---------------------------------------------------------------- softmax (warps 0-7)
    const int t = warp >> 2, quad = warp & 3;
    const int r = quad * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t s_tmem = tmem + lane_off + t * kBlockN;
    const uint32_t o_tmem = tmem + lane_off + C::kOCol + t * D;
    bool ok = true;
    uint32_t phase = 0;  // parities of the waits for s_full (bit 0), o_full (1) and meet_bar (2)
    auto meet = [&]() {  // a bounded barrier of the softmax warps
      __syncwarp();
      if (lane == 0) mbar_arrive(meet_bar);
      const bool r = mbar_wait_warp(meet_bar, (phase >> 2) & 1, kSiteMeet);
      phase ^= 4;
      return r;
    };
    volatile Walk* walk = walks + warp;
    if (lane == 0) {
      walk->it.b = first.b, walk->it.hk = first.hk, walk->it.pair = first.pair;
      walk->it.units = first.units, walk->it.keys = first.keys, walk->it.visible = first.visible;
      walk->j0 = j_first, walk->done = 0, walk->todo = todo, walk->c = c, walk->line_id = line_id;
      walk->item = !w.prefix_pass ? 0 : (w.lines > 1 ? first.hk : first.hk * w.pairs + first.pair);
      walk->unit = u0;
      walk->line.q = line.q, walk->line.more = line.more, walk->line.nc = line.nc;
    }
    __syncwarp();
    auto item_now = [&]() {
      Item i;
      i.b = walk->it.b, i.hk = walk->it.hk, i.pair = walk->it.pair;
      i.units = walk->it.units, i.keys = walk->it.keys, i.visible = walk->it.visible;
      return i;
    };
    while (ok && walk->done < walk->todo) {
      int from, to, lim;
      {
        // What an item needs outside the softmax loop is derived from these copies, which the
        // compiler cannot see through: what it could hoist out of the walk would sit in the loop's
        // registers (a row of S takes 128 of 168) and push others into memory, 20% of its time.
        int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        asm volatile("" : "+r"(lane), "+r"(warp));
        const int t = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
        const Item it = item_now();
        const int j0 = walk->j0, seg = min(it.units - j0, walk->todo - walk->done);
        tile_range(it, t, j0, j0 + seg, from, to);
        const int row_begin = tile_rows_begin(it, t), row = row_begin + r;
        const bool live = row < w.rows;
        const Row at = query_row(w, it, live ? row : 0);
        // Keys that this row sees; -1 in a warp without a query.
        lim = row_begin + quad * 32 >= w.rows ? -1 : !live ? 0 : (w.prefix_pass ? it.keys : max(0, it.keys - p.n + at.i + 1));
        // Q_t is written for every share that its MMAs take part in.  (With two halves both tiles
        // read Q_0, and the halves meet at the end of each item, so it is idle here.)
        if (step == 2 ? t == 0 : from < to) {
          // A warp copies its 32 rows, whole rows at a time; all the copies are in flight at once (a
          // round trip to memory is over a microsecond here, and this one is on the way of every
          // share).
          constexpr int kPieces = D / 8;  // 16-byte pieces of a row
          const int piece = lane % kPieces;
#pragma unroll 4
          for (int x = lane / kPieces; x < 32; x += 32 / kPieces) {
            const int tile_row = quad * 32 + x;
            const bool in = row_begin + tile_row < w.rows && piece * 8 < p.D;
            const Row from_q = query_row(w, it, in ? row_begin + tile_row : 0);
            const uint16_t* src = static_cast<const uint16_t*>(p.q) + (in ? from_q.b * p.q_sb + from_q.i * p.q_ss +
                                                                                from_q.head * p.q_sh + piece * 8
                                                                          : 0);
            cp16(smem_u32(sQ + t * C::kTile + (piece >> 3) * (kTileM * 128) + tile_row * 128) +
                     (((piece & 7) ^ (tile_row & 7)) << 4),
                 src, in);
          }
          cp_commit();
          cp_wait<0>();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[t]);
        }
      }
      const bool any = from < to;
      float m_used = -INFINITY, l = 0.f;
      if (lim < 0) {  // no query in this warp's rows: what P holds there reaches no result
#pragma unroll 1
        for (int j = from; j < to && ok; j += step) {
          ok = mbar_wait_warp(&s_full[t], phase & 1, kSiteS);
          phase ^= 1;
          if (ok && lane == 0) {
            mbar_arrive(&p_half[t]);
            mbar_arrive(&p_full[t]);
          }
        }
        from = to;
      }
#pragma unroll 1
      for (int j = from; j < to; j += step) {
        if (!mbar_wait_warp(&s_full[t], phase & 1, kSiteS)) {
          ok = false;
          break;
        }
        phase ^= 1;
        tc_fence_after();
        uint32_t sr[kBlockN];
        const int n0 = j * kBlockN;
#pragma unroll
        for (int x = 0; x < kBlockN / 32; ++x) tmem_ld32(s_tmem + x * 32, *reinterpret_cast<uint32_t(*)[32]>(&sr[x * 32]));
        tmem_wait_ld();
        if (n0 + kBlockN > lim) {
#pragma unroll
          for (int x = 0; x < kBlockN; ++x)
            if (n0 + x >= lim) sr[x] = __float_as_uint(-INFINITY);
        }
        const float m_new = row_max<kBlockN>(sr) * p.scale_log2;
        const bool need = m_new > m_used + kLazy;
        // A row without a maximum so far holds nothing (in its first block, not even O).
        const bool warp_rescale = __any_sync(0xffffffffu, need && m_used != -INFINITY);
        float alpha = 1.f;
        if (need) {
          alpha = fa::ex2(m_used - m_new);  // 0 where m_used is -inf
          m_used = m_new;
        }
        l *= alpha;
        const float ref = m_used == -INFINITY ? 0.f : m_used;
        const uint64_t sc2 = f2(p.scale_log2, p.scale_log2);
        const uint64_t ng2 = f2(-ref, -ref);
        uint64_t rs2 = f2(0.f, 0.f);
        uint32_t pk[kBlockN / 2];
#pragma unroll
        for (int e = 0; e < kBlockN / 2; ++e) {
          const uint64_t x2 = fma2(f2(__uint_as_float(sr[2 * e]), __uint_as_float(sr[2 * e + 1])), sc2, ng2);
          float x0, x1;
          uf2(x2, x0, x1);
          const float p0 = fa::ex2(x0), p1 = fa::ex2(x1);
          rs2 = add2(rs2, f2(p0, p1));
          pk[e] = pack2<kBf16>(p0, p1);  // rounded for the matrix product; the sum is of the unrounded
          if (e == kBlockN / 4 - 1) {
            tmem_st32(s_tmem, *reinterpret_cast<const uint32_t(*)[32]>(&pk[0]));
            if (warp_rescale) {
#pragma unroll 1
              for (int x = 0; x < D / 32; ++x) {
                uint32_t ov[32];
                tmem_ld32(o_tmem + x * 32, ov);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
                tmem_st32(o_tmem + x * 32, ov);
              }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_half[t]);
          }
        }
        float rs0, rs1;
        uf2(rs2, rs0, rs1);
        l += rs0 + rs1;
        tmem_st32(s_tmem + 32, *reinterpret_cast<const uint32_t(*)[32]>(&pk[32]));
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      if (any) {
        if (!(ok = mbar_wait_warp(&o_full[t], (phase >> 1) & 1, kSiteO))) break;
        phase ^= 2;
        tc_fence_after();
      }
      // A row that saw no key has m = -inf, l = 0; one whose scores were not numbers stays so.
      if (l != l) m_used = fmaxf(m_used, 0.f);

      // ------------------------------------------------------------ results of the share
      int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
      asm volatile("" : "+r"(lane), "+r"(warp));
      const int t = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
      const uint32_t lane_off = (uint32_t)(quad * 32) << 16, s_tmem = tmem + lane_off + t * kBlockN;
      const Item it = item_now();
      const int j0 = walk->j0, seg = min(it.units - j0, walk->todo - walk->done), item = walk->item;
      Line ln;
      ln.q = walk->line.q, ln.more = walk->line.more, ln.nc = walk->line.nc;
      const int item0 = walk->unit - j0;
      const int me = walk->c, cf = ln.block_of(item0), cl = ln.block_of(item0 + it.units - 1);
      // A whole item is written at once.  A part of one is left as a share in the workspace, and
      // the warp that leaves the last share of its rows (and columns; each warp has a counter of
      // its own, nobody waits for anybody) joins them, in block order.  The later of only two
      // adds the other's share to the O that it has: that sum is the same either way round.
      const bool split = !w.prefix_pass && cf != cl, two = cl - cf == 1;
      int* counter = p.counters + cf * 8 + warp;
      bool all_in = false;
      if (split && two) {
        int arrived = 0;
        if (lane == 0) arrived = ld_acquire_gpu(counter);
        all_in = __shfl_sync(~0u, arrived, 0) != 0;
        __threadfence();
      }
      const bool leave = w.prefix_pass || (split && !all_in);
      const int row_begin = tile_rows_begin(it, step == 2 ? 0 : t);
      const int quad_rows = max(0, min(32, w.rows - row_begin - quad * 32));  // queries among this warp's rows
      auto slot_of = [&](int x) {
        return w.prefix_pass ? prefix_slot<D>(p.pre, p.Hk, walk->line_id, item, x)
                             : p.partial + (int64_t)(2 * x + (x == cf ? 1 : 0)) * kSlotFloats<D>;
      };
      // With two halves the tiles' warps read both O_0 and O_1 (the same TMEM lanes).
      float m_row = m_used, l_row = l, w0 = 1.f, w1 = 0.f;
      bool any0 = t == 0 && any, any1 = t == 1 && any;
      if (step == 2) {
        uint32_t ml[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) ml[i] = 0;
        ml[0] = __float_as_uint(m_used), ml[1] = __float_as_uint(l);
        tmem_st32(s_tmem, ml);  // S_t is idle: every MMA of the item is complete
        tmem_wait_st();
        tc_fence_before();
        if (!(ok = meet())) break;
        tc_fence_after();
        tmem_ld32(tmem + lane_off + (1 - t) * kBlockN, ml);
        tmem_wait_ld();
        const float m_o = __uint_as_float(ml[0]), l_o = __uint_as_float(ml[1]);
        m_row = fmaxf(m_used, m_o);
        const float mine = weight(m_used, m_row), other = weight(m_o, m_row);
        l_row = mine * l + other * l_o;
        w0 = t == 0 ? mine : other, w1 = t == 0 ? other : mine;
        // Whether a tile took a block at all: the same for all its rows.
        any0 = j0 + (j0 & 1) < j0 + seg, any1 = j0 + 1 - (j0 & 1) < j0 + seg;
      } else {
        w0 = w1 = m_used == -INFINITY ? 0.f : 1.f;
      }
      HandOn<D> h;
      h.w = &w, h.it = it, h.sQ = sQ, h.tmem = tmem;
      h.m_row = m_row, h.l_row = l_row, h.w0 = w0, h.w1 = w1, h.any0 = any0, h.any1 = any1;
      h.row_begin = row_begin, h.quad_rows = quad_rows;
      h.cf = cf, h.cl = cl, h.me = me;
      if (quad_rows > 0) {
        bool result = !leave;
#pragma unroll 1
        for (bool again = true; again;) {
          hand_on<D, kBf16>(h, result ? nullptr : slot_of(me), lane, warp);
          again = false;
          if (!split) break;
          if (result) {
            if (lane == 0) *counter = 0;
          } else {
            int last = 0;
            if (lane == 0) {
              __threadfence();
              last = atomicAdd(counter, 1) == cl - cf;
            }
            // All shares are there now: join them (of two, the other's, O being still here).
            result = again = __shfl_sync(~0u, last, 0) != 0;
            if (again) __threadfence();
          }
        }
      }
      // O_t has been read: the next item's first PV_t may overwrite it once p_half says so.  With
      // two halves the other tile's warps read it too, and Q_0 is shared.
      tc_fence_before();
      if (step == 2)
        if (!(ok = meet())) break;
      // Past this item's share.
      Item nx = it;
      const bool more = walk->done + seg < walk->todo;
      if (more) next_item(w, nx);
      __syncwarp();
      if (lane == 0) {
        walk->it.b = nx.b, walk->it.hk = nx.hk, walk->it.pair = nx.pair;
        walk->it.units = nx.units, walk->it.keys = nx.keys, walk->it.visible = nx.visible;
        walk->j0 = 0, walk->item = item + 1;
        walk->unit = walk->unit + seg;
        walk->done = walk->done + seg;
      }
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
  // The join of the prefix's shares waits for this kernel, and by its first block for the prefix pass
  // before it.
  if (!w.prefix_pass && p.row_share && blockIdx.x == 0) griddep_wait();
}

template <int D, bool kBf16>
int launch(const CUtensorMap& tk, const CUtensorMap& tv, const WideParams& w, int grid, bool dependent, cudaStream_t s) {
  auto kern = paged_wide_kernel<D, kBf16>;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem);
    if (e != cudaSuccess) return cuda_status(e);
    configured.fetch_or(bit);
  }
  return launch_kernel(kern, grid, kThreads, Cfg<D>::kSmem, dependent, s, tk, tv, w);
}

// Cache pages as a [page][head][row][d] tensor, boxes of 64 values x box_rows rows.
int page_map(CUtensorMap* map, bool bf16, const void* base, const Params& p, int64_t sp, int64_t ss, int64_t sh, int box_rows) {
  const uint64_t dims[4] = {(uint64_t)p.D, (uint64_t)p.page_size, (uint64_t)p.Hk, (uint64_t)p.num_pages};
  const uint64_t strides[3] = {(uint64_t)ss * 2, (uint64_t)sh * 2, (uint64_t)sp * 2};
  const uint32_t box[4] = {64, (uint32_t)box_rows, 1, 1};
  return make_tmap(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims, strides, box,
                   CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

int wide_box_rows(int page_size) {
  int r = 1;
  while (r < 128 && page_size % (2 * r) == 0) r *= 2;
  return r >= 8 ? r : 0;
}

int launch_wide(const Params& p, bool bf16, bool prefix_pass, int64_t max_units, cudaStream_t s) {
  WideParams w{};
  w.p = p;
  w.prefix_pass = prefix_pass;
  w.rows = prefix_pass ? p.B * p.rows : p.rows;
  w.halves = w.rows <= kTileM ? 2 : 1;
  const int64_t tile = w.halves == 2 ? kTileM : 2 * kTileM;
  w.pairs = (int)((w.rows + tile - 1) / tile);
  w.box_rows = wide_box_rows(p.page_size);
  w.lines = 1;
  int64_t grid = sm_count();
  if (prefix_pass) {
    w.lines = p.pre.lines;
    grid = (int64_t)p.pre.lines * p.pre.nc;
  } else if (grid > max_units) {
    grid = max_units;
  }
  // Test hook (lk_debug_inject): boxes of half the rows bring fewer bytes than the barriers wait for.
  const Injection inj = take_injection(LK_INJECT_PAGED_DROP_LOAD);
  auto rows_of = [&](int which) { return inj.kind && inj.item == which ? w.box_rows / 2 : w.box_rows; };
  CUtensorMap tk, tv;
  if (int st = page_map(&tk, bf16, p.k, p, p.k_sp, p.k_ss, p.k_sh, rows_of(0))) return st;
  if (int st = page_map(&tv, bf16, p.v, p, p.v_sp, p.v_ss, p.v_sh, rows_of(1))) return st;
  const bool dependent = !prefix_pass && p.row_share != nullptr;
  if (p.D > 64)
    return bf16 ? launch<128, true>(tk, tv, w, (int)grid, dependent, s) : launch<128, false>(tk, tv, w, (int)grid, dependent, s);
  return bf16 ? launch<64, true>(tk, tv, w, (int)grid, dependent, s) : launch<64, false>(tk, tv, w, (int)grid, dependent, s);
}

}  // namespace paged
}  // namespace lk
