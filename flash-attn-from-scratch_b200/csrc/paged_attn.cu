// paged_attn.cu — attention of each sequence's newest tokens to its pages of a key/value cache:
// the kernel for up to 16 query rows per K/V head (single tokens, drafted tokens).
//
// Query i of the n newest tokens of a sequence of L keys sees its keys below L - n + i + 1 (and,
// with a shared prefix, all of the prefix):  o = sum_j p_j v_j / sum_j p_j with
// p_j = exp(scale q.k_j - m), lse = m + ln sum_j p_j; a row that sees nothing gives 0 and -inf.
//
// Bound: memory.  Each key and value is read once for at most 16 rows (4 D bytes for 64 D flops
// per key and head at 16 rows: 16 flop/byte, and the card's balance is ~250), so the work is to
// keep reads in flight.  The warps of a block run without any barrier between them until an item
// ends: a warp takes 16 keys a step, has its own ring of stages in shared memory, filled by
// 16-byte cp.async -- row by row through the block table, so pages of any size and caches of any
// stride take the same path, and rows behind the last key are filled with zeros instead of read
// -- and its own running (m, l, O), kept in registers.  The rows of a K/V head's query group fill
// the 16 rows of mma.sync's A operand, and S's accumulator layout is P's operand layout, so P
// never leaves registers.  (tcgen05 would need 128 rows and a trip
// through tensor memory for the same 16; its throughput is not what bounds this kernel.)
// Loads run ahead across the ends of items, so short sequences do not drain the ring.
//
// A team is the warps that share an item: four where there are few items (their shares meet in
// shared memory, a quarter as many go through the workspace), one where there are many (an item's
// end then holds up one warp, not four).
//
// Measured (B200, 32/8 heads, D = 128, bf16): 64 sequences of 200-8192 keys 188-195 us, 5.8-5.9 TB/s of
// K and V (a copy runs at 6.5); at 6000 keys each time grows by 6.6 TB/s, on top of 16-18 us that the
// chain lengths -> table -> first keys, the joins and the launch take.  One sequence of 1000 keys:
// 7.5 us, all of it such chains.
#include <atomic>

#include "lk_abi.h"
#include "paged_common.cuh"

namespace lk {
namespace paged {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kGroup = 16;             // keys of one warp's step
// log2 of the keys of a team's step, its unit: 16 keys a warp.
constexpr int team_shift(int team) { return team == 1 ? 4 : 6; }
static_assert(1 << team_shift(1) == kGroup && 1 << team_shift(kWarps) == kWarps * kGroup, "units of a team's warps");
constexpr float kLazy = 8.0f;  // log2 units that the maximum may grow by before O is rescaled
// Units of 64 prefix keys, over all sequences, K/V heads and tiles of 16 query rows, above which the
// prefix pass pays; below, each tile reads the prefix itself, mostly from L2, in one kernel.  One tile
// alone shares nothing.  (32/8 heads, D = 128, one kernel against the pass.  16 single tokens: 256 keys
// 17 us against 19, 1024 keys, 2048 units, 21 either way, 4096 keys 46 against 23.  20 tokens of each of
// two sequences: 512 keys, 640 units, 19 either way, 4096 keys 38 against 25.  One piece of 500 tokens:
// 64 keys 53 against 61, 256 keys, 4000 units, 63 either way, 8192 keys 484 against 126.  Of 252 calls
// of 1-32 sequences, 1-500 tokens, 64-16384 keys and five head layouts the rule's choice takes 2.5% more
// than the better one, 41% at most; at 2048 units it is 2.7%, 96% at most, at 6144 4.5%.)
constexpr int64_t kPrefixPass = 3072;
// Items from which a team is one warp.  (4 tokens of each of 16 sequences of 4-2999 keys, 16/16 heads, D = 64:
// 31 us against 41 with teams of four; 32 sequences of 500 keys, 32/8 heads, 21 against 23; 64 of 6000 keys 266
// against 270; one sequence of 1000 keys 23 with teams of one, 10 with teams of four.)
constexpr int64_t kManyItems = 256;
// Two tiles of 16 rows read their keys twice, but this kernel starts and joins faster than the one
// of 256 rows: up to so many keys times K/V heads they take this one.  (32 rows: 8 heads of 8000 keys
// 29 us against 54, 64 of 2000 33 against 44, 64 of 8000 104 against 83, 512 of 2000 191 against 156.)
constexpr int64_t kTwoTileKeys = 1 << 18;

template <int DP>
struct Cfg {
  static constexpr int kStages = DP == 128 ? 3 : 6;          // of a warp's ring: 24 KB
  static constexpr int kTile = kGroup * DP * 2;              // bytes of a warp's K or V tile
  static constexpr int kRing = kWarps * kStages * 2 * kTile;
  static constexpr int kJoin = kWarps * 8 * DP * 4;          // 8 rows of every warp's O
  static constexpr int kSmem = kRing + kJoin + kWarps * kRows * 2 * 4;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A place on the line of units: a team's step is 2^kShift keys.
template <int kShift>
struct Place {
  int b, hk, rt;  // item: sequence, K/V head, tile of 16 rows
  int j, units;   // unit of the item, and how many it has
  int keys;       // prefix + own keys of the sequence
  __device__ __forceinline__ void enter(const Params& p) {
    keys = b < p.B ? p.prefix + own_length(p, b) : 0;
    units = units_of(keys, kShift);
  }
  __device__ __forceinline__ void advance(const Params& p, int tiles) {
    if (++j < units) return;
    j = 0;
    if (++rt < tiles) return;
    rt = 0;
    if (++hk < p.Hk) return;
    hk = 0;
    ++b;
    enter(p);
  }
};

template <int DP, bool kBf16, int kTeam>
__global__ void __launch_bounds__(kThreads, 2) paged_rows16_kernel(const Params p) {
  using C = Cfg<DP>;
  constexpr int kStages = C::kStages;
  constexpr int kShift = team_shift(kTeam), kUnit = 1 << kShift;
  constexpr int kTeams = kWarps / kTeam;   // of a block
  constexpr int kChunks = DP / 8;          // 16-byte pieces of a row
  constexpr int kPerCopy = 32 / kChunks;   // rows that one copy instruction of a warp covers
  constexpr int kPer = DP / 32;            // columns of a lane where a warp has whole rows
  griddep_launch_dependents();
  extern __shared__ __align__(128) uint8_t smem[];
  float* sO = reinterpret_cast<float*>(smem + C::kRing);              // [kWarps][8][DP], swizzled
  float* sM = reinterpret_cast<float*>(smem + C::kRing + C::kJoin);   // [kWarps][kRows]
  float* sL = sM + kWarps * kRows;
  __shared__ int s_last;
  __shared__ int2 s_found[kTeams];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int in_team = warp % kTeam;  // this warp's place in its team
  const int tiles = (p.rows + kRows - 1) / kRows;
  const int per_seq = own_items(p);
  const int c = blockIdx.x * kTeams + warp / kTeam;  // this warp's team
  Line line;
  locate<kThreads, kTeams>(
      p.B, blockIdx.x * kTeams, reinterpret_cast<int*>(sM), s_found, line,
      [&](int b) { return units_of(p.prefix + own_length(p, b), kShift) * per_seq; }, [&](int units) {
        // Beside a prefix pass that yields: as many blocks as run at once on the SMs it leaves (a
        // second wave of them would begin when it ends), unless this pass is much the longer one.
        const int line_units = p.pre.units * (p.pre.lines > 1 ? p.Hk : p.Hk * p.pre.pairs);
        if (!p.row_share || !yields(p.pre, line_units)) return (int)gridDim.x * kTeams;
        const float bytes = own_bytes(p, units, per_seq);
        const int kept = yielding_blocks(p.pre, p.sms, line_units, bytes), left = max(p.sms - kept * p.pre.lines, p.sms / kLeastShare);
        return bytes < kMuchLonger * left * kSmBytesPerNs * prefix_ns(p.pre, line_units, kept) ? left * 2 * kTeams
                                                                                       : (int)gridDim.x * kTeams;
      });
  if (c >= line.nc) return;
  Place<kShift> at;
  at.b = s_found[warp / kTeam].x;
  at.enter(p);
  const int offset = s_found[warp / kTeam].y;
  at.hk = (int)((unsigned)offset / (unsigned)at.units);
  at.j = offset - at.hk * at.units;
  at.rt = 0;
  if (tiles > 1) {
    const int item = at.hk;
    at.hk = item / tiles;
    at.rt = item - at.hk * tiles;
  }
  const int u0 = line.begin(c);
  const int todo = line.begin(c + 1) - u0;  // units of this team

  // ------------------------------------------------------------------ loads
  const uint32_t ring = smem_u32(smem) + warp * (kStages * 2 * C::kTile);
  const int chunk = lane % kChunks, sub = lane / kChunks;
  const bool chunk_in = chunk * 8 < p.D;
  Place<kShift> ld = at;
  int ld_left = todo;
  // Lane l (and l + 16) looks up the page of key l of this warp's step, one step ahead; the entry
  // is not looked at before its turn.
  auto look_up = [&](int& in) {
    const int t = ld.j * kUnit + in_team * kGroup + (lane & 15);
    in = 0;
    if (ld_left <= 0 || t >= ld.keys) return -1;
    const int o = t - p.prefix, x = o < 0 ? t : o;
    const int col = p.by_page.div(x);
    in = x - col * p.page_size;
    return o < 0 ? p.prefix_pages[col] : p.table[ld.b * p.table_ld + col];
  };
  int in_next;
  int page = look_up(in_next);
  int ld_stage = 0;
  auto load = [&]() {
    if (ld_left > 0) {
      const bool held = (unsigned)page < (unsigned)p.num_pages;
      if (!held && ld.j * kUnit + in_team * kGroup + (lane & 15) < ld.keys) record_bad_index(kSitePage);
      const int64_t ok = held ? page * p.k_sp + in_next * p.k_ss + ld.hk * p.k_sh : -1;
      const int64_t ov = held ? page * p.v_sp + in_next * p.v_ss + ld.hk * p.v_sh : -1;
      const uint32_t dst = ring + ld_stage * (2 * C::kTile);
#pragma unroll
      for (int i = 0; i < kGroup / kPerCopy; ++i) {
        const int r = i * kPerCopy + sub;
        const int64_t rk = __shfl_sync(~0u, ok, r), rv = __shfl_sync(~0u, ov, r);
        const bool read = rk >= 0 && chunk_in;
        const uint32_t at_row = r * (DP * 2) + ((chunk ^ (r & 7)) << 4);
        cp16(dst + at_row, static_cast<const uint16_t*>(p.k) + (read ? rk + chunk * 8 : 0), read);
        cp16(dst + C::kTile + at_row, static_cast<const uint16_t*>(p.v) + (read ? rv + chunk * 8 : 0), read);
      }
      ld.advance(p, tiles);
      --ld_left;
      page = look_up(in_next);
      ld_stage = ld_stage + 1 == kStages ? 0 : ld_stage + 1;
    }
    cp_commit();
  };
#pragma unroll 1
  for (int i = 0; i < kStages - 1; ++i) load();

  // ------------------------------------------------------------------ items
  int stage = 0, unit = u0;
  const int r0 = lane >> 2;  // this lane's rows: r0 and r0 + 8
  for (int done = 0; done < todo;) {
    const int seg = min(at.units - at.j, todo - done);  // units of this item here
    // Q: row r of the tile is query row rt * 16 + r = token i, head g of the group.
    uint32_t qf[DP / 16][4];
    int lim[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = at.rt * kRows + r0 + 8 * h;
      const bool in = row < p.rows;
      const int i = in ? p.by_G.div(row) : 0, g = in ? row - i * p.G : 0;
      // Keys below lim are seen: the prefix and the own keys up to the token's own.
      lim[h] = p.prefix + max(0, at.keys - p.prefix - p.n + i + 1);
      const uint16_t* src = static_cast<const uint16_t*>(p.q) + at.b * p.q_sb + i * p.q_ss +
                            (int64_t)(at.hk * p.G + g) * p.q_sh + 2 * (lane & 3);
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        const int d = ks * 16 + 2 * (lane & 3);
        qf[ks][h] = in && d < p.D ? *reinterpret_cast<const uint32_t*>(src + ks * 16) : 0u;
        qf[ks][2 + h] = in && d + 8 < p.D ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8) : 0u;
      }
    }
    // Tokens see at least this many keys: steps below need no mask.
    const int all_see = p.prefix + max(0, at.keys - p.prefix - p.n + 1);
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

#pragma unroll 1
    for (int s = 0; s < seg; ++s) {
      cp_wait<kStages - 2>();
      __syncwarp();
      load();  // into the stage that the step before this one has read
      const uint32_t sk = ring + stage * (2 * C::kTile), sv = sk + C::kTile;
      stage = stage + 1 == kStages ? 0 : stage + 1;
      float x[2][4] = {};
      {
        // K rows are the B operand's columns: lane l addresses row (l & 7) + 8 (l >> 4) and the
        // 16-byte piece 2 ks + (l >> 3 & 1).
        const int r = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          uint32_t kf[4];
          ldsm4(sk + r * (DP * 2) + (((2 * ks + half) ^ (r & 7)) << 4), kf);
          mma16816<kBf16>(x[0], qf[ks], kf[0], kf[1]);
          mma16816<kBf16>(x[1], qf[ks], kf[2], kf[3]);
        }
      }
      const int t0 = (at.j + s) * kUnit + in_team * kGroup;
      if (t0 + kGroup > all_see) {
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t0 + nt * 8 + 2 * (lane & 3) + (e & 1) >= lim[e >> 1]) x[nt][e] = -INFINITY;
      }
      float top[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float t = fmaxf(fmaxf(x[0][2 * h], x[0][2 * h + 1]), fmaxf(x[1][2 * h], x[1][2 * h + 1]));
        t = fmaxf(t, __shfl_xor_sync(~0u, t, 1));
        t = fmaxf(t, __shfl_xor_sync(~0u, t, 2));
        top[h] = t * p.scale_log2;
      }
      // The maximum in use moves only when it is passed by more than 2^8: P stays below 2^8.
      if (__any_sync(~0u, top[0] > m[0] + kLazy || top[1] > m[1] + kLazy)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float now = fmaxf(m[h], top[h]);
          const float a = weight(m[h], now);
          m[h] = now;
          l[h] *= a;
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) o[i][2 * h] *= a, o[i][2 * h + 1] *= a;
        }
      }
      uint32_t pf[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float ref = m[h] == -INFINITY ? 0.f : m[h];
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = fa::ex2(fmaf(x[i >> 1][2 * h + (i & 1)], p.scale_log2, -ref));
        l[h] += (e[0] + e[1]) + (e[2] + e[3]);
        // P is rounded to the inputs' type for the matrix product; the sum l is of the unrounded.  (The
        // error is then 1.35 times that of a result rounded once.  With P in two parts, and two products,
        // 64 sequences of 200-8192 keys take 194 us instead of 188, one of 1000 keys 9.9 instead of 8.8.)
        pf[h] = pack2<kBf16>(e[0], e[1]);
        pf[2 + h] = pack2<kBf16>(e[2], e[3]);
      }
      {
        const int r = lane & 15, half = lane >> 4;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
          uint32_t vf[4];
          ldsm4_t(sv + r * (DP * 2) + (((2 * i + half) ^ (r & 7)) << 4), vf);
          mma16816<kBf16>(o[2 * i], pf, vf[0], vf[1]);
          mma16816<kBf16>(o[2 * i + 1], pf, vf[2], vf[3]);
        }
      }
      __syncwarp();
    }

    // ---------------------------------------------------------------- end of the item's share
    auto team_sync = [&]() {
      if constexpr (kTeam == 1) __syncwarp();
      else __syncthreads();
    };
    const int item0 = unit - at.j;  // the item's first unit
    const int cf = line.block_of(item0), cl = line.block_of(item0 + at.units - 1);
    const bool split = cf != cl;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(~0u, l[h], 1);
      l[h] += __shfl_xor_sync(~0u, l[h], 2);
      if (l[h] != l[h]) m[h] = fmaxf(m[h], 0.f);  // scores that are no numbers stay so when shares are joined
      if ((lane & 3) == 0) {
        sM[warp * kRows + r0 + 8 * h] = m[h];
        sL[warp * kRows + r0 + 8 * h] = l[h];
      }
    }
    const int rows_here = min(kRows, p.rows - at.rt * kRows);
    // Slot of team x's share of a split item: 2 x if it began before x, else 2 x + 1.
    auto slot_of = [&](int x) { return p.partial + (int64_t)(2 * x + (x == cf ? 1 : 0)) * kRows * (DP + 2); };
    const int col = lane * kPer;  // from here on a warp has whole rows
    auto write_out = [&](int row, float mm, float ll, float (&v)[kPer]) {
      const int q_row = at.rt * kRows + row;
      const int i = p.by_G.div(q_row), g = q_row - i * p.G, head = at.hk * p.G + g;
      if (p.row_share) return leave_row<DP, kPer>(p, (at.b * p.n + i) * p.H + head, col, mm, ll, v);
      const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);
      if (col < p.D) {
        uint16_t* dst = static_cast<uint16_t*>(p.out) + at.b * p.o_sb + i * p.o_ss + head * p.o_sh + col;
        if constexpr (kPer == 4)
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<kBf16>(v[0] * inv, v[1] * inv), pack2<kBf16>(v[2] * inv, v[3] * inv));
        else
          *reinterpret_cast<uint32_t*>(dst) = pack2<kBf16>(v[0] * inv, v[1] * inv);
      }
      if (p.lse && col == 0)
        p.lse[((int64_t)at.b * p.n + i) * p.H + head] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * kLn2;
    };
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half * 8 >= rows_here) break;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        const int d = i * 8 + 2 * (lane & 3);
        *reinterpret_cast<float2*>(sO + (warp * 8 + r0) * DP + (d ^ (r0 * 8 % DP))) =
            make_float2(o[i][half ? 2 : 0], o[i][half ? 3 : 1]);
      }
      team_sync();
#pragma unroll 1
      for (int jr = in_team; jr < min(8, rows_here - half * 8); jr += kTeam) {
        const int row = half * 8 + jr, first = warp - in_team;
        float mw[kTeam], mm = -INFINITY, ll = 0.f, v[kPer] = {};
#pragma unroll
        for (int w = 0; w < kTeam; ++w) mw[w] = sM[(first + w) * kRows + row], mm = fmaxf(mm, mw[w]);
#pragma unroll
        for (int w = 0; w < kTeam; ++w) {
          const float a = weight(mw[w], mm);
          ll += a * sL[(first + w) * kRows + row];
          const float* src = sO + ((first + w) * 8 + jr) * DP + (col ^ (jr * 8 % DP));
#pragma unroll
          for (int e = 0; e < kPer; ++e) v[e] += a * src[e];
        }
        if (!split) {
          write_out(row, mm, ll, v);
        } else {
          float* dst = slot_of(c);
          if (col == 0) *reinterpret_cast<float2*>(dst + kRows * DP + 2 * row) = make_float2(mm, ll);
          if constexpr (kPer == 4)
            *reinterpret_cast<float4*>(dst + row * DP + col) = make_float4(v[0], v[1], v[2], v[3]);
          else
            *reinterpret_cast<float2*>(dst + row * DP + col) = make_float2(v[0], v[1]);
        }
      }
      team_sync();
    }
    if (split) {
      int last = 0;
      if (lane == 0 && in_team == 0) {
        __threadfence();
        last = atomicAdd(&p.counters[cf], 1) == cl - cf;
        if (kTeam > 1) s_last = last;
      }
      if constexpr (kTeam > 1) {
        __syncthreads();
        last = s_last;
      } else {
        last = __shfl_sync(~0u, last, 0);
      }
      if (last) {
        __threadfence();
        // Rows in flight at a time: four of a warp alone; one or two of each warp of a team, as there are.
        auto join_rows = [&](auto at_once) {
          constexpr int kR = decltype(at_once)::value, kBatch = kR == 4 ? 3 : 8;
#pragma unroll 1
          for (int row0 = in_team * kR; row0 < rows_here; row0 += kTeam * kR) {
            int r[kR];
            float mm[kR], ll[kR], v[kR][kPer];
#pragma unroll
            for (int k = 0; k < kR; ++k) {
              r[k] = min(row0 + k, rows_here - 1);
              mm[k] = -INFINITY, ll[k] = 0.f;
#pragma unroll
              for (int e = 0; e < kPer; ++e) v[k][e] = 0.f;
            }
            join_shares<DP, kPer, kR, kBatch>(cl - cf + 1, [&](int x) { return slot_of(cf + x); }, kRows, r, 0, col, mm, ll, v);
#pragma unroll
            for (int k = 0; k < kR; ++k)
              if (row0 + k < rows_here) write_out(row0 + k, mm[k], ll[k], v[k]);
          }
        };
        if constexpr (kTeam == 1) join_rows(std::integral_constant<int, 4>());
        else if (rows_here > kTeam) join_rows(std::integral_constant<int, 2>());
        else join_rows(std::integral_constant<int, 1>());
        if (lane == 0 && in_team == 0) p.counters[cf] = 0;
      }
    }
    // Past this item.
    done += seg;
    unit += seg;
    at.j += seg - 1;
    at.advance(p, tiles);
  }
  cp_wait<0>();
  // The join of the prefix's shares waits for this kernel, and by its first block for the prefix pass
  // before it.  (If all blocks waited they would hold the SMs that the others are to run on.)
  if (p.row_share && blockIdx.x == 0) griddep_wait();
}

// One warp for each query row: its sums over its own keys and the prefix's shares of it, to `out`.
// Bound: latency of the loads, all of a batch in flight at once; a pass of its own, because a block
// of the kernels over the sequences' own keys would wait for it at the end of every sequence.
template <int DP, bool kBf16>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(const Params p) {
  constexpr int kPer = DP / 32;
  const int lane = threadIdx.x & 31, row = blockIdx.x * kWarps + (threadIdx.x >> 5);
  griddep_wait();
  if (row >= p.B * p.n * p.H) return;
  const int token = row / p.H, head = row - token * p.H, b = token / p.n, i = token - b * p.n;
  const int hk = p.by_G.div(head), col = lane * kPer;
  using V = typename std::conditional<kPer % 4 == 0, float4, float2>::type;
  float v1[1][kPer];
  float(&v)[kPer] = v1[0];
  *reinterpret_cast<V*>(v) = __ldcg(reinterpret_cast<const V*>(p.row_share + (int64_t)row * DP + col));
  const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.row_share + (int64_t)p.B * p.n * p.H * DP + 2 * (int64_t)row));
  float m1[1] = {ml.x}, l1[1] = {ml.y};
  join_prefix<DP, kPer, 8>(p.pre, __ldcg(p.counters + kPrefixBlocks), p.Hk, hk, b * p.rows + i * p.G + head - hk * p.G, col, m1, l1, v1);
  const float mm = m1[0], ll = l1[0];
  const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);
  if (col < p.D) {
    uint16_t* dst = static_cast<uint16_t*>(p.out) + b * p.o_sb + i * p.o_ss + head * p.o_sh + col;
    if constexpr (kPer == 4)
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<kBf16>(v[0] * inv, v[1] * inv), pack2<kBf16>(v[2] * inv, v[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(dst) = pack2<kBf16>(v[0] * inv, v[1] * inv);
  }
  if (p.lse && col == 0) p.lse[row] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * kLn2;
}

template <int DP, bool kBf16>
int launch_join(const Params& p, cudaStream_t s) {
  const int rows = p.B * p.n * p.H;
  return launch_kernel(paged_join_kernel<DP, kBf16>, (rows + kWarps - 1) / kWarps, kThreads, 0, true, s, p);
}

// Units of the line of a launch by teams of `team` warps, at most: sequences of at most `keys` keys.
constexpr int64_t kMostUnits = 0x7FFFFFFF;
int64_t line_units(int64_t items, int64_t keys, int team) {
  const int64_t unit = 1 << team_shift(team);
  return items * (keys > unit ? (keys + unit - 1) / unit : 1);
}

template <int DP, bool kBf16, int kTeam>
int launch_team(const Params& p, int64_t items, int64_t keys, cudaStream_t s) {
  using C = Cfg<DP>;
  auto kern = paged_rows16_kernel<DP, kBf16, kTeam>;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return cuda_status(e);
    configured.fetch_or(bit);
  }
  int64_t grid = 2 * (int64_t)sm_count();
  constexpr int64_t kTeams = kWarps / kTeam;
  const int64_t most = line_units(items, keys, kTeam);
  if (grid * kTeams > most) grid = (most + kTeams - 1) / kTeams;
  if (grid * kTeams > kPrefixBlocks) grid = kPrefixBlocks / kTeams;
  return launch_kernel(kern, (int)grid, kThreads, C::kSmem, p.row_share != nullptr, s, p);
}

// Warps of a team.  Lengths are device data: a line that might not fit 31 bits, by the block table's
// width, takes the longer units of a team of four.
int team_of(int64_t items, int64_t keys) {
  return items >= kManyItems && line_units(items, keys, 1) <= kMostUnits ? 1 : kWarps;
}

template <int DP, bool kBf16>
int launch_rows16(const Params& p, int64_t keys, cudaStream_t s) {
  const int64_t items = (int64_t)p.B * p.Hk * ((p.rows + kRows - 1) / kRows);
  return team_of(items, keys) == 1 ? launch_team<DP, kBf16, 1>(p, items, keys, s)
                                   : launch_team<DP, kBf16, kWarps>(p, items, keys, s);
}

}  // namespace paged
}  // namespace lk

namespace lk {
namespace paged {
namespace {
// How the prefix pass cuts its work (paged_common.cuh); slots is left to the caller.
PrefixShares prefix_shares(int64_t rows, int64_t H_kv, int64_t prefix) {
  PrefixShares s{};
  const int sms = sm_count();
  s.tile = rows <= kWideRows / 2 ? kWideRows / 2 : kWideRows;
  s.pairs = (int)((rows + s.tile - 1) / s.tile);
  s.units = (int)((prefix + 127) / 128);
  // The pairs of a K/V head go side by side where that leaves at most a seventh of the SMs idle: they read
  // the same keys at the same time.  (32/8 heads, D = 128: 600 sequences behind 4096 keys, 10 pairs, 122 us
  // against 127 on one line; 128 sequences of 100 own keys behind 4096, 2 pairs, 40 against 38.  With 30
  // pairs, where 28 SMs would idle, 226 either way.)
  s.lines = s.pairs <= sms && sms / s.pairs * s.pairs * 7 >= sms * 6 ? s.pairs : 1;
  const int64_t items = s.lines > 1 ? H_kv : H_kv * s.pairs;
  s.nc = sms / s.lines;
  if (s.nc > items * s.units) s.nc = (int)(items * s.units);
  return s;
}
int64_t prefix_floats(const PrefixShares& s, int64_t H_kv, int64_t DP) {
  const int64_t items = s.lines > 1 ? H_kv : H_kv * s.pairs;
  return s.lines * (items + s.nc) * kWideRows * (DP + 2);
}
// Floats of the shares of sequences' own keys.
int64_t own_floats(int64_t rows, int64_t DP) {
  const int64_t wide = rows > kRows ? (int64_t)2 * sm_count() * kWideRows * (DP + 2) : 0;
  const int64_t narrow = (int64_t)4 * kWarps * sm_count() * kRows * (DP + 2);
  return wide > narrow ? wide : narrow;
}
}  // namespace
}  // namespace paged
}  // namespace lk

extern "C" int64_t lk_paged_attention_workspace_bytes(int64_t B, int64_t n, int64_t H, int64_t H_kv, int64_t D,
                                                      int64_t prefix_length) {
  using namespace lk::paged;
  if (B < 1 || n < 1 || H < 1 || H_kv < 1 || D < 1 || prefix_length < 0) return 0;
  const int64_t DP = D > 64 ? 128 : 64, rows = n * (H / H_kv);
  int64_t floats = kCounters + own_floats(rows, DP);
  if (prefix_length > 0)
    floats += prefix_floats(prefix_shares(B * rows, H_kv, prefix_length), H_kv, DP) + B * n * H * (DP + 2);
  return (floats * 4 + 255) / 256 * 256;
}

extern "C" int lk_shared_prefix_attention(const void* q, const void* k_cache, const void* v_cache,
                                          const int32_t* prefix_pages, int64_t prefix_length, const int32_t* block_table,
                                          int64_t table_ld, int64_t table_cols, const int32_t* lengths, void* out,
                                          float* lse, const int64_t* strides, int dtype, int64_t B, int64_t n, int64_t H,
                                          int64_t H_kv, int64_t D, int64_t num_pages, int64_t page_size,
                                          float softmax_scale, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace lk;
  if (B < 0 || n < 0 || H < 0 || H_kv < 0 || D < 0 || num_pages < 0 || page_size < 1 || prefix_length < 0 ||
      table_cols < 0)
    return LK_ERR_INVALID_ARG;
  if (H > 0 && (H_kv == 0 || H % H_kv != 0)) return LK_ERR_INVALID_ARG;
  if (B == 0 || n == 0 || H == 0) return LK_OK;
  if (!q || !k_cache || !v_cache || !lengths || !out || !strides || (table_cols > 0 && !block_table) ||
      (prefix_length > 0 && !prefix_pages))
    return LK_ERR_INVALID_ARG;
  if (dtype != LK_F16 && dtype != LK_BF16) return LK_ERR_UNSUPPORTED;
  if (D < 8 || D > 128 || D % 8) return LK_ERR_UNSUPPORTED;
  constexpr int64_t kMax = 1 << 30, kMaxKeys = 1 << 29;
  if (B > kMax || n > kMax || H > kMax || B > kMax / n || B * n > kMax / H || num_pages > 0x7FFFFFFF || page_size > kMax ||
      table_cols > kMaxKeys / page_size || prefix_length > kMaxKeys)
    return LK_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out)) return LK_ERR_ALIGNMENT;
  for (int i = 0; i < 12; ++i)
    if (strides[i] % 8) return LK_ERR_ALIGNMENT;
  // All lines of units fit 31 bits if that of the 16-row kernel by teams of four does: its units are no
  // more keys or rows than any other's.  A batch for which it might not is taken in two halves.
  const int64_t row_tiles = (n * (H / H_kv) + paged::kRows - 1) / paged::kRows;
  if (paged::line_units(B * H_kv * row_tiles, prefix_length + table_cols * page_size, paged::kWarps) > paged::kMostUnits) {
    if (B == 1) return LK_ERR_INVALID_ARG;
    const int64_t half = B / 2;
    for (int i = 0; i < 2; ++i) {
      const int64_t b = i * half;
      const int st = lk_shared_prefix_attention(
          static_cast<const uint16_t*>(q) + b * strides[0], k_cache, v_cache, prefix_pages, prefix_length,
          block_table ? block_table + b * table_ld : nullptr, table_ld, table_cols, lengths + b, static_cast<uint16_t*>(out) + b * strides[3], lse ? lse + b * n * H : nullptr, strides,
          dtype, i ? B - half : half, n, H, H_kv, D, num_pages, page_size, softmax_scale, workspace, workspace_bytes, stream);
      if (st != LK_OK) return st;
    }
    return LK_OK;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const DeviceScope scope(s);
  if (scope.status()) return scope.status();
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
      workspace_bytes < lk_paged_attention_workspace_bytes(B, n, H, H_kv, D, prefix_length))
    return LK_ERR_INVALID_ARG;
  paged::Params p{};
  p.q = q, p.out = out, p.lse = lse, p.k = k_cache, p.v = v_cache;
  p.table = block_table, p.lengths = lengths, p.prefix_pages = prefix_pages;
  p.q_sb = strides[0], p.q_ss = strides[1], p.q_sh = strides[2];
  p.o_sb = strides[3], p.o_ss = strides[4], p.o_sh = strides[5];
  p.k_sp = strides[6], p.k_ss = strides[7], p.k_sh = strides[8];
  p.v_sp = strides[9], p.v_ss = strides[10], p.v_sh = strides[11];
  p.table_ld = table_ld, p.table_cols = (int)table_cols;
  p.B = (int)B, p.n = (int)n, p.H = (int)H, p.Hk = (int)H_kv, p.G = (int)(H / H_kv), p.D = (int)D;
  p.rows = p.n * p.G;
  p.by_G = paged::FastDiv::of(p.G), p.by_rows = paged::FastDiv::of(p.rows), p.by_page = paged::FastDiv::of(page_size);
  p.sms = sm_count();
  p.num_pages = (int)num_pages, p.page_size = (int)page_size, p.prefix = (int)prefix_length;
  const float scale = softmax_scale > 0.f ? softmax_scale : 1.0f / sqrtf((float)D);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.counters = static_cast<int*>(workspace);
  p.partial = reinterpret_cast<float*>(p.counters + paged::kCounters);
  const bool bf16 = dtype == LK_BF16;
  const int64_t DP = D > 64 ? 128 : 64;
  bool wide = paged::wide_box_rows(p.page_size) > 0;  // TMA can read the pages
  for (int i = 6; i < 12; ++i) wide = wide && strides[i] > 0;
  const bool pass = prefix_length > 0 && wide && B * row_tiles > 1 &&
                    B * H_kv * row_tiles * ((prefix_length + 63) / 64) > paged::kPrefixPass;
  const int64_t keys = (pass ? 0 : prefix_length) + table_cols * page_size;  // of a sequence, at most
  const bool few = p.rows <= 2 * paged::kRows && B * H_kv * keys <= paged::kTwoTileKeys;
  const bool own_wide = p.rows > paged::kRows && wide && (pass || prefix_length == 0) && !few;
  if (pass) {
    paged::PrefixShares pre = paged::prefix_shares(B * p.rows, H_kv, prefix_length);
    pre.slots = p.partial + paged::own_floats(p.rows, DP);
    pre.own_shift = own_wide ? 0 : paged::team_shift(paged::team_of(B * H_kv * row_tiles, keys));
    p.pre = pre;
    p.row_share = pre.slots + paged::prefix_floats(pre, H_kv, DP);
    if (int st = paged::launch_wide(p, bf16, true, 0, s)) return st;
    p.prefix = 0;
  }
  int st;
  if (own_wide)
    st = paged::launch_wide(p, bf16, false, B * H_kv * ((p.rows + 127) / 128) * (keys > 128 ? (keys + 127) / 128 : 1), s);
  else if (D > 64)
    st = bf16 ? paged::launch_rows16<128, true>(p, keys, s) : paged::launch_rows16<128, false>(p, keys, s);
  else
    st = bf16 ? paged::launch_rows16<64, true>(p, keys, s) : paged::launch_rows16<64, false>(p, keys, s);
  if (st != LK_OK || !p.row_share) return st;
  if (D > 64) return bf16 ? paged::launch_join<128, true>(p, s) : paged::launch_join<128, false>(p, s);
  return bf16 ? paged::launch_join<64, true>(p, s) : paged::launch_join<64, false>(p, s);
}

extern "C" int lk_paged_attention(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                                  int64_t table_ld, int64_t table_cols, const int32_t* lengths, void* out, float* lse,
                                  const int64_t* strides, int dtype, int64_t B, int64_t n, int64_t H, int64_t H_kv,
                                  int64_t D, int64_t num_pages, int64_t page_size, float softmax_scale, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  return lk_shared_prefix_attention(q, k_cache, v_cache, nullptr, 0, block_table, table_ld, table_cols, lengths, out, lse,
                                    strides, dtype, B, n, H, H_kv, D, num_pages, page_size, softmax_scale, workspace,
                                    workspace_bytes, stream);
}
