// rotary.cu — rotary position embedding of queries and keys, and the append of new keys and
// values to a paged cache with the rotation applied on the way.
//
// Pair i of a head's first 2 * pairs values is (x[i], x[i + pairs]) or, interleaved,
// (x[2i], x[2i + 1]).  With p the token's position on pair i's axis and (c, s) = cos_sin[p][i]:
//     a' = a c - b s,   b' = b c + a s,
// in fp32 from the 16-bit values, rounded once to 16 bits; values past 2 * pairs pass through.
// The map is a rotation, so its gradient is the rotation by -s (inverse).
//
// Bound: memory.  A token's heads are read and written once and nothing is reused but the table
// rows (8 bytes a pair, from L1 / L2).  Measured (B200, bf16, D = 128): 16380 tokens of 32/8 heads
// with three axes and their gradient 112 us, 6.2 TB/s; append of 16384 tokens of 32 heads 132 us,
// 6.2 TB/s (a copy runs at 6.5).  16 tokens: 3.5 us, two round trips to memory and the launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "lk_abi.h"
#include "lk_sm100.cuh"
#include "paged_common.cuh"

namespace lk {
namespace rot {

using paged::cp_commit;
using paged::cp_wait;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) { paged::cp16(dst, src, true); }
__device__ __forceinline__ void cp8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

constexpr int kMaxAxes = 4;
constexpr int kMaxThreads = 256;
constexpr int kHeads = 3;              // heads of a thread
constexpr int kStages = 4;             // of its ring
constexpr int kSmBytes = 200 * 1024;   // shared memory that an SM's blocks may take
constexpr int kPart = 3;  // q, k, v

enum Site : int {
  kSitePosition = 301,  // a position outside the table's rows
  kSiteSlot = 302,      // a slot past the cache's end
};

struct Params {
  const void* src[kPart];
  void* dst[kPart];  // append: dst[1], dst[2] are the cache's K and V pages
  int64_t src_sb[kPart], src_ss[kPart], src_sh[kPart];  // element strides: outer, token, head
  int64_t dst_sb[kPart], dst_ss[kPart], dst_sh[kPart];  // append, parts 1, 2: page, slot in page, head
  int heads[kPart];
  int64_t S;  // tokens per outer index
  int outer, tokens;
  paged::FastDiv by_S;
  int D, pairs;
  const float* table;  // [table_rows][pairs][2] (cos, sin); nullptr: no rotation
  int64_t table_rows;
  const void* pos;
  int64_t pos_sa, pos_sb, pos_ss;  // element strides: axis, outer, token
  int pos64, axes;
  int axis_end[kMaxAxes];  // pair i's axis: the first a with i < axis_end[a]
  int interleaved;
  float sign;  // +1 rotation, -1 its inverse
  const void* slots;
  int slots64;
  int64_t page_size, num_slots;
  int block_heads; // heads of a block (vector form)
  int page_shift;  // log2 of page_size, -1 where it is no power of two
};

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

template <bool kBf16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (kBf16) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

__device__ __forceinline__ int axis_of(const Params& p, int pair) {
  int a = 0;
#pragma unroll
  for (int i = 0; i < kMaxAxes - 1; ++i) a += (i < p.axes - 1 && pair >= p.axis_end[i]) ? 1 : 0;
  return a;
}

// The token's position on each axis, clamped into the table (a position outside it is reported
// unless the token is padding).
__device__ __forceinline__ void load_positions(const Params& p, int64_t b, int64_t s, bool live, int64_t (&row)[kMaxAxes]) {
#pragma unroll
  for (int a = 0; a < kMaxAxes; ++a) {
    row[a] = 0;
    if (a < p.axes) {
      const int64_t v = load_index(p.pos, a * p.pos_sa + b * p.pos_sb + s * p.pos_ss, p.pos64);
      if (live && (v < 0 || v >= p.table_rows)) record_bad_index(kSitePosition);
      row[a] = v < 0 ? 0 : (v >= p.table_rows ? p.table_rows - 1 : v);
    }
  }
}

struct Token {
  int64_t b, s;      // outer index and token
  bool live;         // append: it has a slot
  int64_t page, in;  // append: where the slot lies
};

template <bool kAppend>
__device__ __forceinline__ Token load_token(const Params& p) {
  Token t{};
  const int64_t i = blockIdx.x;
  t.b = i / p.S;
  t.s = i - t.b * p.S;
  t.live = true;
  if constexpr (kAppend) {
    const int64_t slot = load_index(p.slots, i, p.slots64);
    if (slot >= p.num_slots) record_bad_index(kSiteSlot);
    t.live = slot >= 0 && slot < p.num_slots;
    if (t.live) {
      t.page = slot / p.page_size;
      t.in = slot - t.page * p.page_size;
    }
  }
  return t;
}

// Vector form: D and 2 * pairs are multiples of 16 and every row starts on 16 bytes.
// A thread owns two 16-byte vectors (8 pairs, or 16 values that pass through) of each of kHeads heads,
// and a block walks over tokens blockIdx.x, blockIdx.x + gridDim.x, ...  The next kStages - 1 tokens
// are on their way into shared memory: each thread's own vectors, and the token's (cos, sin) of all
// pairs, put together from the rows of its positions (thread i copies pair i's).  So neither the data
// nor the chain position -> table is waited for, and loads in flight cost no registers.  (One head a
// thread spends more instructions on tokens and addresses than on values, and is bound by them.)
template <bool kBf16, bool kAppend>
__global__ void __launch_bounds__(kMaxThreads) rotary_vec_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint4 ring[];  // [kStages][kHeads][2][threads], then [kStages][pairs] (cos, sin)
  const int units = p.D / 16, u = threadIdx.x % units, h_in = threadIdx.x / units;
  const int pairs = p.table != nullptr ? p.pairs : 0;
  const int total = p.heads[0] + p.heads[1] + (kAppend ? p.heads[2] : 0);
  const bool pair_unit = u < pairs / 8;
  // The unit's vectors are 8 values each; those of a unit that is not turned follow one another (so
  // do a value head's, which is turned nowhere).
  const bool apart = pair_unit && !p.interleaved;
  const int v0 = apart ? 8 * u : 16 * u, v_step = apart ? p.pairs : 8;
  const uint16_t* src[kHeads];  // the head's vectors at token 0
  uint16_t* dst[kHeads];        // ... or at slot 0
  int part[kHeads];             // -1: none
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    const int i = k * p.block_heads + h_in, h = blockIdx.y * p.block_heads * kHeads + i;
    part[k] = -1;
    if (h_in >= p.block_heads || h >= total) continue;
    part[k] = h < p.heads[0] ? 0 : (h < p.heads[0] + p.heads[1] ? 1 : 2);
    const int head = h - (part[k] > 0 ? p.heads[0] : 0) - (part[k] > 1 ? p.heads[1] : 0);
    src[k] = static_cast<const uint16_t*>(p.src[part[k]]) + head * p.src_sh[part[k]] + v0;
    dst[k] = static_cast<uint16_t*>(p.dst[part[k]]) + head * p.dst_sh[part[k]] + v0;
  }
  const uint32_t mine = smem_u32(ring + threadIdx.x), row_bytes = blockDim.x * 16;
  const uint32_t table0 = smem_u32(ring + 2 * kHeads * kStages * blockDim.x);
  const bool copies_pair = (int)threadIdx.x < pairs;
  const int64_t pos_axis = copies_pair ? axis_of(p, threadIdx.x) * p.pos_sa : 0;

  auto place = [&](int t, int& b, int& s) {
    b = p.outer > 1 ? p.by_S.div(t) : 0;
    s = t - b * (int)p.S;
  };
  auto position = [&](int t) -> int64_t {  // of pair threadIdx.x's axis
    if (!copies_pair || t >= p.tokens) return 0;
    int b, s;
    place(t, b, s);
    return load_index(p.pos, pos_axis + b * p.pos_sb + s * p.pos_ss, p.pos64);
  };
  auto load = [&](int t, int stage, int64_t pos) {
    if (t < p.tokens) {
      int b, s;
      place(t, b, s);
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        if (part[k] < 0) continue;
        const uint16_t* x = src[k] + b * p.src_sb[part[k]] + s * p.src_ss[part[k]];
        cp16(mine + (2 * (kHeads * stage + k)) * row_bytes, x);
        cp16(mine + (2 * (kHeads * stage + k) + 1) * row_bytes, x + v_step);
      }
      if (copies_pair) {
        if (pos < 0 || pos >= p.table_rows) {
          if (!kAppend || load_index(p.slots, t, p.slots64) >= 0) record_bad_index(kSitePosition);
          pos = pos < 0 ? 0 : p.table_rows - 1;
        }
        cp8(table0 + (stage * pairs + threadIdx.x) * 8, p.table + (pos * pairs + threadIdx.x) * 2);
      }
    }
    cp_commit();
  };
  const int step = gridDim.x;
  int64_t pos[kStages - 1];
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) pos[i] = position(blockIdx.x + i * step);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load(blockIdx.x + i * step, i, pos[i]);
  int64_t pos_next = position(blockIdx.x + (kStages - 1) * step);
  int64_t slot = kAppend ? load_index(p.slots, blockIdx.x, p.slots64) : 0;
  int stage = 0;
#pragma unroll 1
  for (int t = blockIdx.x; t < p.tokens; t += step) {
    cp_wait<kStages - 2>();
    __syncthreads();  // the stage is in for all threads, and the one before it has been read by all
    load(t + (kStages - 1) * step, stage == 0 ? kStages - 1 : stage - 1, pos_next);
    pos_next = position(t + kStages * step);
    const int64_t slot_next = kAppend && t + step < p.tokens ? load_index(p.slots, t + step, p.slots64) : 0;
    int b, s;
    place(t, b, s);
    bool live = true;
    int64_t page = 0, in_page = 0;
    if (kAppend) {
      if (slot >= p.num_slots) record_bad_index(kSiteSlot);
      live = slot >= 0 && slot < p.num_slots;
      page = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
      in_page = slot - page * p.page_size;
    }
    float4 c[4];  // (cos, sin) of pairs 2 e and 2 e + 1 of the unit
    if (pair_unit) {
      const float4* cs = reinterpret_cast<const float4*>(ring + 2 * kHeads * kStages * blockDim.x) + (stage * pairs + 8 * u) / 2;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[e] = cs[e];
        c[e].y *= p.sign, c[e].w *= p.sign;
      }
    }
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      if (part[k] < 0) continue;
      uint4 x0 = ring[2 * (kHeads * stage + k) * blockDim.x + threadIdx.x];
      uint4 x1 = ring[(2 * (kHeads * stage + k) + 1) * blockDim.x + threadIdx.x];
      if (pair_unit && part[k] < 2) {
        uint32_t m[4] = {x0.x, x0.y, x0.z, x0.w}, n[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (p.interleaved) {  // m[0], m[1] .. n[2], n[3]: two pairs each
            uint32_t& lo = e < 2 ? m[2 * e] : n[2 * e - 4];
            uint32_t& hi = e < 2 ? m[2 * e + 1] : n[2 * e - 3];
            const float2 f = unpack2<kBf16>(lo), g = unpack2<kBf16>(hi);
            lo = pack2<kBf16>(f.x * c[e].x - f.y * c[e].y, f.y * c[e].x + f.x * c[e].y);
            hi = pack2<kBf16>(g.x * c[e].z - g.y * c[e].w, g.y * c[e].z + g.x * c[e].w);
          } else {  // m[e] and n[e]: the halves of two pairs
            const float2 f = unpack2<kBf16>(m[e]), g = unpack2<kBf16>(n[e]);
            m[e] = pack2<kBf16>(f.x * c[e].x - g.x * c[e].y, f.y * c[e].z - g.y * c[e].w);
            n[e] = pack2<kBf16>(g.x * c[e].x + f.x * c[e].y, g.y * c[e].z + f.y * c[e].w);
          }
        }
        x0 = make_uint4(m[0], m[1], m[2], m[3]);
        x1 = make_uint4(n[0], n[1], n[2], n[3]);
      }
      const bool cached = kAppend && part[k] > 0;
      if (!cached || live) {
        uint16_t* y = cached ? dst[k] + page * p.dst_sb[part[k]] + in_page * p.dst_ss[part[k]]
                             : dst[k] + b * p.dst_sb[part[k]] + s * p.dst_ss[part[k]];
        *reinterpret_cast<uint4*>(y) = x0;
        *reinterpret_cast<uint4*>(y + v_step) = x1;
      }
    }
    slot = slot_next;
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  cp_wait<0>();
}

// Any D, pairs, stride and alignment: a thread per pair or passed value, 2-byte accesses.
template <bool kBf16, bool kAppend>
__global__ void __launch_bounds__(256) rotary_any_kernel(const Params p) {
  const Token t = load_token<kAppend>(p);
  const int pairs = p.table != nullptr ? p.pairs : 0;
  const int units = p.D - pairs;  // pairs, then the values that pass through
  int64_t row[kMaxAxes] = {0, 0, 0, 0};
  if (pairs) load_positions(p, t.b, t.s, t.live, row);
  const int total = p.heads[0] + p.heads[1] + (kAppend ? p.heads[2] : 0);
  for (int64_t w = threadIdx.x; w < (int64_t)total * p.D; w += blockDim.x) {
    const int h = (int)(w / p.D), u = (int)(w - (int64_t)h * p.D);
    if (u >= units) continue;
    const int part = h < p.heads[0] ? 0 : (h < p.heads[0] + p.heads[1] ? 1 : 2);
    const int head = h - (part > 0 ? p.heads[0] : 0) - (part > 1 ? p.heads[1] : 0);
    if (kAppend && part > 0 && !t.live) continue;
    const uint16_t* src =
        static_cast<const uint16_t*>(p.src[part]) + t.b * p.src_sb[part] + t.s * p.src_ss[part] + head * p.src_sh[part];
    const int64_t db = kAppend && part > 0 ? t.page : t.b, ds = kAppend && part > 0 ? t.in : t.s;
    uint16_t* dst = static_cast<uint16_t*>(p.dst[part]) + db * p.dst_sb[part] + ds * p.dst_ss[part] + head * p.dst_sh[part];
    if (u >= pairs) {
      dst[u + pairs] = src[u + pairs];
      continue;
    }
    const int i0 = p.interleaved ? 2 * u : u, i1 = p.interleaved ? 2 * u + 1 : u + pairs;
    uint32_t x = (uint32_t)src[i0] | ((uint32_t)src[i1] << 16);
    if (part < 2) {
      const float2 cs = reinterpret_cast<const float2*>(p.table)[row[axis_of(p, u)] * p.pairs + u];
      const float2 f = unpack2<kBf16>(x);
      const float sn = cs.y * p.sign;
      x = pack2<kBf16>(f.x * cs.x - f.y * sn, f.y * cs.x + f.x * sn);
    }
    dst[i0] = (uint16_t)x;
    dst[i1] = (uint16_t)(x >> 16);
  }
}

bool vec_rows(const void* p, int64_t sb, int64_t ss, int64_t sh) {
  return aligned16(p) && sb % 8 == 0 && ss % 8 == 0 && sh % 8 == 0;
}

template <bool kAppend>
int launch(Params& p, bool bf16, int64_t tokens, cudaStream_t s) {
  bool vec = p.D % 16 == 0 && (p.table == nullptr || (p.pairs % 8 == 0));
  for (int i = 0; i < kPart; ++i)
    if (p.heads[i] > 0)
      vec = vec && vec_rows(p.src[i], p.src_sb[i], p.src_ss[i], p.src_sh[i]) &&
            vec_rows(p.dst[i], p.dst_sb[i], p.dst_ss[i], p.dst_sh[i]);
  const int units = p.D / 16;
  if (vec && units <= 16) {
    const int pairs = p.table ? p.pairs : 0;
    const int total = p.heads[0] + p.heads[1] + p.heads[2];
    const int block_most = kMaxThreads / units;  // heads of a block, kHeads of them to a thread
    const int y = (total + block_most * kHeads - 1) / (block_most * kHeads);
    p.block_heads = (total + y * kHeads - 1) / (y * kHeads);
    int threads = p.block_heads * units;
    if (threads < pairs) threads = pairs;  // a thread for each pair's (cos, sin)
    threads = (threads + 31) / 32 * 32;
    const int smem = kStages * (kHeads * 2 * 16 * threads + 8 * pairs);
    // As many blocks as the SMs hold at a time walk over the tokens.
    const int per_sm = kSmBytes / smem < 1 ? 1 : kSmBytes / smem;
    int64_t x = (int64_t)sm_count() * per_sm / y;
    if (x < 1) x = 1;
    if (x > tokens) x = tokens;
    if (y > 65535) return LK_ERR_INVALID_ARG;
    auto kern = bf16 ? rotary_vec_kernel<true, kAppend> : rotary_vec_kernel<false, kAppend>;
    if (smem > 48 * 1024) {
      static std::atomic<uint64_t> configured[2] = {{0}, {0}};
      int dev = 0;
      cudaGetDevice(&dev);
      const uint64_t bit = 1ull << (dev & 63);
      if (!(configured[bf16].load() & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmBytes);
        if (e != cudaSuccess) return cuda_status(e);
        configured[bf16].fetch_or(bit);
      }
    }
    kern<<<dim3((unsigned)x, (unsigned)y), threads, smem, s>>>(p);
  } else {
    auto kern = bf16 ? rotary_any_kernel<true, kAppend> : rotary_any_kernel<false, kAppend>;
    kern<<<(unsigned)tokens, 256, 0, s>>>(p);
  }
  return check_launch();
}

// Positions, table and axes, common to both entry points.
int set_angles(Params* p, const void* positions, int pos_dtype, const int64_t* pos_strides, const float* cos_sin,
               int64_t table_rows, int64_t pairs, int64_t axes, const int64_t* sections, int interleaved) {
  if (!positions || !pos_strides || table_rows <= 0 || pairs <= 0 || 2 * pairs > p->D) return LK_ERR_INVALID_ARG;
  if (axes < 1 || axes > kMaxAxes || (axes > 1 && !sections)) return LK_ERR_INVALID_ARG;
  if (pos_dtype != LK_I32 && pos_dtype != LK_I64) return LK_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(cos_sin) & 7) return LK_ERR_ALIGNMENT;
  int64_t end = 0;
  for (int64_t a = 0; a < axes; ++a) {
    const int64_t n = axes > 1 ? sections[a] : pairs;
    if (n < 0 || n > pairs) return LK_ERR_INVALID_ARG;
    end += n;
    p->axis_end[a] = (int)end;
  }
  if (end != pairs) return LK_ERR_INVALID_ARG;
  p->axes = (int)axes;
  p->pos = positions;
  p->pos64 = pos_dtype == LK_I64;
  p->pos_sa = pos_strides[0];
  p->pos_sb = pos_strides[1];
  p->pos_ss = pos_strides[2];
  p->table = cos_sin;
  p->table_rows = table_rows;
  p->pairs = (int)pairs;
  p->interleaved = interleaved ? 1 : 0;
  return LK_OK;
}

constexpr int64_t kMaxHeads = 1 << 20, kMaxDim = 1 << 16;

}  // namespace rot
}  // namespace lk

extern "C" int lk_rotary_embed(const void* q, void* q_out, const void* k, void* k_out, const int64_t* strides, int dtype,
                               int64_t B, int64_t S, int64_t H, int64_t H_kv, int64_t D, const void* positions,
                               int pos_dtype, const int64_t* pos_strides, const float* cos_sin, int64_t table_rows,
                               int64_t pairs, int64_t axes, const int64_t* sections, int interleaved, int inverse,
                               void* stream) {
  using namespace lk;
  if (B < 0 || S < 0 || H < 0 || H_kv < 0 || D < 0 || H > rot::kMaxHeads || H_kv > rot::kMaxHeads || D > rot::kMaxDim)
    return LK_ERR_INVALID_ARG;
  if (B == 0 || S == 0 || H + H_kv == 0 || D == 0) return LK_OK;
  if (!strides || !cos_sin || (H > 0 && (!q || !q_out)) || (H_kv > 0 && (!k || !k_out))) return LK_ERR_INVALID_ARG;
  if (dtype != LK_F16 && dtype != LK_BF16) return LK_ERR_UNSUPPORTED;
  if (S > 0x3FFFFFFF / B) return LK_ERR_INVALID_ARG;
  rot::Params p{};
  p.src[0] = q, p.dst[0] = q_out, p.src[1] = k, p.dst[1] = k_out;
  p.heads[0] = (int)H, p.heads[1] = (int)H_kv;
  for (int i = 0; i < 2; ++i) {
    const int64_t* st = strides + 6 * i;
    p.src_sb[i] = st[0], p.src_ss[i] = st[1], p.src_sh[i] = st[2];
    p.dst_sb[i] = st[3], p.dst_ss[i] = st[4], p.dst_sh[i] = st[5];
  }
  p.S = S;
  p.outer = (int)B, p.tokens = (int)(B * S), p.by_S = paged::FastDiv::of(S);
  p.D = (int)D;
  p.sign = inverse ? -1.f : 1.f;
  if (int st = rot::set_angles(&p, positions, pos_dtype, pos_strides, cos_sin, table_rows, pairs, axes, sections,
                               interleaved))
    return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const DeviceScope scope(s);
  if (scope.status()) return scope.status();
  return rot::launch<false>(p, dtype == LK_BF16, B * S, s);
}

extern "C" int lk_paged_kv_append(const void* q, void* q_out, const void* k, const void* v, void* k_cache, void* v_cache,
                                  const int64_t* strides, int dtype, int64_t T, int64_t H, int64_t H_kv, int64_t D,
                                  int64_t num_pages, int64_t page_size, const void* slots, int slots_dtype,
                                  const void* positions, int pos_dtype, const int64_t* pos_strides,
                                  const float* cos_sin, int64_t table_rows, int64_t pairs, int64_t axes,
                                  const int64_t* sections, int interleaved, void* stream) {
  using namespace lk;
  if (T < 0 || H < 0 || H_kv < 0 || D < 0 || num_pages < 0 || page_size < 0 || T > 0x3FFFFFFF || H > rot::kMaxHeads ||
      H_kv > rot::kMaxHeads || D > rot::kMaxDim)
    return LK_ERR_INVALID_ARG;
  if (T == 0 || H + H_kv == 0 || D == 0) return LK_OK;
  if (!strides || !slots || (H > 0 && (!q || !q_out)) || (H_kv > 0 && (!k || !v))) return LK_ERR_INVALID_ARG;
  if (page_size == 0 || (H_kv > 0 && num_pages > 0 && (!k_cache || !v_cache))) return LK_ERR_INVALID_ARG;
  if (num_pages > (int64_t)0x7FFFFFFF || page_size > (int64_t)0x7FFFFFFF) return LK_ERR_INVALID_ARG;
  if (dtype != LK_F16 && dtype != LK_BF16) return LK_ERR_UNSUPPORTED;
  if (slots_dtype != LK_I32 && slots_dtype != LK_I64) return LK_ERR_UNSUPPORTED;
  if (H > 0 && !cos_sin) return LK_ERR_INVALID_ARG;  // queries are only passed to be rotated
  rot::Params p{};
  p.src[0] = q, p.src[1] = k, p.src[2] = v;
  p.dst[0] = q_out, p.dst[1] = k_cache, p.dst[2] = v_cache;
  p.heads[0] = (int)H, p.heads[1] = p.heads[2] = (int)H_kv;
  // (token, head) of q, q_out, k, v; (page, slot, head) of the two caches
  p.src_ss[0] = strides[0], p.src_sh[0] = strides[1];
  p.dst_ss[0] = strides[2], p.dst_sh[0] = strides[3];
  p.src_ss[1] = strides[4], p.src_sh[1] = strides[5];
  p.src_ss[2] = strides[6], p.src_sh[2] = strides[7];
  for (int i = 0; i < 2; ++i) {
    p.dst_sb[1 + i] = strides[8 + 3 * i], p.dst_ss[1 + i] = strides[9 + 3 * i], p.dst_sh[1 + i] = strides[10 + 3 * i];
  }
  p.S = T;
  p.outer = 1, p.tokens = (int)T, p.by_S = paged::FastDiv::of(T);
  p.D = (int)D;
  p.sign = 1.f;
  p.slots = slots;
  p.slots64 = slots_dtype == LK_I64;
  p.page_size = page_size;
  p.num_slots = num_pages * page_size;
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (page_size == (int64_t)1 << i) p.page_shift = i;
  if (cos_sin)
    if (int st = rot::set_angles(&p, positions, pos_dtype, pos_strides, cos_sin, table_rows, pairs, axes, sections,
                                 interleaved))
      return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const DeviceScope scope(s);
  if (scope.status()) return scope.status();
  return rot::launch<true>(p, dtype == LK_BF16, T, s);
}
