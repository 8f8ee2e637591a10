// paged_attn.cu — attention of each sequence's newest tokens to its pages of a key/value cache.
//
// Query i of the n newest tokens of a sequence of L keys sees its keys below L - n + i + 1 (and,
// with a shared prefix, all of the prefix):  o = sum_j p_j v_j / sum_j p_j with
// p_j = exp(scale q.k_j - m), lse = m + ln sum_j p_j; a row that sees nothing gives 0 and -inf.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lk_abi.h"
#include "lk_sm100.cuh"

namespace lk {
namespace paged {

enum Site : int {
  kSitePage = 311,    // a page id outside the cache
  kSiteLength = 312,  // a length past the block table's room
};

struct Params {
  const void* q;
  void* out;
  float* lse;
  const void *k, *v;
  const int *table, *lengths, *prefix_pages;
  int64_t q_sb, q_ss, q_sh, o_sb, o_ss, o_sh;
  int64_t k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;
  int64_t table_ld;
  int B, n, H, Hk, G, D;
  int num_pages, page_size, table_cols;
  int prefix;  // keys before the sequences' own, common to all
  float scale_log2;
};

template <bool kBf16>
__device__ __forceinline__ float to_float(const uint16_t v) {
  if constexpr (kBf16) return __uint_as_float((uint32_t)v << 16);
  else return __half2float(__ushort_as_half(v));
}

__device__ __forceinline__ int sequence_length(const Params& p, int b) {
  int L = max(0, p.lengths[b]);
  if ((int64_t)L > (int64_t)p.table_cols * p.page_size) {
    record_bad_index(kSiteLength);
    L = p.table_cols * p.page_size;
  }
  return L;
}

// One block per (sequence, token, query head); its warps take every fourth key.
template <bool kBf16>
__global__ void __launch_bounds__(128) paged_simple_kernel(const Params p) {
  const int h = blockIdx.x % p.H, i = blockIdx.x / p.H % p.n, b = blockIdx.x / p.H / p.n;
  const int hk = h / p.G, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint16_t* q = static_cast<const uint16_t*>(p.q) + b * p.q_sb + i * p.q_ss + h * p.q_sh;
  float qr[4], acc[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
  for (int c = 0; c < 4; ++c) qr[c] = lane + 32 * c < p.D ? to_float<kBf16>(q[lane + 32 * c]) : 0.f;
  const int seen = max(0, sequence_length(p, b) - p.n + i + 1);
  for (int j = warp; j < p.prefix + seen; j += 4) {
    const int t = j < p.prefix ? j : j - p.prefix;
    int page = (j < p.prefix ? p.prefix_pages : p.table + b * p.table_ld)[t / p.page_size];
    if (page < 0 || page >= p.num_pages) {
      record_bad_index(kSitePage);
      continue;
    }
    const int in = t % p.page_size;
    const uint16_t* k = static_cast<const uint16_t*>(p.k) + page * p.k_sp + in * p.k_ss + hk * p.k_sh;
    const uint16_t* v = static_cast<const uint16_t*>(p.v) + page * p.v_sp + in * p.v_ss + hk * p.v_sh;
    float x = 0;
    for (int c = 0; c < 4; ++c)
      if (lane + 32 * c < p.D) x += qr[c] * to_float<kBf16>(k[lane + 32 * c]);
    for (int o = 16; o; o /= 2) x += __shfl_xor_sync(~0u, x, o);
    x *= p.scale_log2;
    const float top = fmaxf(m, x), ref = top == -INFINITY ? 0.f : top, a = exp2f(m - ref), e = exp2f(x - ref);
    l = l * a + e;
    for (int c = 0; c < 4; ++c)
      if (lane + 32 * c < p.D) acc[c] = acc[c] * a + e * to_float<kBf16>(v[lane + 32 * c]);
    m = top;
  }
  __shared__ float sm[4], sl[4], so[4][128];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  for (int c = 0; c < 4; ++c) so[warp][lane + 32 * c] = acc[c];
  __syncthreads();
  float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), sum = 0, o = 0;
  for (int w = 0; w < 4 && top > -INFINITY; ++w) {
    const float a = exp2f(sm[w] - top);
    sum += sl[w] * a;
    o += so[w][threadIdx.x] * a;
  }
  if ((int)threadIdx.x < p.D) {
    const float r = sum > 0 ? o / sum : 0.f;
    uint16_t* out = static_cast<uint16_t*>(p.out) + b * p.o_sb + i * p.o_ss + h * p.o_sh;
    if constexpr (kBf16) reinterpret_cast<__nv_bfloat16*>(out)[threadIdx.x] = __float2bfloat16(r);
    else reinterpret_cast<__half*>(out)[threadIdx.x] = __float2half(r);
  }
  if (threadIdx.x == 0 && p.lse)
    p.lse[((int64_t)b * p.n + i) * p.H + h] = sum > 0 ? (top + log2f(sum)) * 0.69314718055994531f : -INFINITY;
}

}  // namespace paged
}  // namespace lk

extern "C" int64_t lk_paged_attention_workspace_bytes(int64_t H, int64_t H_kv, int64_t D) { return 256; }

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
  constexpr int64_t kMax = 1 << 30;
  if (B > kMax || n > kMax || H > kMax || B * n > kMax / H || num_pages > 0x7FFFFFFF || page_size > kMax ||
      table_cols > kMax / page_size || prefix_length > kMax)
    return LK_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out)) return LK_ERR_ALIGNMENT;
  for (int i = 0; i < 12; ++i)
    if (strides[i] % 8) return LK_ERR_ALIGNMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int st = bind_stream(s)) return st;
  paged::Params p{};
  p.q = q, p.out = out, p.lse = lse, p.k = k_cache, p.v = v_cache;
  p.table = block_table, p.lengths = lengths, p.prefix_pages = prefix_pages;
  p.q_sb = strides[0], p.q_ss = strides[1], p.q_sh = strides[2];
  p.o_sb = strides[3], p.o_ss = strides[4], p.o_sh = strides[5];
  p.k_sp = strides[6], p.k_ss = strides[7], p.k_sh = strides[8];
  p.v_sp = strides[9], p.v_ss = strides[10], p.v_sh = strides[11];
  p.table_ld = table_ld, p.table_cols = (int)table_cols;
  p.B = (int)B, p.n = (int)n, p.H = (int)H, p.Hk = (int)H_kv, p.G = (int)(H / H_kv), p.D = (int)D;
  p.num_pages = (int)num_pages, p.page_size = (int)page_size, p.prefix = (int)prefix_length;
  const float scale = softmax_scale > 0.f ? softmax_scale : 1.0f / sqrtf((float)D);
  p.scale_log2 = scale * 1.4426950408889634f;
  if (dtype == LK_BF16) paged::paged_simple_kernel<true><<<(unsigned)(B * n * H), 128, 0, s>>>(p);
  else paged::paged_simple_kernel<false><<<(unsigned)(B * n * H), 128, 0, s>>>(p);
  return check_launch();
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
