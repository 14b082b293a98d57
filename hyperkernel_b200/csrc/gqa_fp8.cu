// Ragged paged GQA attention over the block-scaled e4m3 cache, dense and over selected blocks.
//
//   s_j = scale * ks[page(j)] * (q . k_j),  o = sum_j softmax(s)_j vs[page(j)] v_j,  lse = log sum_j e^{s_j}
//
// over the tokens j <= position of the row (and, sparse, of the row's blocks).
//
// One warp per (row, query head): lanes split the head's dims, online softmax in fp32.
#include "common.cuh"
#include "gqa_fp8.cuh"

namespace {

using hk::GqaArgs;

__device__ __forceinline__ int lane_of_row(const int32_t* __restrict__ cu, int num_lanes, int t) {
  int lo = 0, hi = num_lanes;  // largest b with cu[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

template <bool kF16, int D>
__global__ void __launch_bounds__(128) gqa_fp8_warp_kernel(GqaArgs a) {
  constexpr int P = D / 32;
  const int t = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (h >= a.q_heads || t >= a.cu[a.num_lanes]) return;  // rows behind the last lane stay as they are
  const int g = h / (a.q_heads / a.kv_heads);
  const int b = lane_of_row(a.cu, a.num_lanes, t);
  if (a.cu[b + 1] - a.cu[b] > a.max_rows) {
    if (lane == 0) hk_flag(a.err, hk::kErrLaneRows, (unsigned)b);
    return;
  }
  const int pos = a.positions[t];
  float q[P], acc[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const uint16_t w = a.q[t * a.q_stride + (int64_t)h * D + lane * P + i];
    q[i] = kF16 ? __half2float(*reinterpret_cast<const __half*>(&w)) : bf16_bits_to_f32(w);
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int visible = pos < 0 ? 0 : pos / a.page_size + 1;
  const int n = a.blocks != nullptr ? a.top : visible;
  const int32_t* list = a.blocks != nullptr ? a.blocks + ((int64_t)t * a.kv_heads + g) * a.top : nullptr;
  int last = -1;
  for (int i = 0; i < n; ++i) {
    const int blk = list != nullptr ? list[i] : i;
    if (list != nullptr) {
      if (blk == -1) break;
      if (blk <= last || blk >= visible) {
        if (lane == 0) hk_flag(a.err, hk::kErrBlockList, (unsigned)t);
        continue;
      }
      last = blk;
    }
    const int page = blk < a.bt_stride ? a.bt[(int64_t)b * a.bt_stride + blk] : -1;
    if (page <= 0 || page >= a.num_pages) {
      if (lane == 0) hk_flag(a.err, hk::kErrAttnPage, (unsigned)b);
      continue;
    }
    const int64_t base = ((int64_t)page * a.kv_heads + g) * a.page_size * D;
    const float ks = a.ks[(int64_t)page * a.kv_heads + g] * a.scale, vs = a.vs[(int64_t)page * a.kv_heads + g];
    const int rows = min(a.page_size, pos + 1 - blk * a.page_size);
    for (int r = 0; r < rows; ++r) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < P; ++e) s = fmaf(q[e], e4m3_to_f32(a.kc[base + r * D + lane * P + e]), s);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      s *= ks;
      const float m_new = fmaxf(m, s);
      const float corr = m_new == -INFINITY ? 1.f : expf(m - m_new);
      const float p = s == -INFINITY ? 0.f : expf(s - m_new);
      l = l * corr + p;
#pragma unroll
      for (int e = 0; e < P; ++e) acc[e] = fmaf(p * vs, e4m3_to_f32(a.vc[base + r * D + lane * P + e]), acc[e] * corr);
      m = m_new;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that is not finite stays NaN
#pragma unroll
  for (int i = 0; i < P; i += 2)
    *reinterpret_cast<uint32_t*>(a.out + ((int64_t)t * a.q_heads + h) * D + lane * P + i) = pack2<kF16>(acc[i] * inv, acc[i + 1] * inv);
  if (lane == 0) a.lse[(int64_t)t * a.q_heads + h] = l == 0.f ? -INFINITY : m + logf(l);
}

int check(const char* name, const GqaArgs& a, int32_t dtype) {
  HK_REQUIRE(dtype == HK_BF16 || dtype == HK_F16, "%s: dtype %d", name, dtype);
  HK_REQUIRE(a.num_lanes > 0 && a.num_tokens >= 0 && a.bt_stride > 0 && a.num_pages > 0, "%s: bad sizes (lanes %d, tokens %d, table stride %d, pages %lld)",
             name, a.num_lanes, a.num_tokens, a.bt_stride, (long long)a.num_pages);
  HK_REQUIRE(a.kv_heads > 0 && a.q_heads > 0 && a.q_heads % a.kv_heads == 0 && a.q_heads <= 65536, "%s: %d query heads do not divide into %d KV heads",
             name, a.q_heads, a.kv_heads);
  HK_REQUIRE(a.dim == 64 || a.dim == 128 || a.dim == 256, "%s: head_dim %d not 64, 128 or 256", name, a.dim);
  HK_REQUIRE(a.page_size >= 16 && a.page_size <= 256 && a.page_size % 16 == 0, "%s: page_size %d must be a multiple of 16 up to 256", name, a.page_size);
  HK_REQUIRE(a.q_stride >= (int64_t)a.q_heads * a.dim && a.q_stride % 8 == 0, "%s: q_stride must hold a row and be a multiple of 8 elements", name);
  HK_REQUIRE(a.scale > 0.f && a.scale < 3.0e38f, "%s: scale must be positive and finite", name);
  if (a.num_tokens == 0) return HK_OK;
  HK_REQUIRE(a.q && a.kc && a.vc && a.ks && a.vs && a.bt && a.cu && a.positions && a.out && a.lse, "%s: null pointer", name);
  HK_REQUIRE(((uintptr_t)a.q | (uintptr_t)a.kc | (uintptr_t)a.vc | (uintptr_t)a.out) % 16 == 0, "%s: buffers must be 16-byte aligned", name);
  return HK_OK;
}

int launch(GqaArgs& a, int32_t dtype, cudaStream_t s) {
  a.err = hk::err_word();
  const dim3 grid(a.num_tokens, (a.q_heads + 3) / 4);
#define HK_GQA(D)                                                            \
  case D:                                                                    \
    if (dtype == HK_F16) gqa_fp8_warp_kernel<true, D><<<grid, 128, 0, s>>>(a); \
    else gqa_fp8_warp_kernel<false, D><<<grid, 128, 0, s>>>(a);              \
    break
  switch (a.dim) {
    HK_GQA(64);
    HK_GQA(128);
    HK_GQA(256);
  }
#undef HK_GQA
  HK_TRY_LAUNCH("gqa_fp8_warp_kernel");
  return HK_OK;
}

}  // namespace

extern "C" {

size_t hk_gqa_fp8_workspace_size(int32_t num_tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
  (void)num_tokens, (void)q_heads, (void)kv_heads, (void)head_dim;
  return 256;
}

int hk_gqa_decode_fp8(const uint16_t* q, int64_t q_stride, const uint8_t* k_cache, const uint8_t* v_cache,
                      const float* k_scale, const float* v_scale, const int32_t* block_table, int32_t bt_stride,
                      const int32_t* cu_seqlens, const int32_t* positions, int32_t num_lanes, int32_t num_tokens,
                      int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t page_size, int64_t num_pages,
                      int32_t max_rows, int32_t max_kv_len, float scale, int32_t dtype, uint16_t* out, float* lse,
                      void* workspace, size_t workspace_bytes, void* stream) {
  GqaArgs a = {q, q_stride, k_cache, v_cache, k_scale, v_scale, block_table, bt_stride, cu_seqlens, positions,
               nullptr, 0, num_lanes, num_tokens, q_heads, kv_heads, head_dim, page_size, num_pages, max_rows, scale,
               out, lse, nullptr};
  HK_TRY(check("hk_gqa_decode_fp8", a, dtype));
  HK_REQUIRE(max_rows >= 0 && max_kv_len >= 0, "hk_gqa_decode_fp8: negative max_rows or max_kv_len");
  if (num_tokens == 0) return HK_OK;
  HK_REQUIRE((uintptr_t)workspace % 256 == 0, "hk_gqa_decode_fp8: workspace must be 256-byte aligned");
  if (workspace == nullptr || workspace_bytes < hk_gqa_fp8_workspace_size(num_tokens, q_heads, kv_heads, head_dim))
    return hk::fail(HK_ESPACE, "hk_gqa_decode_fp8: workspace of %zu bytes is too small", workspace_bytes);
  HK_TRY(hk::ensure_device());
  return launch(a, dtype, (cudaStream_t)stream);
}

int hk_gqa_sparse_fp8(const uint16_t* q, int64_t q_stride, const uint8_t* k_cache, const uint8_t* v_cache,
                      const float* k_scale, const float* v_scale, const int32_t* block_table, int32_t bt_stride,
                      const int32_t* cu_seqlens, const int32_t* positions, const int32_t* blocks, int32_t top_blocks,
                      int32_t num_lanes, int32_t num_tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                      int32_t page_size, int64_t num_pages, float scale, int32_t dtype, uint16_t* out, float* lse,
                      void* workspace, size_t workspace_bytes, void* stream) {
  GqaArgs a = {q, q_stride, k_cache, v_cache, k_scale, v_scale, block_table, bt_stride, cu_seqlens, positions,
               blocks, top_blocks, num_lanes, num_tokens, q_heads, kv_heads, head_dim, page_size, num_pages, num_tokens,
               scale, out, lse, nullptr};
  HK_TRY(check("hk_gqa_sparse_fp8", a, dtype));
  HK_REQUIRE(top_blocks > 0 && top_blocks <= 4096, "hk_gqa_sparse_fp8: top_blocks %d not in 1..4096", top_blocks);
  if (num_tokens == 0) return HK_OK;
  HK_REQUIRE(blocks != nullptr, "hk_gqa_sparse_fp8: null pointer");
  HK_REQUIRE((uintptr_t)workspace % 256 == 0, "hk_gqa_sparse_fp8: workspace must be 256-byte aligned");
  if (workspace == nullptr || workspace_bytes < hk_gqa_fp8_workspace_size(num_tokens, q_heads, kv_heads, head_dim))
    return hk::fail(HK_ESPACE, "hk_gqa_sparse_fp8: workspace of %zu bytes is too small", workspace_bytes);
  HK_TRY(hk::ensure_device());
  return launch(a, dtype, (cudaStream_t)stream);
}

}  // extern "C"
