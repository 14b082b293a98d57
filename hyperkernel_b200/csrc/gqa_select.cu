// The blocks each row reads, by a cheap score: q summed over the query heads of a KV head and
// rounded to int8, against each page's int8 centroid (hk_gqa_append_fp8).
//
//   u_d = sum_h q[h][d] (exact, rounded once to fp32),  c_d = rint(u_d * (127 / max|u|))
//   score(block) = fp32(sum_d c_d * centroid[page][d]) * centroid_scale[page]
//
// The dot product is of whole numbers, and each fp32 step has one given order, so a row's
// blocks are the same on every run and in every batch.  The first `sink` and the last `local`
// blocks are always read; the rest of top_blocks go to the highest scores, equal ones to the lower
// block.
//
// One CTA per (row, KV head): scores to the workspace as keys whose unsigned order is the
// scores' order, a radix select for the top_blocks-th key (8 bits a pass), and one ordered pass
// that writes the chosen indices rising.
#include "common.cuh"
#include "gqa_fp8.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct SelectArgs {
  const uint16_t* q;
  int64_t q_stride;
  const int8_t* centroids;
  const float* centroid_scale;
  const int32_t* bt;
  int32_t bt_stride;
  const int32_t* cu;
  const int32_t* positions;
  int32_t num_lanes, num_tokens, q_heads, kv_heads, dim, page_size;
  int64_t num_pages;
  int32_t max_blocks, top, sink, local;
  int32_t* blocks;
  uint32_t* keys;  // [T][kv_heads][max_blocks]
  unsigned long long* err;
};

__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

template <bool kF16>
__global__ void __launch_bounds__(kThreads) gqa_select_kernel(SelectArgs a) {
  __shared__ float u[256];
  __shared__ __align__(16) int8_t c8[256];
  __shared__ float warp_max[kWarps];
  __shared__ int hist[256];
  __shared__ int warp_sum[2][kWarps];
  __shared__ uint32_t s_prefix;
  __shared__ int s_rank;
  const int t = blockIdx.x, g = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (t >= a.cu[a.num_lanes]) return;
  const int pos = a.positions[t];
  int32_t* list = a.blocks + ((int64_t)t * a.kv_heads + g) * a.top;
  int n = pos < 0 ? 0 : pos / a.page_size + 1;
  if (n > a.max_blocks) {
    if (tid == 0) hk_flag(a.err, hk::kErrPosition, (unsigned)t);
    n = 0;
  }
  if (n <= a.top) {
    for (int i = tid; i < a.top; i += kThreads) list[i] = i < n ? i : -1;
    return;
  }
  const int b = hk::lane_of_row(a.cu, a.num_lanes, t);
  const int group = a.q_heads / a.kv_heads;
  float mine = 0.f;
  if (tid < a.dim) {
    double sum = 0.0;
    for (int h = 0; h < group; ++h) {
      const uint16_t w = a.q[t * a.q_stride + (int64_t)(g * group + h) * a.dim + tid];
      sum += (double)(kF16 ? __half2float(*reinterpret_cast<const __half*>(&w)) : bf16_bits_to_f32(w));
    }
    u[tid] = (float)sum;
    mine = fabsf(u[tid]);
    if (!(mine < INFINITY)) mine = INFINITY;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, o));
  if (lane == 0) warp_max[warp] = mine;
  __syncthreads();
  float m = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, warp_max[w]);
  // A row with a value that is not finite scores 0 everywhere: its blocks are the first ones.
  const float r = m > 0.f && m < INFINITY ? __fdiv_rn(127.f, m) : 0.f;
  if (tid < a.dim) c8[tid] = r > 0.f ? (int8_t)rintf(__fmul_rn(u[tid], r)) : (int8_t)0;
  __syncthreads();

  uint32_t* keys = a.keys + ((int64_t)t * a.kv_heads + g) * a.max_blocks;
  const int vec = a.dim / 16;  // 16-byte parts of a centroid
  for (int i = tid; i < n; i += kThreads) {
    uint32_t key;
    if (i < a.sink || i >= n - a.local) {
      key = 0xffffffffu;
    } else {
      const int page = i < a.bt_stride ? a.bt[(int64_t)b * a.bt_stride + i] : -1;
      if (page <= 0 || page >= a.num_pages) {
        hk_flag(a.err, hk::kErrAttnPage, (unsigned)b);
        key = 0;
      } else {
        const int64_t at = (int64_t)page * a.kv_heads + g;
        const int4* cen = reinterpret_cast<const int4*>(a.centroids + at * a.dim);
        int dot = 0;
        for (int v = 0; v < vec; ++v) {
          const int4 x = cen[v], y = reinterpret_cast<const int4*>(c8)[v];
          dot = __dp4a(x.x, y.x, dot), dot = __dp4a(x.y, y.y, dot);
          dot = __dp4a(x.z, y.z, dot), dot = __dp4a(x.w, y.w, dot);
        }
        key = order_key(__fadd_rn(__fmul_rn((float)dot, a.centroid_scale[at]), 0.f));  // -0 becomes 0
        key = min(key, 0xfffffffeu);
      }
    }
    keys[i] = key;
  }
  if (tid == 0) s_prefix = 0, s_rank = a.top;
  // The top-th largest key, from its highest 8 bits down: s_rank = how many of the keys that
  // share the prefix are wanted.
  for (int shift = 24; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix, mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t k = keys[i];
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    // Keys at or above each bin: a scan from the highest bin down.
    const int bin = 255 - tid, here = hist[bin];
    int x = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[0][warp] = x;
    const int want = s_rank;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += warp_sum[0][w];
    const int above = before + x - here;
    if (above < want && above + here >= want) {
      s_prefix = prefix | ((uint32_t)bin << shift);
      s_rank = want - above;
    }
    __syncthreads();
  }
  const uint32_t cut = s_prefix;
  const int ties = s_rank;  // keys equal to `cut` that are taken, the lower blocks first
  int done = 0, tied = 0;
  for (int base = 0; base < n && done < a.top; base += kThreads) {
    const int i = base + tid;
    const uint32_t k = i < n ? keys[i] : 0u;
    const bool eq = i < n && k == cut, gt = i < n && k > cut;
    const unsigned beq = __ballot_sync(0xffffffffu, eq), bgt = __ballot_sync(0xffffffffu, gt);
    __syncthreads();
    if (lane == 0) warp_sum[0][warp] = __popc(beq), warp_sum[1][warp] = __popc(bgt);
    __syncthreads();
    int eq_before = tied, gt_before = done - min(tied, ties), eq_all = tied, gt_all = gt_before;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) eq_before += warp_sum[0][w], gt_before += warp_sum[1][w];
      eq_all += warp_sum[0][w], gt_all += warp_sum[1][w];
    }
    const unsigned low = (1u << lane) - 1u;
    eq_before += __popc(beq & low), gt_before += __popc(bgt & low);
    const bool take = gt || (eq && eq_before < ties);
    if (take) list[gt_before + min(eq_before, ties)] = i;
    tied = eq_all;
    done = gt_all + min(tied, ties);
  }
}

}  // namespace

extern "C" {

size_t hk_gqa_select_workspace_size(int32_t num_tokens, int32_t kv_heads, int32_t page_size, int32_t max_kv_len) {
  if (num_tokens <= 0 || kv_heads <= 0 || page_size <= 0 || max_kv_len <= 0) return 256;
  const size_t blocks = ((size_t)max_kv_len + page_size - 1) / page_size;
  return ((size_t)num_tokens * kv_heads * blocks * 4 + 255) / 256 * 256;
}

int hk_gqa_select_blocks(const uint16_t* q, int64_t q_stride, const int8_t* centroids, const float* centroid_scale,
                         const int32_t* block_table, int32_t bt_stride, const int32_t* cu_seqlens,
                         const int32_t* positions, int32_t num_lanes, int32_t num_tokens, int32_t q_heads,
                         int32_t kv_heads, int32_t head_dim, int32_t page_size, int64_t num_pages, int32_t max_kv_len,
                         int32_t top_blocks, int32_t sink, int32_t local, int32_t dtype, int32_t* blocks,
                         void* workspace, size_t workspace_bytes, void* stream) {
  HK_REQUIRE(dtype == HK_BF16 || dtype == HK_F16, "hk_gqa_select_blocks: dtype %d", dtype);
  HK_REQUIRE(num_lanes > 0 && num_tokens >= 0 && bt_stride > 0 && num_pages > 0 && max_kv_len >= 0,
             "hk_gqa_select_blocks: bad sizes (lanes %d, tokens %d, table stride %d, pages %lld, max_kv_len %d)", num_lanes,
             num_tokens, bt_stride, (long long)num_pages, max_kv_len);
  HK_REQUIRE(kv_heads > 0 && kv_heads <= 65535 && q_heads > 0 && q_heads % kv_heads == 0,
             "hk_gqa_select_blocks: %d query heads do not divide into %d KV heads", q_heads, kv_heads);
  HK_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "hk_gqa_select_blocks: head_dim %d not 64, 128 or 256", head_dim);
  HK_REQUIRE(page_size >= 16 && page_size <= 256 && page_size % 16 == 0,
             "hk_gqa_select_blocks: page_size %d must be a multiple of 16 up to 256", page_size);
  HK_REQUIRE(q_stride >= (int64_t)q_heads * head_dim && q_stride % 8 == 0,
             "hk_gqa_select_blocks: q_stride must hold a row and be a multiple of 8 elements");
  HK_REQUIRE(top_blocks > 0 && top_blocks <= 4096, "hk_gqa_select_blocks: top_blocks %d not in 1..4096", top_blocks);
  HK_REQUIRE(sink >= 0 && local >= 1 && sink <= top_blocks && local <= top_blocks && sink + local <= top_blocks,
             "hk_gqa_select_blocks: sink %d and local %d (at least 1) must fit in top_blocks %d", sink, local, top_blocks);
  if (num_tokens == 0) return HK_OK;
  HK_REQUIRE(q && centroids && centroid_scale && block_table && cu_seqlens && positions && blocks, "hk_gqa_select_blocks: null pointer");
  HK_REQUIRE(((uintptr_t)q | (uintptr_t)centroids) % 16 == 0 && (uintptr_t)workspace % 16 == 0,
             "hk_gqa_select_blocks: buffers must be 16-byte aligned");
  if (workspace == nullptr || workspace_bytes < hk_gqa_select_workspace_size(num_tokens, kv_heads, page_size, max_kv_len))
    return hk::fail(HK_ESPACE, "hk_gqa_select_blocks: workspace of %zu bytes is too small", workspace_bytes);
  HK_TRY(hk::ensure_device());
  SelectArgs a = {q, q_stride, centroids, centroid_scale, block_table, bt_stride, cu_seqlens, positions, num_lanes,
                  num_tokens, q_heads, kv_heads, head_dim, page_size, num_pages,
                  (int32_t)(((int64_t)max_kv_len + page_size - 1) / page_size), top_blocks, sink, local, blocks,
                  (uint32_t*)workspace, hk::err_word()};
  const dim3 grid(num_tokens, kv_heads);
  if (dtype == HK_F16) gqa_select_kernel<true><<<grid, kThreads, 0, (cudaStream_t)stream>>>(a);
  else gqa_select_kernel<false><<<grid, kThreads, 0, (cudaStream_t)stream>>>(a);
  HK_TRY_LAUNCH("gqa_select_kernel");
  return HK_OK;
}

}  // extern "C"
