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
// Two kernels.  The first spreads the scores over CTAs of 256 blocks (a centroid is read by dim / 16
// lanes, 16 bytes each, and dotted by dp4a) and leaves them in the workspace as keys whose unsigned
// order is the scores' order: bound by reading the centroids.  The second has one CTA per (row, KV head),
// whose threads hold the keys in registers and find the lowest chosen key bit by bit from the
// first bit in which the keys differ: counts by warp reductions, so that equal leading bits, which
// scores have, cost no contention.  One scan then places the chosen indices in rising order.
// Measured: 64 of up to 2,048 blocks for 16 rows and 8 KV heads, 18.6 us; with the attention that follows, 65 us in all.
#include "common.cuh"
#include "gqa_fp8.cuh"

namespace {

constexpr int kScoreThreads = 128;
constexpr int kScoreBlocks = 256;  // per CTA
constexpr int kHold = 16;          // keys a thread of the second kernel holds

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

// Blocks in sight of row t; 0 when they pass the call's max_kv_len.
__device__ __forceinline__ int blocks_of(const SelectArgs& a, int t) {
  const int pos = a.positions[t];
  const int n = pos < 0 ? 0 : pos / a.page_size + 1;
  return n <= a.max_blocks ? n : 0;
}

template <bool kF16>
__global__ void __launch_bounds__(kScoreThreads) gqa_score_kernel(SelectArgs a) {
  __shared__ float warp_max[kScoreThreads / 32];
  __shared__ int page_s[kScoreBlocks];
  __shared__ __align__(16) int8_t c8[256];
  const int t = blockIdx.x, g = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  hk::let_next_grid_start();
  if (t >= a.cu[a.num_lanes]) return;
  const int n = blocks_of(a, t), from = blockIdx.z * kScoreBlocks, to = min(n - a.local, from + kScoreBlocks);
  if (n <= a.top || from >= to) return;
  // The pages first: their addresses are what the loop waits for.
  const int b = hk::lane_of_row(a.cu, a.num_lanes, t);
  for (int k = tid; k < kScoreBlocks; k += kScoreThreads) {
    const int i = from + k;
    int page = i < to && i < a.bt_stride ? a.bt[(int64_t)b * a.bt_stride + i] : -1;
    if (page <= 0 || page >= a.num_pages) {
      if (i < to && i >= a.sink) hk_flag(a.err, hk::kErrAttnPage, (unsigned)b);
      page = -1;
    }
    page_s[k] = page;
  }
  const int group = a.q_heads / a.kv_heads;
  float u[2] = {0.f, 0.f}, mine = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = tid + k * kScoreThreads;
    if (d >= a.dim) continue;
    double sum = 0.0;
#pragma unroll 4
    for (int h = 0; h < group; ++h) {
      const uint16_t w = a.q[t * a.q_stride + (int64_t)(g * group + h) * a.dim + d];
      sum += (double)(kF16 ? __half2float(*reinterpret_cast<const __half*>(&w)) : bf16_bits_to_f32(w));
    }
    u[k] = (float)sum;
    const float v = fabsf(u[k]);
    mine = v < INFINITY ? fmaxf(mine, v) : INFINITY;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, o));
  if (lane == 0) warp_max[warp] = mine;
  __syncthreads();
  float m = 0.f;
#pragma unroll
  for (int w = 0; w < kScoreThreads / 32; ++w) m = fmaxf(m, warp_max[w]);
  if (m < 0x1p-64f) {  // 127 / m could pass fp32: a power of two on u and m changes nothing else
    m *= 0x1p64f;
#pragma unroll
    for (int k = 0; k < 2; ++k) u[k] *= 0x1p64f;
  }
  // A row with a value that is not finite scores 0 everywhere.
  const float r = m > 0.f && m < INFINITY ? __fdiv_rn(127.f, m) : 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = tid + k * kScoreThreads;
    if (d < a.dim) c8[d] = r > 0.f ? (int8_t)rintf(__fmul_rn(u[k], r)) : (int8_t)0;
  }
  __syncthreads();

  const int vec = a.dim / 16, sub = tid % vec;  // 4, 8 or 16 lanes per centroid
  const int4 y = reinterpret_cast<const int4*>(c8)[sub];
  uint32_t* keys = a.keys + ((int64_t)t * a.kv_heads + g) * a.max_blocks;
  const int per = kScoreThreads / vec;
#pragma unroll 8
  for (int base = 0; base < to - from; base += per) {
    const int i = base + tid / vec, page = i < kScoreBlocks ? page_s[i] : -1;
    const bool ok = page > 0;
    const int64_t at = (int64_t)(ok ? page : 0) * a.kv_heads + g;
    const int4 x = reinterpret_cast<const int4*>(a.centroids + at * a.dim)[sub];
    const float f = a.centroid_scale[at];
    int dot = __dp4a(x.x, y.x, __dp4a(x.y, y.y, __dp4a(x.z, y.z, __dp4a(x.w, y.w, 0))));
    for (int o = 1; o < vec; o <<= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (sub == 0 && from + i < to) keys[from + i] = ok ? order_key(__fadd_rn(__fmul_rn((float)dot, f), 0.f)) : 0u;  // -0 becomes 0
  }
}

// kThreads threads hold kHold keys each (`kHeld`), or read them again for every count where there are more.
template <int kThreads, bool kHeld>
__global__ void __launch_bounds__(kThreads) gqa_select_kernel(SelectArgs a) {
  constexpr int kWarps = kThreads / 32;
  __shared__ uint32_t and_s, or_s;
  __shared__ int count_s[32];
  __shared__ int64_t sums_s[kWarps];
  const int t = blockIdx.x, g = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  hk::wait_for_grid_before();
  if (t >= a.cu[a.num_lanes]) return;
  int32_t* list = a.blocks + ((int64_t)t * a.kv_heads + g) * a.top;
  const int n = blocks_of(a, t);
  if (n == 0 && a.positions[t] >= 0 && tid == 0) hk_flag(a.err, hk::kErrPosition, (unsigned)t);
  if (n <= a.top) {
    for (int i = tid; i < a.top; i += kThreads) list[i] = i < n ? i : -1;
    return;
  }
  for (int i = tid; i < a.sink; i += kThreads) list[i] = i;
  for (int i = tid; i < a.local; i += kThreads) list[a.top - a.local + i] = n - a.local + i;
  const int want = a.top - a.sink - a.local, m = n - a.sink - a.local;
  if (want == 0) return;
  const uint32_t* keys = a.keys + ((int64_t)t * a.kv_heads + g) * a.max_blocks + a.sink;
  // Thread tid has keys tid * per .. + per - 1.
  const int per = (m + kThreads - 1) / kThreads, first = tid * per, mine = max(0, min(per, m - first));
  uint32_t k[kHeld ? kHold : 1];
  uint32_t all = 0xffffffffu, any = 0;
  if (kHeld) {
#pragma unroll
    for (int j = 0; j < kHold; ++j)
      if (j < mine) k[j] = keys[first + j], all &= k[j], any |= k[j];
  } else {
    for (int j = 0; j < mine; ++j) all &= keys[first + j], any |= keys[first + j];
  }
  auto count = [&](uint32_t at_least) {
    int c = 0;
    if (kHeld) {
#pragma unroll
      for (int j = 0; j < kHold; ++j) c += j < mine && k[j] >= at_least;
    } else {
      for (int j = 0; j < mine; ++j) c += keys[first + j] >= at_least;
    }
    return c;
  };
  if (tid < 32) count_s[tid] = 0;
  if (tid == 0) and_s = 0xffffffffu, or_s = 0;
  __syncthreads();
  all = __reduce_and_sync(0xffffffffu, all), any = __reduce_or_sync(0xffffffffu, any);
  if (lane == 0) atomicAnd(&and_s, all), atomicOr(&or_s, any);
  __syncthreads();
  all = and_s;
  const uint32_t vary = all ^ or_s;
  // The largest value that at least `want` keys reach: bits above the first varying one are common.
  uint32_t cut = vary == 0 ? all : all & ~(0xffffffffu >> __clz(vary));
  int reach = m;  // keys >= cut
  for (int bit = vary == 0 ? -1 : 31 - __clz(vary); bit >= 0 && reach != want; --bit) {
    const uint32_t tryout = cut | (1u << bit);
    const int c = __reduce_add_sync(0xffffffffu, count(tryout));
    if (lane == 0) atomicAdd(&count_s[bit], c);
    __syncthreads();
    if (count_s[bit] >= want) cut = tryout, reach = count_s[bit];
  }
  // All keys above the cut are taken, and of those equal to it the lower blocks, until `want` are.
  const int above = reach == want ? count(cut) : cut == 0xffffffffu ? 0 : count(cut + 1);
  const int equal = reach == want ? 0 : count(cut) - above;
  const int64_t v = (int64_t)above << 32 | equal;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sums_s[warp] = x;
  __syncthreads();
  int64_t before = x - v, total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums_s[w];
    total += sums_s[w];
  }
  const int ties = want - (int)(total >> 32);
  int gt = (int)(before >> 32), eq = (int)(uint32_t)before;
  auto place = [&](int j, uint32_t key) {
    const bool over = reach == want ? key >= cut : key > cut, same = reach != want && key == cut;
    if (over || (same && eq < ties)) list[a.sink + gt + min(eq, ties)] = a.sink + first + j;
    gt += over, eq += same;
  };
  if (kHeld) {
#pragma unroll
    for (int j = 0; j < kHold; ++j)
      if (j < mine) place(j, k[j]);
  } else {
    for (int j = 0; j < mine; ++j) place(j, keys[first + j]);
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
  const cudaStream_t st = (cudaStream_t)stream;
  const int parts = (a.max_blocks + kScoreBlocks - 1) / kScoreBlocks;
  HK_REQUIRE(parts <= 65535, "hk_gqa_select_blocks: max_kv_len %d holds too many blocks", max_kv_len);
  if (a.max_blocks > top_blocks) {  // else every list is the whole range
    const dim3 grid(num_tokens, kv_heads, parts);
    if (dtype == HK_F16) gqa_score_kernel<true><<<grid, kScoreThreads, 0, st>>>(a);
    else gqa_score_kernel<false><<<grid, kScoreThreads, 0, st>>>(a);
    HK_TRY_LAUNCH("gqa_score_kernel");
  }
  const dim3 grid(num_tokens, kv_heads);
  const bool early = a.max_blocks > top_blocks;  // behind the scores
  auto select = [&](auto kernel, int threads) -> cudaError_t {
    if (early) return hk::launch_early(kernel, grid, threads, 0, st, a);
    kernel<<<grid, threads, 0, st>>>(a);
    return cudaSuccess;
  };
  if (a.max_blocks <= 256 * kHold) HK_TRY_CUDA(select(gqa_select_kernel<256, true>, 256));
  else if (a.max_blocks <= 1024 * kHold) HK_TRY_CUDA(select(gqa_select_kernel<1024, true>, 1024));
  else HK_TRY_CUDA(select(gqa_select_kernel<1024, false>, 1024));
  HK_TRY_LAUNCH("gqa_select_kernel");
  return HK_OK;
}

}  // extern "C"
