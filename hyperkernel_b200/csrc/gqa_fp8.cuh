// The block-scaled 8-bit GQA attention: arguments its kernels share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace hk {

struct GqaArgs {
  const uint16_t* q;  // [T][q_heads][dim], rows q_stride elements apart
  int64_t q_stride;
  const uint8_t* kc;  // [num_pages][kv_heads][page_size][dim] e4m3
  const uint8_t* vc;
  const float* ks;    // [num_pages][kv_heads]
  const float* vs;
  const int32_t* bt;
  int32_t bt_stride;
  const int32_t* cu;
  const int32_t* positions;
  const int32_t* blocks;  // [T][kv_heads][top] rising block indices, -1 behind the last; null: every block
  int32_t top;
  int32_t num_lanes, num_tokens, q_heads, kv_heads, dim, page_size;
  int64_t num_pages;
  int32_t max_rows;
  float scale;
  uint16_t* out;  // [T][q_heads][dim]
  float* lse;     // [T][q_heads]
  unsigned long long* err;
};

// The reference M of a row's weights 2^(x - M), x = score + log2 vs, in fp16.  Those have full precision from 2^-14 up to
// 65,504, and 2^-25 absolutely below.  M is set kHead below the largest x in sight, and set anew when an x passes it by
// more than kRoom, or when a whole step of the context has stayed kSlack below it: then what is summed so far is scaled up,
// which fp32 has room for.  So a token of much weight early in a long context (after which everything else would be
// below the range) costs the tokens after it nothing.  M does not come further than kDeep below its highest (there, fp16
// reaches 2^-61 of the largest weight in full), nor where the sum of w / vs is too large to be scaled (vs below 2^-60 or so).
// (Where M lies as deep as it may and the scores are lower still, every step of a chunk looks for a lower one in vain: 168 -> 185 us,
// measured with kDeep at 16 and a token 20 nats above the others; at 40 nothing changes up to 40 nats.)
// (With M at the running maximum, the part of 30,000 tokens 17 nats below a first one was off by up to 3% of itself, and at 24 nats lost.)
constexpr float kNoMax = -3.402823466e38f;  // of a row that has seen no score: the lowest finite value
constexpr float kHead = 7.f, kRoom = 15.f, kSlack = 3.f, kDeep = 40.f, kFullSum = 1e24f;

__device__ __forceinline__ float new_reference(float m, float most, float peak, bool may_fall) {
  if (may_fall && most < m - kSlack && most > kNoMax) return fmaxf(most - kHead, peak - kDeep);
  return fmaxf(m, most - kHead);
}

// A kernel launched by launch_early may start while the one before it in the stream still runs: its launch is hidden, and it
// waits (wait_for_grid_before) before it reads or writes anything.  The one before allows it by let_next_grid_start.
__device__ __forceinline__ void let_next_grid_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_grid_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid, c.blockDim = dim3(threads), c.dynamicSmemBytes = smem, c.stream = stream;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &at, c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, P(args)...);
}

// The lane of row t: the largest b with cu[b] <= t.
__device__ __forceinline__ int lane_of_row(const int32_t* __restrict__ cu, int num_lanes, int t) {
  int lo = 0, hi = num_lanes;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

}  // namespace hk

namespace hk {

// The tcgen05 kernel for prompt chunks (gqa_prefill.cu): the lanes with more than `least` query rows (rows x
// heads of a group) at dims 64 and 128.  `workspace`: gqa_prefill_workspace bytes.
bool gqa_prefill_supported(int32_t dim);
size_t gqa_prefill_workspace(int32_t dim);
int gqa_prefill(const GqaArgs& a, int32_t dtype, int32_t least, int64_t max_kv_len, void* workspace, cudaStream_t stream);

}  // namespace hk
