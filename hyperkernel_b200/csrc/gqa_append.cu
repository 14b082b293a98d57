// Append into the block-scaled 8-bit GQA cache: e4m3 rows, one power-of-two scale for each page and KV head.
//
// The rows of a call that fall in one page form a run (the rows of a lane are consecutive).  For a
// run of rows o .. o + n - 1 of a page, and each KV head, for K and for V:
//   s_new = 2^e, e the least whole number with max|x| <= 448 * 2^e  (max|x| taken as at least 2^-32)
//   s     = s_new if o == 0 (the page starts anew), else max(s_old, s_new)
//   rows 0 .. o - 1 are requantised by s_old / s when s > s_old;  the new rows are e4m3_rn(x / s).
// e4m3 is itself a floating-point format, so a power of two costs no mantissa bits against
// max / 448, x / s is exact before its one rounding, and a page whose scale grows keeps its values
// exactly, except those that become e4m3 subnormals.
//
// A page whose last row is written gets its centroid: the column sums of its stored K values in
// units of 2^-9 (whole numbers, so their order does not matter), scaled to int8.
//
// One warp handles one (run, head, K or V): a decode step has one row in each run and is bound by
// latency (slot -> scale -> store), a prompt chunk has whole pages and is bound by HBM.  The
// warp reads its rows twice, once for the maximum and once to store them; the second read is
// of 16 KB at most that the same warp has just read.
#include "common.cuh"

namespace {

constexpr int kWarps = 8;

struct AppendArgs {
  const uint16_t* x[2];
  int64_t xs[2];
  uint8_t* cache[2];
  float* scale[2];
  const int32_t* slots;
  int32_t num_tokens, heads, dim, page_size;
  int64_t num_pages;
  int8_t* centroids;
  float* centroid_scale;
  unsigned long long* err;
};

// The least power of two s with top <= 448 s, top >= 2^-32.  448 = 1.75 * 2^8.
__device__ __forceinline__ float pow2_scale(float top) {
  const uint32_t b = __float_as_uint(fmaxf(top, 2.3283064365386963e-10f));
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ __forceinline__ uint16_t f32x2_to_e4m3x2(float lo, float hi) {
  return (uint16_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ uint32_t scale_e4m3x4(uint32_t w, float r) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __fmul_rn(e4m3_to_f32((uint8_t)(w >> (8 * i))), r);
  return (uint32_t)f32x2_to_e4m3x2(f[0], f[1]) | ((uint32_t)f32x2_to_e4m3x2(f[2], f[3]) << 16);
}

// Largest finite magnitude of 8 values; *bad is set when one of them is not finite.
__device__ __forceinline__ float finite_max8(const float* x, float top, bool* bad) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = fabsf(x[j]);
    if (v < INFINITY) top = fmaxf(top, v);
    else *bad = true;
  }
  return top;
}

template <bool kF16>
__global__ void __launch_bounds__(kWarps * 32) append_blocks_kernel(AppendArgs a) {
  const int t = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (t >= a.num_tokens) return;
  const int lane = threadIdx.x & 31;
  const int g = blockIdx.y >> 1, which = blockIdx.y & 1;
  const int slot = a.slots[t];
  const int page_size = a.page_size;
  if (slot < 0) return;  // a padding row, or one that hk_pack has reported
  const int64_t page = slot / page_size;
  if (page >= a.num_pages) {
    if (lane == 0) hk_flag(a.err, hk::kErrAppendSlot, (unsigned)t);
    return;
  }
  // A run starts where the row before lies in another page, or is not the row just before.
  if (t > 0) {
    const int before = a.slots[t - 1];
    if (before >= 0 && before / page_size == page) {
      if (before + 1 != slot && lane == 0) hk_flag(a.err, hk::kErrAppendSlot, (unsigned)t);
      return;
    }
  }
  const int o = (int)(slot - page * page_size);
  // Rows of this run: the longest stretch of slots slot, slot + 1, ... inside the page.
  int n = 1;
  for (int base = 1; o + base < page_size; base += 32) {
    const int i = base + lane;
    const bool ok = o + i < page_size && t + i < a.num_tokens && a.slots[t + i] == slot + i;
    const unsigned miss = __ballot_sync(0xffffffffu, !ok);
    if (miss != 0) {
      n = base + __ffs(miss) - 1;
      break;
    }
    n = base + 32;
  }
  const int dim = a.dim, vec = dim / 8;  // lanes per row: 8, 16 or 32
  const int per = 32 / vec;              // rows side by side in a warp
  const int sub = lane % vec, r0 = lane / vec;
  const uint16_t* x = a.x[which] + (int64_t)t * a.xs[which] + (int64_t)g * dim + sub * 8;
  uint8_t* block = a.cache[which] + (page * a.heads + g) * (int64_t)page_size * dim;
  float* scale = a.scale[which] + page * a.heads + g;
  const float old = o > 0 ? *scale : 0.f;

  float top = 0.f;
  bool bad = false;
#pragma unroll 4
  for (int r = r0; r < n; r += per) {
    float f[8];
    unpack8<kF16>(*reinterpret_cast<const uint4*>(x + r * a.xs[which]), f);
    top = finite_max8(f, top, &bad);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (bad) hk_flag(a.err, hk::kErrKvInput, (unsigned)t);
  const float s = fmaxf(pow2_scale(top), old);
  const float inv = __fdiv_rn(1.f, s);
  if (o > 0 && old < s) {
    const float r = __fmul_rn(old, inv);
    uint4* rows = reinterpret_cast<uint4*>(block);
    for (int i = lane; i < o * dim / 16; i += 32) {
      uint4 u = rows[i];
      rows[i] = make_uint4(scale_e4m3x4(u.x, r), scale_e4m3x4(u.y, r), scale_e4m3x4(u.z, r), scale_e4m3x4(u.w, r));
    }
  }
#pragma unroll 4
  for (int r = r0; r < n; r += per) {
    float f[8];
    unpack8<kF16>(*reinterpret_cast<const uint4*>(x + r * a.xs[which]), f);
    uint32_t q[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = f[j] == f[j] ? __fmul_rn(f[j], inv) : 0.f;  // NaN is stored as 0 (and flagged)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      q[j] = (uint32_t)f32x2_to_e4m3x2(f[4 * j], f[4 * j + 1]) | ((uint32_t)f32x2_to_e4m3x2(f[4 * j + 2], f[4 * j + 3]) << 16);
    *reinterpret_cast<uint2*>(block + (int64_t)(o + r) * dim + sub * 8) = make_uint2(q[0], q[1]);
  }
  if (lane == 0) *scale = s;

  if (which == 0 && a.centroids != nullptr && o + n == page_size) {
    __syncwarp();  // the rows that the other lanes stored
    const int words = dim / 4;  // a lane sums 4 neighbouring dims of every row
    int sum[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    int big = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int wd = lane + 32 * k;
      if (wd >= words) continue;
      const uint32_t* col = reinterpret_cast<const uint32_t*>(block) + wd;
#pragma unroll 8
      for (int r = 0; r < page_size; ++r) {
        const uint32_t w = col[(int64_t)r * words];
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[k][j] += (int)(e4m3_to_f32((uint8_t)(w >> (8 * j))) * 512.f);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) big = max(big, abs(sum[k][j]));
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, d));
    const float m = (float)big;
    const float r = big > 0 ? __fdiv_rn(127.f, m) : 0.f;
    int8_t* c = a.centroids + (page * a.heads + g) * (int64_t)dim;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int wd = lane + 32 * k;
      if (wd >= words) continue;
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) w |= (uint32_t)((int)rintf(__fmul_rn((float)sum[k][j], r)) & 0xff) << (8 * j);
      reinterpret_cast<uint32_t*>(c)[wd] = w;
    }
    if (lane == 0)
      a.centroid_scale[page * a.heads + g] = __fmul_rn(s, __fdiv_rn(m, 127.f * 512.f * (float)page_size));
  }
}

}  // namespace

extern "C" int hk_gqa_append_fp8(const uint16_t* k_new, int64_t k_stride, const uint16_t* v_new, int64_t v_stride,
                                 int32_t dtype, const int32_t* slot_mapping, int32_t num_tokens, int32_t kv_heads,
                                 int32_t head_dim, int32_t page_size, int64_t num_pages, uint8_t* k_cache,
                                 uint8_t* v_cache, float* k_scale, float* v_scale, int8_t* centroids,
                                 float* centroid_scale, void* stream) {
  HK_REQUIRE(dtype == HK_BF16 || dtype == HK_F16, "hk_gqa_append_fp8: dtype %d", dtype);
  HK_REQUIRE(num_tokens >= 0 && kv_heads > 0 && kv_heads <= 16384 && num_pages > 0,
             "hk_gqa_append_fp8: bad sizes (tokens %d, kv_heads %d, pages %lld)", num_tokens, kv_heads, (long long)num_pages);
  HK_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "hk_gqa_append_fp8: head_dim %d not 64, 128 or 256", head_dim);
  HK_REQUIRE(page_size >= 16 && page_size <= 256 && page_size % 16 == 0,
             "hk_gqa_append_fp8: page_size %d must be a multiple of 16 up to 256", page_size);
  HK_REQUIRE(k_stride >= (int64_t)kv_heads * head_dim && v_stride >= (int64_t)kv_heads * head_dim && (k_stride | v_stride) % 8 == 0,
             "hk_gqa_append_fp8: row strides must hold a row and be multiples of 8 elements");
  HK_REQUIRE((centroids == nullptr) == (centroid_scale == nullptr), "hk_gqa_append_fp8: centroids need their scales");
  if (num_tokens == 0) return HK_OK;
  HK_REQUIRE(k_new && v_new && slot_mapping && k_cache && v_cache && k_scale && v_scale, "hk_gqa_append_fp8: null pointer");
  HK_REQUIRE(((uintptr_t)k_new | (uintptr_t)v_new | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)centroids) % 16 == 0,
             "hk_gqa_append_fp8: buffers must be 16-byte aligned");
  HK_TRY(hk::ensure_device());
  AppendArgs a;
  a.x[0] = k_new, a.x[1] = v_new, a.xs[0] = k_stride, a.xs[1] = v_stride;
  a.cache[0] = k_cache, a.cache[1] = v_cache, a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.slots = slot_mapping, a.num_tokens = num_tokens, a.heads = kv_heads, a.dim = head_dim, a.page_size = page_size;
  a.num_pages = num_pages, a.centroids = centroids, a.centroid_scale = centroid_scale, a.err = hk::err_word();
  const dim3 grid((num_tokens + kWarps - 1) / kWarps, 2 * kv_heads);
  if (dtype == HK_F16) append_blocks_kernel<true><<<grid, kWarps * 32, 0, (cudaStream_t)stream>>>(a);
  else append_blocks_kernel<false><<<grid, kWarps * 32, 0, (cudaStream_t)stream>>>(a);
  HK_TRY_LAUNCH("append_blocks_kernel");
  return HK_OK;
}
