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
// A CTA looks at 4 or 32 rows of the call for one head and one of K and V.  Runs that start there are short
// (decode steps, verify blocks) or long (prompt chunks): the warps write the short ones, one each,
// then all warps together write the long ones, the rows held in registers between the maximum
// and the store when the run fits them (64 rows at dim 128).  Short runs are bound by latency (slot ->
// scale -> store), long ones by HBM.  The maximum is taken of the 16-bit patterns without their signs, whose
// order is the magnitudes': what is not finite shows in it too, and only then is it taken apart.
// Measured over buffers larger than L2, 8 KV heads of 128, pages of 64: 64 decode rows 4.3 us; 16 prompt chunks, 6,300 rows,
// 28.8 us (1.35 TB/s; 17.6 us where L2 still holds the buffers).
#include "common.cuh"

namespace {

constexpr int kWarps = 4;
constexpr int kShort = 8;  // rows of a run that one warp writes: at most four loads a lane at dim 128
constexpr int kHold = 8;   // 16-byte loads a thread keeps between its two passes

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

// Packed maximum of the sign-less 16-bit patterns of 8 values.
__device__ __forceinline__ uint32_t pattern_max8(const uint4& u, uint32_t top) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
  return top;
}

// Largest finite magnitude of 8 values.
template <bool kF16>
__device__ __forceinline__ float finite_max8(const uint4& u, float top) {
  float f[8];
  unpack8<kF16>(u, f);
#pragma unroll
  for (int j = 0; j < 8; ++j) top = fabsf(f[j]) < INFINITY ? fmaxf(top, fabsf(f[j])) : top;
  return top;
}

// Maximum over a team: a warp, or all warps of the CTA (then `smem` holds a word for each).
template <int kTeam>
__device__ __forceinline__ uint32_t team_max(uint32_t v, uint32_t* smem) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (kTeam == 32) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kTeam / 32; ++w) v = max(v, smem[w]);
  return v;
}

template <int kTeam>
__device__ __forceinline__ void team_sync() {
  if (kTeam == 32) __syncwarp();
  else __syncthreads();
}

// Writes the run of n rows from row t of the call (slot) for head g.  All threads of the team call it.
template <bool kF16, int kTeam>
__device__ __forceinline__ void write_run(const AppendArgs& a, int which, int g, int t, int slot, int n, uint32_t* smem, int* sum_s) {
  const int id = kTeam == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t page = slot / a.page_size;
  const int o = slot - (int)page * a.page_size;
  const int dim = a.dim, vec = dim / 8;  // threads per row: 8, 16 or 32
  const int per = kTeam / vec, sub = id % vec, r0 = id / vec;
  const int64_t stride = which ? a.xs[1] : a.xs[0];  // selected, not indexed: an indexed parameter goes to local memory
  const uint16_t* x = (which ? a.x[1] : a.x[0]) + (int64_t)t * stride + (int64_t)g * dim + sub * 8;
  uint8_t* block = (which ? a.cache[1] : a.cache[0]) + (page * a.heads + g) * (int64_t)a.page_size * dim;
  float* scale = (which ? a.scale[1] : a.scale[0]) + page * a.heads + g;
  const float old = o > 0 ? *scale : 0.f;

  uint4 held[kHold];
  const bool holds = n <= kHold * per;
#pragma unroll
  for (int i = 0; i < kHold; ++i) {
    const int r = r0 + i * per;
    held[i] = r < n ? *reinterpret_cast<const uint4*>(x + r * stride) : make_uint4(0, 0, 0, 0);
  }
  uint32_t pattern = 0;
#pragma unroll
  for (int i = 0; i < kHold; ++i) pattern = pattern_max8(held[i], pattern);
  for (int r = r0 + kHold * per; r < n; r += per) pattern = pattern_max8(*reinterpret_cast<const uint4*>(x + r * stride), pattern);
  pattern = team_max<kTeam>(max(pattern & 0xffffu, pattern >> 16), smem);
  const bool odd = pattern >= (kF16 ? 0x7c00u : 0x7f80u);  // a value that is not finite
  float top = kF16 ? __half2float(__ushort_as_half((uint16_t)pattern)) : __uint_as_float(pattern << 16);
  if (odd) {
    if (id == 0) hk_flag(a.err, hk::kErrKvInput, (unsigned)t);
    top = 0.f;
    for (int r = r0; r < n; r += per) top = finite_max8<kF16>(*reinterpret_cast<const uint4*>(x + r * stride), top);
    top = __uint_as_float(team_max<kTeam>(__float_as_uint(top), smem));
  }
  const float s = fmaxf(pow2_scale(top), old);
  const float inv = __fdiv_rn(1.f, s);
  if (o > 0 && old < s) {
    const float r = __fmul_rn(old, inv);
    uint4* rows = reinterpret_cast<uint4*>(block);
    for (int i = id; i < o * dim / 16; i += kTeam) {
      const uint4 u = rows[i];
      rows[i] = make_uint4(scale_e4m3x4(u.x, r), scale_e4m3x4(u.y, r), scale_e4m3x4(u.z, r), scale_e4m3x4(u.w, r));
    }
  }
  auto put = [&](int r, const uint4& u) {
    float f[8];
    unpack8<kF16>(u, f);
    if (odd) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = f[j] == f[j] ? f[j] : 0.f;  // NaN is stored as 0
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __fmul_rn(f[j], inv);
    uint32_t q[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      q[j] = (uint32_t)f32x2_to_e4m3x2(f[4 * j], f[4 * j + 1]) | ((uint32_t)f32x2_to_e4m3x2(f[4 * j + 2], f[4 * j + 3]) << 16);
    *reinterpret_cast<uint2*>(block + (int64_t)(o + r) * dim + sub * 8) = make_uint2(q[0], q[1]);
  };
#pragma unroll
  for (int i = 0; i < kHold; ++i)
    if (r0 + i * per < n) put(r0 + i * per, held[i]);
  if (!holds)
    for (int r = r0 + kHold * per; r < n; r += per) put(r, *reinterpret_cast<const uint4*>(x + r * stride));
  if (id == 0) *scale = s;

  if (which == 0 && a.centroids != nullptr && o + n == a.page_size) {
    // Thread: 8 neighbouring dims of every `per`-th row.  The values are whole multiples of 2^-9 below 2^9: 32 of them
    // add up exactly in fp32, and the rest of the sum is of whole numbers, so its order is free.
    int sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int i = id; i < dim; i += kTeam) sum_s[i] = 0;
    team_sync<kTeam>();  // also: the rows that other threads stored
    for (int base = r0; base < a.page_size; base += 16 * per) {
      float part[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const int r = base + i * per;
        if (r >= a.page_size) break;
        const uint2 u = *reinterpret_cast<const uint2*>(block + (int64_t)r * dim + sub * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((j < 2 ? u.x : u.y) >> (16 * (j & 1))), __NV_E4M3);
          const float2 f = __half22float2(__half2(h));
          part[2 * j] += f.x, part[2 * j + 1] += f.y;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += (int)(part[j] * 512.f);
    }
    for (int m = vec; m < 32; m <<= 1)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], m);
    if ((id & 31) < vec)
#pragma unroll
      for (int j = 0; j < 8; ++j) atomicAdd(&sum_s[sub * 8 + j], sum[j]);
    team_sync<kTeam>();
    uint32_t big = 0;
    for (int i = id; i < dim; i += kTeam) big = max(big, (uint32_t)abs(sum_s[i]));
    const float m = (float)team_max<kTeam>(big, smem);
    const float r = m > 0.f ? __fdiv_rn(127.f, m) : 0.f;
    int8_t* c = a.centroids + (page * a.heads + g) * (int64_t)dim;
    for (int i = id; i < dim; i += kTeam) c[i] = (int8_t)rintf(__fmul_rn((float)sum_s[i], r));
    if (id == 0) a.centroid_scale[page * a.heads + g] = __fmul_rn(s, __fdiv_rn(m, 127.f * 512.f * (float)a.page_size));
    team_sync<kTeam>();  // sum_s is free again
  }
}

// kRows rows of the call to a CTA.
template <bool kF16, int kRows>
__global__ void __launch_bounds__(kWarps * 32, 6) append_blocks_kernel(AppendArgs a) {
  __shared__ int sum_s[kWarps][256];
  __shared__ uint32_t max_s[kWarps];
  __shared__ unsigned start_s;
  __shared__ int n_s[kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // The heads of the same rows are neighbours in the grid, as they are in memory.
  const unsigned chunk = blockIdx.x / (2u * a.heads), part = blockIdx.x - chunk * (2u * a.heads);
  const int t0 = chunk * kRows, g = part >> 1, which = part & 1;
  const int page_size = a.page_size;
  if (warp == 0) {  // the rows at which runs start
    bool start = false;
    const int t = t0 + lane;
    const int slot = lane < kRows && t < a.num_tokens ? a.slots[t] : -1;
    if (slot >= 0) {  // else: a padding row, or one that hk_pack has reported
      const int page = slot / page_size;
      const int before = t > 0 ? a.slots[t - 1] : -1;
      const bool same = before >= 0 && before / page_size == page;
      if (page >= a.num_pages || (same && before + 1 != slot)) hk_flag(a.err, hk::kErrAppendSlot, (unsigned)t);
      else start = !same;
    }
    const unsigned starts = __ballot_sync(0xffffffffu, start);
    if (lane == 0) start_s = starts;
    if (lane < kRows) n_s[lane] = 0;
  }
  __syncthreads();
  const unsigned starts = start_s;
  int at = 0;
  for (unsigned left = starts; left != 0; left &= left - 1, ++at) {
    if (at % kWarps != warp) continue;
    const int i0 = __ffs(left) - 1, t = t0 + i0, slot = a.slots[t], o = slot % page_size;
    // The longest stretch of slots slot, slot + 1, ... inside the page.
    int n = 0;
    for (int base = 0; n == base && base < page_size - o; base += 32) {
      const int i = base + lane;
      const bool ok = o + i < page_size && t + i < a.num_tokens && a.slots[t + i] == slot + i;
      const unsigned miss = __ballot_sync(0xffffffffu, !ok);
      n = base + (miss != 0 ? __ffs(miss) - 1 : 32);
    }
    if (n <= kShort) write_run<kF16, 32>(a, which, g, t, slot, n, max_s, sum_s[warp]);
    else if (lane == 0) n_s[i0] = n;
  }
  __syncthreads();
  for (unsigned left = starts; left != 0; left &= left - 1) {
    const int i0 = __ffs(left) - 1;
    if (n_s[i0] > 0) write_run<kF16, kWarps * 32>(a, which, g, t0 + i0, a.slots[t0 + i0], n_s[i0], max_s, sum_s[0]);
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
  // Small calls: few rows to a CTA, for their latency; large ones: fewer CTAs that find nothing to do.  4 against 32 rows a CTA: 64 single
  // rows 4.3 us against 16.6, 300 14.4 against 23.1, 1,000 25.1 against 25.9, 1,100 26.6 against 26.0, 8,000 133 against 111;
  // one chunk of 500 rows 10.8 against 13.4, 900 20.0 against 23.1, 1,500 20.9 against 23.8; four of 2,048 rows 57.5 against 31.7;
  // 60 verify blocks of 5 rows 10.8 against 12.9, 250 22.8 against 13.7.
  const bool small = num_tokens <= 1024;
  const int rows = small ? 4 : 32;
  const int64_t ctas = ((int64_t)num_tokens + rows - 1) / rows * 2 * kv_heads;
  HK_REQUIRE(ctas <= INT32_MAX, "hk_gqa_append_fp8: too many rows and heads in one call");
  const unsigned grid = (unsigned)ctas;
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == HK_F16) {
    if (small) append_blocks_kernel<true, 4><<<grid, kWarps * 32, 0, s>>>(a);
    else append_blocks_kernel<true, 32><<<grid, kWarps * 32, 0, s>>>(a);
  } else {
    if (small) append_blocks_kernel<false, 4><<<grid, kWarps * 32, 0, s>>>(a);
    else append_blocks_kernel<false, 32><<<grid, kWarps * 32, 0, s>>>(a);
  }
  HK_TRY_LAUNCH("append_blocks_kernel");
  return HK_OK;
}
