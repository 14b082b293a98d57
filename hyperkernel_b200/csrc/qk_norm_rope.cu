// RMS norm of every query and key head with its gain, and the rotation by the row's position, in
// one pass over the projection's rows.
//
//   y = x / sqrt(mean(x^2) + eps) * gain;   (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)
//
// with (c, s) from the row's line of an hk_rope_table table and (a, b) = (i, i + rot / 2), or
// (2i, 2i + 1) in the interleaved form; dims past rot pass unrotated.  Everything is fp32 from the
// load to the one rounding of the store.
//
// Bound: HBM, each head read and written once.  A head is held by D / 8 lanes (rounded up to a
// power of two), 16 bytes each, so the sum of squares is a few shuffles and the partner of a
// rotated element is either in the same lane (interleaved) or rot / 16 lanes away.  A warp takes
// kHeads heads of one row and issues all their loads first: that keeps enough bytes in flight, and the
// row's cosines and sines are read once for all of them.
#include "common.cuh"

namespace {

constexpr int kWarps = 8;  // per CTA
constexpr int kIters = 4;  // head groups a warp holds at once

struct NormRopeArgs {
  const uint16_t* x[2];   // q, k
  const uint16_t* gain[2];
  uint16_t* y[2];
  int64_t xs[2], ys[2];   // row strides in elements
  int32_t heads[2];
  const float* table;
  int64_t table_rows;
  const int32_t* positions;
  int32_t num_tokens, dim, rot, items;  // items: warps per row
  float eps;
  unsigned long long* err;
};

// LPH lanes per head (8, 16 or 32).
template <bool kF16, int LPH, bool kPairs>
__global__ void __launch_bounds__(kWarps * 32) norm_rope_kernel(NormRopeArgs a) {
  constexpr int kGroups = 32 / LPH;  // heads side by side in a warp
  const uint32_t item = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const uint32_t row = item / (uint32_t)a.items;
  if (row >= (uint32_t)a.num_tokens) return;
  const int64_t t = row;
  const int pos = a.positions[t];
  if (pos < 0) return;  // a padding row
  const int lane = threadIdx.x & 31, sub = lane % LPH, e0 = sub * 8;
  if (pos >= a.table_rows) {
    if (lane == 0) hk_flag(a.err, hk::kErrPosition, (unsigned)t);
    return;
  }
  const bool on = e0 < a.dim;
  const int h0 = (int)(item - row * a.items) * (kGroups * kIters) + lane / LPH;
  const int total = a.heads[0] + a.heads[1];

  uint4 v[kIters];
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int h = h0 + i * kGroups;
    v[i] = make_uint4(0, 0, 0, 0);
    if (on && h < total) {
      const int w = h >= a.heads[0];
      v[i] = *reinterpret_cast<const uint4*>(a.x[w] + t * a.xs[w] + (int64_t)(h - w * a.heads[0]) * a.dim + e0);
    }
  }
  // This lane's 8 cosines and sines (4 of each, twice, when neighbours pair up); 1 and 0 outside the rotated dims.
  float c[8], s[8];
  const float* line = a.table + (int64_t)pos * a.rot;
  const int half = a.rot / 2;
  const bool turned = e0 < a.rot;
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = 1.f, s[j] = 0.f;
  if (turned) {
    const float* f = line + (kPairs ? e0 / 2 : e0 < half ? e0 : e0 - half);
#pragma unroll
    for (int j = 0; j < (kPairs ? 4 : 8); j += 4) {
      const float4 x = *reinterpret_cast<const float4*>(f + j), y = *reinterpret_cast<const float4*>(f + half + j);
      const float cx[4] = {x.x, x.y, x.z, x.w}, sx[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (kPairs) c[2 * e] = c[2 * e + 1] = cx[e], s[2 * e] = s[2 * e + 1] = sx[e];
        else c[j + e] = cx[e], s[j + e] = sx[e];
      }
    }
  }
  const float inv_dim = 1.f / (float)a.dim;
  const int partner = e0 < half ? lane + half / 8 : lane - half / 8;  // halves form: rot % 16 == 0
  const float sign = e0 < half ? -1.f : 1.f;
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int h = h0 + i * kGroups;
    const int w = h >= a.heads[0];
    float x[8];
    unpack8<kF16>(v[i], x);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(fmaf(ss, inv_dim, a.eps));
    float g[8];
    if (a.gain[w] != nullptr && on) {
      unpack8<kF16>(*reinterpret_cast<const uint4*>(a.gain[w] + e0), g);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * r * g[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= r;
    }
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (kPairs) {
        y[j] = (j & 1) ? fmaf(x[j], c[j], x[j ^ 1] * s[j]) : fmaf(x[j], c[j], -(x[j ^ 1] * s[j]));
      } else {
        const float other = __shfl_sync(0xffffffffu, x[j], turned ? partner : lane);
        y[j] = turned ? fmaf(x[j], c[j], sign * (other * s[j])) : x[j];
      }
    }
    if (on && h < total)
      *reinterpret_cast<uint4*>(a.y[w] + t * a.ys[w] + (int64_t)(h - w * a.heads[0]) * a.dim + e0) = pack8<kF16>(y);
  }
}

template <bool kF16, int LPH>
void launch(const NormRopeArgs& a, bool pairs, unsigned grid, cudaStream_t s) {
  if (pairs) norm_rope_kernel<kF16, LPH, true><<<grid, kWarps * 32, 0, s>>>(a);
  else norm_rope_kernel<kF16, LPH, false><<<grid, kWarps * 32, 0, s>>>(a);
}

}  // namespace

extern "C" int hk_qk_norm_rope(const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride,
                               const uint16_t* q_gain, const uint16_t* k_gain, const float* table,
                               int64_t table_rows, int32_t rot_dim, int32_t interleaved,
                               const int32_t* positions, int32_t num_tokens, int32_t q_heads,
                               int32_t kv_heads, int32_t head_dim, float eps, int32_t dtype,
                               uint16_t* q_out, int64_t q_out_stride, uint16_t* k_out,
                               int64_t k_out_stride, void* stream) {
  HK_REQUIRE(dtype == HK_BF16 || dtype == HK_F16, "hk_qk_norm_rope: dtype %d", dtype);
  HK_REQUIRE(num_tokens >= 0 && q_heads >= 0 && kv_heads >= 0 && q_heads <= 65536 && kv_heads <= 65536 &&
                 q_heads + kv_heads > 0,
             "hk_qk_norm_rope: bad sizes (tokens %d, heads %d and %d)", num_tokens, q_heads, kv_heads);
  HK_REQUIRE(head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0,
             "hk_qk_norm_rope: head_dim %d must be a multiple of 8 up to 256", head_dim);
  HK_REQUIRE(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 16 == 0,
             "hk_qk_norm_rope: rot_dim %d must be a multiple of 16 up to head_dim", rot_dim);
  HK_REQUIRE(eps >= 0.f && table_rows >= 0, "hk_qk_norm_rope: negative eps or table_rows");
  const int64_t qd = (int64_t)q_heads * head_dim, kd = (int64_t)kv_heads * head_dim;
  HK_REQUIRE(q_stride >= qd && q_out_stride >= qd && k_stride >= kd && k_out_stride >= kd &&
                 (q_stride | q_out_stride | k_stride | k_out_stride) % 8 == 0,
             "hk_qk_norm_rope: row strides must hold a row and be multiples of 8 elements");
  if (num_tokens == 0) return HK_OK;
  HK_REQUIRE((q_heads == 0 || (q && q_out)) && (kv_heads == 0 || (k && k_out)) && positions && (table || rot_dim == 0),
             "hk_qk_norm_rope: null pointer");
  HK_REQUIRE(((uintptr_t)q | (uintptr_t)k | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)q_gain |
              (uintptr_t)k_gain | (uintptr_t)table) % 16 == 0,
             "hk_qk_norm_rope: buffers must be 16-byte aligned");
  HK_TRY(hk::ensure_device());
  NormRopeArgs a;
  a.x[0] = q, a.x[1] = k, a.gain[0] = q_gain, a.gain[1] = k_gain, a.y[0] = q_out, a.y[1] = k_out;
  a.xs[0] = q_stride, a.xs[1] = k_stride, a.ys[0] = q_out_stride, a.ys[1] = k_out_stride;
  a.heads[0] = q_heads, a.heads[1] = kv_heads;
  a.table = table, a.table_rows = rot_dim == 0 ? INT64_MAX : table_rows, a.positions = positions;
  a.num_tokens = num_tokens, a.dim = head_dim, a.rot = rot_dim, a.eps = eps, a.err = hk::err_word();
  const int lph = head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32;
  const int per = 32 / lph * kIters;
  a.items = (q_heads + kv_heads + per - 1) / per;
  const int64_t ctas = ((int64_t)num_tokens * a.items + kWarps - 1) / kWarps;
  HK_REQUIRE(ctas * kWarps <= INT32_MAX, "hk_qk_norm_rope: too many heads in one call");
  const cudaStream_t s = (cudaStream_t)stream;
  const bool pairs = interleaved != 0;
  if (dtype == HK_F16) {
    if (lph == 8) launch<true, 8>(a, pairs, (unsigned)ctas, s);
    else if (lph == 16) launch<true, 16>(a, pairs, (unsigned)ctas, s);
    else launch<true, 32>(a, pairs, (unsigned)ctas, s);
  } else {
    if (lph == 8) launch<false, 8>(a, pairs, (unsigned)ctas, s);
    else if (lph == 16) launch<false, 16>(a, pairs, (unsigned)ctas, s);
    else launch<false, 32>(a, pairs, (unsigned)ctas, s);
  }
  HK_TRY_LAUNCH("norm_rope_kernel");
  return HK_OK;
}
