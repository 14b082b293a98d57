// RMS norm of every query and key head with its gain, and the rotation by the row's position, in
// one pass over the projection's rows.
//
//   y = x / sqrt(mean(x^2) + eps) * gain;   (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)
//
// with (c, s) from the row's line of an hk_rope_table table and (a, b) = (i, i + rot / 2), or
// (2i, 2i + 1) in the interleaved form; dims past rot pass unrotated.  Everything is fp32 from the
// load to the one rounding of the store.
//
// Bound: HBM, each head read and written once.  D / 8 lanes (rounded up to a power of two) hold a head, eight
// elements each as two runs of four: four of the first half of the rotated dims and their four partners
// (interleaved: eight neighbours), or eight dims past them.  So partners meet in one thread, and a lane's
// products of gain with cosine and sine, the same for all heads, are formed once:
//   out_j = (r x_j) A_j + (r x_p(j)) B_j,  A = gain * c,  B = -+ gain_p * s,  r = 1 / sqrt(mean + eps).
// A warp takes kIters groups of heads of one row and issues all their loads first.  Measured: 8192 rows of 64 + 8 heads of
// 128, 59.7 us, 5.1 TB/s (80% of the measured copy rate); 64 rows 2.8 us.
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
  int32_t num_tokens, dim, rot, items, q_items;  // warps per row, and those of q among them
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
  const int part = (int)(item - row * a.items);  // the first items of a row are of q, the others of k
  const int w = part >= a.q_items;
  const int heads = w ? a.heads[1] : a.heads[0];
  const int h0 = (part - (w ? a.q_items : 0)) * (kGroups * kIters) + lane / LPH;
  const int half = a.rot / 2;
  const bool on = e0 < a.dim, turned = e0 < a.rot;
  // This lane's two runs of four.
  const int at0 = kPairs || !turned ? e0 : e0 / 2, at1 = kPairs || !turned ? e0 + 4 : half + e0 / 2;
  const uint16_t* x = (w ? a.x[1] : a.x[0]) + t * (w ? a.xs[1] : a.xs[0]);
  uint16_t* y = (w ? a.y[1] : a.y[0]) + t * (w ? a.ys[1] : a.ys[0]);

  uint2 v[kIters][2];
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int h = h0 + i * kGroups;
    v[i][0] = v[i][1] = make_uint2(0, 0);
    if (on && h < heads) {
      v[i][0] = *reinterpret_cast<const uint2*>(x + h * a.dim + at0);
      v[i][1] = *reinterpret_cast<const uint2*>(x + h * a.dim + at1);
    }
  }
  constexpr int kPartner = kPairs ? 1 : 4;
  float A[8], B[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) A[j] = 1.f, B[j] = 0.f;
  const uint16_t* gain = w ? a.gain[1] : a.gain[0];
  if (gain != nullptr && on) {
    const uint2 lo = *reinterpret_cast<const uint2*>(gain + at0), hi = *reinterpret_cast<const uint2*>(gain + at1);
    unpack8<kF16>(make_uint4(lo.x, lo.y, hi.x, hi.y), A);
  }
  if (turned) {
    // Four angles: those of the first run (halves), or of the pairs (0, 1) (2, 3) (4, 5) (6, 7).
    const float* line = a.table + (int64_t)pos * a.rot + e0 / 2;
    const float4 cv = *reinterpret_cast<const float4*>(line), sv = *reinterpret_cast<const float4*>(line + half);
    const float c[4] = {cv.x, cv.y, cv.z, cv.w}, s[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int f = kPairs ? j / 2 : j % 4;
      B[j] = (j & kPartner) ? A[j ^ kPartner] * s[f] : -(A[j ^ kPartner] * s[f]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) A[j] *= c[kPairs ? j / 2 : j % 4];
  }
  const float inv_dim = 1.f / (float)a.dim;
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int h = h0 + i * kGroups;
    float f[8];
    unpack8<kF16>(make_uint4(v[i][0].x, v[i][0].y, v[i][1].x, v[i][1].y), f);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(f[j], f[j], ss);
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(fmaf(ss, inv_dim, a.eps));
    float g[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= r;
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = f[j] * A[j];
    if (turned) {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = fmaf(f[j ^ kPartner], B[j], g[j]);
    }
    if (on && h < heads) {
      const uint4 u = pack8<kF16>(g);
      *reinterpret_cast<uint2*>(y + h * a.dim + at0) = make_uint2(u.x, u.y);
      *reinterpret_cast<uint2*>(y + h * a.dim + at1) = make_uint2(u.z, u.w);
    }
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
  a.q_items = (q_heads + per - 1) / per;
  a.items = a.q_items + (kv_heads + per - 1) / per;
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
