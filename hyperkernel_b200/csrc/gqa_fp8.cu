// Ragged paged GQA attention over the block-scaled e4m3 cache, dense and over selected blocks.
//
//   s_j = scale * ks[page(j)] * (q . k_j),  o = sum_j softmax(s)_j vs[page(j)] v_j,  lse = log sum_j e^{s_j}
//
// over the tokens j <= position of the row (and, sparse, of the row's blocks).
//
// Bound: HBM, the cache read once (2 * dim bytes a token and KV head).  The query rows that share a KV
// head (rows of the lane x heads of the group) are the narrow side of the products, so the
// tokens take the M side of mma.m16n8k16 and 8 x NT query rows the N side:
//   S^T = K Q^T,  O^T += V^T P^T.
// e4m3 is exact in fp16, and so is q once each row is scaled by a power of two (but for values below 2^-21 of
// the row's largest, which keep an absolute error of 2^-32 of it), so the products are those of the
// stored values; P is rounded to fp16 (2^-11; below 2^-14 of 2^M to 2^-25 of it).
//
// Every warp streams 16-token chunks through a ring of its own in shared memory, filled by TMA (a chunk
// of one page and head is contiguous: 16 * dim bytes), so bytes in flight cost no registers and
// no barrier joins warps.  The order of k inside a product, and of the dims among the M tiles of
// the second one, is free, so each thread's fragments are runs of 16 bytes of a token (8 for V at
// dim 64), and TMA's 128-byte swizzle keeps those reads free of bank conflicts (2-way at most
// for V at dims 64 and 256).  For V the bytes of two tokens are interleaved by prmt before the
// conversion, which makes the transposed fragment.  P^T reaches the layout of a B fragment by
// movmatrix.
//
// With vs folded into the exponent, w_j = 2^(s_j + log2 vs - M), one reference M serves pages of
// any scale, and sum_j w_j / vs is the softmax's denominator.  M follows the row's largest weights (gqa_fp8.cuh); every
// 16 chunks a warp looks whether it has to come down.
//
// Work split: the 16-token chunks of all (lane, KV head, row tile) problems lie end to end in
// units of kWarps chunks, and every CTA takes an equal contiguous range of units.  Problems cut by
// a range's end leave fp32 partials, two at most for each CTA, which gqa_merge_kernel joins in
// the order of the ranges: results do not depend on timing.
//
// Measured: 64 lanes of 1K to 32K tokens, 64 query and 8 KV heads of 128: 217 us, 5.6 TB/s (87% of the measured copy rate); 32
// query and 8 KV heads of 64: 132 us, 4.6 TB/s; 5 rows of 32 heads over a million tokens: 474 us, 4.5 TB/s; one
// row over 778 tokens: 11 us, two launches and their dependent loads.
#include "common.cuh"
#include "gqa_fp8.cuh"
#include "sm100.cuh"

namespace {

using hk::GqaArgs;
namespace sm100 = hk::sm100;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = kWarps * 16;  // tokens
constexpr int kMaxCtasPerSm = 4;

// CTAs that an SM holds (by registers: 128 threads of at most 128, 168 or 255; by shared memory: see stages).  Three N tiles at
// dim 128 in 168 registers spill: 481 us against 474 us for 5 rows of 4 heads over a million tokens.  Two and four N tiles at
// dim 64 and four at dim 128 spill 4 to 60 bytes.  One N tile at dim 64 in five CTAs of 96 registers
// and four stages: 132.0 us against 130.1 us for 64 lanes of 1K to 32K tokens, 32 query and 8 KV heads.
constexpr int ctas_per_sm(int d, int nt) {
  return d == 256 ? 2 : d * nt <= 128 ? 4 : d * nt <= 320 ? 3 : 2;
}
constexpr int kLook = 16;           // chunks whose pages and scales are looked up at once
// Shared memory of a CTA: the ring, up to 1 KB for its alignment, the fixed arrays (Q's fragments, the rows' sums, lookups and barriers),
// and 1 KB that the device takes for itself; an SM has 228 KB.
constexpr int kSmBytes = 228 * 1024, kCtaBytes = 1024, kAlignBytes = 1024;
constexpr int fixed_bytes(int d, int nt) {
  return 16 * nt * d + 8 * nt * (4 * (3 + 2 * kWarps) + 8) + kWarps * (2 * kLook * 20 + 8 * kLook + 16) + 64;
}
// Chunks a warp keeps in flight: what is left for the ring.
constexpr int stages(int d, int nt) {
  return (kSmBytes / ctas_per_sm(d, nt) - kCtaBytes - kAlignBytes - fixed_bytes(d, nt)) / (kWarps * 32 * d);
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
using hk::kNoMax;

// What CTA i leaves for the merge: the problem its last range starts and does not finish, and whether the
// problem it continues from the CTA before ends in it.
struct Rec {
  int32_t item, sub;   // problem of the open last segment (item < 0: none)
  int32_t ends;        // the first segment was continued from the CTA before, and ends here
  int32_t pad;
};

struct SplitArgs {
  GqaArgs a;
  int32_t is_f16;
  int32_t group, tiles_max;
  int32_t items;  // lanes (dense) or rows (sparse)
  int32_t most;   // dense: query rows (rows x group) of a lane above which it is not this kernel's
  Rec* rec;       // [grid]
  float* part;    // [grid][2][R * D + 2 R]
};

struct Item {
  int rows, t0, len;  // query rows (tokens), first row, KV tokens (sparse: of the list)
  int pos;            // sparse: the row's position
  int tiles;
  int64_t nu;         // units of one (row tile, head)
};

template <int R, bool kSparse>
__device__ __forceinline__ Item item_of(const SplitArgs& s, int i, bool report) {
  const GqaArgs& a = s.a;
  Item x;
  if (kSparse) {
    const int total = min(a.cu[a.num_lanes], a.num_tokens);
    x.t0 = i;
    x.rows = i < total ? 1 : 0;
    x.pos = x.rows ? a.positions[i] : -1;
    x.len = x.pos < 0 ? 0 : min(a.top, x.pos / a.page_size + 1) * a.page_size;
  } else {
    x.t0 = a.cu[i];
    const int t1 = min(a.cu[i + 1], a.num_tokens);
    x.rows = x.t0 >= 0 ? max(0, t1 - x.t0) : 0;
    if (x.rows > a.max_rows) {
      if (report) hk_flag(a.err, hk::kErrLaneRows, (unsigned)i);
      x.rows = 0;
    }
    if ((int64_t)x.rows * s.group > s.most) x.rows = 0;
    x.pos = 0;
    x.len = x.rows ? max(0, a.positions[t1 - 1] + 1) : 0;
  }
  x.tiles = (x.rows * s.group + R - 1) / R;
  x.nu = max(1, (x.len + kUnit - 1) / kUnit);
  return x;
}

__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same onto zero.
__device__ __forceinline__ void mma_f16_first(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Four e4m3 bytes as two fp16 pairs (exact).
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Where fragments lie.  A chunk's 16 tokens x D bytes are 16 D / 128 lines of 128 bytes, 16-byte part p of line y
// stored at part p ^ (y & 7).  K: thread (r, c) reads parts k_part(c, i) of tokens r and r + 8, 4 k steps
// each; V: 16 bytes (8 at dim 64) at v_dim(r, 4 i) of tokens 2c, 2c + 1, 2c + 8, 2c + 9.
template <int D>
__device__ __forceinline__ int k_part(int c, int i) {  // of a token's D / 16
  return D == 64 ? c : D == 128 ? 2 * c + i : (i >> 1) * 8 + (c & 1) + (c >> 1) * 4 + (i & 1) * 2;
}
template <int D>
__device__ __forceinline__ int v_dim(int r, int w) {
  return D == 64 ? r * 8 + 4 * w : (w >> 2) * 128 + r * 16 + (w & 3) * 4;
}
// Offset of 16-byte part `part` of token t in a chunk.
template <int D>
__device__ __forceinline__ uint32_t part_at(int t, int part) {
  const int at = t * (D / 16) + part, line = at >> 3;
  return (uint32_t)(line * 128 + (((at & 7) ^ (line & 7)) << 4));
}

__device__ __forceinline__ uint4 lds16(uint32_t p) {
  uint4 u;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(p));
  return u;
}
__device__ __forceinline__ uint2 lds8(uint32_t p) {
  uint2 u;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(u.x), "=r"(u.y) : "r"(p));
  return u;
}

// A thread's offsets in a chunk: K parts of token r (and r + 8), V parts of its tokens 2c and 2c + 1 (and + 8).  Eight
// tokens on is the same line pattern 8 D bytes on, but for dim 64, where the lines' parity in the swizzle turns.
template <int D>
struct Offsets {
  uint32_t k[2][D / 64], v[4][D == 64 ? 1 : D / 128];
  __device__ __forceinline__ Offsets(int r, int c) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < D / 64; ++i) k[h][i] = part_at<D>(r + (D == 64 ? 8 * h : 0), k_part<D>(c, i)) + (D == 64 ? 0 : h * 8 * D);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = 2 * c + (j & 1), up = j >> 1;
      if (D == 64) {
        v[j][0] = 16 * D + part_at<D>(t + 8 * up, r >> 1) + (r & 1) * 8;
      } else {
#pragma unroll
        for (int i = 0; i < D / 128; ++i) v[j][i] = 16 * D + part_at<D>(t, i * 8 + r) + up * 8 * D;
      }
    }
  }
};

template <int D>
__device__ __forceinline__ void read_k(uint32_t (&x)[2][D / 16], uint32_t chunk, const Offsets<D>& at) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const uint4 u = lds16(chunk + at.k[h][i]);
      x[h][4 * i] = u.x, x[h][4 * i + 1] = u.y, x[h][4 * i + 2] = u.z, x[h][4 * i + 3] = u.w;
    }
}

template <int D>
__device__ __forceinline__ void read_v(uint32_t (&x)[4][D / 32], uint32_t chunk, const Offsets<D>& at) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (D == 64) {
      const uint2 u = lds8(chunk + at.v[j][0]);
      x[j][0] = u.x, x[j][1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < D / 128; ++i) {
        const uint4 u = lds16(chunk + at.v[j][i]);
        x[j][4 * i] = u.x, x[j][4 * i + 1] = u.y, x[j][4 * i + 2] = u.z, x[j][4 * i + 3] = u.w;
      }
    }
  }
}

// What the chunks' loop needs of a chunk: its scales and first token.
struct Look {
  float kf, lsv, isv;  // ks * scale * log2 e, log2 vs, 1 / vs
  int p0;
};

// A warp's running state: 8 NT query rows (columns 2c, 2c + 1 of each N tile in this thread).
template <int D, int NT>
struct State {
  float o[D / 16][NT][4];
  float m[NT][2], l[NT][2];
};

// S = K Q^T of one chunk: column n * 8 + 2c + (e & 1), token r + 8 (e >> 1).  q: this lane's B fragments, two k
// steps to 16 bytes.
template <int D, int NT>
__device__ __forceinline__ void scores(float (&s)[NT][4], const uint32_t (&k)[2][D / 16], uint32_t q) {
#pragma unroll
  for (int i = 0; i < D / 16; i += 2) {
    uint32_t a[2][4];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      e4m3x4_to_f16x4(k[0][i + y], a[y][0], a[y][2]);
      e4m3x4_to_f16x4(k[1][i + y], a[y][1], a[y][3]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint4 b = lds16(q + (n * (D / 32) + i / 2) * 512);
      if (i == 0) mma_f16_first(s[n], a[0][0], a[0][1], a[0][2], a[0][3], b.x, b.y);
      else mma_f16(s[n], a[0][0], a[0][1], a[0][2], a[0][3], b.x, b.y);
      mma_f16(s[n], a[1][0], a[1][1], a[1][2], a[1][3], b.z, b.w);
    }
  }
}

// The scores of one chunk become weights (B fragments of P) and enter the running sums.  y: the chunk's
// scales; `edge`: some token is past a row's position; `settle`: M may come down here.  M starts at a finite
// value far below any score, so that a masked score (-inf) weighs 0 with no further test.  top_s: the highest M a
// row has had.
template <int D, int NT>
__device__ __forceinline__ void weigh(State<D, NT>& st, float (&s)[NT][4], uint32_t (&b)[NT][2], const float (&rowf)[NT][2],
                                      const Look& y, bool edge, bool settle, const int* pos_s, float* top_s, int r, int c) {
  float p[NT][4];
  float most = -INFINITY;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float f0 = rowf[n][0] * y.kf, f1 = rowf[n][1] * y.kf;
#pragma unroll
    for (int e = 0; e < 4; ++e) s[n][e] = fmaf(s[n][e], e & 1 ? f1 : f0, y.lsv);
    if (edge) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (y.p0 + r + 8 * (e >> 1) > pos_s[n * 8 + 2 * c + (e & 1)]) s[n][e] = -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) p[n][e] = s[n][e] - st.m[n][e & 1];
    most = fmaxf(most, fmaxf(fmaxf(p[n][0], p[n][1]), fmaxf(p[n][2], p[n][3])));
  }
  if (settle) {  // does every row have a weight near M?
    uint32_t near = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) near |= (uint32_t)(fmaxf(p[n][e], p[n][e + 2]) >= -hk::kSlack) << (2 * n + e);
    if (__reduce_or_sync(0xffffffffu, near << (2 * NT * c)) != 0xffffffffu >> (32 - 8 * NT)) most = INFINITY;
  }
  if (__any_sync(0xffffffffu, most > hk::kRoom)) {
    bool full = false;  // a sum that coming down could carry past fp32
#pragma unroll
    for (int n = 0; n < NT; ++n) full |= st.l[n][0] > hk::kFullSum || st.l[n][1] > hk::kFullSum;
    settle = settle && !__any_sync(0xffffffffu, full);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float t = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
        const int row = n * 8 + 2 * c + e;
        const float peak = top_s[row];
        __syncwarp();
        const float m = hk::new_reference(st.m[n][e], t, peak, settle);
        if (r == 0) top_s[row] = fmaxf(peak, m);
        p[n][e] = s[n][e] - m, p[n][e + 2] = s[n][e + 2] - m;
        const float f = exp2_approx(st.m[n][e] - m);
        st.m[n][e] = m;
        st.l[n][e] *= f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) st.o[j][n][e] *= f, st.o[j][n][e + 2] *= f;
      }
    __syncwarp();
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) p[n][e] = exp2_approx(p[n][e]);
    st.l[n][0] = fmaf(p[n][0] + p[n][2], y.isv, st.l[n][0]);
    st.l[n][1] = fmaf(p[n][1] + p[n][3], y.isv, st.l[n][1]);
    b[n][0] = transpose8x8(pack2<true>(p[n][0], p[n][1]));
    b[n][1] = transpose8x8(pack2<true>(p[n][2], p[n][3]));
  }
}

// O += V^T P of one chunk.
template <int D, int NT>
__device__ __forceinline__ void values(State<D, NT>& st, const uint32_t (&v)[4][D / 32], const uint32_t (&b)[NT][2]) {
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    uint32_t a[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      e4m3x4_to_f16x4(__byte_perm(v[2 * h][w], v[2 * h + 1][w], 0x5140), a[0][2 * h], a[0][2 * h + 1]);
      e4m3x4_to_f16x4(__byte_perm(v[2 * h][w], v[2 * h + 1][w], 0x7362), a[1][2 * h], a[1][2 * h + 1]);
    }
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16(st.o[2 * w + y][n], a[y][0], a[y][1], a[y][2], a[y][3], b[n][0], b[n][1]);
  }
}

// Block-wide exclusive scan of one 64-bit value per thread.
__device__ __forceinline__ int64_t block_excl_scan(int64_t v, int64_t* sums, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  *total = all;
  return before + x - v;
}

template <int D, int NT>
constexpr int split_smem() {
  constexpr int ring = kWarps * stages(D, NT) * 32 * D, joined = kWarps * NT * (D / 16) * 32 * 16;  // O of every warp
  static_assert(stages(D, NT) >= 2 && stages(D, NT) <= kLook && joined <= ring, "ring");
  return ring + kAlignBytes;  // lines are swizzled from 1 KB boundaries
}

template <int D, int NT, bool kSparse>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(D, NT)) gqa_split_kernel(SplitArgs s, const __grid_constant__ CUtensorMap kmap,
                                                                                     const __grid_constant__ CUtensorMap vmap) {
  constexpr int R = 8 * NT;
  extern __shared__ uint8_t dyn_raw[];
  uint8_t* dyn = dyn_raw + (1024 - (__cvta_generic_to_shared(dyn_raw) & 1023)) % 1024;
  constexpr int S = stages(D, NT);
  float4* o_s = reinterpret_cast<float4*>(dyn);  // [kWarps][D / 16][NT][32], over the ring once it is read
  __shared__ __align__(16) uint4 q_s[NT * (D / 32) * 32];  // B fragments of Q: [N tile][two k steps][lane]
  __shared__ float rowf_s[R], m_s[kWarps][R], l_s[kWarps][R];
  __shared__ int pos_s[R];
  __shared__ float inv_s[R];
  __shared__ int64_t row_s[R];
  __shared__ int64_t scan_s[kWarps];
  __shared__ int64_t at_s;
  __shared__ int item_s;
  __shared__ int32_t line_s[kWarps][2 * kLook];  // first 128-byte line of a chunk in the cache, -1: not to be read
  __shared__ __align__(8) uint64_t full_s[kWarps][S];
  __shared__ volatile int stop_s[kWarps];  // a wait of this warp ran out
  __shared__ __align__(16) Look look_s[kWarps][2 * kLook];
  static_assert(sizeof q_s + sizeof rowf_s + sizeof m_s + sizeof l_s + sizeof pos_s + sizeof inv_s + sizeof row_s + sizeof scan_s + sizeof at_s +
                        sizeof item_s + sizeof line_s + sizeof full_s + sizeof stop_s + sizeof look_s <= fixed_bytes(D, NT),
                "fixed arrays");
  static_assert(ctas_per_sm(D, NT) * (split_smem<D, NT>() + fixed_bytes(D, NT) + kCtaBytes) <= kSmBytes, "CTAs an SM holds");
  const GqaArgs& a = s.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  const int G = a.kv_heads, group = s.group;
  hk::let_next_grid_start();
  if (tid == 0) {
    for (int i = 0; i < kWarps; ++i) stop_s[i] = 0;
    for (int i = 0; i < kWarps * S; ++i) sm100::mbar_init(sm100::smem_u32(&full_s[0][0] + i), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // The stage (and, for reads, the phase) this warp fills and reads next, and how many are filled and not yet read.
  int fill = 0, take = 0, filled = 0;
  uint32_t phase = 0;
  bool dead = false;  // a wait ran out: ask for no more
  const Offsets<D> at(r, c);
  // (the barriers are seen by all after the scan's first __syncthreads)

  // This CTA's range of units, and the item it begins in.  (With more items than threads the scan is run again to find it.)
  int64_t total = 0, mine = 0, before = 0;
  for (int base = 0; base < s.items; base += kThreads) {
    const int i = base + tid;
    int64_t all;
    mine = 0;
    if (i < s.items) {
      const Item x = item_of<R, kSparse>(s, i, blockIdx.x == 0);
      mine = x.nu * x.tiles * G;
    }
    before = total + block_excl_scan(mine, scan_s, &all);
    total += all;
  }
  // One range for each resident CTA: two to four ranges, which even out the SMs, measured 4 to 11% slower
  // (more starts, and more partials to join).
  const int64_t ranges = min((int64_t)gridDim.x, total), cta = blockIdx.x;
  const int64_t u0 = cta < ranges ? total * cta / ranges : 0, u1 = cta < ranges ? total * (cta + 1) / ranges : 0;
  Rec rec = {-1, 0, 0, 0};
  if (u0 < u1) {
    if (s.items <= kThreads) {
      if (before <= u0 && u0 < before + mine) item_s = tid, at_s = before;
    } else {
      int64_t carry = 0;
      for (int base = 0; base < s.items; base += kThreads) {
        const int i = base + tid;
        int64_t all;
        mine = 0;
        if (i < s.items) {
          const Item x = item_of<R, kSparse>(s, i, false);
          mine = x.nu * x.tiles * G;
        }
        before = carry + block_excl_scan(mine, scan_s, &all);
        if (before <= u0 && u0 < before + mine) item_s = i, at_s = before;
        carry += all;
        if (carry > u0) break;
      }
    }
    __syncthreads();
    int i = item_s;
    int64_t begin = at_s;  // unit at which item i begins
    Item x = item_of<R, kSparse>(s, i, false);
    for (int64_t u = u0; u < u1;) {
      while (u >= begin + x.nu * x.tiles * G) {
        begin += x.nu * x.tiles * G;
        x = item_of<R, kSparse>(s, ++i, false);
      }
      const int sub = (int)((u - begin) / x.nu);
      const int first = (int)(u - begin - sub * x.nu);
      const int last = (int)min(x.nu, first + (u1 - u));
      const int g = sub / x.tiles, row0 = sub % x.tiles * R;
      const int tok0 = first * kUnit, tok1 = min(x.len, last * kUnit);
      const int lane_b = kSparse ? hk::lane_of_row(a.cu, a.num_lanes, x.t0) : i;
      __syncthreads();
      // The query rows of this warp, asked for now and used after the lookups below: lane y finds row warp + kWarps y.
      constexpr int kMine = R / kWarps;
      uint32_t qw[kMine][D / 64];
      int my_pos = INT32_MAX;
      {
        if (tid < R && row0 + tid < x.rows * group) my_pos = a.positions[x.t0 + (row0 + tid) / group];
        const int row = row0 + warp + kWarps * (lane % kMine);
        const int t = row / group;
        const int64_t at = row < x.rows * group ? (x.t0 + t) * a.q_stride + (int64_t)(g * group + row - t * group) * D : -1;
#pragma unroll
        for (int y = 0; y < kMine; ++y) {
          const int64_t from = __shfl_sync(0xffffffffu, at, y);
#pragma unroll
          for (int e = 0; e < D / 64; ++e) qw[y][e] = 0;
          if (from >= 0) {
            const uint16_t* src = a.q + from + lane * (D / 32);
            if (D == 64) {
              qw[y][0] = *reinterpret_cast<const uint32_t*>(src);
            } else if (D == 128) {
              const uint2 u = *reinterpret_cast<const uint2*>(src);
              qw[y][0] = u.x, qw[y][1 % (D / 64)] = u.y;
            } else {
              const uint4 u = *reinterpret_cast<const uint4*>(src);
              qw[y][0] = u.x, qw[y][1 % (D / 64)] = u.y, qw[y][2 % (D / 64)] = u.z, qw[y][3 % (D / 64)] = u.w;
            }
          }
        }
      }
      // This warp's chunks: tokens tok0 + 16 warp + kUnit e.
      const int32_t* row_bt = a.bt + (int64_t)lane_b * a.bt_stride;
      const int32_t* list = kSparse ? a.blocks + ((int64_t)x.t0 * G + g) * a.top : nullptr;
      if (kSparse && first == 0 && x.len > 0) {  // nothing may stand behind as many entries as blocks are in sight
        for (int e = x.len / a.page_size + tid; e < a.top; e += kThreads)
          if (list[e] != -1) hk_flag(a.err, hk::kErrBlockList, (unsigned)x.t0);
      }
      const int nchunk = tok1 > tok0 + 16 * warp ? (tok1 - tok0 - 16 * warp + kUnit - 1) / kUnit : 0;
      auto look = [&](int e0) {  // pages and scales of chunks e0 .. e0 + kLook - 1, a lane each
        __syncwarp();  // every lane has read the places of the chunks before (skipped ones among them)
        if (lane < kLook && e0 + lane < nchunk) {
          int32_t line = -1;
          Look y = {0.f, 0.f, 1.f, 0};
          const int j = tok0 + 16 * warp + kUnit * (e0 + lane);
          const int idx = j / a.page_size, r16 = j - idx * a.page_size;
          int blk = idx;
          if (kSparse) {
            blk = list[idx];
            const int before = idx > 0 ? list[idx - 1] : -1;
            if (blk != -1 && (blk <= before || (idx > 0 && before < 0) || blk > x.pos / a.page_size)) {
              hk_flag(a.err, hk::kErrBlockList, (unsigned)x.t0);
              blk = -1;
            }
          }
          if (blk >= 0) {
            y.p0 = blk * a.page_size + r16;
            const int page = blk < a.bt_stride ? row_bt[blk] : -1;
            if (page <= 0 || page >= a.num_pages) {
              hk_flag(a.err, hk::kErrAttnPage, (unsigned)lane_b);
            } else {
              const int64_t at = (int64_t)page * G + g;
              line = (int32_t)((at * a.page_size + r16) * D / 128);
              y.kf = a.ks[at] * (a.scale * kLog2e);
              const float vs = fmaxf(a.vs[at], 7.8886090522101181e-31f);
              y.lsv = __log2f(vs), y.isv = __frcp_rn(vs);
            }
          }
          line_s[warp][(e0 + lane) % (2 * kLook)] = line;
          look_s[warp][(e0 + lane) % (2 * kLook)] = y;
        }
        __syncwarp();
      };
      const uint32_t ring = sm100::smem_u32(dyn) + warp * (S * 32 * D), bars = sm100::smem_u32(&full_s[warp][0]);
      const uint32_t q_frag = sm100::smem_u32(q_s + lane);
      auto ask = [&](int e) {
        const int line = e < nchunk ? line_s[warp][e % (2 * kLook)] : -1;
        if (line < 0 || dead) return;
        if (lane == 0) {
          const uint32_t bar = bars + fill * 8, dst = ring + fill * (32 * D);
          sm100::mbar_expect_tx(bar, 32 * D);
          sm100::tma_load_2d(dst, &kmap, bar, 0, line);
          sm100::tma_load_2d(dst + 16 * D, &vmap, bar, 0, line);
        }
        fill = fill + 1 == S ? 0 : fill + 1;
        ++filled;
      };
#pragma unroll 1
      for (int e = 0; e < 2 * kLook; e += kLook) look(e);
#pragma unroll 1
      for (int e = 0; e < S - 1; ++e) ask(e);
      // Query rows: scaled by a power of two so that fp16 holds them exactly, in the order of the fragments.
#pragma unroll
      for (int y = 0; y < kMine; ++y) {
        const int n = warp + kWarps * y;
        float f[D / 32], top = 0.f;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          const uint16_t bits = (uint16_t)(qw[y][e / 2] >> (16 * (e & 1)));
          f[e] = s.is_f16 ? __half2float(__ushort_as_half(bits)) : bf16_bits_to_f32(bits);
          top = fmaxf(top, fabsf(f[e]));
        }
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));  // (magnitudes: their bits are in order)
        const int ex = (int)((__float_as_uint(top) >> 23) & 255);  // 0: zero or subnormal, 255: not finite
        const int up = ex == 255 ? 0 : min(134 - ex, 120);
        const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          const int d = lane * (D / 32) + e;
          const int part = d / 16, half = D == 256 ? part & 7 : part;  // the inverse of k_part
          const int cc = D == 64 ? part : D == 128 ? part >> 1 : (half & 1) | (half >> 2) << 1;
          const int i = D == 64 ? 0 : D == 128 ? part & 1 : (part >> 3) * 2 + (half >> 1 & 1);
          const int k = i * 4 + (d % 16) / 4;
          reinterpret_cast<__half*>(q_s + ((n >> 3) * (D / 32) + k / 2) * 32 + (n & 7) * 4 + cc)[(k & 1) * 4 + (d & 3)] = __float2half_rn(f[e] * mul);
        }
        if (lane == 0) rowf_s[n] = __uint_as_float((uint32_t)(127 - up) << 23);
      }
      if (tid < R) {
        pos_s[tid] = my_pos;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m_s[w][tid] = kNoMax;
      }
      __syncthreads();
      float rowf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) rowf[n][0] = rowf_s[n * 8 + 2 * c], rowf[n][1] = rowf_s[n * 8 + 2 * c + 1];
      const int pos_min = kSparse ? x.pos : pos_s[0];  // the first row's: positions rise
      const int len = kSparse ? x.pos + 1 : x.len;

      State<D, NT> st;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        st.m[n][0] = st.m[n][1] = kNoMax;
        st.l[n][0] = st.l[n][1] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) st.o[j][n][0] = st.o[j][n][1] = st.o[j][n][2] = st.o[j][n][3] = 0.f;
      }

#pragma unroll 1
      for (int e = 0; e < nchunk; ++e) {
        const bool again = e > 0 && e % kLook == 0;
        if (again) look(e + kLook);
        ask(e + S - 1);  // into the stage that the step before has read
        if (line_s[warp][e % (2 * kLook)] < 0 || filled == 0) continue;
        const Look y = look_s[warp][e % (2 * kLook)];
        const bool ok = __all_sync(0xffffffffu, sm100::mbar_wait(bars + take * 8, phase, &stop_s[warp], a.err, 0x60));
        const uint32_t mine = ring + take * (32 * D);
        if (ok) {
          const bool edge = y.p0 + 15 > pos_min;
          float sc[NT][4];
          uint32_t pb[NT][2];
          {
            uint32_t k[2][D / 16];
            read_k<D>(k, mine, at);
            scores<D, NT>(sc, k, q_frag);
          }
          weigh<D, NT>(st, sc, pb, rowf, y, edge, again && !edge, pos_s, m_s[warp], r, c);
          uint32_t v[4][D / 32];
          read_v<D>(v, mine, at);
          if (edge) {  // tokens past the lane's end may hold anything, NaN codes among it
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (y.p0 + 2 * c + (j & 1) + 8 * (j >> 1) >= len) {
#pragma unroll
                for (int w = 0; w < D / 32; ++w) v[j][w] = 0;
              }
          }
          values<D, NT>(st, v, pb);
        }
        dead |= !ok;
        --filled;
        if (++take == S) take = 0, phase ^= 1;
        __syncwarp();
      }

      // Join the warps through shared memory (over the ring, which is read): each warp's maxima and sums, then its O under the
      // common maximum; the threads add the warps' parts in order and write the rows.  (The code after the loop is kept
      // short: a small call's time is in good part that of fetching it.)
      const bool starts = first == 0, ends = last == x.nu;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float l = st.l[n][e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
          if (r == 0) m_s[warp][n * 8 + 2 * c + e] = st.m[n][e], l_s[warp][n * 8 + 2 * c + e] = l;
        }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = n * 8 + 2 * c + e;
          float m = kNoMax;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) m = fmaxf(m, m_s[w][row]);
          f[e] = exp2_approx(st.m[n][e] - m);
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
          o_s[((warp * (D / 16) + j) * NT + n) * 32 + lane] =
              make_float4(st.o[j][n][0] * f[0], st.o[j][n][1] * f[1], st.o[j][n][2] * f[0], st.o[j][n][3] * f[1]);
      }
      float* part = s.part + ((int64_t)blockIdx.x * 2 + (starts ? 1 : 0)) * (R * D + 2 * R);
      const bool whole = starts && ends;
      if (tid < R) {  // a row's denominator, and where it goes
        float m = kNoMax, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, m_s[w][tid]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) l += l_s[w][tid] * exp2_approx(m_s[w][tid] - m);
        const int at = row0 + tid;
        int64_t y = -1;
        if (at < x.rows * group) {
          y = (int64_t)(x.t0 + at / group) * a.q_heads + g * group + at % group;
          if (whole) a.lse[y] = l == 0.f ? -INFINITY : fmaf(m, kLn2, logf(l));
          else part[R * D + tid] = m, part[R * D + R + tid] = l;
        }
        row_s[tid] = y;
        inv_s[tid] = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
      }
      __syncthreads();
#pragma unroll 1
      for (int k = tid; k < D / 32 * NT * 32; k += kThreads) {  // four dims of two rows
        const int ln = k & 31, n = k / 32 % NT, w = k / 32 / NT, cc = ln & 3, d = v_dim<D>(ln >> 2, w);
        float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
#pragma unroll
        for (int e = 0; e < kWarps; ++e) {
          const float4 p = o_s[((e * (D / 16) + 2 * w) * NT + n) * 32 + ln], q = o_s[((e * (D / 16) + 2 * w + 1) * NT + n) * 32 + ln];
          u.x += p.x, u.y += p.z, u.z += q.x, u.w += q.z;
          v.x += p.y, v.y += p.w, v.z += q.y, v.w += q.w;
        }
#pragma unroll 1
        for (int e = 0; e < 2; ++e, u = v) {
          const int row = n * 8 + 2 * cc + e;
          const int64_t y = row_s[row];
          if (y < 0) continue;
          const float f = inv_s[row];
          if (!whole) *reinterpret_cast<float4*>(part + row * D + d) = u;
          else if (s.is_f16) *reinterpret_cast<uint2*>(a.out + y * D + d) = make_uint2(pack2<true>(u.x * f, u.y * f), pack2<true>(u.z * f, u.w * f));
          else *reinterpret_cast<uint2*>(a.out + y * D + d) = make_uint2(pack2<false>(u.x * f, u.y * f), pack2<false>(u.z * f, u.w * f));
        }
      }
      // O lay where the next copies go: order those writes before them.
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (starts && !ends) rec.item = i, rec.sub = sub;
      if (!starts && ends) rec.ends = 1;
      u += last - first;
    }
  }
  if (tid == 0) s.rec[blockIdx.x] = rec;
  if (dead) {  // a wait has run out: copies still in flight get time to land before the CTA ends
    const unsigned long long t0 = sm100::globaltimer();
    while (sm100::globaltimer() - t0 < 100000000ull) {
    }
  }
}

// Joins the partials of the problems that CTAs of the split kernel began and left open (their records), row blockIdx.y of
// each.  A warp takes one record and joins its pieces in order, a lane holding D / 32 dims; problems of many
// pieces (one long lane) are left to all warps of the CTA together, each taking every eighth piece.
constexpr int kMergeWarps = 8;
constexpr int kMergeAlone = 32;  // pieces up to which one warp joins them: a few rounds of loads

struct Joined {
  float m, l;
};

template <int D, int R>
__device__ __forceinline__ Joined join_pieces(const float* part, int row, int from, int step, int to, int lane, float (&o)[D / 32]) {
  constexpr int P = D / 32;
  constexpr int64_t kPart = R * D + 2 * R;
  Joined j = {kNoMax, 0.f};
#pragma unroll
  for (int e = 0; e < P; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int i = from; i < to; i += step) {
    const float* p = part + ((int64_t)i * 2 + (i == 0 ? 1 : 0)) * kPart;
    const float pm = p[R * D + row], pl = p[R * D + R + row];
    const float top = fmaxf(j.m, pm), f = exp2_approx(j.m - top), pf = exp2_approx(pm - top);
    j.m = top;
    j.l = j.l * f + pl * pf;
#pragma unroll
    for (int e = 0; e < P; ++e) o[e] = o[e] * f + p[row * D + lane * P + e] * pf;
  }
  return j;
}

template <int D, int NT, bool kSparse>
__global__ void __launch_bounds__(kMergeWarps * 32) gqa_merge_kernel(SplitArgs s, int ctas) {
  constexpr int R = 8 * NT, P = D / 32;
  constexpr int64_t kPart = R * D + 2 * R;
  __shared__ float o_s[kMergeWarps][D], m_s[kMergeWarps], l_s[kMergeWarps];
  __shared__ int pieces_s[kMergeWarps];
  __shared__ int64_t row_s[kMergeWarps];
  const GqaArgs& a = s.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.y;
  const int first = blockIdx.x * kMergeWarps + warp;
  int pieces = 0;
  int64_t y = 0;  // (row, head) of the output
  hk::wait_for_grid_before();
  const Rec rec = first < ctas ? s.rec[first] : Rec{-1, 0, 0, 0};
  if (rec.item >= 0) {
    const Item x = item_of<R, kSparse>(s, rec.item, false);
    const int g = rec.sub / x.tiles, at = rec.sub % x.tiles * R + row;
    if (at < x.rows * s.group) {
      y = (int64_t)(x.t0 + at / s.group) * a.q_heads + g * s.group + at % s.group;
      // The last piece: the first CTA after this one in which a continued problem ends.
      for (int base = first + 1; pieces == 0; base += 32) {
        const unsigned hit = __ballot_sync(0xffffffffu, base + lane >= ctas || s.rec[min(base + lane, ctas - 1)].ends);
        if (hit) pieces = min(base + __ffs(hit) - 1, ctas - 1) - first + 1;
      }
    }
  }
  if (pieces > 0 && pieces <= kMergeAlone) {
    float o[P];
    const Joined j = join_pieces<D, R>(s.part + (int64_t)first * 2 * kPart, row, 0, 1, pieces, lane, o);
    const float inv = j.l == 0.f ? 0.f : 1.f / j.l;
#pragma unroll
    for (int e = 0; e < P; e += 2)
      *reinterpret_cast<uint32_t*>(a.out + y * D + lane * P + e) =
          s.is_f16 ? pack2<true>(o[e] * inv, o[e + 1] * inv) : pack2<false>(o[e] * inv, o[e + 1] * inv);
    if (lane == 0) a.lse[y] = j.l == 0.f ? -INFINITY : fmaf(j.m, kLn2, logf(j.l));
  }
  if (lane == 0) pieces_s[warp] = pieces, row_s[warp] = y;
  __syncthreads();
  for (int w = 0; w < kMergeWarps; ++w) {
    if (pieces_s[w] <= kMergeAlone) continue;
    float o[P];
    const Joined j = join_pieces<D, R>(s.part + (int64_t)(blockIdx.x * kMergeWarps + w) * 2 * kPart, row, warp, kMergeWarps, pieces_s[w], lane, o);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < P; ++e) o_s[warp][lane * P + e] = o[e];
    if (lane == 0) m_s[warp] = j.m, l_s[warp] = j.l;
    __syncthreads();
    if (tid < D / 2) {
      float top = kNoMax, sum = 0.f, v[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < kMergeWarps; ++e) top = fmaxf(top, m_s[e]);
#pragma unroll
      for (int e = 0; e < kMergeWarps; ++e) {
        const float f = exp2_approx(m_s[e] - top);
        sum += l_s[e] * f;
        v[0] = fmaf(o_s[e][2 * tid], f, v[0]), v[1] = fmaf(o_s[e][2 * tid + 1], f, v[1]);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint32_t*>(a.out + row_s[w] * D + 2 * tid) = s.is_f16 ? pack2<true>(v[0] * inv, v[1] * inv) : pack2<false>(v[0] * inv, v[1] * inv);
      if (tid == 0) a.lse[row_s[w]] = sum == 0.f ? -INFINITY : fmaf(top, kLn2, logf(sum));
    }
  }
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

// N tiles for `rows` query rows of a problem: 1 to 4, at most 2 at dim 256 (registers).
int n_tiles(int64_t rows, int dim) {
  const int64_t n = (rows + 7) / 8, most = dim == 256 ? 2 : 4;
  return (int)(n < most ? n : most);
}

// Query rows (rows x heads of a group) of a lane above which the tcgen05 kernel takes it: above 32 the split kernel reads the
// cache once for each 32 rows.  8 lanes of 20,000 tokens, 8 KV heads, 4 query heads each: 40 query rows 216 us (split) against
// 176 us, 96 rows 312 against 180, 256 rows 796 against 213.
constexpr int32_t kFewRows = 32;

size_t split_workspace(int64_t rows, int dim);

size_t part_floats(int nt, int dim) { return (size_t)8 * nt * dim + 16 * nt; }

template <int D, int NT, bool kSparse>
int launch_one(SplitArgs& s, int64_t units, cudaStream_t stream) {
  constexpr int smem = split_smem<D, NT>();
  const int64_t resident = hk::sm_count() * ctas_per_sm(D, NT);
  const int grid = (int)(units < resident ? units : resident);
  // (set on every call: cheap, and right on every device)
  HK_TRY_CUDA(cudaFuncSetAttribute(gqa_split_kernel<D, NT, kSparse>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  CUtensorMap kmap, vmap;
  const uint64_t lines = (uint64_t)s.a.num_pages * s.a.kv_heads * s.a.page_size * D / 128;
  HK_REQUIRE(lines <= INT32_MAX, "the cache's K and V arrays must be below 2^38 bytes each");
  HK_TRY(hk::sm100::make_map_u8(&kmap, s.a.kc, lines, 128, 16 * D / 128));
  HK_TRY(hk::sm100::make_map_u8(&vmap, s.a.vc, lines, 128, 16 * D / 128));
  gqa_split_kernel<D, NT, kSparse><<<grid, kThreads, smem, stream>>>(s, kmap, vmap);
  HK_TRY_LAUNCH("gqa_split_kernel");
  if (grid > 1) {
    HK_TRY_CUDA(hk::launch_early(gqa_merge_kernel<D, NT, kSparse>, dim3((grid + kMergeWarps - 1) / kMergeWarps, 8 * NT), kMergeWarps * 32, 0, stream, s, grid));
    HK_TRY_LAUNCH("gqa_merge_kernel");
  }
  return HK_OK;
}

template <bool kSparse>
int launch(const GqaArgs& a, int32_t dtype, int64_t rows, int64_t units, int32_t most, void* workspace, cudaStream_t stream) {
  SplitArgs s;
  s.a = a;
  s.most = most;
  s.is_f16 = dtype == HK_F16;
  s.group = a.q_heads / a.kv_heads;
  s.items = kSparse ? a.num_tokens : a.num_lanes;
  s.rec = (Rec*)workspace;
  s.part = (float*)((uint8_t*)workspace + (size_t)hk::sm_count() * kMaxCtasPerSm * sizeof(Rec));
  const int nt = n_tiles(rows * s.group, a.dim);
  switch (a.dim * 8 + nt) {
#define HK_GQA(D, NT) \
  case D * 8 + NT:    \
    return launch_one<D, NT, kSparse>(s, units, stream)
    HK_GQA(64, 1);
    HK_GQA(64, 2);
    HK_GQA(64, 3);
    HK_GQA(64, 4);
    HK_GQA(128, 1);
    HK_GQA(128, 2);
    HK_GQA(128, 3);
    HK_GQA(128, 4);
    HK_GQA(256, 1);
    HK_GQA(256, 2);
#undef HK_GQA
  }
  return hk::fail(HK_EINVAL, "no kernel for dim %d", a.dim);
}

}  // namespace

namespace {

// Bytes of the split kernel's records and partials for problems of up to `rows` query rows.
size_t split_workspace(int64_t rows, int head_dim) {
  const int nt = n_tiles(rows, head_dim);
  size_t most = 0;  // over the tile counts that a call with these sizes can pick
  for (int n = 1; n <= nt; ++n) {
    const size_t part = ctas_per_sm(head_dim, n) * 2 * part_floats(n, head_dim) * sizeof(float);
    most = most > part ? most : part;
  }
  return ((size_t)hk::sm_count() * (kMaxCtasPerSm * sizeof(Rec) + most) + 255) / 256 * 256;
}

}  // namespace

extern "C" {

size_t hk_gqa_fp8_workspace_size(int32_t num_tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
  if (num_tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 256;
  const int64_t rows = (int64_t)num_tokens * (q_heads / kv_heads > 0 ? q_heads / kv_heads : 1);
  size_t bytes = split_workspace(rows, head_dim);
  if (rows > kFewRows && hk::gqa_prefill_supported(head_dim)) bytes += (hk::gqa_prefill_workspace(head_dim) + 255) / 256 * 256;
  return bytes;
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
  a.err = hk::err_word();
  const int group = q_heads / kv_heads;
  int64_t rows = max_rows < num_tokens ? max_rows : num_tokens;
  int32_t most = INT32_MAX;
  if (rows * group > kFewRows && hk::gqa_prefill_supported(head_dim)) {
    void* at = (uint8_t*)workspace + split_workspace((int64_t)num_tokens * group, head_dim);
    HK_TRY(hk::gqa_prefill(a, dtype, kFewRows, max_kv_len, at, (cudaStream_t)stream));
    most = kFewRows;
    if (kFewRows / group == 0) return HK_OK;  // one row is already above it
    rows = kFewRows / group;
  }
  const int64_t tiles = rows * group / 8 + 1;
  const int64_t units = (int64_t)(num_lanes < num_tokens ? num_lanes : num_tokens) * kv_heads * tiles * (max_kv_len / kUnit + 1);
  return launch<false>(a, dtype, rows > 0 ? rows : 1, units, most, workspace, (cudaStream_t)stream);
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
  const int group = q_heads / kv_heads;
  const int64_t units = (int64_t)num_tokens * kv_heads * (group / 8 + 1) * ((int64_t)top_blocks * page_size / kUnit + 1);
  a.err = hk::err_word();
  return launch<true>(a, dtype, 1, units, INT32_MAX, workspace, (cudaStream_t)stream);
}

}  // extern "C"
