// Attention of prompt chunks (many query rows of a lane) over the block-scaled e4m3 cache, on tcgen05.
//
// Query rows that share a KV head (rows of the lane x heads of the group) are laid end to end and cut
// into tiles of 256, two halves of 128 TMEM lanes.  Per 128 tokens of the cache, for each half w:
//   S_w = Q_w K^T            M = 128, N = 128, K = dim, fp16 operands from shared memory
//   P_w = 2^(S_w f + log2 vs - M)   one thread per row; fp16, written over S_w in tensor memory
//   O_w += P_w V             M = 128, N = dim, K = 128, P from tensor memory, V from shared memory
// While the softmax warps of one half work, the tensor core runs the other half's products.
//
// e4m3 is exact in fp16, and so is q once each row is scaled by a power of two, so the products are those of
// the stored values.  K and V come as e4m3 by TMA into a ring of 64-token stages, and four
// warps convert them into the swizzled fp16 tiles the products read (1/13 of the softmax's work, as
// 256 rows share it).  Scales of pages enter as one factor and one addend for each 16 tokens, and with log2 vs in
// the exponent one running maximum serves pages of any scale (sum w / vs is the denominator).
// M is raised, and O rescaled, only when a value passes it by more than 2^8.
//
// Work split: the (row tile, head) problems' 128-token steps lie end to end, and every SM takes an
// equal contiguous range of them.  Problems cut by a range's end leave fp32 partials, two at
// most for each SM, which the merge kernel joins in the order of the ranges.
//
// Roles (16 warps): 0-3 and 4-7 softmax of the two halves, 8-11 conversion, 12 product issue, 13 TMA.
#include "common.cuh"
#include "gqa_fp8.cuh"
#include "sm100.cuh"

namespace {

using hk::GqaArgs;
using namespace hk::sm100;

constexpr int kThreads = 512;
constexpr int kRows = 256;    // query rows of a problem
constexpr int kTok = 128;     // tokens of a step
constexpr int kStages = 4;    // raw ring: 64 tokens of K or V each
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoMax = -1e30f;
// Registers: 512 threads x 128 = 2 x 128 x 184 (softmax) + 2 x 128 x 72 (the rest).
constexpr int kSoftmaxRegs = 184, kOtherRegs = 72;

// Scales of 16 tokens: ks * scale * log2 e, log2 vs, 1 / vs; ok: the tokens are there.
struct Scale {
  float kf, lsv, isv;
  int ok;
};

struct Rec {
  int32_t lane, g, row0;  // the problem its last range starts and does not finish (lane < 0: none)
  int32_t ends;           // the first problem was continued from the CTA before, and ends here
};

struct PrefillArgs {
  GqaArgs a;
  int32_t is_f16, group;
  int32_t least;   // query rows (rows x group) above which a lane is this kernel's
  int32_t box;     // tokens of a TMA box: the largest of 16, 32, 64 that divides the page
  Rec* rec;        // [grid]
  float* part;     // [grid][2][256 * (D + 2)]
};

template <int D>
struct Layout {
  static constexpr int kHalf = kTok * 128;           // [128 rows][64 fp16]
  static constexpr int kTile = kHalf * (D / 64);     // a K, V or half-Q tile
  static constexpr int kRaw = 64 * D;                // a raw stage
  static constexpr int kQ = 0, kK = 2 * kTile, kV = kK + 2 * kTile, kRing = kV + 2 * kTile, kCtl = kRing + kStages * kRaw;
  static constexpr int kBytes = kCtl + 2048;
};

// Control block, byte offsets.
constexpr int kRawFull = 0, kRawEmpty = 32, kKFull = 64, kKEmpty = 80, kVFull = 96, kVEmpty = 112, kQFull = 128, kSFull = 144,
              kPFull = 160, kOFull = 176, kDrain = 192, kSlot = 200, kAbort = 204, kScales = 256 /* [4][8] */,
              kScan = 768 /* [16] */, kFound = 896 /* unit, lane */;

constexpr uint32_t idesc_f16(int n, int b_mn_major) {  // D fp32, A and B fp16, M = 128
  return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void umma_f16_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
      "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

// A lane's rows of this kernel, 0 when it has none.
struct Lane {
  int t0, rows, pos0;
};

__device__ __forceinline__ Lane lane_at(const PrefillArgs& s, int b) {
  Lane x;
  x.t0 = s.a.cu[b];
  const int t1 = min(s.a.cu[b + 1], s.a.num_tokens);
  x.rows = x.t0 >= 0 ? max(0, t1 - x.t0) : 0;
  if (x.rows > s.a.max_rows || (int64_t)x.rows * s.group <= s.least) x.rows = 0;
  x.pos0 = x.rows ? s.a.positions[x.t0] : 0;
  return x;
}

// Steps of one (row tile, head): up to the position of the tile's last row.
__device__ __forceinline__ int steps_of(const PrefillArgs& s, const Lane& x, int tile) {
  const int64_t upto = min((int64_t)x.rows, ((int64_t)(tile + 1) * kRows + s.group - 1) / s.group);
  return (int)max((int64_t)1, (x.pos0 + upto + kTok - 1) / kTok);
}

__device__ __forceinline__ int tiles_of(const PrefillArgs& s, const Lane& x) {
  return (int)(((int64_t)x.rows * s.group + kRows - 1) / kRows);
}

// Walks a CTA's range of steps problem by problem.  Every role walks on its own.
struct Walk {
  int u, end;           // next step and end of the range, from its start
  int begin;            // step at which the current tile begins (its heads follow one another)
  int lane, tile, tiles, steps;
  Lane x;
  // The current problem.
  int g, row0, first, last, rows_left;

  __device__ __forceinline__ bool next(const PrefillArgs& s) {
    if (u >= end) return false;
    while (u - begin >= steps * s.a.kv_heads) {
      begin += steps * s.a.kv_heads;
      if (++tile >= tiles) {
        do {
          x = lane_at(s, ++lane);
        } while (x.rows == 0);
        tile = 0, tiles = tiles_of(s, x);
      }
      steps = steps_of(s, x, tile);
    }
    g = (u - begin) / steps;
    first = u - begin - g * steps;
    last = min(steps, first + (end - u));
    row0 = tile * kRows;
    rows_left = x.rows * s.group - row0;
    u += last - first;
    return true;
  }
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1) gqa_prefill_kernel(PrefillArgs s, const __grid_constant__ CUtensorMap kmap,
                                                                  const __grid_constant__ CUtensorMap vmap) {
  using L = Layout<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const GqaArgs& a = s.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* ctl = smem + L::kCtl;
  volatile int* abort = reinterpret_cast<volatile int*>(ctl + kAbort);
  const uint32_t base = smem_u32(smem), bars = smem_u32(ctl);
  auto bar = [&](int off, int i = 0) { return bars + off + 8 * i; };

  if (base & 1023) {  // the swizzles count from 1 KB boundaries
    if (tid == 0) hk_flag(a.err, hk::kErrWaitTimeout, 0x7f), s.rec[blockIdx.x] = Rec{-1, 0, 0, 0};
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(bar(kRawFull, i), 1), mbar_init(bar(kRawEmpty, i), 128);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kKFull, i), 128), mbar_init(bar(kKEmpty, i), 1);
      mbar_init(bar(kVFull, i), 128), mbar_init(bar(kVEmpty, i), 1);
      mbar_init(bar(kQFull, i), 128), mbar_init(bar(kSFull, i), 1);
      mbar_init(bar(kPFull, i), 128), mbar_init(bar(kOFull, i), 1);
    }
    mbar_init(bar(kDrain), 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) tmem_alloc(bar(kSlot), 512);

  // This CTA's range of steps, and the lane in which it begins.
  int64_t* scan = reinterpret_cast<int64_t*>(ctl + kScan);
  int64_t* found = reinterpret_cast<int64_t*>(ctl + kFound);
  auto lane_steps = [&](int b) {
    int64_t n = 0;
    if (b < a.num_lanes) {
      if (blockIdx.x == 0 && a.cu[b + 1] - a.cu[b] > a.max_rows) hk_flag(a.err, hk::kErrLaneRows, (unsigned)b);
      const Lane x = lane_at(s, b);
      if (x.rows)
        for (int i = 0, m = tiles_of(s, x); i < m; ++i) n += steps_of(s, x, i);
    }
    return n * a.kv_heads;
  };
  auto scan_block = [&](int64_t v, int64_t* total) {  // exclusive, over the CTA
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += scan[w];
      all += scan[w];
    }
    *total = all;
    return before + x - v;
  };
  int64_t total = 0;
  for (int b0 = 0; b0 < a.num_lanes; b0 += kThreads) {
    int64_t all;
    scan_block(lane_steps(b0 + tid), &all);
    total += all;
  }
  const int64_t ranges = min((int64_t)gridDim.x, total), cta = blockIdx.x;
  const int64_t u0 = cta < ranges ? total * cta / ranges : 0, u1 = cta < ranges ? total * (cta + 1) / ranges : 0;
  if (u0 < u1) {
    int64_t carry = 0;
    for (int b0 = 0; b0 < a.num_lanes; b0 += kThreads) {
      const int64_t n = lane_steps(b0 + tid);
      int64_t all;
      const int64_t before = carry + scan_block(n, &all);
      if (before <= u0 && u0 < before + n) found[0] = before, found[1] = b0 + tid;
      carry += all;
      if (carry > u0) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(ctl + kSlot);
  Walk w;
  w.u = 0, w.end = (int)(u1 - u0), w.steps = 1, w.tiles = 0, w.tile = 0, w.lane = 0, w.begin = 0;
  if (u0 < u1) {
    int64_t at = found[0] - u0;  // where the lane begins, at or before the range
    w.lane = (int)found[1];
    w.x = lane_at(s, w.lane);
    w.tiles = tiles_of(s, w.x);
    w.steps = steps_of(s, w.x, 0);
    while (at + (int64_t)w.steps * a.kv_heads <= 0) {  // the tile in which the range begins
      at += (int64_t)w.steps * a.kv_heads;
      w.steps = steps_of(s, w.x, ++w.tile);
    }
    w.begin = (int)at;
  }
  Scale* scales = reinterpret_cast<Scale*>(ctl + kScales);

  if (warp < 8) {
    // ---- softmax: thread = row ----------------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lanes + half * 128, o_col = tmem + lanes + 256 + half * 128;
    uint8_t* q_row = smem + L::kQ + half * L::kTile + row * 128;
    uint32_t n_s = 0, n_o = 0, step = 0;
    bool live = true;
    while (live && w.next(s)) {
      if (w.rows_left <= half * 128) {  // no rows for this half
        step += w.last - w.first;
        continue;
      }
      const int r = half * 128 + row;
      const bool on = r < w.rows_left;
      const int at = w.row0 + r, t = w.x.t0 + (on ? at / s.group : 0);
      const int64_t y = (int64_t)t * a.q_heads + w.g * s.group + (on ? at - at / s.group * s.group : 0);
      const int pos = on ? a.positions[t] : INT32_MAX;
      float rowf;
      {  // this row of Q, scaled by a power of two so that fp16 holds it exactly
        const uint4* src = reinterpret_cast<const uint4*>(a.q + t * a.q_stride + (y - (int64_t)t * a.q_heads) * D);
        float top = 0.f;
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
          float f[8];
          const uint4 u = on ? src[i] : make_uint4(0, 0, 0, 0);
          if (s.is_f16) unpack8<true>(u, f);
          else unpack8<false>(u, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[e]));
        }
        const int ex = (int)((__float_as_uint(top) >> 23) & 255);
        const int up = ex == 255 ? 0 : min(134 - ex, 120);
        const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
        rowf = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
          float f[8];
          const uint4 u = on ? src[i] : make_uint4(0, 0, 0, 0);
          if (s.is_f16) unpack8<true>(u, f);
          else unpack8<false>(u, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= mul;
          *reinterpret_cast<uint4*>(q_row + (i >> 3) * L::kHalf + (((i & 7) ^ (row & 7)) << 4)) = pack8<true>(f);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(bar(kQFull, half));
      // The smallest position of this half: rows of a lane rise.
      const int pos_min = w.x.pos0 + (w.row0 + half * 128) / s.group;

      float m = kNoMax, l = 0.f;
      for (int i = w.first; i < w.last; ++i, ++n_s, ++step) {
        live = live && mbar_wait(bar(kSFull, half), n_s & 1, abort, a.err, 0x70);
        live = __all_sync(0xffffffffu, live);
        if (!live) break;
        tc_fence_after();
        float v[128];
        tmem_ld64(s_col, v);
        tmem_ld64(s_col + 64, v + 64);
        const Scale* sc = scales + (step & 3) * 8;
        const bool edge = (i + 1) * kTok - 1 > pos_min;
        float top = -INFINITY;
        if (!edge) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float x = v[16 * k];
#pragma unroll
            for (int e = 1; e < 16; ++e) x = fmaxf(x, v[16 * k + e]);
            top = fmaxf(top, fmaf(x, sc[k].kf * rowf, sc[k].lsv));  // the factor is positive
          }
        } else {
          const int seen = pos - i * kTok;  // tokens after it are masked
#pragma unroll
          for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float x = fmaf(v[16 * k + e], sc[k].kf * rowf, sc[k].lsv);
              v[16 * k + e] = 16 * k + e > seen ? -INFINITY : x;
              top = fmaxf(top, v[16 * k + e]);
            }
        }
        // S is complete, so the product before it (which this row's O is from) is too.
        const bool over = top > m + 8.f;
        if (__any_sync(0xffffffffu, over)) {
          const float m_new = over ? top : m, f = exp2_approx(m - m_new);
          m = m_new;
          l *= f;
          if (i > w.first) {
#pragma unroll 1
            for (int k = 0; k < D / 16; ++k) {
              float o[16];
              tmem_ld16(o_col + 16 * k, o);
              uint32_t x[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(o[e] * f);
              asm volatile(
                  "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(o_col + 16 * k),
                  "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(x[8]), "r"(x[9]), "r"(x[10]),
                  "r"(x[11]), "r"(x[12]), "r"(x[13]), "r"(x[14]), "r"(x[15])
                  : "memory");
            }
          }
        }
        uint32_t p[32];  // 64 tokens' weights at a time, over columns of S that are read already
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float f = edge ? 1.f : sc[k].kf * rowf, c = (edge ? 0.f : sc[k].lsv) - m;
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const float x0 = exp2_approx(fmaf(v[16 * k + e], f, c)), x1 = exp2_approx(fmaf(v[16 * k + e + 1], f, c));
            sum += x0 + x1;
            p[8 * (k & 3) + e / 2] = pack2<true>(x0, x1);
          }
          l = fmaf(sum, sc[k].isv, l);
          if ((k & 3) == 3) tmem_st32(s_col + 8 * (k - 3), p);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        mbar_arrive(bar(kPFull, half));
      }
      live = live && mbar_wait(bar(kOFull, half), n_o & 1, abort, a.err, 0x71);
      live = __all_sync(0xffffffffu, live);
      if (!live) break;
      ++n_o;
      tc_fence_after();
      const bool starts = w.first == 0;
      if (starts && w.last == w.steps) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          float o[32];
          tmem_ld32(o_col + 32 * k, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= inv;
          if (on) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              *reinterpret_cast<uint4*>(a.out + y * D + 32 * k + e) = s.is_f16 ? pack8<true>(o + e) : pack8<false>(o + e);
          }
        }
        if (on) a.lse[y] = l == 0.f ? -INFINITY : fmaf(m, kLn2, logf(l));
      } else {
        float* part = s.part + ((int64_t)blockIdx.x * 2 + (starts ? 1 : 0)) * (kRows * (D + 2));
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          float o[32];
          tmem_ld32(o_col + 32 * k, o);
          if (on) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(part + r * D + 32 * k + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (on) part[kRows * D + r] = m, part[kRows * (D + 1) + r] = l;
      }
      tc_fence_before();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp < 12) {
      // ---- conversion: raw e4m3 -> swizzled fp16 -----------------------------------------------
      const int id = tid - 256;
      constexpr int kPer = 64 * D / 16 / 128;  // 16-byte parts of a stage a thread converts
      uint32_t n = 0, step = 0;                // stages read
      bool live = true;
      while (live && w.next(s)) {
        const int len = w.x.pos0 + w.x.rows;  // tokens of the lane: what lies past them may be anything
        for (int i = w.first; i < w.last && live; ++i, ++step) {
          const Scale* sc = scales + (step & 3) * 8;
#pragma unroll 1
          for (int kv = 0; kv < 2 && live; ++kv) {
            live = mbar_wait(bar(kv ? kVEmpty : kKEmpty, step & 1), (step >> 1 & 1) ^ 1, abort, a.err, 0x72);
            uint8_t* tile = smem + (kv ? L::kV : L::kK) + (step & 1) * L::kTile;
#pragma unroll 1
            for (int h = 0; h < 2 && live; ++h, ++n) {
              const int stage = n % kStages;
              live = mbar_wait(bar(kRawFull, stage), n / kStages & 1, abort, a.err, 0x73);
              if (!live) break;
              const uint8_t* raw = smem + L::kRing + stage * L::kRaw;
              uint4 u[kPer];
#pragma unroll
              for (int k = 0; k < kPer; ++k) {
                const int part = id + 128 * k, t = part / (D / 16), line = part >> 3;
                const bool ok = sc[h * 4 + t / 16].ok && i * kTok + h * 64 + t < len;
                u[k] = ok ? *reinterpret_cast<const uint4*>(raw + line * 128 + (((part & 7) ^ (line & 7)) << 4)) : make_uint4(0, 0, 0, 0);
              }
              mbar_arrive(bar(kRawEmpty, stage));
#pragma unroll
              for (int k = 0; k < kPer; ++k) {
                const int part = id + 128 * k, t = h * 64 + part / (D / 16), p = part % (D / 16);
                uint4 lo, hi;
                e4m3x4_to_f16x4(u[k].x, lo.x, lo.y), e4m3x4_to_f16x4(u[k].y, lo.z, lo.w);
                e4m3x4_to_f16x4(u[k].z, hi.x, hi.y), e4m3x4_to_f16x4(u[k].w, hi.z, hi.w);
                uint8_t* dst = tile + (p >> 2) * L::kHalf + t * 128;
                const int c = 2 * (p & 3), x = t & 7;
                // The second 64 dims in the other order: the two halves of a row share banks.
                const bool second = p >= 4;
                *reinterpret_cast<uint4*>(dst + (((c + second) ^ x) << 4)) = second ? hi : lo;
                *reinterpret_cast<uint4*>(dst + (((c + !second) ^ x) << 4)) = second ? lo : hi;
              }
            }
            if (!live) break;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(bar(kv ? kVFull : kKFull, step & 1));
          }
        }
      }
    } else if (warp == 12) {
      // ---- product issue ----------------------------------------------------------------------
      if (lane == 0) {
        const uint64_t q_desc = sdesc_sw128(base + L::kQ, 16, 1024), k_desc = sdesc_sw128(base + L::kK, 16, 1024),
                       v_desc = sdesc_sw128(base + L::kV, L::kHalf, 1024);
        uint32_t step = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0};
        bool live = true;
        auto scores = [&](int h, uint32_t st) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t off = ((k >> 2) * L::kHalf + (k & 3) * 32) >> 4;
            umma_f16(tmem + h * 128, q_desc + (h * L::kTile >> 4) + off, k_desc + ((st & 1) * L::kTile >> 4) + off, idesc_f16(kTok, 0), k != 0);
          }
          umma_commit(bar(kSFull, h));
        };
        while (live && w.next(s)) {
          const int halves = w.rows_left > 128 ? 2 : 1, n = w.last - w.first;
          live = live && mbar_wait(bar(kKFull, step & 1), step >> 1 & 1, abort, a.err, 0x74);
          for (int h = 0; h < halves && live; ++h) {
            live = mbar_wait(bar(kQFull, h), n_q[h]++ & 1, abort, a.err, 0x75);
            if (!live) break;
            tc_fence_after();
            scores(h, step);
          }
          if (live) umma_commit(bar(kKEmpty, step & 1));
          for (int i = 0; i < n && live; ++i, ++step) {
            live = mbar_wait(bar(kVFull, step & 1), step >> 1 & 1, abort, a.err, 0x76);
            const bool more = i + 1 < n;
            for (int h = 0; h < halves && live; ++h) {
              live = mbar_wait(bar(kPFull, h), n_p[h]++ & 1, abort, a.err, 0x77);
              if (!live) break;
              tc_fence_after();
#pragma unroll
              for (int k = 0; k < kTok / 16; ++k)
                umma_f16_tmem(tmem + 256 + h * 128, tmem + h * 128 + k * 8, v_desc + (((step & 1) * L::kTile + k * 2048) >> 4), idesc_f16(D, 1),
                              i > 0 || k > 0);
              if (more) {
                if (h == 0) live = mbar_wait(bar(kKFull, (step + 1) & 1), (step + 1) >> 1 & 1, abort, a.err, 0x74);
                if (!live) break;
                scores(h, step + 1);
              } else {
                umma_commit(bar(kOFull, h));
              }
            }
            if (!live) break;
            umma_commit(bar(kVEmpty, step & 1));
            if (more) umma_commit(bar(kKEmpty, (step + 1) & 1));
          }
        }
        // Every product issued is complete before tensor memory is freed.
        umma_commit(bar(kDrain));
        *abort = *abort || !live;
        const unsigned long long t0 = globaltimer();
        while (!mbar_try_wait(bar(kDrain), 0) && globaltimer() - t0 < 1000000000ull) {
        }
      }
    } else if (warp == 13) {
      // ---- TMA: lanes 0-7 hold 16 tokens of the step each -----------------------------------------
      uint32_t n = 0, step = 0;
      bool live = true;
      const int boxes = s.box / 16;
      Rec rec = {-1, 0, 0, 0};
      while (live && w.next(s)) {
        if (w.first == 0 && w.last < w.steps) rec.lane = w.lane, rec.g = w.g, rec.row0 = w.row0;
        if (w.first > 0 && w.last == w.steps) rec.ends = 1;
        const int len = w.x.pos0 + w.x.rows;
        const int32_t* row_bt = a.bt + (int64_t)w.lane * a.bt_stride;
        auto page_at = [&](int i) {  // page of this lane's tokens in step i; -1: none, -2: not in the pool
          const int tok = i * kTok + 16 * lane;
          if (lane >= 8 || i >= w.last || tok >= len) return -1;
          const int blk = tok / a.page_size;
          const int page = blk < a.bt_stride ? row_bt[blk] : 0;
          return page > 0 && page < a.num_pages ? page : -2;
        };
        // One step ahead: its scales are loaded while this one is issued; two ahead: its page.
        int page = page_at(w.first), page_next = page_at(w.first + 1);
        float ks = 0.f, vs = 1.f;
        if (page >= 0) ks = a.ks[(int64_t)page * a.kv_heads + w.g], vs = a.vs[(int64_t)page * a.kv_heads + w.g];
        for (int i = w.first; i < w.last && live; ++i, ++step) {
          const int page_after = page_at(i + 2);
          float ks_next = 0.f, vs_next = 1.f;
          if (page_next >= 0) ks_next = a.ks[(int64_t)page_next * a.kv_heads + w.g], vs_next = a.vs[(int64_t)page_next * a.kv_heads + w.g];
          if (page == -2) hk_flag(a.err, hk::kErrAttnPage, (unsigned)w.lane);
          int32_t line = 0;
          if (page >= 0) line = (int32_t)((((int64_t)page * a.kv_heads + w.g) * a.page_size + (i * kTok + 16 * lane) % a.page_size) * D / 128);
          const unsigned there = __ballot_sync(0xffffffffu, page >= 0 && lane % boxes == 0);
          vs = fmaxf(vs, 7.8886090522101181e-31f);
#pragma unroll 1
          for (int part = 0; part < 4 && live; ++part, ++n) {  // K, K, V, V: 64 tokens each
            const int stage = n % kStages, h = part & 1;
            live = mbar_wait(bar(kRawEmpty, stage), (n / kStages & 1) ^ 1, abort, a.err, 0x78);
            live = __all_sync(0xffffffffu, live);
            if (!live) break;
            // The step's scales: their place was last read four steps ago, before the products that freed this stage.
            if (part == 0 && lane < 8) scales[(step & 3) * 8 + lane] = page >= 0 ? Scale{ks * (a.scale * kLog2e), log2f(vs), 1.f / vs, 1} : Scale{1.f, -INFINITY, 0.f, 0};
            __syncwarp();
            if (lane == 0) mbar_expect_tx(bar(kRawFull, stage), (uint32_t)__popc(there & (0xfu << (4 * h))) * s.box * D);
            __syncwarp();
            if ((there >> lane & 1) && lane / 4 == h)
              tma_load_2d(base + L::kRing + stage * L::kRaw + (lane & 3) * 16 * D, part < 2 ? &kmap : &vmap, bar(kRawFull, stage), 0, line);
          }
          page = page_next, page_next = page_after, ks = ks_next, vs = vs_next;
        }
      }
      if (lane == 0) s.rec[blockIdx.x] = rec;
    }
  }
  __syncthreads();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

// Joins the partials of the problem that CTA blockIdx.x began and left open: a warp for each row.
template <int D>
__global__ void __launch_bounds__(256) gqa_prefill_merge_kernel(PrefillArgs s, int ctas) {
  constexpr int P = D / 32;
  constexpr int64_t kPart = kRows * (D + 2);
  const GqaArgs& a = s.a;
  const Rec rec = s.rec[blockIdx.x];
  if (rec.lane < 0) return;
  const Lane x = lane_at(s, rec.lane);
  const int lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5), at = rec.row0 + r;
  if (at >= x.rows * s.group) return;
  float m = kNoMax, l = 0.f, o[P];
#pragma unroll
  for (int e = 0; e < P; ++e) o[e] = 0.f;
  for (int i = blockIdx.x; i < ctas; ++i) {
    const float* part = s.part + ((int64_t)i * 2 + (i == blockIdx.x ? 1 : 0)) * kPart;
    const float pm = part[kRows * D + r], pl = part[kRows * (D + 1) + r];
    const float top = fmaxf(m, pm), f = exp2_approx(m - top), pf = exp2_approx(pm - top);
    m = top;
    l = l * f + pl * pf;
#pragma unroll
    for (int e = 0; e < P; ++e) o[e] = o[e] * f + part[r * D + lane * P + e] * pf;
    if (i > blockIdx.x && s.rec[i].ends) break;
  }
  const int64_t y = (int64_t)(x.t0 + at / s.group) * a.q_heads + rec.g * s.group + at % s.group;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < P; e += 2)
    *reinterpret_cast<uint32_t*>(a.out + y * D + lane * P + e) = s.is_f16 ? pack2<true>(o[e] * inv, o[e + 1] * inv) : pack2<false>(o[e] * inv, o[e + 1] * inv);
  if (lane == 0) a.lse[y] = l == 0.f ? -INFINITY : fmaf(m, kLn2, logf(l));
}

template <int D>
int launch(PrefillArgs& s, int64_t steps, cudaStream_t stream) {
  using L = Layout<D>;
  static_assert(L::kBytes <= 232448, "shared memory");
  const int64_t most = hk::sm_count();
  const int grid = (int)(steps < most ? steps : most);
  const uint64_t lines = (uint64_t)s.a.num_pages * s.a.kv_heads * s.a.page_size * D / 128;
  HK_REQUIRE(lines <= INT32_MAX, "the cache's K and V arrays must be below 2^38 bytes each");
  CUtensorMap kmap, vmap;
  HK_TRY(make_map_u8(&kmap, s.a.kc, lines, 128, s.box * D / 128));
  HK_TRY(make_map_u8(&vmap, s.a.vc, lines, 128, s.box * D / 128));
  HK_TRY_CUDA(cudaFuncSetAttribute(gqa_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes));
  gqa_prefill_kernel<D><<<grid, kThreads, L::kBytes, stream>>>(s, kmap, vmap);
  HK_TRY_LAUNCH("gqa_prefill_kernel");
  if (grid > 1) {
    gqa_prefill_merge_kernel<D><<<dim3(grid, kRows / 8), 256, 0, stream>>>(s, grid);
    HK_TRY_LAUNCH("gqa_prefill_merge_kernel");
  }
  return HK_OK;
}

}  // namespace

namespace hk {

bool gqa_prefill_supported(int32_t dim) { return dim == 64 || dim == 128; }

size_t gqa_prefill_workspace(int32_t dim) {
  return (size_t)sm_count() * (sizeof(Rec) + 2 * sizeof(float) * kRows * (dim + 2));
}

int gqa_prefill(const GqaArgs& a, int32_t dtype, int32_t least, int64_t max_kv_len, void* workspace, cudaStream_t stream) {
  PrefillArgs s;
  s.a = a;
  s.is_f16 = dtype == HK_F16;
  s.group = a.q_heads / a.kv_heads;
  s.least = least;
  s.box = a.page_size % 64 == 0 ? 64 : a.page_size % 32 == 0 ? 32 : 16;
  s.rec = (Rec*)workspace;
  s.part = (float*)((uint8_t*)workspace + (size_t)sm_count() * sizeof(Rec));
  // At most this many steps: each lane's last row tile may be partly filled.
  const int64_t rows = (int64_t)a.num_tokens * s.group;
  const int64_t tiles = rows / kRows + (a.num_lanes < a.num_tokens ? a.num_lanes : a.num_tokens);
  const int64_t steps = tiles * a.kv_heads * (max_kv_len / kTok + 1);
  return a.dim == 64 ? launch<64>(s, steps, stream) : launch<128>(s, steps, stream);
}

}  // namespace hk
