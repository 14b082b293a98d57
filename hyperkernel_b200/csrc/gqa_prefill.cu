// Attention of prompt chunks (many query rows of a lane) over the block-scaled e4m3 cache, on tcgen05.
//
// Query rows that share a KV head (rows of the lane x heads of the group) are laid end to end and cut
// into tiles of 256, two halves of 128 TMEM lanes.  Per 128 tokens of the cache, for each half w:
//   S_w = Q_w K^T            M = 128, N = 128, K = dim, fp16 operands from shared memory
//   P_w = 2^(S_w f + log2 vs - M)   one thread per row; fp16, written over S_w in tensor memory
//   O_w += P_w V             M = 128, N = dim, K = 128, P from tensor memory, V from shared memory
// While the softmax warps of one half work, the tensor core runs the other half's products.
//
// e4m3 is exact in fp16, and so is q once each row is scaled by a power of two (but for values below 2^-21 of the
// row's largest, which keep an absolute error of 2^-32 of it), so the products are those of the stored values.
// P is rounded to fp16 (2^-11; below 2^-14 of 2^M to 2^-25 of it).  K and V come as e4m3 by TMA into a ring of 64-token stages, and four
// warps convert them into the swizzled fp16 tiles the products read (a third of the softmax's instructions, as
// 256 rows share it).  Scales of pages enter as one factor and one addend for each 16 tokens, and with log2 vs in
// the exponent one reference M serves pages of any scale (sum w / vs is the denominator).  M follows the row's largest
// weights (gqa_fp8.cuh), step by step.
//
// Work split: the (row tile, head) problems' 128-token steps lie end to end, and every SM takes an
// equal contiguous range of them.  Problems cut by a range's end leave fp32 partials, two at
// most for each SM, which the merge kernel joins in the order of the ranges.
//
// Bound by the softmax and the products it waits for in turn.  Measured, 32 query and 8 KV heads of 128: 2048 rows behind
// 30,000 tokens 1.08 ms, 960 TFLOP/s (56% of the measured bf16 burst rate); four chunks of 512 to 2048 rows behind
// 1,000 to 6,000 tokens 459 us, 701 TFLOP/s.
//
// Roles (16 warps): 0-3 and 4-7 softmax of the two halves, 8-11 conversion, 12 and 14 product issue of the
// halves, 13 TMA.
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
constexpr int kStart = 2;     // what a problem costs besides its steps, in steps
constexpr int kParts = 4;     // a step's weights are handed over 32 tokens at a time
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
using hk::kNoMax;
// Registers: 512 threads x 128 = 2 x 128 x 184 (softmax) + 2 x 128 x 72 (the rest).
constexpr int kSoftmaxRegs = 184, kOtherRegs = 72;

// Scales of 16 tokens (equal over the tokens of a box): ks * scale * log2 e, log2 vs, 1 / vs; ok: 1 where the tokens are
// there, 2 where all of the step's are.
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
              kPFull = 160 /* [half][part] */, kOFull = 224, kDrain = 240, kTurn = 256, kSlot = 272, kAbort = 276, kScales = 512 /* [4][8] */,
              kScan = 1024 /* [16] */, kFound = 1152 /* step and lane, tile and its first step */;

constexpr uint32_t idesc_f16(int n, int b_mn_major) {  // D fp32, A and B fp16, M = 128
  return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// Products by one thread; descriptors as their low words (address, leading offset), which is all that changes.
__device__ __forceinline__ void umma_f16(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 x, y;\nsetp.ne.b32 p, %5, 0;\nmov.b64 x, {%1, %3};\nmov.b64 y, {%2, %3};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p;\n}" ::"r"(d), "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void umma_f16_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 y;\nsetp.ne.b32 p, %5, 0;\nmov.b64 y, {%2, %3};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n}" ::"r"(d), "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// 128 columns in one wait.
__device__ __forceinline__ void tmem_ld128(uint32_t addr, float* v) {
  uint32_t r[128];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%128];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%129];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]), "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]), "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]), "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]), "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]), "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]), "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]), "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]), "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(addr), "r"(addr + 64)
      : "memory");
#pragma unroll
  for (int i = 0; i < 128; ++i) v[i] = __uint_as_float(r[i]);
}

// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpair(uint64_t d, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(d)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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

// A wait of at most kTries tries: short, as the kernel's code has to stay in the instruction cache (at 150 KB of code a step
// took 1.2 times as long as at 100 KB).  When it runs out it raises `abort`, which ends the others' waits.
constexpr uint32_t kTries = 1u << 22;
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile int* abort, unsigned long long* err, unsigned site) {
  uint32_t n = 0;
  bool ok;
#pragma unroll 1
  while (!(ok = mbar_try_wait(bar, parity)) && !*abort && ++n < kTries) {
  }
  if (n == kTries) *abort = 1, hk_flag(err, hk::kErrWaitTimeout, site);
  return ok;
}

// A warp's arrival: what its lanes did before is seen by who waits.
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// 8 values of a row of Q (kLanes neighbouring lanes hold the row) scaled by a power of two, as fp16; *back undoes it.
template <int kLanes>
__device__ __forceinline__ uint4 scaled_row(uint4 u, int is_f16, float* back) {
  float f[8], top = 0.f;
  if (is_f16) unpack8<true>(u, f);
  else unpack8<false>(u, f);
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[e]));
#pragma unroll
  for (int d = 1; d < kLanes; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const int ex = (int)((__float_as_uint(top) >> 23) & 255);  // 0: zero or subnormal, 255: not finite
  const int up = ex == 255 ? 0 : min(134 - ex, 120);
  const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] *= mul;
  *back = __uint_as_float((uint32_t)(127 - up) << 23);
  return pack8<true>(f);
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

// (Products of rows and heads fit 31 bits: Q itself takes 128 bytes or more for each.)
__device__ __forceinline__ int tiles_of(const PrefillArgs& s, const Lane& x) { return (x.rows * s.group + kRows - 1) / kRows; }

// Steps of one (row tile, head): up to the position of the tile's last row.  (Negative positions count as 0: their rows
// see nothing.)
__device__ __forceinline__ int steps_of(const PrefillArgs& s, const Lane& x, int tile) {
  const int upto = min(x.rows, (int)(((unsigned)(tile + 1) * kRows + s.group - 1) / (unsigned)s.group));
  return (int)(((unsigned)max(x.pos0, 0) + upto + kTok - 1) / kTok);
}

// Units (steps and starts) of the first n tiles of a lane.  The last row of a tile but the lane's last is ceil(256 (tile + 1) / group) - 1, and
// floor((floor(x / g) + b) / m) = floor((x + b g) / (m g)), so the steps are floors of a line: summed by the Euclidean
// algorithm.
__device__ __noinline__ int64_t units_before(int group, int rows, int pos0, int n, int tiles) {
  int64_t sum = (int64_t)n * kStart;
  if (n == tiles && n > 0) sum += ((int64_t)max(pos0, 0) + rows + kTok - 1) / kTok, --n;
  int64_t count = n, m = (int64_t)kTok * group, step = kRows, at = kRows + group - 1 + ((int64_t)max(pos0, 0) + kTok - 1) * group;
  while (count > 0) {
    sum += (count - 1) * count / 2 * (step / m) + count * (at / m);
    step %= m, at %= m;
    const int64_t top = step * count + at;
    if (top < m) break;
    count = top / m, at = top % m;
    const int64_t swap = m;
    m = step, step = swap;
  }
  return sum;
}

// Walks a CTA's range problem by problem.  Every role walks on its own.  A problem counts kStart units for its beginning and
// end (Q, the pipeline's filling, the output) before its steps.
struct Walk {
  int u, end;           // next unit and end of the range, from its start
  int begin;            // unit at which the current tile begins (its heads follow one another)
  int lane, tile, tiles, steps;
  Lane x;
  // The current problem, and its steps in this range.
  int g, row0, first, last, rows_left;

  __device__ __forceinline__ bool next(const PrefillArgs& s) {
    do {
      if (u >= end) return false;
      while (u - begin >= (steps + kStart) * s.a.kv_heads) {
        begin += (steps + kStart) * s.a.kv_heads;
        if (++tile >= tiles) {
          do {
            x = lane_at(s, ++lane);
          } while (x.rows == 0);
          tile = 0, tiles = tiles_of(s, x);
        }
        steps = steps_of(s, x, tile);
      }
      g = (u - begin) / (steps + kStart);
      const int lo = u - begin - g * (steps + kStart), hi = min(steps + kStart, lo + (end - u));
      first = max(0, lo - kStart), last = max(0, hi - kStart);
      u += hi - lo;
    } while (first == last);  // the range ends before the problem's first step
    row0 = tile * kRows;
    rows_left = x.rows * s.group - row0;
    return true;
  }
};

// Query row `at` of a lane as (token, head of the group), stepped without divisions.
struct RowAt {
  int t, h;
  __device__ __forceinline__ RowAt(int at, int group) : t(at / group), h(at - at / group * group) {}
  __device__ __forceinline__ void add(const RowAt& d, int group) {
    t += d.t, h += d.h;
    if (h >= group) h -= group, ++t;
  }
};

// kBox: tokens that share a page for sure (16, 32 or 64), and so a pair of scales.
template <int D, int kBox>
__global__ void __launch_bounds__(kThreads, 1) gqa_prefill_kernel(PrefillArgs s, const __grid_constant__ CUtensorMap kmap,
                                                                  const __grid_constant__ CUtensorMap vmap) {
  using L = Layout<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const GqaArgs& a = s.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* ctl = smem + L::kCtl;
  volatile int* abort = reinterpret_cast<volatile int*>(ctl + kAbort);
  const uint32_t base = smem_u32(smem), bars = smem_u32(ctl);
  hk::let_next_grid_start();
  auto bar = [&](int off, int i = 0) { return bars + off + 8 * i; };

  if (base & 1023) {  // the swizzles count from 1 KB boundaries
    if (tid == 0) hk_flag(a.err, hk::kErrWaitTimeout, 0x7f), s.rec[blockIdx.x] = Rec{-1, 0, 0, 0};
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(bar(kRawFull, i), 1), mbar_init(bar(kRawEmpty, i), 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kKFull, i), 4), mbar_init(bar(kKEmpty, i), 2);  // (empty: both halves' products)
      mbar_init(bar(kVFull, i), 4), mbar_init(bar(kVEmpty, i), 2);
      mbar_init(bar(kDrain, i), 1), mbar_init(bar(kTurn, i), 4);
      mbar_init(bar(kQFull, i), 4), mbar_init(bar(kSFull, i), 1), mbar_init(bar(kOFull, i), 1);
      for (int k = 0; k < kParts; ++k) mbar_init(bar(kPFull, kParts * i + k), 4);
    }
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) tmem_alloc(bar(kSlot), 512);

  // This CTA's range of steps, and the lane in which it begins.
  int64_t* scan = reinterpret_cast<int64_t*>(ctl + kScan);
  int64_t* found = reinterpret_cast<int64_t*>(ctl + kFound);
  auto lane_units = [&](int b) {
    int64_t n = 0;
    if (b < a.num_lanes) {
      if (blockIdx.x == 0 && a.cu[b + 1] - a.cu[b] > a.max_rows) hk_flag(a.err, hk::kErrLaneRows, (unsigned)b);
      const Lane x = lane_at(s, b);
      if (x.rows) n = units_before(s.group, x.rows, x.pos0, tiles_of(s, x), tiles_of(s, x));
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
    scan_block(lane_units(b0 + tid), &all);
    total += all;
  }
  const int64_t ranges = min((int64_t)gridDim.x, total), cta = blockIdx.x;
  const int64_t u0 = cta < ranges ? total * cta / ranges : 0, u1 = cta < ranges ? total * (cta + 1) / ranges : 0;
  if (u0 < u1) {
    int64_t carry = 0;
    for (int b0 = 0; b0 < a.num_lanes; b0 += kThreads) {
      const int64_t n = lane_units(b0 + tid);
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
    w.lane = (int)found[1];
    w.x = lane_at(s, w.lane);
    w.tiles = tiles_of(s, w.x);
    // The tile in which the range begins: every thread tries its own.
    const int64_t into = u0 - found[0];
    for (int i = tid; i < w.tiles; i += kThreads) {
      const int64_t from = units_before(s.group, w.x.rows, w.x.pos0, i, w.tiles) * a.kv_heads;
      if (from <= into && into < from + (int64_t)(steps_of(s, w.x, i) + kStart) * a.kv_heads) found[2] = i, found[3] = from - into;
    }
    __syncthreads();
    w.tile = (int)found[2];
    w.begin = (int)found[3];
    w.steps = steps_of(s, w.x, w.tile);
  }
  Scale* scales = reinterpret_cast<Scale*>(ctl + kScales);

  if (warp < 8) {
    // ---- softmax: thread = row ----------------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lanes + half * 128, o_col = tmem + lanes + 256 + half * 128;
    uint8_t* q_rows = smem + L::kQ + half * L::kTile + (warp & 3) * 32 * 128;  // of this warp
    uint32_t n_s = 0, n_o = 0, n_turn = 0, step = 0, skipped = 0;
    constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;  // lanes of a row of Q, rows a warp copies at once
    const int part = lane % kLanes;
    // The next problem of this half, and the copy of this warp's 32 rows of its Q, as they are, to their places.
    int next_pos = 0;
    auto next = [&]() {
      while (true) {
        if (!w.next(s)) return false;
        if (w.rows_left > half * 128) break;
        skipped += w.last - w.first;  // no rows for this half
      }
      const int r = half * 128 + row;
      RowAt at(w.row0 + r - lane + lane / kLanes, s.group);
      const RowAt by(kAtOnce, s.group);
#pragma unroll 4
      for (int i = 0; i < 32 / kAtOnce; ++i) {
        const int wr = i * kAtOnce + lane / kLanes;
        const bool on = r - lane + wr < w.rows_left;
        const uint16_t* src = a.q + (on ? (w.x.t0 + at.t) * a.q_stride + (int64_t)(w.g * s.group + at.h) * D + part * 8 : 0);
        const uint32_t dst = smem_u32(q_rows) + (part >> 3) * L::kHalf + wr * 128 + (((part & 7) ^ (wr & 7)) << 4);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
        at.add(by, s.group);
      }
      next_pos = r < w.rows_left ? a.positions[w.x.t0 + (w.row0 + r) / s.group] : INT32_MAX;
      return true;
    };
    bool live = true, have = next();
    step = skipped, skipped = 0;
    while (live && have) {
      // The current problem, as the walk moves on before its end.
      const int first = w.first, last = w.last, r = half * 128 + row;
      const bool both = w.rows_left > 128, on = r < w.rows_left;
      const bool starts = w.first == 0, whole = starts && w.last == w.steps;
      const int pos = next_pos;
      const int pos_min = w.x.pos0 + (w.row0 + half * 128) / s.group;  // rows of a lane rise
      const RowAt mine(w.row0 + r, s.group);
      const int64_t y = (int64_t)(w.x.t0 + mine.t) * a.q_heads + w.g * s.group + mine.h;
      // Q to fp16: each row scaled by a power of two, so that fp16 holds it exactly.  (A lane converts what it copied.)
      float rowf = 1.f;
      asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 2
      for (int i = 0; i < 32 / kAtOnce; ++i) {
        const int wr = i * kAtOnce + lane / kLanes;
        uint4* at = reinterpret_cast<uint4*>(q_rows + (part >> 3) * L::kHalf + wr * 128 + (((part & 7) ^ (wr & 7)) << 4));
        float back;
        *at = scaled_row<kLanes>(*at, s.is_f16, &back);
        back = __shfl_sync(0xffffffffu, back, lane % kAtOnce * kLanes);
        if (lane / kAtOnce == i) rowf = back;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      warp_arrive(bar(kQFull, half));

      float m = kNoMax, l = 0.f, peak = kNoMax, soft = 1.f, soft_m = kNoMax;
      for (int i = first; i < last; ++i, ++n_s, ++step) {
        live = live && wait_bar(bar(kSFull, half), n_s & 1, abort, a.err, 0x70);
        live = __all_sync(0xffffffffu, live);
        if (!live) break;
        // The halves take turns: while one half's weights are computed, the other half's products run.
        if (both) {
          live = wait_bar(bar(kTurn, half), (n_turn & 1) ^ (half ^ 1), abort, a.err, 0x79);
          live = __all_sync(0xffffffffu, live);
          if (!live) break;
          ++n_turn;
        }
        tc_fence_after();
        if (i + 1 == last) have = next();  // this half's products with Q are complete: its next rows can come
        float v[128];
        tmem_ld128(s_col, v);
        constexpr int kGroups = kTok / kBox;
        const Scale* sc = scales + (step & 3) * 8;
        // Few groups keep their scales in registers; many read them again (shared memory) for each of the two passes.
        constexpr bool kKeep = kGroups <= 2;
        float f_kept[2] = {1.f, 1.f}, lsv_kept[2] = {0.f, 0.f};
        if (kKeep) {
#pragma unroll
          for (int k = 0; k < 2; ++k) f_kept[k] = fmaxf(sc[4 * k].kf * rowf, 1.1754944e-38f), lsv_kept[k] = sc[4 * k].lsv;
        }
        auto factor = [&](int k) { return kKeep ? f_kept[k & 1] : fmaxf(sc[k * (kBox / 16)].kf * rowf, 1.1754944e-38f); };  // above 0: a masked -inf stays one
        auto addend = [&](int k) { return kKeep ? lsv_kept[k & 1] : sc[k * (kBox / 16)].lsv; };
        const bool edge = (i + 1) * kTok - 1 > pos_min;
        if (edge) {
          const int seen = pos - i * kTok;  // tokens after it are masked
#pragma unroll
          for (int e = 0; e < 128; ++e) v[e] = e > seen ? -INFINITY : v[e];
        }
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
          float x[4];  // chains
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = max3(v[kBox * k + e], v[kBox * k + 4 + e], v[kBox * k + 8 + e]);
#pragma unroll
          for (int e = 12; e < kBox - 4; e += 8)
#pragma unroll
            for (int y = 0; y < 4; ++y) x[y] = max3(x[y], v[kBox * k + e + y], v[kBox * k + e + 4 + y]);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = fmaxf(x[e], v[kBox * k + kBox - 4 + e]);
          const float most = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          top = fmaxf(top, fmaf(most, factor(k), addend(k)));  // the factor is positive
        }
        // S is complete, so the product before it (which this row's O is from) is too.
        if (__any_sync(0xffffffffu, top > m + hk::kRoom || (top < m - hk::kSlack && !edge))) {
          const float m_new = hk::new_reference(m, top, peak, !edge && l < hk::kFullSum), down = exp2_approx(m - m_new);
          m = m_new, peak = fmaxf(peak, m);
          // A weight's exponent is one fused product and sum, M a rounded one: from 2^26 on their difference could pass fp16's room.  Scores
          // of that size are good to 2^-20 of it, so distances from M are taken in units of 2^-24 of it.
          const uint32_t size = __float_as_uint(m) >> 23 & 255;
          soft = size < 127 + 26 ? 1.f : __uint_as_float((127 + 24 + 127 - size) << 23);
          soft_m = m * soft;
          l *= down;
          if (i > first) {
#pragma unroll 1
            for (int k = 0; k < D / 16; ++k) {
              float o[16];
              tmem_ld16(o_col + 16 * k, o);
              uint32_t x[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(o[e] * down);
              tmem_st16(o_col + 16 * k, x);
            }
          }
        }
        // 32 tokens' weights at a time, over columns of S that are read already: their product starts while the others are
        // weighed.
        uint64_t sum = 0;  // two zeros
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const int t = 32 * j + e, k = t / kBox;
            const float f = factor(k) * soft, c = fmaf(addend(k), soft, -soft_m);
            const uint64_t x = fma2(pair(v[t], v[t + 1]), pair(f, f), pair(c, c));
            float x0, x1;
            unpair(x, x0, x1);
            x0 = exp2_approx(x0), x1 = exp2_approx(x1);
            sum = add2(sum, pair(x0, x1));
            p[e / 2] = pack2<true>(x0, x1);
            if ((t + 2) % kBox == 0) {
              float s0, s1;
              unpair(sum, s0, s1);
              l = fmaf(s0 + s1, sc[k * (kBox / 16)].isv, l);
              sum = 0;
            }
          }
          tmem_st16(s_col + 16 * j, p);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tc_fence_before();
          warp_arrive(bar(kPFull, half * kParts + j));
        }
        if (both) warp_arrive(bar(kTurn, half ^ 1));
      }
      live = live && wait_bar(bar(kOFull, half), n_o & 1, abort, a.err, 0x71);
      live = __all_sync(0xffffffffu, live);
      if (!live) break;
      ++n_o;
      tc_fence_after();
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int k = 0; k < D / 32; ++k) {
          float o[32];
          tmem_ld32(o_col + 32 * k, o);
          if (on) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= inv;
            uint4* to = reinterpret_cast<uint4*>(a.out + y * D + 32 * k);
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e] = s.is_f16 ? pack8<true>(o + 8 * e) : pack8<false>(o + 8 * e);
          }
          __syncwarp();
        }
        if (on) a.lse[y] = l == 0.f ? -INFINITY : fmaf(m, kLn2, logf(l));
      } else {
        float* piece = s.part + ((int64_t)blockIdx.x * 2 + (starts ? 1 : 0)) * (kRows * (D + 2));
#pragma unroll 1
        for (int k = 0; k < D / 32; ++k) {
          float o[32];
          tmem_ld32(o_col + 32 * k, o);
          if (on) {
            float4* to = reinterpret_cast<float4*>(piece + r * D + 32 * k);
#pragma unroll
            for (int e = 0; e < 8; ++e) to[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
          __syncwarp();
        }
        if (on) piece[kRows * D + r] = m, piece[kRows * (D + 1) + r] = l;
      }
      step += skipped, skipped = 0;
      tc_fence_before();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp < 12) {
      // ---- conversion: raw e4m3 -> swizzled fp16 -----------------------------------------------
      const int id = tid - 256;
      constexpr int kPer = 64 * D / 16 / 128;  // 16-byte parts of a stage a thread converts: id, id + 128, ...
      // Part id: its place in the raw lines, its token and dims, and its two places in the fp16 tile (the second 64 dims are
      // written in the other order: the two halves of a row share banks).  The next parts lie at fixed distances.
      const int src = (id >> 3) * 128 + (((id & 7) ^ (id >> 3 & 7)) << 4);
      const int t0 = id / (D / 16), p0 = id % (D / 16), c0 = 2 * (p0 & 3);
      const bool second = p0 >= 4;
      const int dst = (p0 >> 2) * L::kHalf + t0 * 128, dst_first = dst + (((c0 + second) ^ (t0 & 7)) << 4), dst_other = dst + (((c0 + !second) ^ (t0 & 7)) << 4);
      uint32_t n = 0, step = 0;                // stages read
      bool live = true;
      while (live && w.next(s)) {
        const int len = w.x.pos0 + w.x.rows;  // tokens of the lane: what lies past them may be anything
        for (int i = w.first; i < w.last && live; ++i, ++step) {
          const Scale* sc = scales + (step & 3) * 8;
#pragma unroll 1
          for (int kv = 0; kv < 2 && live; ++kv) {
            live = __all_sync(0xffffffffu, wait_bar(bar(kv ? kVEmpty : kKEmpty, step & 1), (step >> 1 & 1) ^ 1, abort, a.err, 0x72));
            uint8_t* tile = smem + (kv ? L::kV : L::kK) + (step & 1) * L::kTile;
#pragma unroll 1
            for (int h = 0; h < 2 && live; ++h, ++n) {
              const int stage = n % kStages;
              live = live && __all_sync(0xffffffffu, wait_bar(bar(kRawFull, stage), n / kStages & 1, abort, a.err, 0x73));
              if (!live) break;
              const uint8_t* raw = smem + L::kRing + stage * L::kRaw + src;
              uint4 u[kPer];
#pragma unroll
              for (int k = 0; k < kPer; ++k) u[k] = *reinterpret_cast<const uint4*>(raw + k * 2048);
              if (sc[0].ok != 2) {  // some tokens are not there, or past the lane's end
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                  const int t = h * 64 + t0 + k * (128 * 16 / D);
                  if (!sc[t / 16].ok || i * kTok + t >= len) u[k] = make_uint4(0, 0, 0, 0);
                }
              }
              warp_arrive(bar(kRawEmpty, stage));
              uint8_t* to = tile + h * (64 * 128);
#pragma unroll
              for (int k = 0; k < kPer; ++k) {
                uint4 lo, hi;
                e4m3x4_to_f16x4(u[k].x, lo.x, lo.y), e4m3x4_to_f16x4(u[k].y, lo.z, lo.w);
                e4m3x4_to_f16x4(u[k].z, hi.x, hi.y), e4m3x4_to_f16x4(u[k].w, hi.z, hi.w);
                *reinterpret_cast<uint4*>(to + dst_first + k * (128 * 16 / D * 128)) = second ? hi : lo;
                *reinterpret_cast<uint4*>(to + dst_other + k * (128 * 16 / D * 128)) = second ? lo : hi;
              }
            }
            if (!live) break;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            warp_arrive(bar(kv ? kVFull : kKFull, step & 1));
          }
        }
      }
    } else if (warp == 12 || warp == 14) {
      // ---- product issue: a warp for each half, so that neither waits for the other's weights ---------
      const int h = (warp - 12) / 2;
      if (lane == 0) {
        const uint64_t desc = sdesc_sw128(base, 16, 1024);
        const uint32_t hi = (uint32_t)(desc >> 32), q = (uint32_t)desc + ((L::kQ + h * L::kTile) >> 4), k0 = (uint32_t)desc + (L::kK >> 4);
        const uint32_t v0 = (uint32_t)sdesc_sw128(base + L::kV, L::kHalf, 1024);
        const uint32_t s_at = tmem + h * 128, o_at = tmem + 256 + h * 128;
        uint32_t step = 0, n_q = 0, n_p = 0;
        bool live = true;
        auto scores = [&](uint32_t st) {
          const uint32_t k = k0 + ((st & 1) ? (uint32_t)(L::kTile >> 4) : 0u);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const uint32_t off = ((i >> 2) * L::kHalf + (i & 3) * 32) >> 4;
            umma_f16(s_at, q + off, k + off, hi, idesc_f16(kTok, 0), i != 0);
          }
          umma_commit(bar(kSFull, h));
          umma_commit(bar(kKEmpty, st & 1));
        };
        auto full = [&](int which, uint32_t st) { return wait_bar(bar(which, st & 1), st >> 1 & 1, abort, a.err, 0x74); };
        while (live && w.next(s)) {
          const int n = w.last - w.first;
          if (w.rows_left <= h * 128) {  // no rows for this half: its share of the buffers is free as soon as they are full
            for (int i = 0; i < n && live; ++i, ++step) {
              live = full(kKFull, step);
              if (live) mbar_arrive(bar(kKEmpty, step & 1));
              live = live && full(kVFull, step);
              if (live) mbar_arrive(bar(kVEmpty, step & 1));
            }
            continue;
          }
          live = full(kKFull, step) && wait_bar(bar(kQFull, h), n_q++ & 1, abort, a.err, 0x75);
          if (!live) break;
          tc_fence_after();
          scores(step);
          for (int i = 0; i < n && live; ++i, ++step, ++n_p) {
            const uint32_t v = v0 + ((step & 1) ? (uint32_t)(L::kTile >> 4) : 0u);
            live = full(kVFull, step);
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              live = live && wait_bar(bar(kPFull, h * kParts + part), n_p & 1, abort, a.err, 0x77);
              if (!live) break;
              tc_fence_after();
#pragma unroll
              for (int k = 2 * part; k < 2 * part + 2; ++k)
                umma_f16_tmem(o_at, s_at + k * 8, v + (k * 2048 >> 4), hi, idesc_f16(D, 1), k > 0 ? 1u : (uint32_t)(i > 0));
            }
            if (!live) break;
            umma_commit(bar(kVEmpty, step & 1));
            if (i + 1 < n) {
              live = full(kKFull, step + 1);
              if (!live) break;
              tc_fence_after();
              scores(step + 1);
            } else {
              umma_commit(bar(kOFull, h));
            }
          }
        }
        // Every product issued is complete before tensor memory is freed.
        umma_commit(bar(kDrain, h));
        const unsigned long long t0 = globaltimer();
        while (!mbar_try_wait(bar(kDrain, h), 0) && globaltimer() - t0 < 1000000000ull) {
        }
      }
    } else if (warp == 13) {
      // ---- TMA: lanes 0-7 hold 16 tokens of the step each -----------------------------------------
      uint32_t n = 0, step = 0;
      bool live = true;
      constexpr int boxes = kBox / 16;
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
          const unsigned pages = __ballot_sync(0xffffffffu, page >= 0);
          const unsigned there = pages & (boxes == 1 ? 0xffu : boxes == 2 ? 0x55u : 0x11u);
          const int ok = pages == 0xffu && (i + 1) * kTok <= len ? 2 : 1;
          vs = fmaxf(vs, 7.8886090522101181e-31f);
#pragma unroll 1
          for (int part = 0; part < 4 && live; ++part, ++n) {  // K, K, V, V: 64 tokens each
            const int stage = n % kStages, h = part & 1;
            live = wait_bar(bar(kRawEmpty, stage), (n / kStages & 1) ^ 1, abort, a.err, 0x78);
            live = __all_sync(0xffffffffu, live);
            if (!live) break;
            // The step's scales: their place was last read four steps ago, before the products that freed this stage.
            if (part == 0 && lane < 8) scales[(step & 3) * 8 + lane] = page >= 0 ? Scale{ks * (a.scale * kLog2e), log2f(vs), 1.f / vs, ok} : Scale{1.f, -INFINITY, 0.f, 0};
            __syncwarp();
            if (lane == 0) mbar_expect_tx(bar(kRawFull, stage), (uint32_t)__popc(there & (0xfu << (4 * h))) * (kBox * D));
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
  if (*abort) {  // a wait has run out: copies still in flight get time to land before the CTA ends
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 100000000ull) {
    }
  }
  if (warp == 12) tmem_dealloc(tmem, 512);
}

// Joins the partials of the problem that CTA blockIdx.x began and left open: a warp for each row.
template <int D>
__global__ void __launch_bounds__(256) gqa_prefill_merge_kernel(PrefillArgs s, int ctas) {
  constexpr int P = D / 32;
  constexpr int64_t kPart = kRows * (D + 2);
  const GqaArgs& a = s.a;
  hk::wait_for_grid_before();
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

template <int D, int kBox>
int launch(PrefillArgs& s, int64_t steps, cudaStream_t stream) {
  using L = Layout<D>;
  static_assert(L::kBytes <= 232448, "shared memory");
  const int64_t most = hk::sm_count();
  const int grid = (int)(steps < most ? steps : most);
  const uint64_t lines = (uint64_t)s.a.num_pages * s.a.kv_heads * s.a.page_size * D / 128;
  HK_REQUIRE(lines <= INT32_MAX, "the cache's K and V arrays must be below 2^38 bytes each");
  CUtensorMap kmap, vmap;
  HK_TRY(make_map_u8(&kmap, s.a.kc, lines, 128, kBox * D / 128));
  HK_TRY(make_map_u8(&vmap, s.a.vc, lines, 128, kBox * D / 128));
  HK_TRY_CUDA(cudaFuncSetAttribute(gqa_prefill_kernel<D, kBox>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes));
  gqa_prefill_kernel<D, kBox><<<grid, kThreads, L::kBytes, stream>>>(s, kmap, vmap);
  HK_TRY_LAUNCH("gqa_prefill_kernel");
  if (grid > 1) {
    HK_TRY_CUDA(hk::launch_early(gqa_prefill_merge_kernel<D>, dim3(grid, kRows / 8), 256, 0, stream, s, grid));
    HK_TRY_LAUNCH("gqa_prefill_merge_kernel");
  }
  return HK_OK;
}

template <int D>
int launch(PrefillArgs& s, int64_t steps, cudaStream_t stream) {
  // The largest box of 16, 32 or 64 tokens that divides the page.
  if (s.a.page_size % 64 == 0) return launch<D, 64>(s, steps, stream);
  if (s.a.page_size % 32 == 0) return launch<D, 32>(s, steps, stream);
  return launch<D, 16>(s, steps, stream);
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
  s.rec = (Rec*)workspace;
  s.part = (float*)((uint8_t*)workspace + (size_t)sm_count() * sizeof(Rec));
  // At most this many steps: each lane's last row tile may be partly filled.
  const int64_t rows = (int64_t)a.num_tokens * s.group;
  const int64_t tiles = rows / kRows + (a.num_lanes < a.num_tokens ? a.num_lanes : a.num_tokens);
  const int64_t steps = tiles * a.kv_heads * (max_kv_len / kTok + 1);
  return a.dim == 64 ? launch<64>(s, steps, stream) : launch<128>(s, steps, stream);
}

}  // namespace hk
