// b2g_cache_attention.cu — one query token per request over the paged 8-bit
// cache (b2g_cache_attention).
//
// out[j] = sum_n exp(z_n - max z) V_n / sum_n exp(z_n - max z),
// z_n = scale * q_j . K_n, one pass over K and V with the running maximum and
// sum.  With c the codes and a scale for each block and head, z_n = (scale *
// kscale) * (q . c_n), and the products run on the codes, which fp16 holds
// exactly: a warp's m16n8k16 products take 16 tokens' codes, widened in
// registers, as the 16 rows and up to 8 (or 2 x 8) of the query heads that
// share the kv head as the columns, S^T = K Q^T and O^T = V^T P^T, so that a
// group of 8 heads fills a product (a group of more than 16 is taken 16 at a
// time, and the cache read once for each 16).  q is brought to [-2^15, 2^15] by a power of
// two (exact in fp16 down to 2^-28 of a row's largest value), the weights
// times their value scales are fp16 of at most 2^15, the largest of a head
// near 2^7 (11 bits down to 2^-21 of it), sums, maxima and the output are fp32.
//
// Bound by memory: 2 * dim bytes a token and kv head.  A producer warp keeps
// a ring of stages of 64 to 128 tokens filled by TMA (boxes of whole rows of a
// block in the 128-byte or 64-byte swizzle, which the fragments' shared loads
// read without bank conflicts), with the blocks' scales beside them; four or
// five consumer warps take 16 or 32 tokens each of every stage.  The (request,
// head, stage) tiles are laid end to end and cut into equal ranges, one a CTA, so ragged
// lengths fill the GPU evenly; what a cut divides is joined by a second small
// kernel.
//
// Measured in a stream of calls (in brackets: on the GPU alone, a graph of 20
// calls; GB/s of codes, 6547 being the card's copy rate):
//   64 requests of 14000 to 31000 tokens, 8 kv heads, 32 heads, dim 128, int8:
//   501 us, 6040 GB/s (472, 6410; the power limit lowers the clock in longer runs)
//   1 request of 150001 tokens, 4 kv heads, 32 heads, e4m3: 39.5 us, 3890 GB/s
//   (37; some 10 us are start, the cuts' partial results and their join)
//   48 ragged requests up to 6000 tokens, 56 heads on 8, dim 64, e4m3: 42.9 us,
//   3090 GB/s (41; the consumers' chains of dependent products, not the loads)
//   1 request of 997 tokens: 10.3 us (9.1), two launches and a handful of
//   dependent loads
// K as the first operand instead of q halves the products (8 heads of 16 rows
// were empty): 822 -> 475 us together with the TMA ring, whose place registers
// had before.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "../../include/b2g_serving.h"
#include "b2g_internal.h"
#include "ptx_sm100.cuh"

namespace {

namespace ptx = b2g::ptx;

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Consumer warps of a CTA; the producer is one more.  Two CTAs of six warps
// fill an SM's registers where 16 heads' sums of 128 dims take 168 a thread.
// (16 heads of 64 dims, int8, with a fifth warp: 64 requests of 20000 tokens
// 175 -> 163 us, but 16 of 10000 39.8 -> 44.7.)
__host__ __device__ constexpr int consumers(int dp, int rows) { return dp == 128 && rows == 16 ? 5 : 4; }
// Pieces of 16 tokens that a consumer warp takes from a stage: with rows of 64
// bytes two at once, so that their chains of dependent products overlap.
__host__ __device__ constexpr int pieces(int dp) { return dp == 64 ? 2 : 1; }
// Tokens of a stage.
__host__ __device__ constexpr int tile_tokens(int dp, int rows) {
  return 16 * consumers(dp, rows) * pieces(dp);
}
constexpr float kGrow = 8.f;           // a maximum may be passed by 2^8 before the sums are rescaled
constexpr float kLift = 7.f;           // the largest weight times value scale stands at 2^7 in fp16
constexpr uint64_t kDrainLimitNs = 100000000ull;
constexpr int kJoin = 4;                     // rows of parts that a joining warp loads at once
constexpr uint32_t kNoBlock = 0xffffffffu;   // in the place of a key scale
// What the maxima start from: below every score, yet finite, so that differences of two are no NaN.
constexpr float kNothing = -FLT_MAX;
constexpr float kLeastScale = -100.f;        // log2 of the least value scale that bounds the weights
enum : int { kErrFull = 0x311, kErrEmpty = 0x312 };

// Shared memory of a CTA: the ring, the stages' scales, the barriers, and the
// warps' results of a segment.
template <int DP, int ROWS>
struct Smem {
  // Multiprocessor's CTAs and their stages: with rows of 64 bytes and 8 heads the products' chains
  // want a fourth CTA's warps more than the ring its third stage (64 requests of 20000 tokens, int8:
  // 247 -> 226 us; 48 ragged ones: 41.7 -> 39.3).
  static constexpr bool kFour = DP == 64 && ROWS == 8;
  static constexpr int kCtas = kFour ? 4 : ROWS == 8 ? 3 : 2;
  static constexpr int kStages = kFour ? 2 : 3;
  static constexpr int kWarps = consumers(DP, ROWS), kThreads = (kWarps + 1) * 32;
  static constexpr int kTile = tile_tokens(DP, ROWS);
  static constexpr int kPieces = kTile / 16;
  static constexpr int kSideBytes = kTile * DP;             // K or V of a stage
  static constexpr int kStageBytes = 2 * kSideBytes;
  static constexpr int kOffScales = kStages * kStageBytes;  // [stage][piece]{k scale, v scale}
  static constexpr int kOffBars = kOffScales + kStages * kPieces * 8;
  static constexpr int kOffMisc = kOffBars + 2 * kStages * 8;
  static constexpr int kOffJoin = (kOffMisc + 64 + 15) / 16 * 16;   // m, l, b: [warp][ROWS]; o: [warp][ROWS][DP]
  static constexpr int kOffO = kOffJoin + 3 * kWarps * ROWS * 4;
  static constexpr int kBytes = kOffO + kWarps * ROWS * DP * 4 + 1024;
  static_assert(kSideBytes % 1024 == 0 && kOffScales % 8 == 0 && kOffBars % 8 == 0 && kOffO % 16 == 0,
                "swizzle atoms, float2 scales, barriers, float4 sums");
  static_assert(kCtas * (kBytes + 1024) <= 227 * 1024 + 1024, "shared memory of an SM");
};

struct Args {
  const void* q;
  int64_t q_row, q_head;
  const float* k_scale;
  const float* v_scale;
  const int32_t* table;
  int64_t width, ld;
  const int32_t* seq_lens;
  int requests, kv_heads, group, row_groups, dim, lg_block, bf16;
  int box_rows;                  // rows of a TMA box: the part of a block that a stage holds
  int64_t num_blocks;
  float scale_log2;
  void* out;
  float* lse;
  // workspace: tiles before each request (requests + 1), then the partial results, two a CTA
  int* prefix;
  float* part_m;
  float* part_l;
  float* part_b;
  float* part_o;
  int grid;
  long long wait_limit_ns;
  int* err;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ int length_of(const Args& a, int r) {
  const int64_t n = a.seq_lens[r], most = a.width << a.lg_block;
  return static_cast<int>(n < 0 ? 0 : (n < most ? n : most));
}
template <int TILE>
__device__ __forceinline__ int tiles_of(const Args& a, int r) {
  return (length_of(a, r) + TILE - 1) / TILE;
}

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// An int8 code c, with its sign bit turned c + 128, in the low byte of an fp16
// is the subnormal number (c + 128) 2^-24: what the sum of the products has to
// lose again is 128 times the query's own sum.  (With an offset of 1152, as
// normal numbers have it, the log sums of queries with a common part of 10 were
// off by 1.3e-3, with this one by 2.5e-5; without one, for 32 subtractions a
// piece, 64 requests of 24000 tokens take 521 us for 504.)  The 2^24 comes back in two parts, with the query's power of
// two and with the key scale, neither of which then leaves fp32's range.
constexpr float kI8Offset = 128.f * 0x1p-24f, kI8Query = 0x1p15f, kI8Scale = 0x1p9f;

// Four codes to two fp16 pairs.  OFFSET: int8 codes come as (128 + c) 2^-24 (and the
// caller takes the offset out of the sum), else as c.
template <bool E4M3, bool OFFSET>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    // 0x6400 + u is 1024 + u.
    lo = __byte_perm(u, OFFSET ? 0u : 0x64646464u, 0x4140);
    hi = __byte_perm(u, OFFSET ? 0u : 0x64646464u, 0x4342);
    if (!OFFSET) {
      const __half2 off = __half2half2(__ushort_as_half(0x6480));   // 1152
      const __half2 hx = __hsub2(*reinterpret_cast<__half2*>(&lo), off);
      const __half2 hy = __hsub2(*reinterpret_cast<__half2*>(&hi), off);
      lo = *reinterpret_cast<const uint32_t*>(&hx);
      hi = *reinterpret_cast<const uint32_t*>(&hy);
    }
  }
}

// A warp's running state.  Lane (g, c) = (lane / 4, lane % 4).
template <int DP, int ROWS>
struct State {
  static constexpr int N = ROWS / 8;   // columns of 8 query heads
  uint32_t q[N][DP / 16][2];           // head 8 n + g, the lane's dims
  // Of heads 8 n + 2 c, 8 n + 2 c + 1:
  float rf[N][2];                      // scale * log2(e) * the powers of two that q and the codes were divided by
  float start[N][2];                   // what S starts from: the int8 offset's share
  float m[N][2], l[N][2];              // maximum so far (log2 units), this lane's part of the sum
  float b[N][2];                       // o is in units of 2^b, l in units of 2^m: b is the largest of
                                       // z + log2(value scale) so far, less kLift
  float o[N][DP / 16][4];              // dims DP/8 g + 2 t, + 1 (index / 2) of those heads (index % 2)
};

// One warp's 16 (32) tokens, `left` of them there.  k, v: their rows in shared
// memory, swizzled; sc: the pieces' scales.
template <int DP, int ROWS, bool E4M3>
__device__ __forceinline__ void compute_pieces(State<DP, ROWS>& s, const uint8_t* k, const uint8_t* v,
                                               float2 (&sc)[pieces(DP)], int left, int lane) {
  constexpr int N = ROWS / 8, P = pieces(DP);
  constexpr int kChunk = DP == 128 ? 8 : 4;      // 16-byte chunks of a row
  const int g = lane >> 2, c = lane & 3;
  // Chunk `at` of a row, in the 128-byte (64-byte) swizzle: XOR of row % 8 ((row / 2) % 4).
  auto place = [&](int row, int at) {
    return row * DP + ((at ^ (DP == 128 ? row & 7 : (row >> 1) & 3)) << 4);
  };
  float z[P][N][4];
#pragma unroll
  for (int x = 0; x < P; ++x) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      z[x][n][0] = z[x][n][2] = s.start[n][0];
      z[x][n][1] = z[x][n][3] = s.start[n][1];
    }
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) {
      const int at = kChunk / 4 * c + j;
      const uint4 lo = *reinterpret_cast<const uint4*>(k + place(16 * x + g, at));
      const uint4 hi = *reinterpret_cast<const uint4*>(k + place(16 * x + g + 8, at));
      const uint32_t ls[4] = {lo.x, lo.y, lo.z, lo.w}, hs[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a[4];
        widen4<E4M3, true>(ls[i], a[0], a[2]);
        widen4<E4M3, true>(hs[i], a[1], a[3]);
#pragma unroll
        for (int n = 0; n < N; ++n) mma_16816(z[x][n], a, s.q[n][4 * j + i][0], s.q[n][4 * j + i][1]);
      }
    }
  }
  bool part = left < 16 * P;
#pragma unroll
  for (int x = 0; x < P; ++x) {
    const bool out = __float_as_uint(sc[x].x) == kNoBlock;     // a block outside the cache
    part |= out;
    if (out) sc[x].y = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float r = s.rf[n][h] * sc[x].x;
        z[x][n][h] *= r;
        z[x][n][2 + h] *= r;
      }
  }
  if (part) {                            // the last tokens, or a block outside the cache
#pragma unroll
    for (int x = 0; x < P; ++x) {
      const int here = __float_as_uint(sc[x].x) == kNoBlock ? 0 : left - 16 * x;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (g >= here) z[x][n][h] = -INFINITY;
          if (g + 8 >= here) z[x][n][2 + h] = -INFINITY;
        }
      if (here <= 0) sc[x].y = 0.f;
    }
  }
  // Two maxima: of z for the sums l, and of z + log2 of the value scale for the
  // weights in fp16, which then keep the bits that the output needs however
  // far the blocks' value scales lie apart.
  float top[N][2], tall[N][2], lg[P];
#pragma unroll
  for (int x = 0; x < P; ++x) lg[x] = fmaxf(log2_fast(fabsf(sc[x].y)), kLeastScale);
  bool grow = false;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[n][h] = fmaxf(z[0][n][h], z[0][n][2 + h]);
      tall[n][h] = top[n][h] + lg[0];
#pragma unroll
      for (int x = 1; x < P; ++x) {
        const float t = fmaxf(z[x][n][h], z[x][n][2 + h]);
        top[n][h] = fmaxf(top[n][h], t);
        tall[n][h] = fmaxf(tall[n][h], t + lg[x]);
      }
      grow |= top[n][h] > s.m[n][h] + kGrow || tall[n][h] > s.b[n][h] + (kLift + kGrow);
    }
  if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float t = top[n][h], b = tall[n][h];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
          b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, o));
        }
        t = fmaxf(t, s.m[n][h]);
        b = fmaxf(b - kLift, s.b[n][h]);
        s.l[n][h] *= exp2_fast(s.m[n][h] - t);
        const float corr = exp2_fast(s.b[n][h] - b);
        s.m[n][h] = t;
        s.b[n][h] = b;
#pragma unroll
        for (int t16 = 0; t16 < DP / 16; ++t16) {
          s.o[n][t16][h] *= corr;
          s.o[n][t16][2 + h] *= corr;
        }
      }
  }
  // The weight in fp16 is 2^(z - b) times the value scale, of at most 2^(kLift + kGrow) by the test
  // above.  2^(z - b) alone stays finite too (b takes no scale for less than 2^kLeastScale); a factor
  // 2^(m - b) in its place would not beside a larger scale: where blocks of zeros lead, b lies 107 below m.
  uint32_t p[P][N][2];
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int x = 0; x < P; ++x) {
      float w[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s.l[n][h] += exp2_fast(z[x][n][h] - s.m[n][h]) + exp2_fast(z[x][n][2 + h] - s.m[n][h]);
        w[h] = exp2_fast(z[x][n][h] - s.b[n][h]) * sc[x].y;
        w[2 + h] = exp2_fast(z[x][n][2 + h] - s.b[n][h]) * sc[x].y;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const __half2 hv = __floats2half2_rn(w[2 * t], w[2 * t + 1]);
        p[x][n][t] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hv));
      }
    }
  }
  // V: tokens 2c, 2c+1, 2c+8, 2c+9, dims DP/8 g ... of each.  Loaded here and not
  // before the weights, which then have its registers (16 heads of 128 dims, int8: 67.2 -> 64.8 us
  // at 16 requests of 10000 tokens; 8 heads: 63.8 -> 62.1).
  uint32_t w[P][4][DP / 32];
#pragma unroll
  for (int x = 0; x < P; ++x)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int row = 16 * x + 2 * c + (t & 1) + (t >> 1) * 8;
      if (DP == 128) {
        const uint4 y = *reinterpret_cast<const uint4*>(v + place(row, g));
        w[x][t][0] = y.x, w[x][t][1] = y.y, w[x][t][DP / 32 - 2] = y.z, w[x][t][DP / 32 - 1] = y.w;
      } else {
        const uint2 y = *reinterpret_cast<const uint2*>(v + place(row, g >> 1) + (g & 1) * 8);
        w[x][t][0] = y.x, w[x][t][1] = y.y;
      }
    }
  // What stands behind the last token may be NaN in e4m3, and 0 * NaN must not reach the sums.
  if (E4M3 && part)
#pragma unroll
    for (int x = 0; x < P; ++x) {
      const int here = __float_as_uint(sc[x].x) == kNoBlock ? 0 : left - 16 * x;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (2 * c + (t & 1) + (t >> 1) * 8 >= here)
#pragma unroll
          for (int j = 0; j < DP / 32; ++j) w[x][t][j] = 0;
    }
#pragma unroll
  for (int x = 0; x < P; ++x)
#pragma unroll
    for (int j = 0; j < DP / 32; ++j) {
      const uint32_t(&u)[4][DP / 32] = w[x];
      uint32_t a[2][4];
      widen4<E4M3, false>(__byte_perm(u[0][j], u[1][j], 0x5140), a[0][0], a[0][1]);
      widen4<E4M3, false>(__byte_perm(u[0][j], u[1][j], 0x7362), a[1][0], a[1][1]);
      widen4<E4M3, false>(__byte_perm(u[2][j], u[3][j], 0x5140), a[0][2], a[0][3]);
      widen4<E4M3, false>(__byte_perm(u[2][j], u[3][j], 0x7362), a[1][2], a[1][3]);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        mma_16816(s.o[n][2 * j], a[0], p[x][n][0], p[x][n][1]);
        mma_16816(s.o[n][2 * j + 1], a[1], p[x][n][0], p[x][n][1]);
      }
    }
}

// A segment's queries as they stand in memory: head 8 n + g, dims DP/4 c ...
template <int DP, int ROWS>
__device__ __forceinline__ void fetch_query(uint4 (&raw)[ROWS / 8][DP / 32], const Args& a, int r, int head,
                                            int rg, int lane) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int n = 0; n < ROWS / 8; ++n) {
    const int row = rg * ROWS + 8 * n + g, d0 = DP / 4 * c;
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + r * a.q_row +
                        static_cast<int64_t>(head * a.group + row) * a.q_head + d0;
#pragma unroll
    for (int j = 0; j < DP / 32; ++j)
      raw[n][j] = row < a.group && d0 + 8 * j < a.dim ? __ldg(reinterpret_cast<const uint4*>(q + 8 * j))
                                                      : make_uint4(0, 0, 0, 0);
  }
}

template <int DP, int ROWS, bool E4M3>
__device__ __forceinline__ void take_query(State<DP, ROWS>& s, const uint4 (&raw)[ROWS / 8][DP / 32],
                                           const Args& a, int lane) {
  constexpr int N = ROWS / 8;
  const int c = lane & 3;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float x[DP / 4];
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < DP / 32; ++j) {
      const uint4 w = raw[n][j];
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 v;
        if (a.bf16)
          v = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
        else
          v = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[8 * j + 2 * i] = v.x;
        x[8 * j + 2 * i + 1] = v.y;
        most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
      }
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // The largest comes to [2^14, 2^15): the row's others have fp16's whole range below it.
    const int e = max(static_cast<int>(__float_as_uint(most) >> 23) - 141, -127);
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    // (2^(e + 8) and 2^-8: 2^e itself may be subnormal)
    const float rf =
        a.scale_log2 * __uint_as_float(static_cast<uint32_t>(135 + e) << 23) * (E4M3 ? 0x1p-8f : 0x1p-8f * kI8Query);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const __half2 lo = __floats2half2_rn(x[4 * i] * down, x[4 * i + 1] * down);
      const __half2 hi = __floats2half2_rn(x[4 * i + 2] * down, x[4 * i + 3] * down);
      s.q[n][i][0] = *reinterpret_cast<const uint32_t*>(&lo);
      s.q[n][i][1] = *reinterpret_cast<const uint32_t*>(&hi);
      const float2 fl = __half22float2(lo), fh = __half22float2(hi);
      sum += (fl.x + fl.y) + (fh.x + fh.y);
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s.rf[n][h] = __shfl_sync(0xffffffffu, rf, (2 * c + h) * 4);
      const float t = __shfl_sync(0xffffffffu, sum, (2 * c + h) * 4);
      s.start[n][h] = E4M3 ? 0.f : -kI8Offset * t;
    }
  }
}

__device__ __forceinline__ void store_out(const Args& a, int64_t at, float v) {
  if (a.bf16)
    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(a.out)[at] = __float2half_rn(v);
}

// o 2^shift / l; zeros where no token was seen, NaN where the sum is NaN.  The
// power in two steps: it alone may pass fp32's range, the result not.
__device__ __forceinline__ float quotient(float o, float shift, float l) {
  const float half = exp2_fast(0.5f * shift);
  return l > 0.f ? o * half / l * half : (l == 0.f ? 0.f : l);
}

// Tiles before each request: every thread sums a run of requests, the runs'
// sums are scanned.  Returns the total; *run is the sum before this thread's
// run, *lo and *hi the run.
template <int TILE, int THREADS>
__device__ __forceinline__ int scan_tiles(const Args& a, int* warp_sum, int* lo, int* hi, int* run) {
  const int per = (a.requests + THREADS - 1) / THREADS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  *lo = min(a.requests, static_cast<int>(threadIdx.x) * per);
  *hi = min(a.requests, *lo + per);
  int mine = 0;
  for (int r = *lo; r < *hi; ++r) mine += tiles_of<TILE>(a, r);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  *run = before + incl - mine;
  return total;
}

// The segments of a CTA's range of tiles, in order: tiles t0 .. t1 of one
// request and (virtual) head.
template <int TILE>
struct Segments {
  int64_t u, end;
  int r, before;          // request, tiles before it
  int heads;
  int len, tiles, head, t0, t1;
  __device__ __forceinline__ bool next(const Args& a) {
    if (u >= end) return false;
    while (true) {
      len = length_of(a, r);
      tiles = (len + TILE - 1) / TILE;
      if (u < static_cast<int64_t>(before + tiles) * heads) break;
      before += tiles;
      ++r;
    }
    const int64_t in = u - static_cast<int64_t>(before) * heads;
    head = static_cast<int>(in / tiles);
    t0 = static_cast<int>(in % tiles);
    t1 = static_cast<int>(min(static_cast<int64_t>(tiles), t0 + (end - u)));
    u += t1 - t0;
    return true;
  }
};

__device__ __forceinline__ void fail(int* err, volatile int* abort, int code) {
  atomicCAS(err, 0, code);
  *abort = 1;
}

template <int DP, int ROWS, bool E4M3>
__global__ void __launch_bounds__(Smem<DP, ROWS>::kThreads, Smem<DP, ROWS>::kCtas)
    cache_attention_kernel(const __grid_constant__ CUtensorMap map_k,
                           const __grid_constant__ CUtensorMap map_v, const Args a) {
  using L = Smem<DP, ROWS>;
  constexpr int N = ROWS / 8, kWarps = L::kWarps;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float2* scales = reinterpret_cast<float2*>(smem + L::kOffScales);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
  uint64_t* empty = full + L::kStages;
  int* misc = reinterpret_cast<int*>(smem + L::kOffMisc);
  volatile int* abort_flag = misc;
  int* warp_sum = misc + 1;              // [kThreads / 32]
  int* start = misc + 8;                 // request, tiles before it
  float* sm_m = reinterpret_cast<float*>(smem + L::kOffJoin);
  float* sm_l = sm_m + kWarps * ROWS;
  float* sm_b = sm_l + kWarps * ROWS;
  float* sm_o = reinterpret_cast<float*>(smem + L::kOffO);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  ptx::griddep_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      ptx::mbar_init(&full[i], 1);
      ptx::mbar_init(&empty[i], kWarps);
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }

  int lo, hi, run;
  const int total = scan_tiles<L::kTile, L::kThreads>(a, warp_sum, &lo, &hi, &run);
  Segments<L::kTile> seg;
  seg.heads = a.kv_heads * a.row_groups;
  const int64_t units = static_cast<int64_t>(total) * seg.heads;
  const int64_t share = (units + a.grid - 1) / a.grid;
  seg.u = blockIdx.x * share;
  seg.end = min(seg.u + share, units);
  if (blockIdx.x == 0) {
    int p = run;
    for (int r = lo; r < hi; ++r) {
      a.prefix[r] = p;
      p += tiles_of<L::kTile>(a, r);
    }
    if (tid == 0) a.prefix[a.requests] = total;
  }
  if (seg.u >= seg.end) return;
  {
    int p = run;
    for (int r = lo; r < hi; ++r) {
      const int t = tiles_of<L::kTile>(a, r);
      if (seg.u >= static_cast<int64_t>(p) * seg.heads &&
          seg.u < static_cast<int64_t>(p + t) * seg.heads) {
        start[0] = r;
        start[1] = p;
      }
      p += t;
    }
  }
  __syncthreads();
  seg.r = start[0];
  seg.before = start[1];

  if (warp == kWarps) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      ptx::prefetch_tmap(&map_k);
      ptx::prefetch_tmap(&map_v);
    }
    uint32_t n = 0;                      // stages filled
    bool ok = true;
    int had = -1;                        // request and first tile of the ids in `id`
    int had_tile = 0, id = -1;
    const int boxes = L::kTile / a.box_rows;     // of a stage
    constexpr int kBatch = 32 / L::kPieces;      // stages whose blocks the lanes hold
    const int box_pieces = a.box_rows / 16;
    const int box_bytes = a.box_rows * DP;
    while (ok && seg.next(a)) {
      const int32_t* row = a.table + seg.r * a.ld;
      const int head = seg.head / a.row_groups;
      float ks = 0.f, vs = 0.f;
      for (int t = seg.t0; t < seg.t1 && ok; ++t) {
        const int slot = n % L::kStages;
        if (t == seg.t0 || t - had_tile >= kBatch) {
          // Several stages' blocks and scales at a time, one 16-token piece a lane.
          if (had != seg.r || t < had_tile || t - had_tile >= kBatch) {
            had = seg.r;
            had_tile = t;
            const int64_t token = static_cast<int64_t>(t) * L::kTile + 16 * lane;
            id = token < seg.len ? __ldg(row + (token >> a.lg_block)) : -1;
            if (static_cast<uint32_t>(id) >= a.num_blocks) id = -1;
          }
          ks = vs = 0.f;
          if (id >= 0) {
            ks = __ldg(a.k_scale + static_cast<int64_t>(id) * a.kv_heads + head) * (E4M3 ? 1.f : kI8Scale);
            vs = __ldg(a.v_scale + static_cast<int64_t>(id) * a.kv_heads + head);
          }
        }
        const bool come =
            ptx::mbar_wait_suspended(&empty[slot], ((n / L::kStages) & 1) ^ 1, abort_flag, a.wait_limit_ns);
        if (!__all_sync(0xffffffffu, come)) {
          if (lane == 0) fail(a.err, abort_flag, kErrEmpty);
          ok = false;
          break;
        }
        const int first = (t - had_tile) * L::kPieces;   // lane of the stage's first piece
        const int box_id = __shfl_sync(0xffffffffu, id, (first + lane * box_pieces) & 31);
        const bool load = lane < boxes && box_id >= 0;
        const unsigned loads = __ballot_sync(0xffffffffu, load);
        if (lane == 0) ptx::mbar_expect_tx(&full[slot], __popc(loads) * 2 * box_bytes);
        __syncwarp();
        if (load) {
          uint8_t* to = smem + slot * L::kStageBytes + lane * box_bytes;
          const int off = (t * L::kTile + lane * a.box_rows) & ((1 << a.lg_block) - 1);
          const int y = ((box_id * a.kv_heads + head) << a.lg_block) + off;
          ptx::tma_load_2d(to, &map_k, &full[slot], 0, y);
          ptx::tma_load_2d(to + L::kSideBytes, &map_v, &full[slot], 0, y);
        }
        // The scales, which may still be on their way, complete the stage.
        if (lane >= first && lane < first + L::kPieces)
          // A block outside the cache leaves its tokens out.  (kNoBlock is one of the NaN: a scale that
          // is NaN goes on as another one.)
          scales[slot * L::kPieces + lane - first] =
              make_float2(id >= 0 ? (ks == ks ? ks : NAN) : __uint_as_float(kNoBlock), vs);
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&full[slot]);
        __syncwarp();
        ++n;
      }
    }
    // Every load has landed before the CTA may leave (at once, but after a failure).
    volatile int never = 0;
    for (uint32_t e = n > L::kStages ? n - L::kStages : 0; e < n; ++e)
      ptx::mbar_wait_suspended(&full[e % L::kStages], (e / L::kStages) & 1, &never, kDrainLimitNs);
    return;
  }

  // -------------------------------------------------------------- consumers
  const int g = lane >> 2, c = lane & 3;
  uint32_t n = 0;
  bool first = true;
  // With rows of 64 bytes the next segment's queries are fetched before this one is joined (48
  // ragged requests: 44.3 -> 42.2 us when it was taken); with 128 the registers for it are not there (60.5 -> 64.0).
  constexpr bool kAhead = DP == 64;
  uint4 raw[N][DP / 32];
  auto fetch = [&]() {
    fetch_query<DP, ROWS>(raw, a, seg.r, seg.head / a.row_groups, seg.head % a.row_groups, lane);
  };
  bool more = seg.next(a);
  if (more && kAhead) fetch();
  while (more) {
    const int head = seg.head / a.row_groups, rg = seg.head % a.row_groups;
    const int r = seg.r, len = seg.len, t0 = seg.t0, t1 = seg.t1;
    const bool whole = t0 == 0 && t1 == seg.tiles;
    State<DP, ROWS> s;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) s.m[i][h] = s.b[i][h] = kNothing, s.l[i][h] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) s.o[i][t][0] = s.o[i][t][1] = s.o[i][t][2] = s.o[i][t][3] = 0.f;
    if (!kAhead) fetch();
    take_query<DP, ROWS, E4M3>(s, raw, a, lane);
    for (int t = t0; t < t1; ++t, ++n) {
      const int slot = n % L::kStages;
      // (one answer for the warp: it stays converged; after a failure the waits to come fail at once)
      const bool come =
          ptx::mbar_wait_suspended(&full[slot], (n / L::kStages) & 1, abort_flag, a.wait_limit_ns);
      if (!__all_sync(0xffffffffu, come)) {
        if (lane == 0) fail(a.err, abort_flag, kErrFull);
        break;
      }
      constexpr int P = pieces(DP);
      const int left = len - t * L::kTile - warp * 16 * P;
      float2 sc[P];
#pragma unroll
      for (int x = 0; x < P; ++x) sc[x] = scales[slot * L::kPieces + warp * P + x];
      if (left > 0) {
        const uint8_t* k = smem + slot * L::kStageBytes + warp * 16 * P * DP;
        compute_pieces<DP, ROWS, E4M3>(s, k, k + L::kSideBytes, sc, left, lane);
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&empty[slot]);
    }

    more = seg.next(a);
    if (more && kAhead) fetch();

    // Join the warps.  Sums and outputs keep their own units, 2^m and 2^b, through both joins: 2^(b - m)
    // has no place in 32 bits where blocks that weigh nothing lead by 2^126.
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int y = warp * ROWS + 8 * i + 2 * c + h;
        float l = s.l[i][h];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (g == 0) {
          sm_m[y] = s.m[i][h];
          sm_l[y] = l;
          sm_b[y] = s.b[i][h];
        }
#pragma unroll
        for (int t = 0; t < DP / 16; t += 2)
          *reinterpret_cast<float4*>(sm_o + y * DP + DP / 8 * g + 2 * t) =
              make_float4(s.o[i][t][h], s.o[i][t][2 + h], s.o[i][t + 1][h], s.o[i][t + 1][2 + h]);
      }
    asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (first ? 0 : 1);
    const int rows = min(ROWS, a.group - rg * ROWS);
    // Four dims a thread (2 x, 2 x + 1 and those DP / 2 behind): the units' powers once for all of them.
    for (int i = tid; i < rows * (DP / 4); i += kWarps * 32) {
      const int y = i / (DP / 4), d = 2 * (i % (DP / 4));
      float m = -INFINITY, b = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        m = fmaxf(m, sm_m[w * ROWS + y]);
        b = fmaxf(b, sm_b[w * ROWS + y]);
      }
      float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float e = exp2_fast(sm_b[w * ROWS + y] - b);
        l += exp2_fast(sm_m[w * ROWS + y] - m) * sm_l[w * ROWS + y];
        const float2* from = reinterpret_cast<const float2*>(sm_o + (w * ROWS + y) * DP + d);
        const float2 lo = from[0], hi = from[DP / 4];
        o[0] += e * lo.x, o[1] += e * lo.y, o[2] += e * hi.x, o[3] += e * hi.y;
      }
      if (whole) {
        const int64_t j =
            static_cast<int64_t>(r) * a.kv_heads * a.group + head * a.group + rg * ROWS + y;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int at = d + (x & 1) + (x >> 1) * (DP / 2);
          if (at < a.dim) store_out(a, j * a.dim + at, quotient(o[x], b - m, l));
        }
        if (d == 0 && a.lse) a.lse[j] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      } else {
        float2* to = reinterpret_cast<float2*>(a.part_o + (slot * ROWS + y) * DP + d);
        to[0] = make_float2(o[0], o[1]);
        to[DP / 4] = make_float2(o[2], o[3]);
        if (d == 0) {
          a.part_m[slot * ROWS + y] = m;
          a.part_l[slot * ROWS + y] = l;
          a.part_b[slot * ROWS + y] = b;
        }
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
    first = false;
  }
}

// Joins the parts of what the cuts divided, and writes the zeros of requests
// without tokens.  SPREAD (few heads, so many parts each): a CTA for each
// query head, its warps take every warps-th part.  Else a CTA for each
// request and virtual head, and a warp for each of its rows.
template <int DP, int ROWS, bool SPREAD>
__global__ void cache_join_kernel(const Args a) {
  extern __shared__ float sm[];          // SPREAD: [warps][DP + 1]
  ptx::griddep_wait();
  const int heads = a.kv_heads * a.row_groups;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int all = SPREAD ? a.kv_heads * a.group : heads;
  const int r = blockIdx.x / all, j = blockIdx.x % all;
  const int head = SPREAD ? j / a.group : j / a.row_groups;
  const int rg = SPREAD ? j % a.group / ROWS : j % a.row_groups;
  const int before = a.prefix[r], tiles = a.prefix[r + 1] - before;
  const int64_t units = static_cast<int64_t>(a.prefix[a.requests]) * heads;
  const int64_t share = (units + a.grid - 1) / a.grid;
  const int64_t u0 = static_cast<int64_t>(before) * heads +
                     static_cast<int64_t>(head * a.row_groups + rg) * tiles;
  int c0 = 0, c1 = 0;
  bool late = false;                     // the first part is not its CTA's first segment
  if (tiles > 0) {
    c0 = static_cast<int>(u0 / share), c1 = static_cast<int>((u0 + tiles - 1) / share);
    late = u0 != c0 * share;
    if (c0 == c1) return;                // one CTA did it all
  }
  const int first = SPREAD ? warp : 0, step = SPREAD ? warps : 1;
  const int last_row = SPREAD ? j % a.group % ROWS + 1 : min(ROWS, a.group - rg * ROWS);
  for (int y = SPREAD ? last_row - 1 : warp; y < last_row; y += SPREAD ? ROWS : warps) {
    const int64_t at = static_cast<int64_t>(r) * a.kv_heads * a.group + head * a.group + rg * ROWS + y;
    auto slot_of = [&](int c) { return (2ll * c + (c == c0 && late ? 1 : 0)) * ROWS + y; };
    float m = -INFINITY, b = -INFINITY, l = 0.f, acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] = 0.f;
    if (tiles > 0) {
      for (int c = c0 + lane; c <= c1; c += 32) {
        m = fmaxf(m, a.part_m[slot_of(c)]);
        b = fmaxf(b, a.part_b[slot_of(c)]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, o));
      }
      // A warp's parts: their weights side by side in the lanes, their rows kJoin at a time.
      for (int base = c0 + first; base <= c1; base += 32 * step) {
        const int own = base + lane * step;
        float e = 0.f;
        if (own <= c1) {
          e = exp2_fast(a.part_b[slot_of(own)] - b);
          l += exp2_fast(a.part_m[slot_of(own)] - m) * a.part_l[slot_of(own)];
        }
        const int n = min(32, (c1 - base) / step + 1);
        for (int k = 0; k < n; k += kJoin) {
          float v[kJoin][DP / 32];
#pragma unroll
          for (int x = 0; x < kJoin; ++x) {
            const int64_t slot = slot_of(base + (k + x) * step);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
              v[x][i] = k + x < n ? a.part_o[slot * DP + lane + 32 * i] : 0.f;
          }
#pragma unroll
          for (int x = 0; x < kJoin; ++x) {
            const float w = __shfl_sync(0xffffffffu, e, (k + x) & 31);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) acc[i] += (k + x < n ? w : 0.f) * v[x][i];
          }
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    }
    if (SPREAD) {
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) sm[warp * (DP + 1) + lane + 32 * i] = acc[i];
      if (lane == 0) sm[warp * (DP + 1) + DP] = l;
      __syncthreads();
      if (warp > 0) return;
      l = 0.f;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) acc[i] = 0.f;
      for (int w = 0; w < warps; ++w) {
        l += sm[w * (DP + 1) + DP];
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) acc[i] += sm[w * (DP + 1) + lane + 32 * i];
      }
    }
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
      const int d = lane + 32 * i;
      if (d < a.dim) store_out(a, at * a.dim + d, quotient(acc[i], b - m, l));
    }
    if (lane == 0 && a.lse) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
}

int check(const b2g_cache_attention_desc* d) {
  if (!d || d->requests < 0 || d->heads < 0 || d->kv_heads < 0 || d->dim <= 0 ||
      d->num_blocks < 0 || d->table_width < 0 || d->table_ld < d->table_width ||
      (d->dtype != B2G_F16 && d->dtype != B2G_BF16) ||
      (d->codes != B2G_I8 && d->codes != B2G_E4M3) || !(d->scale >= 0.f && std::isfinite(d->scale)))
    return B2G_ERR_INVALID_ARG;
  if (d->heads > 0 && (d->kv_heads == 0 || d->heads % d->kv_heads)) return B2G_ERR_INVALID_ARG;
  if (d->block_size < 16 || d->block_size > 256 || (d->block_size & (d->block_size - 1)) ||
      d->dim % 16 || d->dim > 128)
    return B2G_ERR_UNSUPPORTED;
  // (each factor before the products that it stands in)
  if (d->num_blocks > 0x7fffffff || d->heads > (1 << 16) || d->kv_heads > (1 << 16) ||
      d->requests > (1 << 20) || d->table_width > 0x7fffffff ||
      d->table_width * d->block_size > 0x7fffff00 ||
      d->num_blocks * d->kv_heads * d->block_size > 0x7fffffff || d->requests * d->heads > 0x7fffffff)
    return B2G_ERR_UNSUPPORTED;
  // The kernel counts the tiles of all requests in 32 bits: requests that share blocks, or wrong
  // lengths, may fill whole rows of a wide table.
  const int rows = d->kv_heads > 0 && d->heads / d->kv_heads > 8 ? 16 : 8;
  const int64_t tiles = cdiv(d->table_width * d->block_size, tile_tokens(d->dim <= 64 ? 64 : 128, rows));
  if (d->requests * tiles > 0x7fffffff) return B2G_ERR_UNSUPPORTED;
  return B2G_OK;
}

struct Layout {
  int rows, dp, row_groups, grid;
  int64_t off_m, off_l, off_b, off_o, bytes;
};

Layout layout_of(const b2g_cache_attention_desc* d, int sms) {
  Layout w;
  const int64_t group = d->heads / d->kv_heads;
  w.rows = group <= 8 ? 8 : 16;
  w.dp = d->dim <= 64 ? 64 : 128;
  w.row_groups = static_cast<int>(cdiv(group, w.rows));
  const int64_t most = d->requests * d->kv_heads * w.row_groups *
                       std::max<int64_t>(cdiv(d->table_width * d->block_size, tile_tokens(w.dp, w.rows)), 1);
  const int ctas = w.dp == 64 ? (w.rows == 8 ? Smem<64, 8>::kCtas : Smem<64, 16>::kCtas)
                              : (w.rows == 8 ? Smem<128, 8>::kCtas : Smem<128, 16>::kCtas);
  w.grid = static_cast<int>(std::min<int64_t>(std::max<int64_t>(most, 1), static_cast<int64_t>(sms) * ctas));
  auto pad = [](int64_t n) { return cdiv(n, 256) * 256; };
  w.off_m = pad((d->requests + 1) * 4);
  w.off_l = w.off_m + pad(2ll * w.grid * w.rows * 4);
  w.off_b = w.off_l + pad(2ll * w.grid * w.rows * 4);
  w.off_o = w.off_b + pad(2ll * w.grid * w.rows * 4);
  w.bytes = w.off_o + 2ll * w.grid * w.rows * w.dp * 4;
  return w;
}

// The codes of a cache as rows of dim bytes; a box is box_rows rows of DP
// bytes (zeros past dim) in the swizzle of that width.
bool make_map(CUtensorMap* map, const void* base, int64_t dim, int64_t rows, int dp, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(dim)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(dp), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  return b2g::encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, estr,
                           dp == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

template <int DP, int ROWS, bool E4M3>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, cudaStream_t stream) {
  using L = Smem<DP, ROWS>;
  static thread_local int configured = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured != dev) {
    if (cudaFuncSetAttribute(cache_attention_kernel<DP, ROWS, E4M3>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes) != cudaSuccess)
      return B2G_ERR_LAUNCH;
    configured = dev;
  }
  // The join may be set up while the kernel before it runs, and waits for it before it reads.  (Not
  // so the attention itself: started among the join's CTAs of the call before, its own can end up
  // unevenly spread, 16 requests of 20000 tokens then took 152 us for 111.)
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.grid), 1, 1);
  cfg.blockDim = dim3(L::kThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (cudaLaunchKernelEx(&cfg, cache_attention_kernel<DP, ROWS, E4M3>, mk, mv, a) != cudaSuccess)
    return B2G_ERR_LAUNCH;
  // Parts of a head, were all lengths alike: from 8 on they are spread over 4 warps, from 32 over 16.
  const int64_t heads = static_cast<int64_t>(a.requests) * a.kv_heads * a.row_groups;
  const bool spread = a.grid > 8 * heads;
  const int warps = a.grid > 32 * heads ? 16 : 4;
  cfg.numAttrs = b2g::pdl_enabled() ? 1 : 0;
  cfg.gridDim = dim3(static_cast<unsigned>(spread ? static_cast<int64_t>(a.requests) * a.kv_heads * a.group : heads), 1, 1);
  cfg.blockDim = dim3(warps * 32, 1, 1);
  cfg.dynamicSmemBytes = spread ? warps * (DP + 1) * sizeof(float) : 0;
  auto* join = spread ? cache_join_kernel<DP, ROWS, true> : cache_join_kernel<DP, ROWS, false>;
  if (cudaLaunchKernelEx(&cfg, join, a) != cudaSuccess) return B2G_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? B2G_OK : B2G_ERR_LAUNCH;
}

}  // namespace

extern "C" int64_t b2g_cache_attention_workspace_bytes(const b2g_cache_attention_desc* d) {
  if (check(d) != B2G_OK) return -1;
  if (d->requests == 0 || d->heads == 0) return 0;
  b2g::Device dev;
  return layout_of(d, b2g::current_device(&dev) == B2G_OK ? dev.num_sms : 148).bytes;
}

extern "C" int b2g_cache_attention(const b2g_cache_attention_desc* d, b2g_stream_t stream_handle) {
  int rc = check(d);
  if (rc != B2G_OK) return rc;
  if (d->requests == 0 || d->heads == 0) return B2G_OK;
  if (!d->q || !d->out || !d->seq_lens || (d->table_width > 0 && !d->block_table) ||
      (d->num_blocks > 0 && (!d->k_cache || !d->v_cache || !d->k_scale || !d->v_scale)))
    return B2G_ERR_INVALID_ARG;
  if (d->q_row_stride % 8 || d->q_head_stride % 8) return B2G_ERR_UNSUPPORTED;
  for (const void* p : {d->q, d->k_cache, d->v_cache})
    if (reinterpret_cast<uintptr_t>(p) % 16) return B2G_ERR_UNSUPPORTED;
  b2g::Device dev;
  rc = b2g::current_device(&dev);
  if (rc != B2G_OK) return rc;
  const Layout w = layout_of(d, dev.num_sms);
  if (!d->workspace || d->workspace_bytes < w.bytes || reinterpret_cast<uintptr_t>(d->workspace) % 16)
    return B2G_ERR_WORKSPACE;
  Args a;
  a.q = d->q;
  a.q_row = d->q_row_stride;
  a.q_head = d->q_head_stride;
  a.k_scale = d->k_scale;
  a.v_scale = d->v_scale;
  a.table = d->block_table;
  // Without a block there is no token either.
  a.width = d->num_blocks > 0 ? d->table_width : 0;
  a.ld = d->table_ld;
  a.seq_lens = d->seq_lens;
  a.requests = static_cast<int>(d->requests);
  a.kv_heads = static_cast<int>(d->kv_heads);
  a.group = static_cast<int>(d->heads / d->kv_heads);
  a.row_groups = w.row_groups;
  a.dim = static_cast<int>(d->dim);
  a.lg_block = 0;
  while ((1 << a.lg_block) < d->block_size) ++a.lg_block;
  a.bf16 = d->dtype == B2G_BF16;
  a.num_blocks = d->num_blocks;
  a.scale_log2 = (d->scale > 0.f ? d->scale : 1.f / std::sqrt(static_cast<float>(d->dim))) *
                 1.4426950408889634f;
  a.out = d->out;
  a.lse = d->lse;
  char* ws = static_cast<char*>(d->workspace);
  a.prefix = reinterpret_cast<int*>(ws);
  a.part_m = reinterpret_cast<float*>(ws + w.off_m);
  a.part_l = reinterpret_cast<float*>(ws + w.off_l);
  a.part_b = reinterpret_cast<float*>(ws + w.off_b);
  a.part_o = reinterpret_cast<float*>(ws + w.off_o);
  a.grid = w.grid;
  a.wait_limit_ns = b2g::current_wait_limit_ns();
  a.err = dev.error_word;
  // (a stage of 80 tokens is a whole number of 16 rows only)
  a.box_rows = consumers(w.dp, w.rows) == 4
                   ? static_cast<int>(std::min<int64_t>(d->block_size, tile_tokens(w.dp, w.rows)))
                   : 16;
  CUtensorMap mk = {}, mv = {};
  const int64_t cache_rows = d->num_blocks * d->kv_heads * d->block_size;
  if (d->num_blocks > 0 && (!make_map(&mk, d->k_cache, d->dim, cache_rows, w.dp, a.box_rows) ||
                            !make_map(&mv, d->v_cache, d->dim, cache_rows, w.dp, a.box_rows)))
    return B2G_ERR_UNSUPPORTED;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  const bool e4 = d->codes == B2G_E4M3;
  if (w.dp == 64)
    return w.rows == 8 ? (e4 ? launch<64, 8, true>(mk, mv, a, stream) : launch<64, 8, false>(mk, mv, a, stream))
                       : (e4 ? launch<64, 16, true>(mk, mv, a, stream) : launch<64, 16, false>(mk, mv, a, stream));
  return w.rows == 8 ? (e4 ? launch<128, 8, true>(mk, mv, a, stream) : launch<128, 8, false>(mk, mv, a, stream))
                     : (e4 ? launch<128, 16, true>(mk, mv, a, stream) : launch<128, 16, false>(mk, mv, a, stream));
}
