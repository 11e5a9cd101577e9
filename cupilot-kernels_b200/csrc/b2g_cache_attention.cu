// b2g_cache_attention.cu — one query token per request over the paged 8-bit
// cache (b2g_cache_attention).
//
// out[j] = sum_n exp(z_n - max z) V_n / sum_n exp(z_n - max z),
// z_n = scale * q_j . K_n, one pass over K and V with the running maximum and
// sum.  With c the codes and a scale for each block and head, z_n = (scale *
// kscale) * (q . c_n), and the products run on the codes: int8 and e4m3 are
// exact in fp16, so a warp's m16n8k16 product takes q (16 rows: the query
// heads that share the kv head) against 16 tokens' codes widened in
// registers.  q is brought to [-1, 1] by a power of two (exact in fp16, where
// the row's small values may go subnormal), the weights are <= 2^12 in fp16,
// sums, maxima and the output are fp32.
//
// Bound by memory: 2 * dim bytes a token and kv head, read once by 16-byte
// loads into registers one step ahead of their use.  The (request, head,
// 64-token) tiles are laid end to end and cut into equal ranges, one a CTA,
// so ragged lengths fill the GPU evenly; what a cut divides is joined by a
// second small kernel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/b2g_serving.h"
#include "b2g_internal.h"
#include "ptx_sm100.cuh"

namespace {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 16 * kWarps;     // tokens of a CTA's step, 16 a warp
// By the registers that a warp's state and its two steps take.
constexpr int ctas_per_sm(int dp, int rows) { return dp == 64 ? (rows == 8 ? 5 : 4) : (rows == 8 ? 3 : 2); }
constexpr float kGrow = 8.f;           // a maximum may be passed by 2^8 before the sums are rescaled

struct Args {
  const void* q;
  int64_t q_row, q_head;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int32_t* table;
  int64_t width, ld;
  const int32_t* seq_lens;
  int requests, kv_heads, group, row_groups, dim, lg_block, bf16;
  int64_t num_blocks;
  float scale_log2;
  void* out;
  float* lse;
  // workspace: tiles before each request (requests + 1), then the partial results, two a CTA
  int* prefix;
  float* part_m;
  float* part_l;
  float* part_o;
  int grid;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ int length_of(const Args& a, int r) {
  const int64_t n = a.seq_lens[r], most = a.width << a.lg_block;
  return static_cast<int>(n < 0 ? 0 : (n < most ? n : most));
}
__device__ __forceinline__ int tiles_of(const Args& a, int r) {
  return (length_of(a, r) + kTile - 1) / kTile;
}

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with rows 8-15 of A zero: their sums are neither kept nor read.
__device__ __forceinline__ void mma_16816(float (&d)[2], uint32_t a0, uint32_t, uint32_t a2,
                                          uint32_t, uint32_t b0, uint32_t b1) {
  asm("{\n\t.reg .f32 x, y;\n\t"
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,x,y}, {%2,%3,%4,%3}, {%5,%6}, "
      "{%0,%1,%7,%7};\n\t}"
      : "+f"(d[0]), "+f"(d[1])
      : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1), "f"(0.f));
}

// Four codes to two fp16 pairs.  int8: with the sign bit flipped a byte u is
// 128 + c, and the fp16 with bits 0x6400 | u is 1024 + u, exactly.
template <bool E4M3>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));   // 1152
    uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
    __half2 hx = __hsub2(*reinterpret_cast<__half2*>(&x), off);
    __half2 hy = __hsub2(*reinterpret_cast<__half2*>(&y), off);
    lo = *reinterpret_cast<uint32_t*>(&hx);
    hi = *reinterpret_cast<uint32_t*>(&hy);
  }
}

__device__ __forceinline__ uint4 load16(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load8(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// One warp's 16 tokens of one head.  Lane (g, c) = (lane / 4, lane % 4) holds
// of K, for tokens g and 8 + g, the dims 64 j + 16 c .. + 15 (the k index of
// a product may be any order of the dims that q has too), and of V, for the
// tokens 2c, 2c+1, 2c+8, 2c+9 that it needs as pairs, DP / 8 dims from
// DP / 8 * g (its n index, in any order that the output is read back in).
template <int DP>
struct Step {
  uint4 k[2][DP / 64];
  uint32_t v[4][DP / 32];
  float ks, vs;
  bool bad;
};

template <int DP>
__device__ __forceinline__ void load_step(Step<DP>& f, const Args& a, int head, int id, int off,
                                          int lane) {
  const int g = lane >> 2, c = lane & 3;
  f.bad = static_cast<uint32_t>(id) >= a.num_blocks;
  const int64_t bh = static_cast<int64_t>(f.bad ? 0 : id) * a.kv_heads + head;
  const int64_t at = ((bh << a.lg_block) + off) * a.dim;
  const uint8_t* kp = a.k_cache + at;
  const uint8_t* vp = a.v_cache + at;
  f.ks = __ldg(a.k_scale + bh);
  f.vs = __ldg(a.v_scale + bh);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) {
      const int d = 64 * j + 16 * c;
      f.k[t][j] = d < a.dim ? load16(kp + (8 * t + g) * a.dim + d) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int tok = 2 * c + (t & 1) + (t >> 1) * 8;
    const int d = DP / 8 * g;
    const uint8_t* p = vp + tok * a.dim + d;
    if (DP == 128) {
      const uint4 w = d < a.dim ? load16(p) : make_uint4(0, 0, 0, 0);
      f.v[t][0] = w.x, f.v[t][1] = w.y, f.v[t][DP / 32 - 2] = w.z, f.v[t][DP / 32 - 1] = w.w;
    } else {
      const uint2 w = d < a.dim ? load8(p) : make_uint2(0, 0);
      f.v[t][0] = w.x, f.v[t][1] = w.y;
    }
  }
}

// The warp's running state: row g (and 8 + g with ROWS == 16).
template <int DP, int ROWS>
struct State {
  static constexpr int H = ROWS / 8;
  uint32_t q[DP / 16][2 * H];
  float rf[H];        // scale * log2(e) * the power of two that q was divided by
  float m[H], l[H];   // maximum so far (log2 units), this lane's part of the sum
  float unit, per;    // o is in units of `unit` (a block's value scale), per = 1 / unit
  float o[DP / 8][2 * H];
};

template <int DP, int ROWS, bool E4M3>
__device__ __forceinline__ void compute_step(State<DP, ROWS>& s, Step<DP>& f, int left, int lane) {
  constexpr int H = ROWS / 8;
  const int c = lane & 3;
  float z[2][2 * H];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int i = 0; i < 2 * H; ++i) z[t][i] = 0.f;
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) {
      const uint32_t w[4] = {f.k[t][j].x, f.k[t][j].y, f.k[t][j].z, f.k[t][j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t b0, b1;
        widen4<E4M3>(w[i], b0, b1);
        const uint32_t* qa = s.q[4 * j + i];
        mma_16816(z[t], qa[0], H == 2 ? qa[H - 1] : 0u, qa[H], H == 2 ? qa[2 * H - 1] : 0u, b0, b1);
      }
    }
  }
  if (left < 16 || f.bad) {            // the last tokens, or a block outside the cache
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2 * H; ++i)
        if (f.bad || 8 * t + 2 * c + (i & 1) >= left) z[t][i] = -INFINITY;
    // What is not a token's may hold anything: 0 * NaN must not reach the sums.
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (f.bad || 2 * c + (t & 1) + (t >> 1) * 8 >= left)
#pragma unroll
        for (int j = 0; j < DP / 32; ++j) f.v[t][j] = 0;
    if (f.bad) f.vs = 0.f, f.ks = 0.f;
  }
  float top[H];
  bool grow = f.vs > 16.f * s.unit;
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const float r = s.rf[h] * f.ks;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float& x = z[t][2 * h + i];
        x = x == -INFINITY ? x : x * r;
      }
    top[h] = fmaxf(fmaxf(z[0][2 * h], z[0][2 * h + 1]), fmaxf(z[1][2 * h], z[1][2 * h + 1]));
    grow |= top[h] > s.m[h] + kGrow;
  }
  if (__any_sync(0xffffffffu, grow)) {
    const float unit = fmaxf(s.unit, f.vs);
    const float ratio = unit > 0.f ? s.unit / unit : 0.f;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      float t = top[h];
      t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
      t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
      t = fmaxf(t, s.m[h]);
      const float corr = s.m[h] == -INFINITY ? 0.f : exp2_fast(s.m[h] - t);
      s.m[h] = t;
      s.l[h] *= corr;
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        s.o[n][2 * h] *= corr * ratio;
        s.o[n][2 * h + 1] *= corr * ratio;
      }
    }
    s.unit = unit;
    s.per = unit > 0.f ? 1.f / unit : 0.f;
  }
  const float w = f.vs * s.per;
  uint32_t p[2][H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const float m = s.m[h] == -INFINITY ? 0.f : s.m[h];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float e0 = exp2_fast(z[t][2 * h] - m), e1 = exp2_fast(z[t][2 * h + 1] - m);
      s.l[h] += e0 + e1;
      const __half2 hv = __floats2half2_rn(e0 * w, e1 * w);
      p[t][h] = *reinterpret_cast<const uint32_t*>(&hv);
    }
  }
  const uint32_t a0 = p[0][0], a1 = H == 2 ? p[0][H - 1] : 0u, a2 = p[1][0],
                 a3 = H == 2 ? p[1][H - 1] : 0u;
#pragma unroll
  for (int j = 0; j < DP / 32; ++j) {
    const uint32_t x01 = __byte_perm(f.v[0][j], f.v[1][j], 0x5140);
    const uint32_t y01 = __byte_perm(f.v[0][j], f.v[1][j], 0x7362);
    const uint32_t x23 = __byte_perm(f.v[2][j], f.v[3][j], 0x5140);
    const uint32_t y23 = __byte_perm(f.v[2][j], f.v[3][j], 0x7362);
    uint32_t b0, b1, b2, b3, c0, c1, c2, c3;
    widen4<E4M3>(x01, b0, b1);
    widen4<E4M3>(y01, b2, b3);
    widen4<E4M3>(x23, c0, c1);
    widen4<E4M3>(y23, c2, c3);
    mma_16816(s.o[4 * j], a0, a1, a2, a3, b0, c0);
    mma_16816(s.o[4 * j + 1], a0, a1, a2, a3, b1, c1);
    mma_16816(s.o[4 * j + 2], a0, a1, a2, a3, b2, c2);
    mma_16816(s.o[4 * j + 3], a0, a1, a2, a3, b3, c3);
  }
}

template <int DP, int ROWS>
__device__ __forceinline__ void load_query(State<DP, ROWS>& s, const Args& a, int r, int head,
                                           int rg, int lane) {
  constexpr int H = ROWS / 8;
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const int row = rg * ROWS + 8 * h + g;
    float x[DP / 4];
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) {
      const int d = 64 * j + 16 * c;
      uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      if (row < a.group && d < a.dim) {
        const uint4* p = reinterpret_cast<const uint4*>(
            static_cast<const uint16_t*>(a.q) + r * a.q_row +
            static_cast<int64_t>(head * a.group + row) * a.q_head + d);
        w[0] = __ldg(p);
        w[1] = __ldg(p + 1);
      }
      const uint32_t u[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float2 v;
        if (a.bf16)
          v = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
        else
          v = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[16 * j + 2 * i] = v.x;
        x[16 * j + 2 * i + 1] = v.y;
        most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
      }
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23) - 126, -126), 126);
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    s.rf[h] = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const __half2 lo = __floats2half2_rn(x[4 * i] * down, x[4 * i + 1] * down);
      const __half2 hi = __floats2half2_rn(x[4 * i + 2] * down, x[4 * i + 3] * down);
      s.q[i][h] = *reinterpret_cast<const uint32_t*>(&lo);
      s.q[i][H + h] = *reinterpret_cast<const uint32_t*>(&hi);
    }
  }
}

__device__ __forceinline__ void store_out(const Args& a, int64_t at, float v) {
  if (a.bf16)
    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(a.out)[at] = __float2half_rn(v);
}

// Tiles before each request: every thread sums a run of requests, the runs'
// sums are scanned.  Returns the total; *run is the sum before this thread's
// run, *lo and *hi the run.
__device__ __forceinline__ int scan_tiles(const Args& a, int* warp_sum, int* lo, int* hi, int* run) {
  const int per = (a.requests + kThreads - 1) / kThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  *lo = min(a.requests, static_cast<int>(threadIdx.x) * per);
  *hi = min(a.requests, *lo + per);
  int mine = 0;
  for (int r = *lo; r < *hi; ++r) mine += tiles_of(a, r);
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
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  *run = before + incl - mine;
  return total;
}

template <int DP, int ROWS, bool E4M3>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(DP, ROWS)) cache_attention_kernel(const Args a) {
  constexpr int H = ROWS / 8;
  __shared__ float sm_o[kWarps][ROWS][DP];
  __shared__ float sm_m[kWarps][ROWS], sm_l[kWarps][ROWS];
  __shared__ int warp_sum[kWarps], start_r, start_p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  b2g::ptx::griddep_launch_dependents();

  int lo, hi, run;
  const int total = scan_tiles(a, warp_sum, &lo, &hi, &run);
  const int heads = a.kv_heads * a.row_groups;
  const int64_t units = static_cast<int64_t>(total) * heads;
  const int64_t share = (units + a.grid - 1) / a.grid;
  int64_t u = blockIdx.x * share;
  const int64_t end = min(u + share, units);
  if (blockIdx.x == 0) {
    int p = run;
    for (int r = lo; r < hi; ++r) {
      a.prefix[r] = p;
      p += tiles_of(a, r);
    }
    if (tid == 0) a.prefix[a.requests] = total;
  }
  if (u >= end) return;
  {
    int p = run;
    for (int r = lo; r < hi; ++r) {
      const int t = tiles_of(a, r);
      if (u >= static_cast<int64_t>(p) * heads && u < static_cast<int64_t>(p + t) * heads) {
        start_r = r;
        start_p = p;
      }
      p += t;
    }
  }
  __syncthreads();
  int r = start_r, p = start_p;
  bool first = true;
  while (u < end) {
    const int len = length_of(a, r), tiles = (len + kTile - 1) / kTile;
    const int64_t base = static_cast<int64_t>(p) * heads;
    if (u >= base + static_cast<int64_t>(tiles) * heads) {
      p += tiles;
      ++r;
      continue;
    }
    const int vh = static_cast<int>((u - base) / tiles);
    const int t0 = static_cast<int>((u - base) % tiles);
    const int t1 = static_cast<int>(min(static_cast<int64_t>(tiles), t0 + (end - u)));
    const int head = vh / a.row_groups, rg = vh % a.row_groups;

    State<DP, ROWS> s;
#pragma unroll
    for (int h = 0; h < H; ++h) s.m[h] = -INFINITY, s.l[h] = 0.f;
    s.unit = s.per = 0.f;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int i = 0; i < 2 * H; ++i) s.o[n][i] = 0.f;

    // This warp's tokens: 16 at t * kTile + warp * 16, t0 <= t < t1.
    const int32_t* row = a.table + r * a.ld;
    const int mask = (1 << a.lg_block) - 1;
    const int w0 = warp * 16;
    const int tend = min(t1, (len - w0 + kTile - 1) / kTile);   // tiles with tokens of this warp
    auto block_at = [&](int t) { return t < tend ? __ldg(row + ((t * kTile + w0) >> a.lg_block)) : 0; };
    Step<DP> f0, f1;
    if (t0 < tend) {
      int id = block_at(t0), next = block_at(t0 + 1);
      load_step<DP>(f0, a, head, id, (t0 * kTile + w0) & mask, lane);
      load_query<DP, ROWS>(s, a, r, head, rg, lane);
      for (int t = t0; t < tend; t += 2) {
        if (t + 1 < tend) load_step<DP>(f1, a, head, next, ((t + 1) * kTile + w0) & mask, lane);
        next = block_at(t + 2);
        compute_step<DP, ROWS, E4M3>(s, f0, len - t * kTile - w0, lane);
        if (t + 1 >= tend) break;
        if (t + 2 < tend) load_step<DP>(f0, a, head, next, ((t + 2) * kTile + w0) & mask, lane);
        next = block_at(t + 3);
        compute_step<DP, ROWS, E4M3>(s, f1, len - (t + 1) * kTile - w0, lane);
      }
    }

    // Join the four warps.
#pragma unroll
    for (int h = 0; h < H; ++h) {
      float l = s.l[h];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (c == 0) {
        sm_m[warp][8 * h + g] = s.m[h];
        sm_l[warp][8 * h + g] = l;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < DP / 8; i += 4)
          *reinterpret_cast<float4*>(&sm_o[warp][8 * h + g][DP / 8 * (2 * c + n) + i]) =
              make_float4(s.o[i][2 * h + n] * s.unit, s.o[i + 1][2 * h + n] * s.unit,
                          s.o[i + 2][2 * h + n] * s.unit, s.o[i + 3][2 * h + n] * s.unit);
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == tiles;
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (first ? 0 : 1);
    const int rows = min(ROWS, a.group - rg * ROWS);
    for (int i = tid; i < rows * DP; i += kThreads) {
      const int y = i / DP, d = i % DP;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sm_m[w][y]);
      float l = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float e = sm_m[w][y] == -INFINITY ? 0.f : exp2_fast(sm_m[w][y] - m);
        l += e * sm_l[w][y];
        o += e * sm_o[w][y][d];
      }
      if (whole) {
        const int64_t j = static_cast<int64_t>(r) * a.kv_heads * a.group + head * a.group + rg * ROWS + y;
        if (d < a.dim) store_out(a, j * a.dim + d, l > 0.f ? o / l : (l == 0.f ? 0.f : l));
        if (d == 0 && a.lse) a.lse[j] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      } else {
        a.part_o[(slot * ROWS + y) * DP + d] = o;
        if (d == 0) {
          a.part_m[slot * ROWS + y] = m;
          a.part_l[slot * ROWS + y] = l;
        }
      }
    }
    __syncthreads();
    u += t1 - t0;
    first = false;
  }
}

// Joins the parts of what the cuts divided, one CTA for each query head; a
// warp takes every warps-th part, a lane DP / 32 dims.  Requests without
// tokens get their zeros here.
template <int DP, int ROWS>
__global__ void cache_join_kernel(const Args a) {
  extern __shared__ float sm[];          // [warps][DP + 1]
  b2g::ptx::griddep_wait();
  const int heads = a.kv_heads * a.row_groups;
  const int j = blockIdx.x % (a.kv_heads * a.group), r = blockIdx.x / (a.kv_heads * a.group);
  const int head = j / a.group, row = j % a.group, rg = row / ROWS, y = row % ROWS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int before = a.prefix[r], tiles = a.prefix[r + 1] - before;
  const int64_t at = static_cast<int64_t>(blockIdx.x);
  if (tiles == 0) {
    for (int d = threadIdx.x; d < a.dim; d += blockDim.x) store_out(a, at * a.dim + d, 0.f);
    if (threadIdx.x == 0 && a.lse) a.lse[at] = -INFINITY;
    return;
  }
  const int64_t units = static_cast<int64_t>(a.prefix[a.requests]) * heads;
  const int64_t share = (units + a.grid - 1) / a.grid;
  const int64_t u0 = static_cast<int64_t>(before) * heads +
                     static_cast<int64_t>(head * a.row_groups + rg) * tiles;
  const int c0 = static_cast<int>(u0 / share), c1 = static_cast<int>((u0 + tiles - 1) / share);
  if (c0 == c1) return;
  // The first part is its CTA's first segment only where it begins there.
  auto slot_of = [&](int c) {
    return (2ll * c + (c == c0 && u0 != c0 * share ? 1 : 0)) * ROWS + y;
  };
  float m = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) m = fmaxf(m, a.part_m[slot_of(c)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float l = 0.f, acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = 0.f;
  for (int c = c0 + warp; c <= c1; c += warps) {
    const int64_t slot = slot_of(c);
    const float pm = a.part_m[slot];
    const float e = pm == -INFINITY ? 0.f : exp2_fast(pm - m);
    l += e * a.part_l[slot];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] += e * a.part_o[slot * DP + lane + 32 * i];
  }
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) sm[warp * (DP + 1) + lane + 32 * i] = acc[i];
  if (lane == 0) sm[warp * (DP + 1) + DP] = l;
  __syncthreads();
  for (int d = threadIdx.x; d < a.dim; d += blockDim.x) {
    float lt = 0.f, ot = 0.f;
    for (int w = 0; w < warps; ++w) {
      lt += sm[w * (DP + 1) + DP];
      ot += sm[w * (DP + 1) + d];
    }
    store_out(a, at * a.dim + d, lt > 0.f ? ot / lt : (lt == 0.f ? 0.f : lt));
    if (d == 0 && a.lse) a.lse[at] = lt == 0.f ? -INFINITY : (m + log2f(lt)) * 0.6931471805599453f;
  }
}

int check(const b2g_cache_attention_desc* d) {
  if (!d || d->requests < 0 || d->heads < 0 || d->kv_heads < 0 || d->dim <= 0 ||
      d->num_blocks < 0 || d->table_width < 0 || d->table_ld < d->table_width ||
      (d->dtype != B2G_F16 && d->dtype != B2G_BF16) ||
      (d->codes != B2G_I8 && d->codes != B2G_E4M3) || !(d->scale >= 0.f))
    return B2G_ERR_INVALID_ARG;
  if (d->heads > 0 && (d->kv_heads == 0 || d->heads % d->kv_heads)) return B2G_ERR_INVALID_ARG;
  if (d->block_size < 16 || d->block_size > 256 || (d->block_size & (d->block_size - 1)) ||
      d->dim % 16 || d->dim > 128 || d->num_blocks > 0x7fffffff ||
      d->table_width * d->block_size > 0x7fffffc0 || d->requests > (1 << 20) ||
      d->heads > (1 << 16) || d->requests * d->heads > 0x7fffffff)
    return B2G_ERR_UNSUPPORTED;
  return B2G_OK;
}

struct Layout {
  int rows, dp, row_groups, grid;
  int64_t off_m, off_l, off_o, bytes;
};

Layout layout_of(const b2g_cache_attention_desc* d, int sms) {
  Layout w;
  const int64_t group = d->heads / d->kv_heads;
  w.rows = group <= 8 ? 8 : 16;
  w.dp = d->dim <= 64 ? 64 : 128;
  w.row_groups = static_cast<int>(cdiv(group, w.rows));
  const int64_t most = d->requests * d->kv_heads * w.row_groups *
                       std::max<int64_t>(cdiv(d->table_width * d->block_size, kTile), 1);
  w.grid = static_cast<int>(std::min<int64_t>(
      std::max<int64_t>(most, 1), static_cast<int64_t>(sms) * ctas_per_sm(w.dp, w.rows)));
  auto pad = [](int64_t n) { return cdiv(n, 256) * 256; };
  w.off_m = pad((d->requests + 1) * 4);
  w.off_l = w.off_m + pad(2ll * w.grid * w.rows * 4);
  w.off_o = w.off_l + pad(2ll * w.grid * w.rows * 4);
  w.bytes = w.off_o + 2ll * w.grid * w.rows * w.dp * 4;
  return w;
}

template <int DP, int ROWS, bool E4M3>
int launch(const Args& a, cudaStream_t stream) {
  cache_attention_kernel<DP, ROWS, E4M3><<<a.grid, kThreads, 0, stream>>>(a);
  if (cudaGetLastError() != cudaSuccess) return B2G_ERR_LAUNCH;
  const int64_t heads = static_cast<int64_t>(a.kv_heads) * a.group;
  // Parts of a head, were all lengths alike.
  const int warps = a.grid > 16 * a.requests * a.kv_heads * a.row_groups ? 16 : 4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.requests * heads), 1, 1);
  cfg.blockDim = dim3(warps * 32, 1, 1);
  cfg.dynamicSmemBytes = warps * (DP + 1) * sizeof(float);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = b2g::pdl_enabled() ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, cache_join_kernel<DP, ROWS>, a) != cudaSuccess) return B2G_ERR_LAUNCH;
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
  a.k_cache = static_cast<const uint8_t*>(d->k_cache);
  a.v_cache = static_cast<const uint8_t*>(d->v_cache);
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
  a.part_o = reinterpret_cast<float*>(ws + w.off_o);
  a.grid = w.grid;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  const bool e4 = d->codes == B2G_E4M3;
  if (w.dp == 64)
    return w.rows == 8 ? (e4 ? launch<64, 8, true>(a, stream) : launch<64, 8, false>(a, stream))
                       : (e4 ? launch<64, 16, true>(a, stream) : launch<64, 16, false>(a, stream));
  return w.rows == 8 ? (e4 ? launch<128, 8, true>(a, stream) : launch<128, 8, false>(a, stream))
                     : (e4 ? launch<128, 16, true>(a, stream) : launch<128, 16, false>(a, stream));
}
