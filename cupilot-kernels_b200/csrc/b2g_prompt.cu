// b2g_prompt.cu — causal attention of packed prompts with grouped heads on
// tcgen05 (b2g_prompt_attention).
//
// o_i = sum_j exp(z_ij - m_i) v_j / sum_j exp(z_ij - m_i), z = scale * q k^T,
// in one pass over the keys: with S a tile of 128 rows by 128 keys,
//   m' = max(m, rowmax S),  P = exp(S - m'),  l = l exp(m - m') + rowsum P,
//   O = O exp(m - m') + P V.
// The rows of a tile are tokens times the query heads that share a kv head
// (row = token * group + head, one TMA box), so K and V are read once for the
// group and a group's short prompt still fills a tile.  A work item is two
// such tiles of one sequence and kv head; a CTA does one after another, the
// later ones taken over from CTAs that have not started.  S, P and O live in
// tensor memory: S0 S1 O0 O1, 128 columns each, P over the first half of its
// S.
//   warps 0-3, 4-7   softmax of tile 0 / 1, a thread a row: S from tensor
//                    memory, P back in 16 bits, at the end O / l to memory
//   warp 8           the products: while one tile's softmax runs, the other
//                    tile's P V and next Q K^T keep the tensor cores busy
//   warp 9           TMA loads: Q, then K and V tiles through a ring
//   warp 10          the next work item
//   warp 11          clears the rows of a V tile past the end of its sequence
// The maximum is taken over only where it grew by more than 2^8 (P stays
// within 16 bits' range, l and O are fp32): then, rarely, the softmax warps
// rescale O themselves.
// What bounds it: a pair of tiles has 2^15 exponentials against 2048 cycles of
// tensor core work (dim 128); the special function unit gives 16 a cycle, so
// 3 of 16 are computed on the FMA units (0: 1 to 2 % slower, 5: 5 %).  Beside
// that a tile's chain softmax - P V - Q K^T, some 1500 + 1024 cycles and four
// barriers, sets the pace of a step (2700 to 3000 cycles; a third tile has no
// room in tensor memory).  Measured:
//   16384 tokens, 16 heads on 4, dim 128, bf16: 0.97 ms, 1130 TFLOP/s, in a
//   stream of calls, where the power limit holds the clock at 1.6 GHz (cuBLAS
//   then: 1384); 0.83 ms, 1320, in a short burst (cuBLAS: 1658)
//   6 prompts of 700 to 2300 tokens, 32 heads on 8: 0.143 ms, 770 TFLOP/s in a
//   stream of calls; 0.121 ms, 910, in a short burst
// Tried and slower: two threads to a row (four softmax warps a scheduler: S
// read twice or registers spilled, +15 %), a thread for each tile's products
// (both tiles' softmax then fall on the same cycles, +25 %), branches around
// key columns past the diagonal (+4 %, the compiler no longer interleaves the
// columns), O staged through shared memory for whole-line stores (-3 % where
// items are short, +2 % where they are long), 64 keys at a time in a loop of
// half the code (-8 % for short prompts, +5 to +19 % for long ones), P beside S
// up to 64 dims (both softmaxes at once: +16 %).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/b2g_serving.h"
#include "b2g_internal.h"
#include "ptx_sm100.cuh"

namespace b2g {
namespace prompt {

constexpr int kRows = 128;            // rows of a tile
constexpr int kKeys = 128;            // keys of a tile
constexpr int kSoftmaxWarps = 8;
constexpr int kMmaWarp = 8, kLoadWarp = 9, kNextWarp = 10, kTailWarp = 11;
constexpr int kThreads = 12 * 32;     // a whole third warpgroup, for the register split
// Registers: 384 threads start with 168 each; the third warpgroup gives 96 of
// each thread's to the softmax warps (2 * 128 * 216 + 128 * 72 = 384 * 168).
// 208 / 88 was 9 % slower (a row's 128 scores no longer fit), 224 / 56 1 %.
constexpr int kRegsSoftmax = 216, kRegsOther = 72;
constexpr int kAskAhead = 2;          // key tiles left to load when the next item is asked for
constexpr int kItemReaders = kSoftmaxWarps + 3;
// Of 16 pairs of exponentials, how many run on the FMA units.
constexpr int kPolyPairs = 3;
constexpr float kGrow = 8.f;
constexpr uint64_t kDrainLimitNs = 100000000ull;
constexpr int kBoxBytes = 128 * 128;  // 64 columns x 128 rows of 16 bits

enum : int { kErrFull = 0x301, kErrEmpty = 0x302, kErrS = 0x303, kErrP = 0x304, kErrO = 0x305,
             kErrQ = 0x306, kErrItem = 0x307, kErrNext = 0x308 };

template <int DP>
struct Smem {
  static constexpr int kBoxes = DP / 64;
  static constexpr int kTileBytes = kBoxes * kBoxBytes;     // a Q, K or V tile
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr int kOffRing = 2 * kTileBytes;
  static constexpr int kOffBars = kOffRing + kStages * kTileBytes;
  static constexpr int kNumBars = 2 * kStages + 2 * 6 + 4 + 5;
  static constexpr int kOffNext = (kOffBars + kNumBars * 8 + 15) / 16 * 16;   // 16-byte answer
  static constexpr int kOffItems = kOffNext + 16;
  static constexpr int kOffMisc = kOffItems + 2 * 48;
  static constexpr int kBytes = kOffMisc + 16 + 1024;
};
static_assert(Smem<128>::kBytes <= 232448 && Smem<64>::kBytes <= 232448, "shared memory budget");

struct Params {
  const int32_t* cu_q;
  const int32_t* cu_k;
  int sequences, tokens, tokens_k, heads, kv_heads, group, dim;
  int tile_tokens;                    // tokens of a tile: 128 / group
  int span;                           // tokens of a work item: two tiles, or one
  int causal;
  int slots;                          // upper bound of tile pairs over all sequences
  float scale_log2;
  uint16_t* out;
  int64_t out_token, out_head;
  float* lse;
  long long wait_limit_ns;
  int* err;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void fail(int* err, volatile int* abort, int code) {
  atomicCAS(err, 0, code);
  *abort = 1;
}

// The halves of a shared-memory matrix descriptor (ptx::smem_desc) in the
// 128-byte swizzle, rows of 8 x 128 bytes: the low one (address and leading
// offset) moves with the tile, the high one is the same for all.  One thread
// issues every product, between waits, so what it computes for each of them
// counts: an addition.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (ptx::kLayoutSw128 << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo_bytes) {
  return (saddr >> 4) | ((lbo_bytes >> 4) << 16);
}
// D (+)= A B^T, A and B in shared memory.
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_low), "r"(b_low), "r"(kDescHigh), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D (+)= A B with A in tensor memory (16-bit pairs, 128 lanes).
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_low), "r"(kDescHigh), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_regs(uint32_t (&r)[32]) {
  ptx::tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Pairs of fp32 in one register pair.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Maxima that keep a NaN.
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x of a pair by range reduction and a polynomial: x = n + f, |f| <= 1/2,
// 2^f by its best relative approximation of degree 3 (error 7.5e-5, for P in
// bf16 with its rounding of 2e-3) or 4 (2.6e-6, for fp16 with 2.4e-4), the
// coefficients found by Remez exchange; n goes into the exponent.  From -127
// on the result is 0: a masked score, -infinity, has to weigh nothing beside
// the largest values that bf16 holds (2^-126 of those is 4).
template <bool BF16>
__device__ __forceinline__ void exp2_poly(uint64_t x2, float& a, float& b) {
  float x, y;
  unpair(x2, x, y);
  x2 = pair(fmaxf(x, -127.f), fmaxf(y, -127.f));
  const float big = 12582912.f;                     // 1.5 * 2^23: the sum's low bits are n
  const uint64_t n2 = add2(x2, pair(big, big));
  const uint64_t back = add2(n2, pair(-big, -big));
  const uint64_t f2 = fma2(back, pair(-1.f, -1.f), x2);
  uint64_t y2;
  if (BF16) {
    y2 = fma2(f2, pair(0.05517167f, 0.05517167f), pair(0.24261113f, 0.24261113f));
    y2 = fma2(f2, y2, pair(0.69326097f, 0.69326097f));
    y2 = fma2(f2, y2, pair(0.99992806f, 0.99992806f));
  } else {
    y2 = fma2(f2, pair(0.009570102f, 0.009570102f), pair(0.05591786f, 0.05591786f));
    y2 = fma2(f2, y2, pair(0.24024744f, 0.24024744f));
    y2 = fma2(f2, y2, pair(0.6931218f, 0.6931218f));
    y2 = fma2(f2, y2, pair(0.9999993f, 0.9999993f));
  }
  float na, nb;
  unpair(n2, na, nb);
  unpair(y2, a, b);
  // 2^f is just below 1 at f = 0, so that the sum is negative there for n = -127.
  a = __int_as_float(max(static_cast<int>(__float_as_uint(a) + (__float_as_uint(na) << 23)), 0));
  b = __int_as_float(max(static_cast<int>(__float_as_uint(b) + (__float_as_uint(nb) << 23)), 0));
}

// Two tiles of one sequence and kv head; all lengths cut to the tensors' sizes.
struct Item {
  int q0, qlen, k0, klen, first;      // first: token of tile 0's row 0, within the sequence
  int head;
  int n0, n1;                         // key tiles of each row tile (0: no rows, or they see nothing)
  int more;                           // 0: no work is left
};
static_assert(sizeof(Item) <= 48, "item slot");

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Keys that token `tok` of the sequence sees.
__device__ __forceinline__ int keys_of(const Params& p, const Item& it, int tok) {
  if (!p.causal) return it.klen;
  return clampi(tok + it.klen - it.qlen + 1, 0, it.klen);
}

// Tile pair x of all sequences: sequence s owns the places from
// cu[s] / span + s on, at least as many as it has pairs; some stay empty.
__device__ __forceinline__ bool find_item(const Params& p, int x, int head, Item* it) {
  const int span = p.span;
  int lo = 0, hi = p.sequences;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (clampi(p.cu_q[mid], 0, p.tokens) / span + mid <= x) lo = mid;
    else hi = mid;
  }
  it->head = head;
  it->q0 = clampi(p.cu_q[lo], 0, p.tokens);
  it->qlen = clampi(p.cu_q[lo + 1], 0, p.tokens) - it->q0;
  it->k0 = clampi(p.cu_k[lo], 0, p.tokens_k);
  it->klen = max(clampi(p.cu_k[lo + 1], 0, p.tokens_k) - it->k0, 0);
  it->first = (x - it->q0 / span - lo) * span;
  auto tiles = [&](int t0) {
    const int last = min(t0 + p.tile_tokens, it->qlen) - 1;
    return t0 < it->qlen ? (keys_of(p, *it, last) + kKeys - 1) / kKeys : 0;
  };
  it->n0 = tiles(it->first);
  it->n1 = span > p.tile_tokens ? tiles(it->first + p.tile_tokens) : 0;
  return it->first >= 0 && it->first < it->qlen;
}

// Rows of no sequence: zeros, a share for each of the first work indices.
__device__ __forceinline__ void zero_rows(const Params& p, int w, int lane) {
  constexpr int kShares = 64;
  const int shares = min(kShares, p.slots * p.kv_heads);
  if (w >= shares) return;
  const int before = p.sequences ? clampi(p.cu_q[0], 0, p.tokens) : 0;
  const int after = p.sequences ? clampi(p.cu_q[p.sequences], before, p.tokens) : 0;
  const int64_t n = static_cast<int64_t>(before + p.tokens - after) * p.heads;
  for (int64_t i = static_cast<int64_t>(w) * 32 + lane; i < n; i += shares * 32) {
    int64_t t = i / p.heads;
    const int h = static_cast<int>(i % p.heads);
    if (t >= before) t += after - before;
    uint16_t* o = p.out + t * p.out_token + h * p.out_head;
    for (int d = 0; d < p.dim; d += 8) *reinterpret_cast<uint4*>(o + d) = make_uint4(0, 0, 0, 0);
    if (p.lse) p.lse[t * p.heads + h] = -INFINITY;
  }
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const Params p) {
  using L = Smem<DP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
  uint64_t* empty = full + L::kStages;
  uint64_t* q_full = empty + L::kStages;     // [2]
  uint64_t* q_empty = q_full + 2;            // [2] the tile's last Q K^T has read Q
  uint64_t* s_full = q_full + 4;             // [2] S of the tile is complete
  uint64_t* p_half = q_full + 6;             // [2] P of the tile's first 64 keys is stored
  uint64_t* p_ready = q_full + 8;            // [2] and that of the others
  uint64_t* o_done = q_full + 10;            // [2] P V of the tile is added to O
  uint64_t* item_full = q_full + 12;         // [2]
  uint64_t* item_empty = q_full + 14;        // [2]
  uint64_t* next_wanted = q_full + 16;       // the loads come to an item's end
  uint64_t* next_full = q_full + 17;
  uint64_t* tail_there = q_full + 18;        // the item's last V tile, of a sequence that ends in it
  uint64_t* tail_done = q_full + 19;         // it is cleared past the sequence
  uint64_t* drain = q_full + 20;
  uint8_t* next_answer = smem + L::kOffNext;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  auto item_at = [&](uint32_t k) { return reinterpret_cast<Item*>(smem + L::kOffItems + (k & 1) * 48); };

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&q_full[i], 1);
      ptx::mbar_init(&q_empty[i], 1);
      ptx::mbar_init(&s_full[i], 1);
      ptx::mbar_init(&p_half[i], kSoftmaxWarps / 2);
      ptx::mbar_init(&p_ready[i], kSoftmaxWarps / 2);
      ptx::mbar_init(&o_done[i], 1);
      ptx::mbar_init(&item_full[i], 1);
      ptx::mbar_init(&item_empty[i], kItemReaders);
    }
    ptx::mbar_init(next_wanted, 1);
    ptx::mbar_init(next_full, 1);
    ptx::mbar_init(tail_there, 1);
    ptx::mbar_init(tail_done, 1);
    ptx::mbar_init(drain, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // A wait of a whole warp: one answer, so that it stays converged where a wait gives up.
  auto warp_wait = [&](uint64_t* bar, uint32_t parity, volatile int* abort) {
    const bool come = ptx::mbar_wait_suspended(bar, parity, abort, p.wait_limit_ns);
    return __all_sync(0xffffffffu, come) != 0;
  };
  // The k-th item of this CTA, for the warps that work on it.
  auto get_item = [&](uint32_t k, Item* it) {
    if (!warp_wait(&item_full[k & 1], (k >> 1) & 1, abort_flag)) {
      if (lane == 0) fail(p.err, abort_flag, kErrItem);
      return false;
    }
    *it = *item_at(k);
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(&item_empty[k & 1]);
    return it->more != 0;
  };

  if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == kNextWarp) {
      // ---------------------------------------------------------- next item
      int w = blockIdx.x;
      uint32_t k = 0, asked = 0;
      bool more = true;
      while (more) {
        zero_rows(p, w, lane);
        Item it;
        // Late tiles see the most keys: they go first.
        if (p.sequences > 0 && find_item(p, p.slots - 1 - w / p.kv_heads, w % p.kv_heads, &it)) {
          it.more = 1;
          if (!warp_wait(&item_empty[k & 1], ((k >> 1) & 1) ^ 1, abort_flag)) {
            if (lane == 0) fail(p.err, abort_flag, kErrItem);
            break;
          }
          if (lane == 0) {
            *item_at(k) = it;
            ptx::mbar_arrive(&item_full[k & 1]);
          }
          // Another CTA's work is taken over when this item's last key tiles are on their way: early
          // enough to hide the question, late enough that whoever is done first takes what is left.
          if (!warp_wait(next_wanted, k & 1, abort_flag)) {
            if (lane == 0) fail(p.err, abort_flag, kErrNext);
            break;
          }
          ++k;
        }
        if (lane == 0) {
          ptx::fence_proxy_async_smem();
          ptx::mbar_arrive_expect_tx(next_full, 16);
          ptx::clc_try_cancel(next_answer, next_full);
        }
        volatile int never = 0;                  // (the answer lands before the CTA leaves)
        if (!warp_wait(next_full, asked & 1, &never)) {
          if (lane == 0) fail(p.err, abort_flag, kErrNext);
          break;
        }
        ++asked;
        more = ptx::clc_answer(next_answer, &w);
        __syncwarp();
      }
      if (warp_wait(&item_empty[k & 1], ((k >> 1) & 1) ^ 1, abort_flag)) {
        if (lane == 0) {
          item_at(k)->more = 0;
          ptx::mbar_arrive(&item_full[k & 1]);
        }
      }
      __syncwarp();
    } else if (warp == kLoadWarp) {
      // ---------------------------------------------------------- loads
      if (lane == 0) {
        ptx::prefetch_tmap(&map_q);
        ptx::prefetch_tmap(&map_k);
        ptx::prefetch_tmap(&map_v);
      }
      const uint32_t q_bytes = L::kBoxes * p.group * p.tile_tokens * 128;
      uint32_t q_issued[2] = {0, 0}, issued = 0;
      bool ok = true;
      Item it;
      for (uint32_t k = 0; ok && get_item(k, &it); ++k) {
        if (ptx::elect_one()) {
          auto load_q = [&](int i) {
            if (!ptx::mbar_wait_suspended(&q_empty[i], (q_issued[i] & 1) ^ 1, abort_flag, p.wait_limit_ns)) {
              fail(p.err, abort_flag, kErrEmpty);
              return false;
            }
            ptx::mbar_arrive_expect_tx(&q_full[i], q_bytes);
            for (int b = 0; b < L::kBoxes; ++b)
              ptx::tma_load_3d(smem + i * L::kTileBytes + b * kBoxBytes, &map_q, &q_full[i], b * 64,
                               it.head * p.group, it.q0 + it.first + i * p.tile_tokens);
            ++q_issued[i];
            return true;
          };
          auto load_kv = [&](const CUtensorMap* map, int j) {
            const uint32_t s = issued % L::kStages;
            if (!ptx::mbar_wait_suspended(&empty[s], ((issued / L::kStages) & 1) ^ 1, abort_flag, p.wait_limit_ns)) {
              fail(p.err, abort_flag, kErrEmpty);
              return false;
            }
            ptx::mbar_arrive_expect_tx(&full[s], L::kTileBytes);
            for (int b = 0; b < L::kBoxes; ++b)
              ptx::tma_load_3d(smem + L::kOffRing + s * L::kTileBytes + b * kBoxBytes, map, &full[s],
                               b * 64, it.head, it.k0 + j * kKeys);
            ++issued;
            return true;
          };
          const int n = max(it.n0, it.n1);
          if (it.n0 > 0) ok = load_q(0);
          if (n > 0) ok = ok && load_kv(&map_k, 0);
          if (it.n1 > 0) ok = ok && load_q(1);
          if (n > 0) ok = ok && load_kv(&map_v, 0);
          const int ask = max(n - kAskAhead, 0);
          if (ask == 0) ptx::mbar_arrive(next_wanted);
          for (int j = 1; j < n && ok; ++j) {
            if (j == ask) ptx::mbar_arrive(next_wanted);
            ok = load_kv(&map_k, j) && load_kv(&map_v, j);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
      // Every load has landed before the CTA may leave.
      if (ptx::elect_one()) {
        volatile int never = 0;
        for (int i = 0; i < 2; ++i)
          if (q_issued[i]) ptx::mbar_wait_suspended(&q_full[i], (q_issued[i] - 1) & 1, &never, kDrainLimitNs);
        for (uint32_t e = issued > L::kStages ? issued - L::kStages : 0; e < issued; ++e)
          ptx::mbar_wait_suspended(&full[e % L::kStages], (e / L::kStages) & 1, &never, kDrainLimitNs);
      }
      __syncwarp();
    } else if (warp == kTailWarp) {
      // ---------------------------------------------------------- tails
      // Rows of a V tile past its sequence hold the next one's values (or nothing): their weights
      // are 0, but 0 * inf is not.  They are cleared before the products read them.
      uint32_t used = 0, tails = 0;
      Item it;
      bool ok = true;
      for (uint32_t k = 0; ok && get_item(k, &it); ++k) {
        const int n = max(it.n0, it.n1);
        if (n * kKeys > it.klen) {
          const uint32_t e = used + 2 * (n - 1) + 1;
          if (!warp_wait(tail_there, tails++ & 1, abort_flag)) {
            if (lane == 0) fail(p.err, abort_flag, kErrFull);
            ok = false;
            break;
          }
          uint8_t* v = smem + L::kOffRing + (e % L::kStages) * L::kTileBytes;
          const int from = (it.klen - (n - 1) * kKeys) * 128;
          for (int b = 0; b < L::kBoxes; ++b)
            for (int x = from + lane * 16; x < kBoxBytes; x += 512)
              *reinterpret_cast<uint4*>(v + b * kBoxBytes + x) = make_uint4(0, 0, 0, 0);
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(tail_done);
        }
        used += 2 * n;
      }
    } else if (warp == kMmaWarp) {
      // ---------------------------------------------------------- products
      // One thread does it all, and between two products of a tile pair its own instructions are
      // what the tensor cores wait for: barriers by shared address, ring positions that move on
      // without a division, the next tiles' arrival looked at while a softmax still runs.
      constexpr uint32_t kType = BF16 ? (1u << 7) | (1u << 10) : 0u;
      const uint32_t idesc_s = ptx::idesc_f16(kRows, kKeys, false, false) | kType;
      const uint32_t idesc_o = ptx::idesc_f16(kRows, p.dim, false, true) | kType;
      constexpr uint32_t kTileLow = L::kTileBytes >> 4;
      const uint32_t q_low = desc_low(ptx::smem_addr(smem), 16);
      const uint32_t k_low = desc_low(ptx::smem_addr(smem + L::kOffRing), 16);
      const uint32_t v_low = desc_low(ptx::smem_addr(smem + L::kOffRing), kBoxBytes);
      if (ptx::elect_one()) {
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
          if (!ptx::mbar_wait_suspended(bar, parity, abort_flag, p.wait_limit_ns)) {
            fail(p.err, abort_flag, code);
            ok = false;
          }
        };
        uint32_t slot = 0, ring_phase = 0;     // of the next ring entry
        // Waits for the next ring entry; its slot.
        auto take = [&]() {
          const uint32_t at = slot;
          wait(&full[at], ring_phase, kErrFull);
          if (++slot == L::kStages) slot = 0, ring_phase ^= 1;
          return at;
        };
        auto scores = [&](int i, uint32_t at, bool last) {      // S_i = Q_i K^T, K in ring slot `at`
          const uint32_t sq = q_low + i * kTileLow, sk = k_low + at * kTileLow;
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            const uint32_t off = ((k >> 2) * kBoxBytes + (k & 3) * 32) >> 4;
            if (k * 16 < p.dim) mma_ss(tmem + i * kKeys, sq + off, sk + off, idesc_s, k > 0);
          }
          ptx::mma_commit(&s_full[i]);
          if (last) ptx::mma_commit(&q_empty[i]);
        };
        auto values = [&](int i, uint32_t at, int half, bool add) {   // O_i += P_i V, V in slot `at`
          const uint32_t sv = v_low + at * kTileLow;
#pragma unroll
          for (int x = 0; x < kKeys / 32; ++x) {
            const int k = half * (kKeys / 32) + x;
            mma_ts(tmem + 256 + i * 128, tmem + i * kKeys + k * 8, sv + k * (16 * 128 >> 4), idesc_o,
                   add || x > 0);
          }
          if (half) ptx::mma_commit(&o_done[i]);
        };
        uint32_t q_phase[2] = {0, 0}, p_phase[2] = {0, 0}, tail_phase = 0;
        for (uint32_t k = 0; ok; ++k) {
          wait(&item_full[k & 1], (k >> 1) & 1, kErrItem);
          if (!ok) break;
          const Item* it = item_at(k);
          const int n0 = it->n0, n1 = it->n1, klen = it->klen, more = it->more;
          ptx::mbar_arrive(&item_empty[k & 1]);
          if (!more) break;
          const int n = max(n0, n1);
          if (n == 0) continue;
          const bool tail = n * kKeys > klen;
          const uint32_t first = take();
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int ni = i ? n1 : n0;
            if (ni > 0 && ok) {
              wait(&q_full[i], q_phase[i], kErrQ);
              q_phase[i] ^= 1;
              if (ok) scores(i, first, ni == 1);
            }
          }
          ptx::mma_commit(&empty[first]);
          uint32_t v = take();
          if (tail && n == 1) ptx::mbar_arrive(tail_there);
          uint32_t kk = n > 1 ? take() : 0;
          for (int j = 0; j < n && ok; ++j) {
            if (tail && j == n - 1) {
              wait(tail_done, tail_phase, kErrFull);
              tail_phase ^= 1;
            }
            uint32_t v_next = 0, k_next = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int ni = i ? n1 : n0;
              if (j < ni && ok) {
                wait(&p_half[i], p_phase[i], kErrP);
                ptx::tc_fence_after();
                if (ok) values(i, v, 0, j > 0);
                wait(&p_ready[i], p_phase[i], kErrP);
                p_phase[i] ^= 1;
                ptx::tc_fence_after();
                if (ok) {
                  values(i, v, 1, true);
                  if (j + 1 < ni) scores(i, kk, j + 2 == ni);
                }
              }
              if (i == 0 && ok) {
                if (j + 1 < n) v_next = take();
                if (tail && j + 2 == n) ptx::mbar_arrive(tail_there);
                if (j + 2 < n) k_next = take();
              }
            }
            ptx::mma_commit(&empty[v]);
            if (j + 1 < n) ptx::mma_commit(&empty[kk]);
            v = v_next;
            kk = k_next;
          }
        }
        // No product may still write tensor memory when it is freed.
        ptx::mma_commit(drain);
        volatile int never = 0;
        ptx::mbar_wait(drain, 0, &never, kDrainLimitNs);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int i = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + i * kKeys, to = tmem + lanes + 256 + i * 128;
    const int row_tok = row / p.group, g = row % p.group;
    const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
    uint32_t steps = 0;
    bool ok = true;
    Item it;
    for (uint32_t k = 0; ok && get_item(k, &it); ++k) {
      const int ni = i ? it.n1 : it.n0;
      const int t0 = it.first + i * p.tile_tokens;
      const int tok = t0 + row_tok;
      const bool mine = row_tok < p.tile_tokens && tok < it.qlen && t0 < it.first + p.span;
      const int limit = keys_of(p, it, tok);
      const int least = keys_of(p, it, t0);      // no row of the tile sees fewer keys
      float m = -INFINITY;                       // in log2 units
      uint64_t l2 = 0;                           // the sum, in two parts
      for (int j = 0; j < ni; ++j, ++steps) {
        if (!warp_wait(&s_full[i], steps & 1, abort_flag)) {
          if (lane == 0) fail(p.err, abort_flag, kErrS);
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32b_x32(ts + c * 32, s[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_wait_regs(s[c]);
        if ((j + 1) * kKeys > least) {
          const int seen = limit - j * kKeys;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (c * 32 + x >= seen) s[c][x] = 0xff800000u;   // -infinity
        }
        float tops[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tops[c] = max2(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]));
#pragma unroll
          for (int x = 2; x < 32; x += 2)
            tops[c] = max3(tops[c], __uint_as_float(s[c][x]), __uint_as_float(s[c][x + 1]));
        }
        const float top = max2(max3(tops[0], tops[1], tops[2]), tops[3]) * p.scale_log2;
        // (also where a NaN or an infinity makes the whole row NaN, whichever unit its weights take)
        if (__any_sync(0xffffffffu, !(top <= m + kGrow))) {
          const float now = max2(m, top);
          const float corr = now == m ? 1.f : exp2_fast(m - now);
          m = now == INFINITY ? NAN : now;
          float la, lb;
          unpair(l2, la, lb);
          l2 = pair(la * corr, lb * corr);
          if (j > 0) {
            if (!warp_wait(&o_done[i], (steps - 1) & 1, abort_flag)) {
              if (lane == 0) fail(p.err, abort_flag, kErrO);
              ok = false;
              break;
            }
            ptx::tc_fence_after();
#pragma unroll 1
            for (int d = 0; d < p.dim; d += 32) {
              uint32_t o[32];
              ptx::tmem_ld_32x32b_x32(to + d, o);
              tmem_wait_regs(o);
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * corr);
              tmem_st_x32(to + d, o);
            }
            tmem_st_wait();
          }
        }
        const float off = m == -INFINITY ? 0.f : -m;
        const uint64_t off2 = pair(off, off);
        uint64_t odd2 = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const uint64_t z2 = fma2(pair(__uint_as_float(s[c][2 * x]), __uint_as_float(s[c][2 * x + 1])),
                                     scale2, off2);
            float a, b;
            if ((x + 1) * kPolyPairs / 16 != x * kPolyPairs / 16) {
              exp2_poly<BF16>(z2, a, b);
            } else {
              unpair(z2, a, b);
              a = exp2_fast(a);
              b = exp2_fast(b);
            }
            // (two chains: one of 64 dependent additions a step was 4 % of the time)
            uint64_t& sum2 = x & 1 ? odd2 : l2;
            sum2 = add2(sum2, pair(a, b));
            w[x] = pack<BF16>(a, b);
          }
          tmem_st_x16(ts + c * 16, w);
          if (c == 3) l2 = add2(l2, odd2);
          if (c & 1) {
            tmem_st_wait();
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(c == 1 ? &p_half[i] : &p_ready[i]);
          }
        }
      }
      const int64_t t = it.q0 + tok;
      const int h = it.head * p.group + g;
      uint16_t* out = p.out + t * p.out_token + h * p.out_head;
      if (ok && ni > 0) {
        if (!warp_wait(&o_done[i], (steps - 1) & 1, abort_flag)) {
          if (lane == 0) fail(p.err, abort_flag, kErrO);
          ok = false;
        }
      }
      if (!ok) break;
      ptx::tc_fence_after();
      float la, lb;
      unpair(l2, la, lb);
      const float l = la + lb;
      const bool some = m != -INFINITY && limit > 0;
      const float inv = 1.f / l;
#pragma unroll 1
      for (int d = 0; d < p.dim; d += 32) {
        uint32_t o[32];
        if (ni > 0) {
          ptx::tmem_ld_32x32b_x32(to + d, o);
          tmem_wait_regs(o);
        }
        if (mine) {
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            if (d + x < p.dim) {
              uint32_t w[4] = {0, 0, 0, 0};
              if (some)
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  w[y] = pack<BF16>(__uint_as_float(o[x + 2 * y]) * inv,
                                    __uint_as_float(o[x + 2 * y + 1]) * inv);
              *reinterpret_cast<uint4*>(out + d + x) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      }
      ptx::tc_fence_before();                    // O is read before the next item's products write it
      if (mine && p.lse)
        p.lse[t * p.heads + h] = some ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// {dim, heads, tokens} in 16 bits; a box is 64 columns of box_heads heads of
// box_tokens tokens, rows of 128 bytes in the 128-byte swizzle.
bool make_map(CUtensorMap* map, const void* base, bool bf16, int64_t dim, int64_t heads, int64_t tokens,
              int64_t head_stride, int64_t token_stride, int box_heads, int box_tokens) {
  if (heads == 1) head_stride = dim;
  if (tokens == 1) token_stride = std::max<int64_t>(heads * dim, head_stride);
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads),
                        static_cast<cuuint64_t>(tokens)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_stride) * 2,
                           static_cast<cuuint64_t>(token_stride) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
  cuuint32_t estr[3] = {1, 1, 1};
  return encode_tiled(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                      3, base, dims, strides, box, estr, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int DP, bool BF16>
int launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const Params& p,
           unsigned grid, cudaStream_t stream) {
  static thread_local int configured = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (configured != dev) {
    if (cudaFuncSetAttribute(prompt_kernel<DP, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Smem<DP>::kBytes) != cudaSuccess)
      return B2G_ERR_LAUNCH;
    configured = dev;
  }
  prompt_kernel<DP, BF16><<<grid, kThreads, Smem<DP>::kBytes, stream>>>(q, k, v, p);
  return cudaGetLastError() == cudaSuccess ? B2G_OK : B2G_ERR_LAUNCH;
}

}  // namespace prompt
}  // namespace b2g

extern "C" int b2g_prompt_attention(const b2g_prompt_attention_desc* d, b2g_stream_t stream_handle) {
  using namespace b2g::prompt;
  if (!d || d->tokens < 0 || d->tokens_k < 0 || d->sequences < 0 || d->heads < 0 ||
      d->kv_heads < 0 || d->dim <= 0 || (d->dtype != B2G_F16 && d->dtype != B2G_BF16) ||
      !(d->scale >= 0.f && std::isfinite(d->scale)))
    return B2G_ERR_INVALID_ARG;
  if (d->heads > 0 && (d->kv_heads == 0 || d->heads % d->kv_heads)) return B2G_ERR_INVALID_ARG;
  if (d->tokens == 0 || d->heads == 0) return B2G_OK;
  if (d->dim % 16 || d->dim > 128 || d->heads / d->kv_heads > kRows || d->heads > (1 << 16) ||
      d->tokens > 0x3fffffff || d->tokens_k > 0x3fffffff || d->sequences > 0x3fffffff)
    return B2G_ERR_UNSUPPORTED;
  if (!d->q || !d->out || (d->sequences > 0 && !d->cu_q) || (d->tokens_k > 0 && (!d->k || !d->v)) ||
      (!d->cu_k && d->tokens_k != d->tokens))
    return B2G_ERR_INVALID_ARG;
  for (int64_t s : {d->q_token_stride, d->q_head_stride, d->k_token_stride, d->k_head_stride,
                    d->v_token_stride, d->v_head_stride, d->out_token_stride, d->out_head_stride})
    if (s < 0 || s % 8) return B2G_ERR_UNSUPPORTED;
  for (const void* ptr : {d->q, d->k, d->v, static_cast<const void*>(d->out)})
    if (reinterpret_cast<uintptr_t>(ptr) % 16) return B2G_ERR_UNSUPPORTED;
  b2g::Device dev;
  const int rc = b2g::current_device(&dev);
  if (rc != B2G_OK) return rc;
  Params p;
  p.cu_q = d->cu_q;
  p.cu_k = d->cu_k ? d->cu_k : d->cu_q;
  // Without a key no tile is loaded, but the maps want memory: the queries' stands in.
  const bool no_keys = d->tokens_k == 0;
  p.sequences = static_cast<int>(d->sequences);
  p.tokens = static_cast<int>(d->tokens);
  p.tokens_k = static_cast<int>(d->tokens_k);
  p.heads = static_cast<int>(d->heads);
  p.kv_heads = static_cast<int>(d->kv_heads);
  p.group = p.heads / p.kv_heads;
  p.dim = static_cast<int>(d->dim);
  p.tile_tokens = kRows / p.group;
  p.causal = d->causal != 0;
  p.scale_log2 = (d->scale > 0.f ? d->scale : 1.f / std::sqrt(static_cast<float>(d->dim))) *
                 1.4426950408889634f;
  p.out = static_cast<uint16_t*>(d->out);
  p.out_token = d->out_token_stride;
  p.out_head = d->out_head_stride;
  p.lse = d->lse;
  p.wait_limit_ns = b2g::current_wait_limit_ns();
  p.err = dev.error_word;
  // Two tiles a work item; one where that still leaves no more items than SMs.
  auto slots_of = [&](int64_t span) { return std::max<int64_t>(d->tokens / span + d->sequences, 1); };
  p.span = slots_of(p.tile_tokens) * p.kv_heads <= dev.num_sms ? p.tile_tokens : 2 * p.tile_tokens;
  const int64_t slots = slots_of(p.span);
  if (slots * p.kv_heads > 0x7fffffff) return B2G_ERR_UNSUPPORTED;
  p.slots = static_cast<int>(slots);
  const bool bf = d->dtype == B2G_BF16;
  CUtensorMap mq, mk, mv;
  if (!make_map(&mq, d->q, bf, d->dim, d->heads, d->tokens, d->q_head_stride, d->q_token_stride,
                p.group, p.tile_tokens) ||
      !make_map(&mk, no_keys ? d->q : d->k, bf, d->dim, no_keys ? 1 : d->kv_heads,
                no_keys ? 1 : d->tokens_k, d->k_head_stride, d->k_token_stride, 1, kKeys) ||
      !make_map(&mv, no_keys ? d->q : d->v, bf, d->dim, no_keys ? 1 : d->kv_heads,
                no_keys ? 1 : d->tokens_k, d->v_head_stride, d->v_token_stride, 1, kKeys))
    return B2G_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>(slots * p.kv_heads);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  if (d->dim <= 64)
    return bf ? launch<64, true>(mq, mk, mv, p, grid, stream) : launch<64, false>(mq, mk, mv, p, grid, stream);
  return bf ? launch<128, true>(mq, mk, mv, p, grid, stream) : launch<128, false>(mq, mk, mv, p, grid, stream);
}
