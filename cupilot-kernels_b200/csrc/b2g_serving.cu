// b2g_serving.cu — what a serving step does to its paged cache before it
// attends to it: block tables and slot map (b2g_block_tables) and the
// quantising cache write (b2g_cache_append).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>

#include "../../include/b2g_serving.h"
#include "b2g_internal.h"

namespace {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool power_of_two(int64_t x) { return x > 0 && (x & (x - 1)) == 0; }

int log2_of(int64_t x) {
  int n = 0;
  while ((int64_t{1} << n) < x) ++n;
  return n;
}

// ------------------------------------------------------------ block tables
// Every CTA scans the lengths of all requests into shared memory (a few KB
// out of L2), then takes its share of the new tokens: a token finds its
// request by bisection of the offsets, its block in the table (a block that
// was there) or on the stack (one taken now), and the token that opens a new
// block writes the table entry.  No CTA reads what another writes, so one
// launch does it all.  Bound by latency: launch, one load of the lengths,
// one dependent load of the block, one store (on the GPU, 8 requests:
// 2.1 us; 1000 requests with 64000 new tokens: 4.5 us; a call takes 6.5 us of
// the host for either).

constexpr int64_t kSmallStep = 256;   // requests of a step that the smaller CTAs take

struct TableArgs {
  const int32_t* context_lens;
  const int32_t* new_lens;
  int requests;
  int32_t* table;
  int64_t width, ld;
  const int32_t* free_blocks;
  int64_t free_capacity;
  const int32_t* free_count;
  int64_t total;
  int lg_block;
  int64_t* slots;
  int32_t* cu;
  int32_t* seq_lens;
  int32_t* free_out;
};

__device__ __forceinline__ int64_t blocks_of(int64_t tokens, int lg, int64_t width) {
  const int64_t n = (tokens + (int64_t{1} << lg) - 1) >> lg;
  return n < width ? n : width;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) block_tables_kernel(const TableArgs a) {
  extern __shared__ int smem[];
  int* cu = smem;                        // requests + 1: new tokens before each request
  int* first = cu + a.requests + 1;      // new blocks before each request
  int* had = first + a.requests;         // tokens that it holds
  __shared__ unsigned long long warp_sum[THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t count = min(static_cast<int64_t>(*a.free_count), a.free_capacity);
  // Scan of (tokens, blocks) as the halves of one 64-bit word.
  unsigned long long carry = 0;
  int next_ctx = 0, next_add = 0;        // of the next round, on their way during this one
  if (tid < a.requests) next_ctx = a.context_lens[tid], next_add = a.new_lens[tid];
  for (int base = 0; base < a.requests; base += THREADS) {
    const int r = base + tid;
    unsigned long long v = 0;
    const int64_t ctx = max(next_ctx, 0), add = max(next_add, 0);
    if (r + THREADS < a.requests)
      next_ctx = a.context_lens[r + THREADS], next_add = a.new_lens[r + THREADS];
    if (r < a.requests) {
      const int64_t need =
          blocks_of(ctx + add, a.lg_block, a.width) - blocks_of(ctx, a.lg_block, a.width);
      had[r] = static_cast<int>(ctx);
      v = static_cast<unsigned long long>(need) << 32 | static_cast<unsigned long long>(add);
      if (blockIdx.x == 0) a.seq_lens[r] = static_cast<int32_t>(ctx + add);
    }
    unsigned long long incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    unsigned long long before = carry;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      const unsigned long long s = warp_sum[w];
      if (w < warp) before += s;
      carry += s;
    }
    const unsigned long long excl = before + incl - v;
    if (r < a.requests) {
      cu[r] = static_cast<int>(excl & 0xffffffffu);
      first[r] = static_cast<int>(excl >> 32);
      if (blockIdx.x == 0) a.cu[r] = cu[r];
    }
    __syncthreads();
  }
  const int64_t sum = static_cast<int64_t>(carry & 0xffffffffu);
  if (tid == 0) {
    cu[a.requests] = static_cast<int>(sum);
    if (blockIdx.x == 0) {
      a.cu[a.requests] = static_cast<int>(sum);
      *a.free_out = *a.free_count - static_cast<int>(carry >> 32);
    }
  }
  __syncthreads();
  const int64_t end = max(sum, a.total);
  const int64_t step = static_cast<int64_t>(gridDim.x) * THREADS;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * THREADS + tid; t < end; t += step) {
    int64_t slot = -1;
    if (t < sum) {
      // The last request that begins at or before t.  One token each is the
      // common step: try that first.
      int lo = 0, hi = a.requests;
      if (t < a.requests && cu[t] == t && cu[t + 1] > t) {
        lo = static_cast<int>(t);
      } else {
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (cu[mid] <= t) lo = mid;
          else hi = mid;
        }
      }
      const int64_t ctx = had[lo];
      const int64_t pos = ctx + (t - cu[lo]);
      const int64_t j = pos >> a.lg_block;
      const int off = static_cast<int>(pos & ((int64_t{1} << a.lg_block) - 1));
      if (j < a.width) {
        const int64_t held = blocks_of(ctx, a.lg_block, a.width);
        int32_t* entry = a.table + lo * a.ld + j;
        int64_t block;
        if (j < held) {
          block = *entry;
        } else {
          const int64_t at = count - 1 - (first[lo] + j - held);
          block = at >= 0 && at < count ? a.free_blocks[at] : -1;
          if (off == 0) *entry = static_cast<int32_t>(block);
        }
        if (block >= 0) slot = (block << a.lg_block) + off;
      }
    }
    if (t < a.total) a.slots[t] = slot;
  }
}

// ------------------------------------------------------------ cache write
// W warps take a chunk of consecutive tokens for one head of the keys or the
// values and do the groups that begin in it, one after another: the largest
// |x| of the group, the block's new scale, the old codes moved to it where it
// grew, the new codes.  The group's owner is the only one that touches the
// block's codes and scale of that head, so nothing is atomic and the result
// does not depend on the order.  Bound by memory (2 bytes read and 1 written a
// value) in the long run, by the warps' chain of loads in a call's few waves,
// and where a group has more rows than a warp holds (16 of 128 dims) its rows are
// read twice: 18000 tokens, 8 heads of 128, blocks of 32: 23.9 us, 3460 GB/s in a
// stream of calls (22.4 on the GPU); 64 single tokens: 4.7 us (2.8).
constexpr int kAppendWarps = 8;
struct AppendArgs {
  const uint16_t* x[2];          // keys, values
  int64_t token_stride[2], head_stride[2];
  uint8_t* cache[2];
  float* scale[2];
  const int64_t* slots;
  int64_t tokens, items, limit;  // limit: slots in the cache
  int heads, dim, lg_block, chunk;
  int lanes_row, rows_warp;      // lanes to a row of dim values, rows that a warp covers at once
};

template <bool BF16>
__device__ __forceinline__ float2 widen(uint32_t w) {
  if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Rounded to nearest even; x*steps is within the range of the codes unless
// the value is not finite (`any`).
template <bool E4M3>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, bool any) {
  if (E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  if (any) {
    auto tame = [](float v) { return v == v ? fminf(fmaxf(v, -127.f), 127.f) : 0.f; };
    a = tame(a), b = tame(b), c = tame(c), d = tame(d);
  }
  // 1.5 * 2^23: the sum's last place is 1, so its low byte is the rounded integer.
  const float big = 12582912.f;
  const uint32_t ia = __float_as_uint(__fadd_rn(a, big)), ib = __float_as_uint(__fadd_rn(b, big));
  const uint32_t ic = __float_as_uint(__fadd_rn(c, big)), id = __float_as_uint(__fadd_rn(d, big));
  return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
}

template <bool E4M3>
__device__ __forceinline__ float decode1(uint32_t byte) {
  if (E4M3) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3);
    return __half2float(__half(h));
  }
  return static_cast<float>(static_cast<int8_t>(byte));
}

template <bool BF16, bool E4M3, int W>
__global__ void __launch_bounds__(kAppendWarps * 32, 3)
    cache_append_kernel(const AppendArgs a) {
  constexpr int kHold = 8;                 // 16-byte vectors that a lane keeps between the passes
  __shared__ uint32_t tops[kAppendWarps];
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5, sub = warp % W;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kAppendWarps / W) + warp / W;
  if (item >= a.items) return;
  // The largest of the item's warps.
  auto largest = [&](uint32_t x) {
    x = __reduce_max_sync(0xffffffffu, x);
    if (W == 1) return x;
    auto meet = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / W), "n"(W * 32) : "memory"); };
    if (lane == 0) tops[warp] = x;
    meet();
#pragma unroll
    for (int w = 0; w < W; ++w) x = max(x, tops[warp / W * W + w]);
    meet();                                // read before it is written again
    return x;
  };
  const int both = 2 * a.heads;
  const int64_t t0 = item / both * a.chunk;
  const int hk = static_cast<int>(item % both);
  const int kv = hk >= a.heads, head = hk - kv * a.heads;
  const int bs = 1 << a.lg_block;
  const uint16_t* x = a.x[kv] + head * a.head_stride[kv];
  const int64_t ts = a.token_stride[kv];
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
  constexpr float kInvQmax = E4M3 ? 1.f / 448.f : 1.f / 127.f;

  // Groups that begin in this chunk, and the slots of 64 tokens from its first on.
  int64_t slot = -1, later = -1;
  bool lead = false;
  if (t0 + lane < a.tokens) {
    slot = a.slots[t0 + lane];
    const int64_t prev = t0 + lane > 0 ? a.slots[t0 + lane - 1] : -2;
    lead = lane < a.chunk && slot >= 0 && slot < a.limit && (prev != slot - 1 || (slot & (bs - 1)) == 0);
  }
  if (t0 + 32 + lane < a.tokens) later = a.slots[t0 + 32 + lane];
  unsigned leads = __ballot_sync(0xffffffffu, lead);
  const int row = lane / a.lanes_row, col = lane % a.lanes_row;
  const bool used = row < a.rows_warp;
  while (leads) {
    const int src = __ffs(leads) - 1;
    leads &= leads - 1;
    const int64_t s0 = __shfl_sync(0xffffffffu, slot, src);
    const int64_t t = t0 + src;
    const int fill = static_cast<int>(s0 & (bs - 1));
    const int64_t block = s0 >> a.lg_block;
    // The group's length: consecutive slots, first among the 64 at hand.
    const uint64_t run =
        (static_cast<uint64_t>(__ballot_sync(0xffffffffu, later == s0 + 32 + lane - src)) << 32 |
         __ballot_sync(0xffffffffu, slot == s0 + lane - src)) >> src;
    int n = min(bs - fill, ~run ? __ffsll(static_cast<long long>(~run)) - 1 : 64);
    if (n == 64 - src)
      while (n < bs - fill) {
        const int i = n + lane;
        const bool same = i < bs - fill && t + i < a.tokens && a.slots[t + i] == s0 + i;
        const unsigned m = __ballot_sync(0xffffffffu, same);
        n += m == 0xffffffffu ? 32 : __ffs(~m) - 1;
        if (m != 0xffffffffu) break;
      }
    const uint16_t* xr = x + t * ts + col * 8;
    uint4 held[kHold];
    uint32_t most = 0;           // largest |x| bits, two halves
    const int step = W * a.rows_warp, span = kHold * step;
    auto load = [&](int base) {
#pragma unroll
      for (int i = 0; i < kHold; ++i) {
        const int rr = base + i * step + sub * a.rows_warp + row;
        held[i] = make_uint4(0, 0, 0, 0);
        if (used && rr < n) held[i] = __ldg(reinterpret_cast<const uint4*>(xr + rr * ts));
      }
    };
    for (int base = 0; base < n; base += span) {
      load(base);
#pragma unroll
      for (int i = 0; i < kHold; ++i) {
        const uint32_t w = __vmaxu2(__vmaxu2(held[i].x & 0x7fff7fffu, held[i].y & 0x7fff7fffu),
                                    __vmaxu2(held[i].z & 0x7fff7fffu, held[i].w & 0x7fff7fffu));
        most = __vmaxu2(most, w);
      }
    }
    uint32_t top = largest(max(most & 0xffffu, most >> 16));
    const bool any = top >= kInf;          // an infinity or NaN: look again without those
    if (any) {
      uint32_t m = 0;
      for (int base = 0; base < n; base += span) {
        load(base);
        for (int i = 0; i < kHold; ++i) {
          const uint32_t v[4] = {held[i].x, held[i].y, held[i].z, held[i].w};
          for (int j = 0; j < 4; ++j) {
            const uint32_t lo = v[j] & 0x7fffu, hi = (v[j] >> 16) & 0x7fffu;
            m = max(m, lo < kInf ? lo : 0u);
            m = max(m, hi < kInf ? hi : 0u);
          }
        }
      }
      top = largest(m);
    }
    const float amax = widen<BF16>(top).x;
    float* sp = a.scale[kv] + block * a.heads + head;
    const float old = fill > 0 ? *sp : 0.f;
    if (W > 1 && fill > 0) largest(0);       // every warp has read the scale
    const float now = fmaxf(old, __fmul_rn(amax, kInvQmax));
    // Without a finite value but 0 the steps are 0; 1 then, so that an infinity stays one.
    const float steps = now > 0.f ? fminf(__fdiv_rn(1.f, now), FLT_MAX) : (any ? 1.f : 0.f);
    __syncwarp();
    if (lane == 0 && sub == 0) *sp = now;
    uint8_t* cp = a.cache[kv] + ((block * a.heads + head) << a.lg_block) * a.dim + col * 8;
    if (fill > 0 && now > old) {
      const float ratio = __fdiv_rn(old, now);
      for (int rr = sub * a.rows_warp + row; rr < fill && used; rr += step) {
        uint2* p = reinterpret_cast<uint2*>(cp + rr * a.dim);
        const uint2 w = *p;
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[j] = __fmul_rn(decode1<E4M3>((w.x >> (8 * j)) & 255u), ratio);
          f[4 + j] = __fmul_rn(decode1<E4M3>((w.y >> (8 * j)) & 255u), ratio);
        }
        *p = make_uint2(encode4<E4M3>(f[0], f[1], f[2], f[3], true),
                        encode4<E4M3>(f[4], f[5], f[6], f[7], true));
      }
    }
    for (int base = 0; base < n; base += span) {
      if (n > span) load(base);   // else still held (a lane's rows past n hold zeros)
#pragma unroll
      for (int i = 0; i < kHold; ++i) {
        const int rr = base + i * step + sub * a.rows_warp + row;
        if (used && rr < n) {
          const float2 p0 = widen<BF16>(held[i].x), p1 = widen<BF16>(held[i].y);
          const float2 p2 = widen<BF16>(held[i].z), p3 = widen<BF16>(held[i].w);
          const uint2 w = make_uint2(
              encode4<E4M3>(__fmul_rn(p0.x, steps), __fmul_rn(p0.y, steps),
                            __fmul_rn(p1.x, steps), __fmul_rn(p1.y, steps), any),
              encode4<E4M3>(__fmul_rn(p2.x, steps), __fmul_rn(p2.y, steps),
                            __fmul_rn(p3.x, steps), __fmul_rn(p3.y, steps), any));
          *reinterpret_cast<uint2*>(cp + (fill + rr) * a.dim) = w;
        }
      }
    }
    __syncwarp();
  }
}

}  // namespace

extern "C" int b2g_block_tables(const int32_t* context_lens, const int32_t* new_lens,
                                int64_t requests, int32_t* block_table, int64_t table_width,
                                int64_t table_ld, const int32_t* free_blocks,
                                int64_t free_capacity, const int32_t* free_count,
                                int64_t total_tokens, int block_size, int64_t* slots,
                                int32_t* cu_seqlens, int32_t* seq_lens, int32_t* free_count_out,
                                b2g_stream_t stream_handle) {
  if (requests < 0 || table_width < 0 || table_ld < table_width || free_capacity < 0 ||
      total_tokens < 0 || !power_of_two(block_size))
    return B2G_ERR_INVALID_ARG;
  if (!free_count || !cu_seqlens || !free_count_out || (total_tokens > 0 && !slots) ||
      (requests > 0 && (!context_lens || !new_lens || !seq_lens)) ||
      (requests > 0 && table_width > 0 && !block_table) || (free_capacity > 0 && !free_blocks))
    return B2G_ERR_INVALID_ARG;
  if (requests > B2G_MAX_TABLE_REQUESTS || total_tokens > 0x7fffffff || block_size > 1 << 20)
    return B2G_ERR_UNSUPPORTED;
  b2g::Device dev;
  const int rc = b2g::current_device(&dev);
  if (rc != B2G_OK) return rc;
  TableArgs a;
  a.context_lens = context_lens;
  a.new_lens = new_lens;
  a.requests = static_cast<int>(requests);
  a.table = block_table;
  a.width = table_width;
  a.ld = table_ld;
  a.free_blocks = free_blocks;
  a.free_capacity = free_capacity;
  a.free_count = free_count;
  a.total = total_tokens;
  a.lg_block = log2_of(block_size);
  a.slots = slots;
  a.cu = cu_seqlens;
  a.seq_lens = seq_lens;
  a.free_out = free_count_out;
  const size_t bytes = (3 * requests + 1) * sizeof(int);
  // Fewer threads start a small step sooner (8 requests: 2.4 us for 2.9), more scan a large one in
  // fewer rounds.
  const bool small = requests <= kSmallStep;
  const int threads = small ? 256 : 512;
  auto* kernel = small ? block_tables_kernel<256> : block_tables_kernel<512>;
  // The larger kernel may take what the largest step needs, whatever this one does: a limit that
  // followed the calls could be lowered between another thread's setting and its launch.
  static thread_local int configured = -1;
  int device = 0;
  cudaGetDevice(&device);
  if (!small && configured != device) {
    constexpr int kMost = (3 * B2G_MAX_TABLE_REQUESTS + 1) * sizeof(int);
    if (cudaFuncSetAttribute(block_tables_kernel<512>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kMost) != cudaSuccess)
      return B2G_ERR_LAUNCH;
    configured = device;
  }
  const int grid = static_cast<int>(
      std::min<int64_t>(std::max<int64_t>(cdiv(total_tokens, threads), 1), dev.num_sms));
  kernel<<<grid, threads, bytes, static_cast<cudaStream_t>(stream_handle)>>>(a);
  return cudaGetLastError() == cudaSuccess ? B2G_OK : B2G_ERR_LAUNCH;
}

extern "C" int b2g_cache_append(const b2g_cache_append_desc* d, b2g_stream_t stream_handle) {
  if (!d || d->tokens < 0 || d->kv_heads < 0 || d->num_blocks < 0 || d->dim <= 0 ||
      (d->dtype != B2G_F16 && d->dtype != B2G_BF16) ||
      (d->codes != B2G_I8 && d->codes != B2G_E4M3) || !power_of_two(d->block_size))
    return B2G_ERR_INVALID_ARG;
  if (d->dim % 16 || d->dim > 128 || d->block_size < 16 || d->block_size > 256 ||
      d->kv_heads > 4096)
    return B2G_ERR_UNSUPPORTED;
  if (d->tokens == 0 || d->kv_heads == 0 || d->num_blocks == 0) return B2G_OK;
  if (!d->k || !d->v || !d->slots || !d->k_cache || !d->v_cache || !d->k_scale || !d->v_scale)
    return B2G_ERR_INVALID_ARG;
  for (int64_t s : {d->k_token_stride, d->k_head_stride, d->v_token_stride, d->v_head_stride})
    if (s % 8) return B2G_ERR_UNSUPPORTED;
  for (const void* p : {d->k, d->v, static_cast<const void*>(d->k_cache),
                        static_cast<const void*>(d->v_cache)})
    if (reinterpret_cast<uintptr_t>(p) % 16) return B2G_ERR_UNSUPPORTED;
  b2g::Device dev;
  const int rc = b2g::current_device(&dev);
  if (rc != B2G_OK) return rc;
  AppendArgs a;
  a.x[0] = static_cast<const uint16_t*>(d->k);
  a.x[1] = static_cast<const uint16_t*>(d->v);
  a.token_stride[0] = d->k_token_stride;
  a.token_stride[1] = d->v_token_stride;
  a.head_stride[0] = d->k_head_stride;
  a.head_stride[1] = d->v_head_stride;
  a.cache[0] = static_cast<uint8_t*>(d->k_cache);
  a.cache[1] = static_cast<uint8_t*>(d->v_cache);
  a.scale[0] = d->k_scale;
  a.scale[1] = d->v_scale;
  a.slots = d->slots;
  a.tokens = d->tokens;
  a.limit = d->num_blocks * d->block_size;
  a.heads = static_cast<int>(d->kv_heads);
  a.dim = static_cast<int>(d->dim);
  a.lg_block = log2_of(d->block_size);
  a.lanes_row = a.dim / 8;
  a.rows_warp = 32 / a.lanes_row;
  // Tokens to a warp: one while that fills the GPU with 16 warps an SM, more for longer calls,
  // where a warp would mostly find that its token begins no group.
  const int64_t per_token = 2 * d->kv_heads;
  a.chunk = static_cast<int>(std::min<int64_t>(
      std::max<int64_t>(d->tokens * per_token / (16ll * dev.num_sms), 1),
      std::min<int64_t>(d->block_size, 32)));
  a.items = cdiv(d->tokens, a.chunk) * per_token;
  // Warps to an item: one, but for whole large blocks, of which there are too few to fill the GPU
  // (18000 tokens in blocks of 16, 32, 64: 20, 22, 22 us with one warp, 20, 25, 30 with more; of
  // 128: 31 and 29).
  const int w = d->block_size < 128 || d->tokens <= d->block_size ? 1 : 4;
  const int64_t grid = cdiv(a.items, kAppendWarps / w);
  if (grid > 0x7fffffff) return B2G_ERR_UNSUPPORTED;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  const bool bf = d->dtype == B2G_BF16, e4 = d->codes == B2G_E4M3;
  auto pick = [&](auto* one, auto* four) { return w == 1 ? one : four; };
  auto* kernel =
      bf ? (e4 ? pick(cache_append_kernel<true, true, 1>, cache_append_kernel<true, true, 4>)
               : pick(cache_append_kernel<true, false, 1>, cache_append_kernel<true, false, 4>))
         : (e4 ? pick(cache_append_kernel<false, true, 1>, cache_append_kernel<false, true, 4>)
               : pick(cache_append_kernel<false, false, 1>, cache_append_kernel<false, false, 4>));
  kernel<<<static_cast<unsigned>(grid), kAppendWarps * 32, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? B2G_OK : B2G_ERR_LAUNCH;
}
