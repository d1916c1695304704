// Kernels around the paged 8-bit cache of a batch of requests: the step's
// block table and slot map (gdsq_build_tables) and the cache write with RoPE
// (gdsq_append_kv8).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gdsq.h"
#include "host.h"
#include "common.cuh"

namespace gdsq {
namespace {

// ---------------------------------------------------------------------------
// Block tables and slot maps.
//
// Request s holds c_s cached tokens in the first ceil(c_s / bs) entries of its
// table row and gets n_s new ones, so it needs
//   need_s = ceil((c_s + n_s) / bs) - ceil(c_s / bs)
// blocks more.  They come from the queue of free blocks in request order:
// request s takes the entries head + sum_{u<s} need_u onwards.
//
// Every CTA makes both running sums (of n and need) over all requests itself,
// in shared memory, so that no CTA waits for another; then the CTAs share out
// the tokens and the table rows.
//
// Bound by latency: 4.6 us on the GPU for 64 requests with a token each, 8.0 for
// 1000 requests with up to 511 tokens each, whose 4 MB take 0.7 us of memory time.

constexpr int kTabThreads = 1024;
constexpr int kTabMaxRequests = 16384;
constexpr int kTabMaxLen = (1 << 30) - (1 << 10);  // of a request, cached or new

struct TablesArgs {
  const int* context;
  const int* fresh;
  int* table;
  const int* free_blocks;
  const int* free_head;
  int* seq_lens;
  int* starts;
  long long* positions;
  long long* slots;
  int* head_out;
  int requests, width, num_free, block, tokens;
};

__global__ void __launch_bounds__(kTabThreads) build_tables_kernel(const TablesArgs p) {
  extern __shared__ int sm[];
  int* starts = sm;                      // [requests + 1]
  int* first = starts + p.requests + 1;  // [requests] index into free_blocks
  __shared__ long long wsum[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int threads = kTabThreads, warps = threads >> 5;
  pdl_launch_dependents();
  pdl_wait_primary();
  const int head = *p.free_head;
  const int per = (p.requests + threads - 1) / threads;
  const int r0 = min(tid * per, p.requests), r1 = min(r0 + per, p.requests);
  bool bad = head < 0, wide = false;
  // Lengths that no table holds are cut off, and sums stop at the largest int, so that no index wraps.
  constexpr int kMost = 0x7fffffff;
  auto cut_off = [&](int length) { return min(max(length, 0), kTabMaxLen); };
  for (int r = r0; r < r1; ++r) {
    const int held = p.context[r], fresh = p.fresh[r];
    const int c = cut_off(held), n = cut_off(fresh);
    bad |= held != c || fresh != n;
    wide |= n > 65535;  // else 2^14 requests' sums fit in 31 bits
    first[r] = c;
    starts[r] = n;
  }
  int tall = 0;
  long long blocks = 0;
  auto running_sums = [&](auto zero) {
    using Sum = decltype(zero);
    Sum tok = 0, blk = 0;
    for (int r = r0; r < r1; ++r) {
      const int c = first[r], n = starts[r];
      starts[r] = (int)min((long long)tok, (long long)kMost);
      first[r] = (int)min((long long)blk, (long long)kMost);
      tok += n;
      blk += (c + n + p.block - 1) / p.block - (c + p.block - 1) / p.block;
    }
    Sum ts = tok, bsum = blk;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const Sum a = __shfl_up_sync(0xffffffffu, ts, d), b = __shfl_up_sync(0xffffffffu, bsum, d);
      if (lane >= d) {
        ts += a;
        bsum += b;
      }
    }
    if (lane == 31) {
      wsum[0][warp] = ts;
      wsum[1][warp] = bsum;
    }
    __syncthreads();
    Sum wt = (Sum)wsum[0][lane], wb = (Sum)wsum[1][lane];
    Sum tb = lane < warp ? wt : 0, bb = lane < warp ? wb : 0;
    if constexpr (sizeof(Sum) == 4) {
      tb = __reduce_add_sync(0xffffffffu, tb);
      bb = __reduce_add_sync(0xffffffffu, bb);
      wt = __reduce_add_sync(0xffffffffu, wt);
      wb = __reduce_add_sync(0xffffffffu, wb);
    } else {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        tb += __shfl_xor_sync(0xffffffffu, tb, d);
        bb += __shfl_xor_sync(0xffffffffu, bb, d);
        wt += __shfl_xor_sync(0xffffffffu, wt, d);
        wb += __shfl_xor_sync(0xffffffffu, wb, d);
      }
    }
    tb += ts - tok;
    bb += bsum - blk;
    bad |= wt > p.tokens;
    tall = (int)min((long long)wt, (long long)kMost);
    blocks = wb;
    for (int r = r0; r < r1; ++r) {
      starts[r] = (int)min((long long)starts[r] + tb, (long long)kMost);
      first[r] = (int)min((long long)first[r] + head + bb, (long long)kMost);
    }
  };
  static_assert(warps == 32, "a lane for each warp's sums");
  if (__syncthreads_or(wide)) running_sums(0ll);
  else running_sums(0);
  if (tid == 0) starts[p.requests] = tall;
  __syncthreads();

  auto free_block = [&](long long i) { return i >= 0 && i < p.num_free ? p.free_blocks[i] : -1; };
  for (int r = blockIdx.x * warps + warp; r < p.requests; r += gridDim.x * warps) {
    const int c = cut_off(p.context[r]), n = min(starts[r + 1] - starts[r], kTabMaxLen);
    const int held = (c + p.block - 1) / p.block, after = (c + n + p.block - 1) / p.block;
    for (int j = held + lane; j < min(after, p.width); j += 32) {
      const int b = free_block((long long)first[r] + j - held);
      bad |= b < 0;
      p.table[(size_t)r * p.width + j] = b;
    }
    bad |= after > p.width;
    if (lane == 0) {
      p.seq_lens[r] = c + n;
      p.starts[r] = starts[r];
      if (r == 0) {
        p.starts[p.requests] = tall;
        *p.head_out = (int)min(head + blocks, (long long)kMost);
      }
    }
  }
  const long long stride = (long long)gridDim.x * threads;
  for (long long i = (long long)blockIdx.x * threads + tid; i < p.tokens; i += stride) {
    long long pos = 0, slot = -1;
    if (i < tall) {
      int lo = 0, hi = p.requests;  // the request with starts[lo] <= i < starts[lo + 1]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= i) lo = mid;
        else hi = mid;
      }
      const int c = cut_off(p.context[lo]);
      pos = c + (i - starts[lo]);
      const int col = (int)(pos / p.block), held = (c + p.block - 1) / p.block;
      if (col < p.width) {
        const int b = col < held ? p.table[(size_t)lo * p.width + col] : free_block((long long)first[lo] + col - held);
        if (b >= 0) slot = (long long)b * p.block + pos % p.block;
        bad |= b < 0;
      }
    }
    p.positions[i] = pos;
    p.slots[i] = slot;
  }
  if (bad) record_device_error(kDevErrBadIndex);
}

// ---------------------------------------------------------------------------
// Cache write.
//
// K (rotated first when a table of angles is given) and V of the new tokens
// become 8-bit codes under one fp32 scale per (block, KV head).  For the new
// tokens of one block, with m their largest magnitude and top = 127 (int8) or
// 448 (e4m3):
//   need = m / top, base = 0 on a block begun by these tokens, else its scale
//   scale = base if need <= base, else max(need, 2 base)
// A scale that grows at least doubles, so int8 codes held before, multiplied by
// base / scale and rounded again, are off by less than one step of the new
// scale after any number of growths.  An e4m3 code is not changed by a growth
// that just doubles (while it stays normal) and is rounded once more by one
// that more than doubles.  A non-finite value makes the block's scale NaN and
// is itself stored as 0.  New tokens of one block are adjacent in the batch.

constexpr int kAppThreads = 256;
constexpr float kSmallestScale = 7.888609052210118e-31f;  // 2^-100

struct AppendArgs {
  const void* q;
  const void* k;
  const void* v;
  long long q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride;
  void* q_out;
  const float2* freqs;
  const long long* positions;
  const long long* slots;
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scale;
  float* v_scale;
  int tokens, heads, kv_heads, num_blocks, block_shift, max_position;
};

// 8 values of a row as fp32.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
      const float2 f = __half22float2(u32_as_h2(ww[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(ww[i] << 16);
      x[2 * i + 1] = __uint_as_float(ww[i] & 0xffff0000u);
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) {
      w[i] = h2_as_u32(__floats2half2_rn(x[2 * i], x[2 * i + 1]));
    } else {
      const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ float value_of_bits(uint32_t bits) {
  if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)bits));
  return __uint_as_float(bits << 16);
}

// The angles of 8 values, 4 (cos, sin) pairs.
struct Angles {
  float4 a, b;
};
__device__ __forceinline__ Angles load_angles(const float2* f) {
  const float4* p = reinterpret_cast<const float4*>(f);
  return {__ldg(p), __ldg(p + 1)};
}
// (x + iy)(c + is) as separate fp32 products and sums: the arithmetic of
// rotating the complex pairs in torch.
__device__ __forceinline__ void rotate8(const Angles& f, float (&x)[8]) {
  const float c[4] = {f.a.x, f.a.z, f.b.x, f.b.z}, s[4] = {f.a.y, f.a.w, f.b.y, f.b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = x[2 * i], b = x[2 * i + 1];
    x[2 * i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
    x[2 * i + 1] = __fadd_rn(__fmul_rn(a, s[i]), __fmul_rn(b, c[i]));
  }
}

// 8 codes of x * f, which is at most the format's largest code, give or take a
// rounding, by the choice of the scale.
template <int F>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float f) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __fmul_rn(x[4 * h + i], f);
    if constexpr (F == GDSQ_CACHE_INT8) {
      // 1.5 * 2^23 + y is rounded to a whole number, half to even, whose two's complement is the low bits
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = __float_as_uint(__fadd_rn(y[i], 12582912.f));
      w[h] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    } else {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
      w[h] = lo | hi << 16;
    }
  }
  return make_uint2(w[0], w[1]);
}
template <int F>
__device__ __forceinline__ void decode8(const uint2& w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = ((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 0xffu;
    if constexpr (F == GDSQ_CACHE_INT8) x[i] = (float)(int8_t)c;
    else x[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
  }
}

// Bound by the bytes of q, k and v and, for single tokens, by latency.  A unit
// is (the new tokens of one block, KV head, K or V): its tokens are held in
// registers, 16 to a warp, between the maximum and the codes, so that k and v
// are read once; a longer run takes 2, 4 or 8 warps.  A CTA takes `chunk` tokens
// and the runs that begin among them, and 8 units or a part of q's heads; the
// groups of one chunk are neighbours, so that a token's row is read at one time
// (173 us with the chunks of a group as neighbours where this order takes 159).
//
// Measured: 20 thousand tokens, 32 heads of 128, blocks of 16, bf16 to int8: 146
// us, 4.7 TB/s (72 % of a copy's rate; 159 with 2 CTAs to an SM); 64 tokens,
// 64 / 8 heads: 3.7 us.
template <typename T, int HD, int F>
__global__ void __launch_bounds__(kAppThreads, HD == 256 ? 2 : 4) append_kv8_kernel(const AppendArgs p, const int chunk, const int kv_groups,
                                                                 const int groups) {
  constexpr float kTop = F == GDSQ_CACHE_INT8 ? 127.f : 448.f;
  constexpr int kLanes = HD / 8;          // lanes per token, 8 values each
  constexpr int kAtOnce = 32 / kLanes;    // tokens per load of a warp
  constexpr int kLoads = 16 / kAtOnce;    // of 16 tokens
  __shared__ uint32_t red[kAppThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = blockIdx.x % groups, i0 = (int)(blockIdx.x / groups) * chunk;
  pdl_launch_dependents();
  pdl_wait_primary();
  const bool rope = p.freqs != nullptr;

  if (group >= kv_groups) {
    // q: a thread takes 8 dims of one token for every heads_step-th head
    const int row = threadIdx.x / kLanes, d = (threadIdx.x % kLanes) * 8;
    constexpr int kRowsAtOnce = kAppThreads / kLanes;
    const int parts = groups - kv_groups, part = group - kv_groups;
    for (int j = row % chunk; j < chunk; j += kRowsAtOnce) {  // chunk is a power of two
      const int i = i0 + j;
      if (i >= p.tokens) break;
      const long long pos = p.positions[i];
      if (pos < 0 || pos >= p.max_position) {
        record_device_error(kDevErrBadIndex);
        continue;
      }
      const Angles f = load_angles(p.freqs + pos * (HD / 2) + d / 2);
      const int step = max(kRowsAtOnce / chunk, 1);
      const T* src = static_cast<const T*>(p.q) + i * p.q_token_stride + d;
      T* dst = static_cast<T*>(p.q_out) + (size_t)i * p.heads * HD + d;
      constexpr int kAhead = 4;
      for (int h0 = part * step + row / chunk; h0 < p.heads; h0 += kAhead * parts * step) {
        uint4 w[kAhead];
#pragma unroll
        for (int y = 0; y < kAhead; ++y) {
          const int h = h0 + y * parts * step;
          if (h < p.heads) w[y] = __ldg(reinterpret_cast<const uint4*>(src + h * p.q_head_stride));
        }
#pragma unroll
        for (int y = 0; y < kAhead; ++y) {
          const int h = h0 + y * parts * step;
          if (h >= p.heads) break;
          float x[8];
          unpack8<T>(w[y], x);
          rotate8(f, x);
          *reinterpret_cast<uint4*>(dst + (size_t)h * HD) = pack8<T>(x);
        }
      }
    }
    return;
  }

  const int bs = 1 << p.block_shift;
  // Tokens that begin a run: the first of their block in the batch.
  const int il = i0 + lane;
  bool begins = false;
  if (lane < chunk && il < p.tokens) {
    const long long slot = p.slots[il], page = slot >> p.block_shift;
    if (slot >= 0) {
      if (page >= p.num_blocks) {
        if (warp == 0) record_device_error(kDevErrBadIndex);
      } else {
        begins = il == 0 || p.slots[il - 1] < 0 || (p.slots[il - 1] >> p.block_shift) != page;
      }
    }
  }
  for (unsigned heads = __ballot_sync(0xffffffffu, begins); heads; heads &= heads - 1) {
    const int i = i0 + __ffs(heads) - 1;
    const long long slot = p.slots[i], page = slot >> p.block_shift;
    const int begin = (int)(slot & (bs - 1));
    int n = 0;  // tokens of the run
    for (;;) {
      const int at = i + n + lane;
      const bool same = at < p.tokens && n + lane < bs && p.slots[at] >= 0 && (p.slots[at] >> p.block_shift) == page;
      const unsigned other = ~__ballot_sync(0xffffffffu, same);
      if (other) {
        n += __ffs(other) - 1;
        break;
      }
      n += 32;
    }
    const int wide = n <= 16 ? 1 : n <= 32 ? 2 : n <= 64 ? 4 : 8;  // warps per unit
    const int sub = warp / wide, part = warp % wide;
    for (int pass = 0; pass < wide; ++pass) {
      const int u = group * 8 + pass * (8 / wide) + sub;
      const bool live_unit = u < 2 * p.kv_heads;
      const bool is_v = u >= p.kv_heads;
      const int h = live_unit ? (is_v ? u - p.kv_heads : u) : 0;
      const T* src = static_cast<const T*>(is_v ? p.v : p.k) + h * (is_v ? p.v_head_stride : p.k_head_stride) + (lane % kLanes) * 8;
      const long long stride = is_v ? p.v_token_stride : p.k_token_stride;
      float* scale = (is_v ? p.v_scale : p.k_scale) + page * p.kv_heads + h;
      uint8_t* dst = (is_v ? p.v_cache : p.k_cache) + ((size_t)page * p.kv_heads + h) * bs * HD + (lane % kLanes) * 8;
      const float base = begin == 0 ? 0.f : *scale;
      uint4 raw[kLoads];
      uint32_t live = 0;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int tk = part * 16 + j * kAtOnce + lane / kLanes;
        raw[j] = make_uint4(0, 0, 0, 0);
        if (live_unit && tk < n) {
          raw[j] = __ldg(reinterpret_cast<const uint4*>(src + (long long)(i + tk) * stride));
          live |= 1u << j;
        }
      }
      uint32_t pair = 0;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        if (j * kAtOnce + part * 16 >= n) break;
        if (rope && (live >> j & 1)) {
          const long long pos = p.positions[i + part * 16 + j * kAtOnce + lane / kLanes];
          if (pos < 0 || pos >= p.max_position) {
            record_device_error(kDevErrBadIndex);
            live &= ~(1u << j);
          } else if (!is_v) {
            float x[8];
            unpack8<T>(raw[j], x);
            rotate8(load_angles(p.freqs + pos * (HD / 2) + (lane % kLanes) * 4), x);
            raw[j] = pack8<T>(x);
          }
        }
        if (live >> j & 1) {
          const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) pair = __vmaxu2(pair, w[e] & 0x7fff7fffu);
        }
      }
      // 16-bit magnitudes order as their bits do, inf and NaN on top; 0 is no token, so 1 more
      uint32_t most = __reduce_max_sync(0xffffffffu, live ? max(pair & 0xffffu, pair >> 16) + 1 : 0);
      if (wide > 1) {
        __syncthreads();
        if (lane == 0) red[warp] = most;
        __syncthreads();
        for (int w = 0; w < wide; ++w) most = max(most, red[sub * wide + w]);
      } else {
        __syncwarp();
      }
      if (most == 0) continue;
      const float top = value_of_bits<T>(most - 1);
      float need = __fmul_rn(top, 1.f / kTop);
      if (need < kSmallestScale) need = 0.f;
      float s = need <= base ? base : fmaxf(need, 2.f * base);
      if (!isfinite(top) || !(base == base)) s = __int_as_float(0x7fc00000);
      const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
      if (s != base && begin > 0) {
        const float ratio = __fmul_rn(base, inv);
        for (int j = part * kAtOnce + lane / kLanes; j < begin; j += wide * kAtOnce) {
          uint2* at = reinterpret_cast<uint2*>(dst + (size_t)j * HD);
          float x[8];
          decode8<F>(*at, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = inv > 0.f && x[e] == x[e] ? x[e] : 0.f;
          *at = encode8<F>(x, inv > 0.f ? ratio : 0.f);
        }
      }
      if (part == 0 && lane == 0) *scale = s;
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        if (live >> j & 1) {
          const int off = (int)(p.slots[i + part * 16 + j * kAtOnce + lane / kLanes] & (bs - 1));
          float x[8];
          unpack8<T>(raw[j], x);
          *reinterpret_cast<uint2*>(dst + (size_t)off * HD) = inv > 0.f ? encode8<F>(x, inv) : make_uint2(0, 0);
        }
    }
  }
}

}  // namespace

cudaError_t serve_error_bits(bool clear, int* bits) {
  int own = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&own, g_device_error, sizeof(int));
  if (e == cudaSuccess) *bits |= own;
  const int zero = 0;
  if (e == cudaSuccess && clear) e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
  return e;
}

namespace {

// A CTA looks at one token where there are few, else at 16, so that runs of a
// block's tokens do not leave most CTAs with nothing to do.
constexpr int kAppManyTokens = 1024;

template <typename T, int F>
int launch_append(const AppendArgs& a, int head_dim, cudaStream_t stream) {
  const int chunk = a.tokens >= kAppManyTokens ? 16 : 1;
  const int kv_groups = (2 * a.kv_heads + 7) / 8;
  // q: 16 vectors of 8 values per thread, or 4 where there are few
  const int q_groups = !a.q_out ? 0 : std::max(1, chunk * a.heads * head_dim / 8 / kAppThreads / (chunk == 1 ? 4 : 16));
  const int groups = kv_groups + q_groups;
  const dim3 grid((unsigned)((a.tokens + chunk - 1) / chunk) * groups);
  auto kernel = head_dim == 64    ? append_kv8_kernel<T, 64, F>
                : head_dim == 128 ? append_kv8_kernel<T, 128, F>
                                  : append_kv8_kernel<T, 256, F>;
  cudaError_t e = launch(kernel, grid, dim3(kAppThreads), 0, stream, g_pdl_enabled != 0, a, chunk, kv_groups, groups);
  return e == cudaSuccess ? GDSQ_OK : cuda_fail(e, "append_kv8 launch");
}

}  // namespace
}  // namespace gdsq

using namespace gdsq;

extern "C" {

int gdsq_build_tables(const int32_t* context_lens, const int32_t* new_lens, int num_requests, int32_t* block_table,
                      int table_width, const int32_t* free_blocks, int num_free, const int32_t* free_head,
                      int block_size, int num_tokens, int32_t* seq_lens, int32_t* query_starts, long long* positions,
                      long long* slots, int32_t* free_head_out, void* stream_v) {
  t_last_error.clear();
  if (num_requests < 1 || num_requests > kTabMaxRequests || table_width < 0 || num_free < 0 || block_size < 1 ||
      block_size > 1024 || num_tokens < 0)
    return fail(GDSQ_ERR_INVALID_VALUE, "build_tables: requests %d (1..%d), table width %d, free blocks %d, block "
                "size %d (1..1024), tokens %d", num_requests, kTabMaxRequests, table_width, num_free, block_size, num_tokens);
  if (!context_lens || !new_lens || (!block_table && table_width) || (!free_blocks && num_free) || !free_head ||
      !seq_lens || !query_starts || (num_tokens && (!positions || !slots)) || !free_head_out)
    return fail(GDSQ_ERR_INVALID_VALUE, "build_tables: null pointer");
  if (free_head == free_head_out)
    return fail(GDSQ_ERR_INVALID_VALUE, "build_tables: free_head_out must not be free_head");
  if (!aligned(context_lens, 4) || !aligned(new_lens, 4) || !aligned(block_table, 4) || !aligned(free_blocks, 4) ||
      !aligned(free_head, 4) || !aligned(seq_lens, 4) || !aligned(query_starts, 4) || !aligned(positions, 8) ||
      !aligned(slots, 8) || !aligned(free_head_out, 4))
    return fail(GDSQ_ERR_MISALIGNED, "build_tables: 4-byte (positions and slots 8-byte) alignment");
  // Other CTAs and later loops read the inputs again after the first outputs are written, so nothing may be both.
  struct Range {
    const char* name;
    const void* at;
    unsigned long long bytes;
    bool overlaps(const Range& o) const {
      const auto a = reinterpret_cast<uintptr_t>(at), b = reinterpret_cast<uintptr_t>(o.at);
      return bytes && o.bytes && a < b + o.bytes && b < a + bytes;
    }
  };
  const unsigned long long r = num_requests, t = num_tokens;
  const Range outputs[] = {{"seq_lens", seq_lens, 4 * r},       {"query_starts", query_starts, 4 * (r + 1)},
                           {"positions", positions, 8 * t},     {"slots", slots, 8 * t},
                           {"free_head_out", free_head_out, 4}, {"block_table", block_table, 4 * r * table_width}};
  const Range inputs[] = {{"context_lens", context_lens, 4 * r},
                          {"new_lens", new_lens, 4 * r},
                          {"free_blocks", free_blocks, 4ull * num_free},
                          {"free_head", free_head, 4}};
  for (const Range& o : outputs) {
    for (const Range& i : inputs)
      if (o.overlaps(i)) return fail(GDSQ_ERR_INVALID_VALUE, "build_tables: %s overlaps %s", o.name, i.name);
    for (const Range& i : outputs)
      if (&i != &o && o.overlaps(i)) return fail(GDSQ_ERR_INVALID_VALUE, "build_tables: %s overlaps %s", o.name, i.name);
  }
  const DeviceInfo* dev = nullptr;
  int st = device_info(&dev);
  if (st != GDSQ_OK) return st;
  const TablesArgs a = {context_lens, new_lens,  block_table, free_blocks,   free_head,
                        seq_lens,     query_starts, positions, slots,        free_head_out,
                        num_requests, table_width, num_free,   block_size,   num_tokens};
  const int smem = (2 * num_requests + 1) * (int)sizeof(int);
  cudaError_t e = ensure_smem(build_tables_kernel, smem, dev->ordinal);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(build_tables)");
  const int grid = std::max(1, std::min(dev->sms, (num_tokens + kTabThreads - 1) / kTabThreads));
  e = launch(build_tables_kernel, dim3(grid), dim3(kTabThreads), smem, static_cast<cudaStream_t>(stream_v),
             g_pdl_enabled != 0, a);
  return e == cudaSuccess ? GDSQ_OK : cuda_fail(e, "build_tables launch");
}

int gdsq_append_kv8(int elem_type, const void* q, long long q_token_stride, long long q_head_stride, const void* k,
                    long long k_token_stride, long long k_head_stride, const void* v, long long v_token_stride,
                    long long v_head_stride, void* q_out, const void* freqs, int max_position,
                    const long long* positions, const long long* slots, int num_tokens, int num_heads,
                    int num_kv_heads, int head_dim, int cache_type, void* k_cache, void* v_cache, float* k_scale,
                    float* v_scale, int num_blocks, int block_size, void* stream_v) {
  t_last_error.clear();
  if (elem_type != GDSQ_ELEM_F16 && elem_type != GDSQ_ELEM_BF16)
    return fail(GDSQ_ERR_INVALID_VALUE, "append_kv8: elem_type %d is not fp16 or bf16", elem_type);
  if (cache_type != GDSQ_CACHE_INT8 && cache_type != GDSQ_CACHE_E4M3)
    return fail(GDSQ_ERR_INVALID_VALUE, "append_kv8: cache_type %d is not int8 or e4m3", cache_type);
  if (num_tokens < 0 || num_heads < 0 || num_kv_heads < 1 || num_blocks < 0 || max_position < 0)
    return fail(GDSQ_ERR_INVALID_VALUE, "append_kv8: tokens %d, heads %d, kv heads %d, blocks %d, positions %d",
                num_tokens, num_heads, num_kv_heads, num_blocks, max_position);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(GDSQ_ERR_UNSUPPORTED, "append_kv8: head_dim %d is not 64, 128 or 256", head_dim);
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128)
    return fail(GDSQ_ERR_UNSUPPORTED, "append_kv8: block_size %d is not 16, 32, 64 or 128", block_size);
  if (num_tokens == 0) return GDSQ_OK;
  if (!k || !v || !slots || !k_cache || !v_cache || !k_scale || !v_scale || (freqs && !positions))
    return fail(GDSQ_ERR_INVALID_VALUE, "append_kv8: null pointer");
  if ((q != nullptr) != (q_out != nullptr) || (q && (!freqs || num_heads < 1)))
    return fail(GDSQ_ERR_INVALID_VALUE, "append_kv8: q and q_out go together, and need freqs and heads");
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(q, 16) || !aligned(q_out, 16) || q_token_stride % 8 != 0 ||
      q_head_stride % 8 != 0 || k_token_stride % 8 != 0 || k_head_stride % 8 != 0 || v_token_stride % 8 != 0 ||
      v_head_stride % 8 != 0)
    return fail(GDSQ_ERR_MISALIGNED, "append_kv8: q, k, v 16-byte alignment and strides multiples of 8 elements");
  if (!aligned(freqs, 16) || !aligned(positions, 8) || !aligned(slots, 8) || !aligned(k_cache, 128) ||
      !aligned(v_cache, 128) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return fail(GDSQ_ERR_MISALIGNED, "append_kv8: freqs 16-byte, positions and slots 8-byte, caches 128-byte, scales "
                "4-byte alignment");
  AppendArgs a = {q,         k,       v,         q_token_stride, q_head_stride, k_token_stride,
                  k_head_stride, v_token_stride, v_head_stride,  q_out,         static_cast<const float2*>(freqs),
                  positions, slots,   static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), k_scale, v_scale,
                  num_tokens, num_heads, num_kv_heads, num_blocks, __builtin_ctz(block_size), max_position};
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (elem_type == GDSQ_ELEM_F16)
    return cache_type == GDSQ_CACHE_INT8 ? launch_append<__half, GDSQ_CACHE_INT8>(a, head_dim, stream)
                                         : launch_append<__half, GDSQ_CACHE_E4M3>(a, head_dim, stream);
  return cache_type == GDSQ_CACHE_INT8 ? launch_append<__nv_bfloat16, GDSQ_CACHE_INT8>(a, head_dim, stream)
                                       : launch_append<__nv_bfloat16, GDSQ_CACHE_E4M3>(a, head_dim, stream);
}

}  // extern "C"
