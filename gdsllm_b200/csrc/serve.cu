// Kernels around the paged 8-bit cache of a batch of requests: the step's
// block table and slot map (gdsq_build_tables), the cache write with RoPE
// (gdsq_append_kv8) and the token choice (gdsq_sample).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
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

constexpr int kTabThreads = 1024;
constexpr int kTabMaxRequests = 16384;

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
  __shared__ int wsum[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait_primary();
  const int head = *p.free_head;
  const int per = (p.requests + kTabThreads - 1) / kTabThreads;
  const int r0 = min(tid * per, p.requests), r1 = min(r0 + per, p.requests);
  int tok = 0, blk = 0;
  bool bad = head < 0;
  for (int r = r0; r < r1; ++r) {
    const int c = max(p.context[r], 0), n = max(p.fresh[r], 0);
    bad |= p.context[r] < 0 || p.fresh[r] < 0;
    starts[r] = tok;
    first[r] = blk;
    tok += n;
    blk += (c + n + p.block - 1) / p.block - (c + p.block - 1) / p.block;
  }
  int ts = tok, bsum = blk;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, ts, d), b = __shfl_up_sync(0xffffffffu, bsum, d);
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
  int tb = ts - tok, bb = bsum - blk, tall = 0, ball = 0;
  for (int w = 0; w < kTabThreads / 32; ++w) {
    if (w < warp) {
      tb += wsum[0][w];
      bb += wsum[1][w];
    }
    tall += wsum[0][w];
    ball += wsum[1][w];
  }
  for (int r = r0; r < r1; ++r) {
    starts[r] += tb;
    first[r] += head + bb;
  }
  if (tid == 0) starts[p.requests] = tall;
  __syncthreads();

  auto free_block = [&](int i) { return i >= 0 && i < p.num_free ? p.free_blocks[i] : -1; };
  const int gw = blockIdx.x * (kTabThreads / 32) + warp;
  for (int r = gw; r < p.requests; r += gridDim.x * (kTabThreads / 32)) {
    const int c = max(p.context[r], 0), n = starts[r + 1] - starts[r];
    const int held = (c + p.block - 1) / p.block, after = (c + n + p.block - 1) / p.block;
    for (int j = held + lane; j < min(after, p.width); j += 32) {
      const int b = free_block(first[r] + j - held);
      bad |= b < 0;
      p.table[(size_t)r * p.width + j] = b;
    }
    bad |= after > p.width;
    if (lane == 0) {
      p.seq_lens[r] = c + n;
      p.starts[r] = starts[r];
      if (r == 0) {
        p.starts[p.requests] = tall;
        *p.head_out = head + ball;
      }
    }
  }
  bad |= tall > p.tokens;
  const long long stride = (long long)gridDim.x * kTabThreads;
  for (long long i = (long long)blockIdx.x * kTabThreads + tid; i < p.tokens; i += stride) {
    long long pos = 0, slot = -1;
    if (i < tall) {
      int lo = 0, hi = p.requests;  // the request with starts[lo] <= i < starts[lo + 1]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= i) lo = mid;
        else hi = mid;
      }
      const int c = max(p.context[lo], 0);
      pos = c + (i - starts[lo]);
      const int col = (int)(pos / p.block), held = (c + p.block - 1) / p.block;
      if (col < p.width) {
        const int b = col < held ? p.table[(size_t)lo * p.width + col] : free_block(first[lo] + col - held);
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

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }

template <int N, typename T>
__device__ __forceinline__ void load_row(const T* src, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = to_f32(src[i]);
}

// (a + ib)(c + id) as separate fp32 products and sums, rounded to T: the
// arithmetic of rotating the complex pairs in torch.
template <typename T, int N>
__device__ __forceinline__ void rotate(const float2* f, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 cs = f[i / 2];
    const float a = x[i], b = x[i + 1];
    x[i] = to_f32(from_f32<T>(__fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y))));
    x[i + 1] = to_f32(from_f32<T>(__fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(b, cs.x))));
  }
}

template <int F>
__device__ __forceinline__ uint8_t encode(float x) {
  if (!(x == x)) x = 0.f;
  if constexpr (F == GDSQ_CACHE_INT8) {
    return (uint8_t)(int8_t)(int)rintf(fminf(fmaxf(x, -127.f), 127.f));
  } else {
    return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  }
}
template <int F>
__device__ __forceinline__ float decode(uint8_t c) {
  if constexpr (F == GDSQ_CACHE_INT8) {
    return (float)(int8_t)c;
  } else {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
  }
}

// Grid (tokens, 1 + (q > 0)).  y = 0: a warp writes the whole of one (block,
// KV head, K or V) when the CTA's token is the first of its block; y = 1: the
// token's q heads are rotated.
template <typename T, int HD, int F>
__global__ void __launch_bounds__(kAppThreads) append_kv8_kernel(const AppendArgs p) {
  constexpr int N = HD / 32;
  constexpr float kTop = F == GDSQ_CACHE_INT8 ? 127.f : 448.f;
  const int i = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait_primary();
  const long long pos = p.freqs ? p.positions[i] : 0;
  const bool bad_pos = p.freqs && (pos < 0 || pos >= p.max_position);
  if (bad_pos && threadIdx.x == 0) record_device_error(kDevErrBadIndex);
  if (blockIdx.y == 1) {
    if (bad_pos) return;
    for (int h = warp; h < p.heads; h += kAppThreads / 32) {
      float x[N];
      load_row<N>(static_cast<const T*>(p.q) + i * p.q_token_stride + h * p.q_head_stride + lane * N, x);
      rotate<T, N>(p.freqs + pos * (HD / 2) + lane * (N / 2), x);
      T* dst = static_cast<T*>(p.q_out) + ((size_t)i * p.heads + h) * HD + lane * N;
#pragma unroll
      for (int e = 0; e < N; ++e) dst[e] = from_f32<T>(x[e]);
    }
    return;
  }
  const long long slot = p.slots[i];
  if (slot < 0) return;
  const long long page = slot >> p.block_shift;
  if (page >= p.num_blocks) {
    if (threadIdx.x == 0) record_device_error(kDevErrBadIndex);
    return;
  }
  if (i > 0 && p.slots[i - 1] >= 0 && (p.slots[i - 1] >> p.block_shift) == page) return;
  int n = 1;
  while (i + n < p.tokens && p.slots[i + n] >= 0 && (p.slots[i + n] >> p.block_shift) == page) ++n;
  const int bs = 1 << p.block_shift;
  const int begin = (int)(slot & (bs - 1));
  for (int u = warp; u < 2 * p.kv_heads; u += kAppThreads / 32) {
    const bool is_v = u >= p.kv_heads;
    const int h = is_v ? u - p.kv_heads : u;
    const T* src = static_cast<const T*>(is_v ? p.v : p.k) + h * (is_v ? p.v_head_stride : p.k_head_stride) + lane * N;
    const long long ts = is_v ? p.v_token_stride : p.k_token_stride;
    float* scale = (is_v ? p.v_scale : p.k_scale) + page * p.kv_heads + h;
    uint8_t* dst = (is_v ? p.v_cache : p.k_cache) + ((size_t)page * p.kv_heads + h) * bs * HD + lane * N;
    auto row = [&](int j, float(&x)[N]) {
      load_row<N>(src + (long long)(i + j) * ts, x);
      if (!is_v && p.freqs) {
        const long long pj = p.positions[i + j];
        if (pj >= 0 && pj < p.max_position) rotate<T, N>(p.freqs + pj * (HD / 2) + lane * (N / 2), x);
      }
    };
    uint32_t most = 0;  // magnitudes order as their bits do, inf and NaN on top
    for (int j = 0; j < n; ++j) {
      float x[N];
      row(j, x);
#pragma unroll
      for (int e = 0; e < N; ++e) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    const float base = begin == 0 ? 0.f : *scale;
    float need = __fmul_rn(__uint_as_float(most), 1.f / kTop);
    if (need < kSmallestScale) need = 0.f;
    float s = need <= base ? base : fmaxf(need, 2.f * base);
    if (most >= 0x7f800000u || !(base == base)) s = __int_as_float(0x7fc00000);
    const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
    __syncwarp();
    if (s != base && begin > 0) {
      const float ratio = __fmul_rn(base, inv);
      for (int j = 0; j < begin; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) dst[(size_t)j * HD + e] = encode<F>(__fmul_rn(decode<F>(dst[(size_t)j * HD + e]), ratio));
    }
    if (lane == 0) *scale = s;
    for (int j = 0; j < n; ++j) {
      float x[N];
      row(j, x);
      const int off = (int)(p.slots[i + j] & (bs - 1));
#pragma unroll
      for (int e = 0; e < N; ++e) dst[(size_t)off * HD + e] = encode<F>(__fmul_rn(x[e], inv));
    }
  }
}

// ---------------------------------------------------------------------------
// Sampling.
//
// e_i = exp((l_i - max) / T) and the whole-number weight w_i = floor(2^31 e_i):
// sums of weights are exact, so neither the order of additions nor the number
// of threads can change the token.  A NaN logit counts as -inf; one equal to
// the maximum has e = 1 (so +inf logits share the choice).  In the order
// (logit descending, index ascending) the kept tokens are the longest prefix
// inside the first top_k, with the weight before it below top_p of the
// top_k's, and with e >= min_p; the first is always kept.  The token is the
// first kept index, in index order, whose running sum exceeds floor(u * sum).

// A row lives in the shared memory of one cluster: thread i of the cluster owns
// the 32 logits from 32 i (counted from the 16-byte boundary below the row), so
// that index order is thread order, and the logits are read once.  The work is
// one exponential per logit where the whole weight is needed (no filter, or
// top-p alone), else a comparison.
//
// With filters few tokens can be kept, and those that can are copied to one
// CTA's list, which chooses alone while the others leave:
//   top_k   each CTA finds a value that ceil(k / CTAs) of its threads' maxima
//           reach; k logits of the row reach the lowest of these values
//   top_p   tokens of weight below (1 - p) W / V cannot add up to what is left out
//   min_p   the value itself
//   any     a token of weight 0 never matters
// A longer list than fits is worked on where it lies, by all of them.
//
// A cut (top_k by count, top_p by weight) is found by histograms over the
// distance of a logit's ordered bit pattern from the maximum's: 2048 bins over
// the span of the candidates, then 2048 inside the bin where the cut falls,
// until a bin is one logit value; ties then follow from counts alone.  A list
// of up to 256 is ordered by comparing all pairs instead, in one pass.

constexpr int kSampleItems = 32;  // logits per thread
constexpr int kSampleBins = 2048;
constexpr int kSampleShort = 256;  // lists up to here are ordered by comparing all pairs
constexpr float kWeightCut = -21.6f;  // floor(2^31 exp(z)) = 0 below (ln 2^-31 = -21.49)

struct SampleArgs {
  const void* logits;
  long long row_stride;
  const float* uniforms;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  long long* tokens;
  float* logprobs;
  int vocab;
};

// Orders floats as unsigned numbers do; NaN becomes -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (!(x == x)) x = -INFINITY;
  x += 0.f;  // -0 equals +0
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The logits of one CTA in shared memory, 16-byte vectors in an order in which
// lanes write neighbouring vectors and read their own stretch of 32 logits
// without bank conflicts.
template <typename T>
struct SampleRow {
  static constexpr int kVec = 16 / sizeof(T);           // logits per vector
  static constexpr int kVecs = kSampleItems / kVec;     // vectors per thread
  static constexpr int kDrop = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16;  // low bits of the fp32 pattern that say nothing
  uint32_t at;  // shared address

  static __device__ __forceinline__ uint32_t place(uint32_t v) { return (v ^ ((v >> 3) & (kVecs - 1))) << 4; }

  // Vectors first .. of the row, counted from the 16-byte boundary at or below its start; what lies outside becomes -inf.
  // Returns the largest of what this thread loaded, NaN aside.
  __device__ __forceinline__ float load(const T* row, int skew, int first, int vocab, int threads) const {
    float most = -INFINITY;
    constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int v = j * threads + threadIdx.x;
      const long long i = (long long)(first + v) * kVec - skew;
      uint4 x = make_uint4(kNone, kNone, kNone, kNone);
      if (i >= 0 && i + kVec <= vocab) {
        x = __ldg(reinterpret_cast<const uint4*>(row + i));
      } else if (i + kVec > 0 && i < vocab) {
        T e[kVec];
#pragma unroll
        for (int y = 0; y < kVec; ++y) e[y] = i + y >= 0 && i + y < vocab ? row[i + y] : from_f32<T>(-INFINITY);
        memcpy(&x, e, 16);
      }
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at + place(v)), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w)
                   : "memory");
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) most = fmaxf(most, __uint_as_float(w[e]));
      } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        T2 m[4];
        memcpy(m, w, 16);
        m[0] = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
        most = fmaxf(most, fmaxf(to_f32(m[0].x), to_f32(m[0].y)));
      }
    }
    return most;
  }

  __device__ __forceinline__ float get(int i) const {  // this thread's i-th
    const uint32_t a = at + place(threadIdx.x * kVecs + i / kVec) + (i % kVec) * (uint32_t)sizeof(T);
    if constexpr (sizeof(T) == 4) {
      return lds32f(a);
    } else {
      unsigned short v;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
      T x;
      memcpy(&x, &v, 2);
      return to_f32(x);
    }
  }

  // f(i, logit) for this thread's 32 logits in index order.
  template <typename Fn>
  __device__ __forceinline__ void each(Fn f) const {
#pragma unroll 1
    for (int j = 0; j < kVecs; ++j) {
      const uint4 x = lds128(at + place(threadIdx.x * kVecs + j));
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        float v;
        if constexpr (sizeof(T) == 4) v = __uint_as_float(w[e]);
        else if constexpr (std::is_same<T, __half>::value) v = __half2float(__ushort_as_half((unsigned short)(w[e >> 1] >> (16 * (e & 1)))));
        else v = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
        f(j * kVec + e, v);
      }
    }
  }
};

struct SampleShared {
  alignas(16) uint32_t lo[kSampleBins];  // counts, or low halves of weights
  alignas(16) uint32_t hi[kSampleBins];  // high halves of weights
  unsigned long long sum[32];
  uint32_t num[32];
  // by cluster rank, each written once
  uint32_t rank_top[16];
  uint32_t rank_bound[16];
  uint32_t rank_count[16];
  unsigned long long rank_total[16];
  unsigned long long rank_sum[16];
  uint32_t rank_ties[16];
  // the histogram's answer, written by the cluster's first CTA
  uint32_t bin;
  uint32_t found;
  unsigned long long before, at;
};

// Tokens that the list of one CTA holds.
template <typename T>
constexpr int kSampleList = sizeof(T) == 4 ? 2048 : 4096;

// Grid: one cluster per row.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) sample_kernel(const SampleArgs p, const int ranks) {
  using Items = SampleRow<T>;
  constexpr int kWarps = kThreads / 32;
  __shared__ SampleShared sh;
  extern __shared__ __align__(16) unsigned char logits_smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = ranks > 1 ? (int)(blockIdx.x % ranks) : 0;
  const int b = blockIdx.x / ranks;
  const int V = p.vocab;
  int team = ranks;   // CTAs that work on the row: all of them, or the first alone
  bool solo = false;  // on the list
  auto everyone = [&] {
    if (team > 1) cluster_sync_all();
    else __syncthreads();
  };
  // Stores `v` to *slot in every CTA of the cluster; one warp calls it.
  auto tell_u64 = [&](unsigned long long* slot, unsigned long long v) {
    if (team == 1) {
      if (lane == 0) *slot = v;
    } else if (lane < team) {
      st_cluster_u64(map_to_rank(slot, lane), v);
    }
  };
  auto tell_u32 = [&](uint32_t* slot, uint32_t v) {
    if (team == 1) {
      if (lane == 0) *slot = v;
    } else if (lane < team) {
      st_cluster_u32(map_to_rank(slot, lane), v);
    }
  };
  // Sum over the cluster, the same in every thread; called once at most.
  auto total = [&](unsigned long long v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if (lane == 0) sh.sum[warp] = v;
    __syncthreads();
    if (warp == 0) {
      v = lane < kWarps ? sh.sum[lane] : 0;
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
      tell_u64(&sh.rank_total[rank], v);
    }
    everyone();
    v = 0;
    for (int r = 0; r < team; ++r) v += sh.rank_total[r];
    return v;
  };

  if (ranks > 1) cluster_arrive_relaxed();  // waited for before the first store to a peer
  pdl_launch_dependents();
  pdl_wait_primary();
  const T* row = static_cast<const T*>(p.logits) + (long long)b * p.row_stride;
  const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int base = (rank * kThreads + tid) * kSampleItems - skew;  // index of this thread's first logit
  const Items x{smem_addr(logits_smem)};
  const float own_most = x.load(row, skew, rank * kThreads * Items::kVecs, V, kThreads);
  uint32_t* list_value = reinterpret_cast<uint32_t*>(logits_smem + kThreads * kSampleItems * sizeof(T));
  int* list_index = reinterpret_cast<int*>(list_value + kSampleList<T>);
  const float temp = p.temperature ? p.temperature[b] : 1.f;
  const bool greedy = !(temp > 0.f);
  const float inv = greedy ? 1.f : __frcp_rn(temp);
  const float mp = p.min_p ? p.min_p[b] : 0.f;
  const float tp = p.top_p ? p.top_p[b] : 1.f;
  const float u = p.uniforms[b];
  int k = p.top_k ? p.top_k[b] : 0;
  if (greedy || mp > 1.f || !(mp == mp)) k = 1;  // min_p above 1: nothing but the first passes
  if (k <= 0 || k > V) k = V;

  // The maximum, and for top_k a value that `share` of this CTA's threads' maxima reach.
  const uint32_t own_top = order_key(own_most);
  const int share = (k + ranks - 1) / ranks;
  const bool by_count = k > 1 && k < V;
  {
    const uint32_t w = __reduce_max_sync(0xffffffffu, own_top);
    if (lane == 0) sh.num[warp] = w;
    if (by_count && share <= kThreads)
      for (int i = tid; i < kSampleBins; i += kThreads) sh.lo[i] = 0;
    if (tid == 0) sh.found = 0;
    __syncthreads();
    const uint32_t cta_top = __reduce_max_sync(0xffffffffu, lane < kWarps ? sh.num[lane] : 0);
    float bound = -INFINITY;
    if (by_count && share <= kThreads) {
      // bins of equal width in the logit, down to where weights vanish
      const float high = key_value(cta_top), width = -kWeightCut / inv / kSampleBins;
      const float d = (high - own_most) / width;
      if (d < (float)kSampleBins) atomicAdd(&sh.lo[(int)d], 1u);
      __syncthreads();
      constexpr int kPer = kSampleBins / kThreads;
      uint32_t n[kPer], sum = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) sum += n[j] = sh.lo[tid * kPer + j];
      uint32_t upto = sum;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, upto, s);
        if (lane >= s) upto += a;
      }
      if (lane == 31) sh.num[warp] = upto;
      __syncthreads();
      uint32_t at = upto - sum;
      for (int w2 = 0; w2 < warp; ++w2) at += sh.num[w2];
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (at < (uint32_t)share && at + n[j] >= (uint32_t)share) {
          sh.bin = tid * kPer + j;
          sh.found = 1;
        }
        at += n[j];
      }
      __syncthreads();
      if (sh.found) {
        const float far = (float)(sh.bin + 1) * width;
        bound = high - far - 1e-5f * (fabsf(high) + far);
        if (!(bound == bound)) bound = -INFINITY;
      }
    }
    if (ranks > 1) cluster_wait();
    if (warp == 0) {
      tell_u32(&sh.rank_top[rank], cta_top);
      tell_u32(&sh.rank_bound[rank], order_key(bound));
    }
    everyone();
  }
  uint32_t top = 0;
  for (int r = 0; r < ranks; ++r) top = max(top, sh.rank_top[r]);
  const float most = key_value(top);
  if (most == -INFINITY) {  // the whole cluster leaves
    if (rank == 0 && tid == 0) {
      p.tokens[b] = -1;
      if (p.logprobs) p.logprobs[b] = -INFINITY;
    }
    return;
  }
  auto z_of = [&](float v) { return __fmul_rn(v - most, inv); };  // NaN for a NaN logit, for inf - inf and for 0 x inf
  auto e_of = [&](float v) { return v == most ? 1.f : expf(z_of(v)); };
  auto w_of = [&](float v) { return (uint32_t)(e_of(v) * 2147483648.f); };
  auto near = [&](float v, float cut) { return v == most || z_of(v) >= cut; };


  // This thread's whole weight.  Where the maximum and 1 / T are finite, the plain formula gives 1 at the maximum and 0 for -inf
  // and NaN by itself.
  const bool regular = isfinite(most) && isfinite(inv);
  auto own_weight = [&] {
    unsigned long long sum = 0;
    if (regular)
      x.each([&](int, float v) { sum += (uint32_t)(expf(z_of(v)) * 2147483648.f); });
    else
      x.each([&](int, float v) {
        if (near(v, kWeightCut)) sum += w_of(v);
      });
    return sum;
  };

  // The value where the running sum over falling logits reaches `want`: its distance
  // `first` from the maximum, `before` the sum over nearer ones, `at` the value's own.  each(f) calls f(logit) for the candidates,
  // which lie at distances below `span`; their share is their weight, or 1.
  // fix(from, to) is taken off the sum of the distances [from, to).
  struct Cut {
    uint32_t first;
    unsigned long long before, at;
    bool found;
  };
  const uint32_t top_key = top >> Items::kDrop;
  auto histogram = [&](unsigned long long want, uint32_t span, bool weights, auto each, auto fix) {
    Cut c{0, 0, 0, true};
    for (;;) {
      const int shift = max(0, 21 - __clz(span - 1));  // span <= 2048 << shift
      for (int i = tid; i < kSampleBins; i += kThreads) {
        sh.lo[i] = 0;
        sh.hi[i] = 0;
      }
      __syncthreads();
      each([&](float v) {
        const uint32_t d = top_key - (order_key(v) >> Items::kDrop) - c.first;
        if (d >= span) return;
        if (weights) {
          const uint32_t w = w_of(v);
          atomicAdd(&sh.lo[d >> shift], w & 0xffffu);
          atomicAdd(&sh.hi[d >> shift], w >> 16);
        } else {
          atomicAdd(&sh.lo[d >> shift], 1u);
        }
      });
      everyone();
      if (rank == 0) {
        constexpr int kPer = kSampleBins / kThreads;
        unsigned long long mine[kPer], sum = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          mine[j] = sh.lo[tid * kPer + j];
          if (weights) mine[j] += (unsigned long long)sh.hi[tid * kPer + j] << 16;
        }
#pragma unroll 4
        for (int r = 1; r < team; ++r)
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            mine[j] += ld_cluster_u32(map_to_rank(&sh.lo[tid * kPer + j], r));
            if (weights) mine[j] += (unsigned long long)ld_cluster_u32(map_to_rank(&sh.hi[tid * kPer + j], r)) << 16;
          }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const uint32_t bin = tid * kPer + j;
          mine[j] -= fix(c.first + (bin << shift), c.first + ((bin + 1) << shift));
          sum += mine[j];
        }
        unsigned long long upto = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const unsigned long long a = __shfl_up_sync(0xffffffffu, upto, d);
          if (lane >= d) upto += a;
        }
        if (lane == 31) sh.sum[warp] = upto;
        if (tid == 0) sh.found = 0;
        __syncthreads();
        unsigned long long at = c.before + upto - sum;
        for (int w = 0; w < warp; ++w) at += sh.sum[w];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (at < want && at + mine[j] >= want) {
            sh.bin = tid * kPer + j;
            sh.before = at;
            sh.at = mine[j];
            sh.found = 1;
          }
          at += mine[j];
        }
        __syncthreads();
        if (warp == 0 && team > 1) {
          const uint32_t bin = sh.bin, found = sh.found;
          const unsigned long long before = sh.before, in = sh.at;
          __syncwarp();
          tell_u32(&sh.bin, bin);
          tell_u32(&sh.found, found);
          tell_u64(&sh.before, before);
          tell_u64(&sh.at, in);
        }
      }
      everyone();
      c.found = sh.found != 0;
      if (!c.found) return c;
      c.before = sh.before;
      c.at = sh.at;
      c.first += sh.bin << shift;
      if (shift == 0) return c;
      span = 1u << shift;
    }
  };
  // Not above any logit with z >= cut.
  auto low_of = [&](float cut) {
    const float far = cut / inv;
    return isfinite(most) ? most + far - 1e-5f * (fabsf(most) + fabsf(far)) : -INFINITY;
  };
  // More than the distance of any logit that is at least `low`.
  auto span_of = [&](float low) { return top_key - min(order_key(low) >> Items::kDrop, top_key) + 2; };
  auto no_fix = [](uint32_t, uint32_t) { return 0ull; };
  const bool by_weight = k > 1 && (tp < 1.f || !(tp == tp));
  const float min_cut = mp > 0.f ? fmaxf(kWeightCut, logf(mp) - 1e-3f) : kWeightCut;
  auto limit_of = [&](unsigned long long all) {
    const double lim = (double)tp * (double)all;
    return lim > 1.0 ? (unsigned long long)ceil(lim) : 1ull;
  };

  auto target_of = [&](unsigned long long whole) {
    const double d = (double)u * (double)whole;
    return min(d > 0.0 ? (unsigned long long)d : 0ull, whole - 1);
  };

  // No candidate lies below `low`; the list.
  float low = low_of(kWeightCut);
  unsigned long long all = 0;
  if (by_count) {
    uint32_t bound = 0xffffffffu;
    for (int r = 0; r < ranks; ++r) bound = min(bound, sh.rank_bound[r]);
    low = fmaxf(low, key_value(bound));
    if (!by_weight) low = fmaxf(low, low_of(min_cut));
  } else if (by_weight) {
    all = total(own_weight());
    const float least = 0.99f * (1.f - tp) * (float)all / (float)V;
    if (least > 1.f) low = fmaxf(low, low_of(logf(least * 4.656612873077393e-10f) - 1e-3f));
    low = fmaxf(low, low_of(min_cut));
  } else if (k > 1) {
    low = fmaxf(low, low_of(min_cut));
  }
  int list = 0;
  if (by_count || by_weight || (k > 1 && mp > 0.f)) {
    uint32_t mask = 0;
    x.each([&](int i, float v) { mask |= (uint32_t)(v >= low) << i; });
    const int n = __popc(mask);
    int upto = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += a;
    }
    __syncthreads();
    if (lane == 31) sh.num[warp] = upto;
    __syncthreads();
    if (warp == 0) {
      const uint32_t c = __reduce_add_sync(0xffffffffu, lane < kWarps ? sh.num[lane] : 0);
      tell_u32(&sh.rank_count[rank], c);
    }
    everyone();
    int at = upto - n;
    for (int w = 0; w < warp; ++w) at += sh.num[w];
    for (int r = 0; r < ranks; ++r) {
      if (r < rank) at += sh.rank_count[r];
      list += sh.rank_count[r];
    }
    if (list <= kSampleList<T>) {
      for (; mask; mask &= mask - 1, ++at) {
        const int i = __ffs(mask) - 1;
        const uint32_t v = __float_as_uint(x.get(i));
        if (ranks == 1) {
          list_value[at] = v;
          list_index[at] = base + i;
        } else {
          st_cluster_u32(map_to_rank(list_value + at, 0), v);
          st_cluster_u32(map_to_rank(list_index + at, 0), (uint32_t)(base + i));
        }
      }
      everyone();
      if (rank != 0) return;
      solo = true;
      team = 1;
    }
  }
  // A short list: one thread per candidate compares it with all others, which gives its place and the weight before it at once.
  if (solo && list <= kSampleShort) {
    const bool live = tid < list;
    const float v = live ? __uint_as_float(list_value[tid]) : -INFINITY;
    const uint32_t key = order_key(v);
    const float e = live ? e_of(v) : 0.f;
    const uint32_t w = (uint32_t)(e * 2147483648.f);
    if (tid < kSampleShort) {
      sh.lo[tid] = live ? key : 0;
      sh.hi[tid] = w;
    }
    __syncthreads();
    uint32_t place = 0;
    unsigned long long ahead = 0;
    if (warp * 32 < list) {
      const uint32_t keys = smem_addr(sh.lo), weights = smem_addr(sh.hi);
      for (int j = 0; j < list; j += 4) {
        const uint4 kj = lds128(keys + 4 * j), wj = lds128(weights + 4 * j);
        const uint32_t kk[4] = {kj.x, kj.y, kj.z, kj.w}, ww[4] = {wj.x, wj.y, wj.z, wj.w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const bool first = kk[y] > key || (kk[y] == key && j + y < tid);
          place += first;
          ahead += first ? ww[y] : 0;
        }
      }
    }
    auto block_sum = [&](unsigned long long s) {
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
      if (lane == 0) sh.sum[warp] = s;
      __syncthreads();
      s = 0;
      for (int i = 0; i < kSampleShort / 32; ++i) s += sh.sum[i];
      return s;
    };
    bool keep = live && place < (uint32_t)k;
    if (by_weight) {
      if (by_count) all = block_sum(keep ? w : 0);
      keep = keep && ahead < limit_of(all);
    }
    keep = keep && (e >= mp || place == 0);
    unsigned long long upto = keep ? w : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned long long a = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += a;
    }
    __syncthreads();
    if (lane == 31) sh.sum[warp] = upto;
    __syncthreads();
    unsigned long long whole = 0;
    for (int i = 0; i < kSampleShort / 32; ++i) {
      if (i < warp) upto += sh.sum[i];
      whole += sh.sum[i];
    }
    const unsigned long long target = target_of(whole);
    if (keep && upto - w <= target && target < upto) {
      p.tokens[b] = list_index[tid];
      if (p.logprobs) p.logprobs[b] = logf((float)((double)w / (double)whole));
    }
    return;
  }
  // fn(i, logit) for the candidates of this thread: a stretch of the list, or its own logits.
  const int list_per = (list + kThreads - 1) / kThreads, list_at = min(tid * list_per, list), list_end = min(list_at + list_per, list);
  auto walk = [&](auto fn) {
    if (solo) {
      for (int i = list_at; i < list_end; ++i) fn(i - list_at, __uint_as_float(list_value[i]));
    } else {
      x.each([&](int i, float v) {
        if (v >= low) fn(i, v);
      });
    }
  };

  // kept: keys above `thr`, and the first `ties` (in index order) of those equal to it
  uint32_t thr = 0, ties = 0xffffffffu;
  unsigned long long tied = 0;  // how many there are
  bool cut_k = false;
  if (k == 1) {
    thr = top_key;
    ties = 1;
    cut_k = true;
  } else if (by_count) {
    const Cut c = histogram(k, span_of(low), false, [&](auto f) {
      walk([&](int, float v) {
        if (near(v, kWeightCut)) f(v);
      });
    }, no_fix);
    if (c.found) {
      thr = top_key - c.first;
      ties = k - (uint32_t)c.before;
      tied = c.at;
      cut_k = true;
    }
  }
  // the logit whose key is `thr`
  auto value_of = [&](uint32_t key) {
    const uint32_t full = key << Items::kDrop;
    return key_value(full & 0x80000000u ? full : full | ((1u << Items::kDrop) - 1));
  };
  if (by_weight) {
    const float at_thr = value_of(thr);
    const unsigned long long w_thr = cut_k ? w_of(at_thr) : 0;
    float from = low;
    if (by_count) {
      unsigned long long own = 0;
      walk([&](int, float v) {
        if ((order_key(v) >> Items::kDrop) > thr && near(v, kWeightCut)) own += w_of(v);
      });
      all = total(own) + (cut_k ? ties * w_thr : 0);
      if (cut_k) from = at_thr;
    }
    const unsigned long long limit = limit_of(all);
    const uint32_t at = top_key - thr;
    const unsigned long long extra = cut_k && near(at_thr, kWeightCut) ? (tied - ties) * w_thr : 0;
    const Cut c = histogram(limit, span_of(from), true, [&](auto f) {
      walk([&](int, float v) {
        if (v >= from && near(v, kWeightCut)) f(v);
      });
    }, [&](uint32_t lo, uint32_t hi) { return extra && lo <= at && at < hi ? extra : 0ull; });
    if (c.found) {
      const uint32_t key = top_key - c.first;
      const unsigned long long w = w_of(value_of(key));
      const uint32_t n = (uint32_t)min((limit - c.before + w - 1) / w, 0xffffffffull);
      ties = cut_k && key == thr ? min(ties, n) : n;
      thr = key;
    }
  }

  // Running sums of the kept weight in index order.
  unsigned long long own = 0;
  uint32_t own_ties = 0;
  if (thr == 0 && !(mp > 0.f) && !solo)
    own = own_weight();
  else
    walk([&](int, float v) {
      const uint32_t key = order_key(v) >> Items::kDrop;
      if (key < thr || !near(v, min_cut)) return;
      const float e = e_of(v);
      if (!(e >= mp) && v != most) return;
      if (key == thr) ++own_ties;
      else own += (uint32_t)(e * 2147483648.f);
    });
  unsigned long long upto = own;
  uint32_t upto_ties = own_ties;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned long long a = __shfl_up_sync(0xffffffffu, upto, d);
    const uint32_t c = __shfl_up_sync(0xffffffffu, upto_ties, d);
    if (lane >= d) {
      upto += a;
      upto_ties += c;
    }
  }
  __syncthreads();
  if (lane == 31) {
    sh.sum[warp] = upto;
    sh.num[warp] = upto_ties;
  }
  __syncthreads();
  if (warp == 0) {
    unsigned long long a = lane < kWarps ? sh.sum[lane] : 0;
    uint32_t c = lane < kWarps ? sh.num[lane] : 0;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) a += __shfl_xor_sync(0xffffffffu, a, m);
    c = __reduce_add_sync(0xffffffffu, c);
    tell_u64(&sh.rank_sum[rank], a);
    tell_u32(&sh.rank_ties[rank], c);
  }
  everyone();
  unsigned long long before = upto - own, sum = 0;
  unsigned long long ties_before = upto_ties - own_ties, ties_all = 0;
  for (int w = 0; w < warp; ++w) {
    before += sh.sum[w];
    ties_before += sh.num[w];
  }
  for (int r = 0; r < team; ++r) {
    if (r < rank) {
      before += sh.rank_sum[r];
      ties_before += sh.rank_ties[r];
    }
    sum += sh.rank_sum[r];
    ties_all += sh.rank_ties[r];
  }
  const unsigned long long w_thr = ties_all ? w_of(value_of(thr)) : 0, most_ties = ties;
  const unsigned long long whole = sum + min(ties_all, most_ties) * w_thr;
  const unsigned long long end = before + own + min(ties_before + own_ties, most_ties) * w_thr;
  before += min(ties_before, most_ties) * w_thr;
  const unsigned long long target = target_of(whole);
  if (before <= target && target < end) {  // this thread holds the token
    int chosen = -1;
    uint32_t weight = 0;
    walk([&](int i, float v) {
      const uint32_t key = order_key(v) >> Items::kDrop;
      if (chosen >= 0 || key < thr || !near(v, min_cut)) return;
      const float e = e_of(v);
      if (!(e >= mp) && v != most) return;
      if (key == thr && ties_before++ >= most_ties) return;
      weight = (uint32_t)(e * 2147483648.f);
      before += weight;
      if (before > target) chosen = i;
    });
    p.tokens[b] = solo ? list_index[list_at + chosen] : base + chosen;
    if (p.logprobs) p.logprobs[b] = logf((float)((double)weight / (double)whole));
  }
}

// Threads per CTA and CTAs per row: as few CTAs as hold the row, so that a row
// of up to 32768 logits needs no barrier across CTAs; smaller CTAs, two to an
// SM, where a row takes a cluster anyway.
template <typename T>
int launch_sample(const SampleArgs& a, int rows, cudaStream_t stream) {
  // and what lies between a row's start and the 16-byte boundary below it
  const int skew = (a.row_stride * sizeof(T)) % 16 == 0 || rows == 1
                       ? (int)((reinterpret_cast<uintptr_t>(a.logits) & 15) / sizeof(T))
                       : SampleRow<T>::kVec - 1;
  const int n = a.vocab + skew;
  const bool small = n <= 512 * kSampleItems, wide = n > 8 * 512 * kSampleItems || (!small && n <= 1024 * kSampleItems);
  const int threads = wide ? 1024 : 512;
  int ranks = 1;
  while (ranks * threads * kSampleItems < n) ranks *= 2;
  auto kernel = wide ? sample_kernel<T, 1024> : sample_kernel<T, 512>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * ranks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = (size_t)threads * kSampleItems * sizeof(T) + (size_t)kSampleList<T> * 8;
  cfg.stream = stream;
  const DeviceInfo* dev = nullptr;
  const int st = device_info(&dev);
  if (st != GDSQ_OK) return st;
  cudaError_t e = ensure_smem(kernel, (int)(cfg.dynamicSmemBytes + sizeof(SampleShared)), dev->ordinal);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(sample)");
  cudaLaunchAttribute attr[2];
  int n_attr = 0;
  if (ranks > 1) {
    attr[n_attr].id = cudaLaunchAttributeClusterDimension;
    attr[n_attr].val.clusterDim.x = ranks;
    attr[n_attr].val.clusterDim.y = 1;
    attr[n_attr].val.clusterDim.z = 1;
    ++n_attr;
  }
  if (g_pdl_enabled) {
    attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n_attr].val.programmaticStreamSerializationAllowed = 1;
    ++n_attr;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n_attr;
  if (ranks > 8) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(sample)");
  }
  e = cudaLaunchKernelEx(&cfg, kernel, a, ranks);
  return e == cudaSuccess ? GDSQ_OK : cuda_fail(e, "sample launch");
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

template <typename T, int F>
int launch_append(const AppendArgs& a, int head_dim, cudaStream_t stream) {
  const dim3 grid(a.tokens, a.q_out ? 2 : 1);
  auto kernel = head_dim == 64    ? append_kv8_kernel<T, 64, F>
                : head_dim == 128 ? append_kv8_kernel<T, 128, F>
                                  : append_kv8_kernel<T, 256, F>;
  cudaError_t e = launch(kernel, grid, dim3(kAppThreads), 0, stream, g_pdl_enabled != 0, a);
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
      num_tokens < 0)
    return fail(GDSQ_ERR_INVALID_VALUE, "build_tables: requests %d (1..%d), table width %d, free blocks %d, block "
                "size %d, tokens %d", num_requests, kTabMaxRequests, table_width, num_free, block_size, num_tokens);
  if (!context_lens || !new_lens || (!block_table && table_width) || (!free_blocks && num_free) || !free_head ||
      !seq_lens || !query_starts || (num_tokens && (!positions || !slots)) || !free_head_out)
    return fail(GDSQ_ERR_INVALID_VALUE, "build_tables: null pointer");
  if (free_head == free_head_out)
    return fail(GDSQ_ERR_INVALID_VALUE, "build_tables: free_head_out must not be free_head");
  if (!aligned(context_lens, 4) || !aligned(new_lens, 4) || !aligned(block_table, 4) || !aligned(free_blocks, 4) ||
      !aligned(free_head, 4) || !aligned(seq_lens, 4) || !aligned(query_starts, 4) || !aligned(positions, 8) ||
      !aligned(slots, 8) || !aligned(free_head_out, 4))
    return fail(GDSQ_ERR_MISALIGNED, "build_tables: 4-byte (positions and slots 8-byte) alignment");
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

int gdsq_sample(int elem_type, const void* logits, long long row_stride, int num_rows, int vocab,
                const float* uniforms, const float* temperature, const int32_t* top_k, const float* top_p,
                const float* min_p, long long* tokens, float* logprobs, void* stream_v) {
  t_last_error.clear();
  if (elem_type != GDSQ_ELEM_F16 && elem_type != GDSQ_ELEM_BF16 && elem_type != GDSQ_ELEM_F32)
    return fail(GDSQ_ERR_INVALID_VALUE, "sample: elem_type %d is not fp16, bf16 or fp32", elem_type);
  if (num_rows < 0 || vocab < 1 || vocab > GDSQ_SAMPLE_MAX_VOCAB || row_stride < 0)
    return fail(GDSQ_ERR_INVALID_VALUE, "sample: rows %d, vocab %d (1..%d), row stride %lld", num_rows, vocab,
                GDSQ_SAMPLE_MAX_VOCAB, row_stride);
  if (num_rows == 0) return GDSQ_OK;
  if (!logits || !uniforms || !tokens) return fail(GDSQ_ERR_INVALID_VALUE, "sample: null pointer");
  if (!aligned(logits, elem_type == GDSQ_ELEM_F32 ? 4 : 2) || !aligned(uniforms, 4) || !aligned(temperature, 4) ||
      !aligned(top_k, 4) || !aligned(top_p, 4) || !aligned(min_p, 4) || !aligned(tokens, 8) || !aligned(logprobs, 4))
    return fail(GDSQ_ERR_MISALIGNED, "sample: logits to their own size, tokens 8-byte, the rest 4-byte alignment");
  const SampleArgs a = {logits, row_stride, uniforms, temperature, top_k, top_p, min_p, tokens, logprobs, vocab};
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (elem_type == GDSQ_ELEM_F16) return launch_sample<__half>(a, num_rows, stream);
  if (elem_type == GDSQ_ELEM_BF16) return launch_sample<__nv_bfloat16>(a, num_rows, stream);
  return launch_sample<float>(a, num_rows, stream);
}

}  // extern "C"
