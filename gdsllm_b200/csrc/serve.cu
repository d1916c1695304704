// Kernels around the paged 8-bit cache of a batch of requests: the step's
// block table and slot map (gdsq_build_tables) and the cache write with RoPE
// (gdsq_append_kv8).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

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

}  // extern "C"
