// Attention over a paged cache held in 8 bits (gdsq_attend_kv8).
//
// The cache is [blocks][kv_heads][block_size][head_dim] of int8 or e4m3
// codes with one fp32 scale per (block, kv head) for K and one for V.  A
// request's tokens sit in the blocks its row of the block table names; its n
// new tokens are the last n of its len tokens, and query i sees the positions
// j <= len - n + i:
//
//   s_ij = scale * ks[page(j)] * sum_d q_id kq_jd
//   o_i  = sum_j softmax_j(s_ij) * vs[page(j)] * vq_j
//
// A query that sees nothing gives zeros.  Query heads h * G .. h * G + G - 1
// share KV head h, so the G heads of the n new tokens are the n * G rows of
// one matrix product per (request, KV head).
//
// Products run on 16-bit matrix instructions with fp32 sums.  Every code is
// exact in fp16 (an e4m3 code as value * 2^-8), and a query row is scaled by a
// power of two to at most 1 before it becomes fp16, so the only operand that
// is rounded is the softmax weight (11 bits, as the output has).
//
// One pass with a running maximum: with lv = log2(vs[page]), a weight is
// p_j = 2^(s_j log2(e) + lv - r), r the running maximum of s_j log2(e) + lv.
// p_j is at most 1 whatever the scales are, sum p_j vq_j needs no scale of its
// own, and the softmax's denominator is sum p_j 2^-lv, kept from the fp32
// weights before they are rounded.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>

#include "gdsq.h"
#include "host.h"
#include "common.cuh"

namespace gdsq {
namespace {

constexpr int kAttWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMaxLogScale = 100.f;  // |log2| of a value scale is held to this

struct AttendArgs {
  const void* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int* table;
  const int* seq_lens;
  const int* starts;
  void* out;
  long long q_token_stride, q_head_stride;      // elements
  long long out_token_stride, out_head_stride;  // elements
  int requests, num_blocks, table_width;
  int kv_heads, group, block_shift;  // block_size = 1 << block_shift
  int tokens;                        // rows of q
  bool bf16;
  float scale;  // softmax scale * log2(e) * the code format's factor
};

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 8-bit codes to fp16 pairs.  kFactor * fp16 value = code value.
template <int F>
struct Code;

template <>
struct Code<GDSQ_CACHE_INT8> {
  static constexpr float kFactor = 1.f;
  static constexpr float kLogFactor = 0.f;
  // Bytes 0,1 and 2,3 of w.  1024 + (code + 128) is an fp16 bit pattern;
  // subtracting 1152 is exact.
  static __device__ __forceinline__ void unpack(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t t = w ^ 0x80808080u;
    const __half2 k1152 = u32_as_h2(0x64806480u);
    lo = h2_as_u32(__hsub2(u32_as_h2(__byte_perm(t, 0x64646464u, 0x4140)), k1152));
    hi = h2_as_u32(__hsub2(u32_as_h2(__byte_perm(t, 0x64646464u, 0x4342)), k1152));
  }
};

template <>
struct Code<GDSQ_CACHE_E4M3> {
  static constexpr float kFactor = 256.f;
  static constexpr float kLogFactor = 8.f;
  // seeeemmm to s0eeeemmm0000000: the fp16 with that exponent field is the
  // code's value * 2^-8, subnormal codes included.  The NaN codes become
  // 480 * 2^-8, so bytes past a request's end cannot reach a sum as NaN.
  static __device__ __forceinline__ uint32_t widen(uint32_t x) {  // codes in the high bytes
    return ((x & 0x7f007f00u) >> 1) | (x & 0x80008000u);
  }
  static __device__ __forceinline__ void unpack(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = widen(__byte_perm(w, 0, 0x1404));
    hi = widen(__byte_perm(w, 0, 0x3424));
  }
};

__device__ __forceinline__ float load_q(const AttendArgs& p, long long i) {
  return p.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.q)[i])
                : __half2float(static_cast<const __half*>(p.q)[i]);
}

// Per-page constants of the softmax: x = kscale factor, y = lv, z = 2^-lv.
__device__ __forceinline__ float3 page_constants(const AttendArgs& p, int page, int h, float log_factor) {
  const size_t i = (size_t)page * p.kv_heads + h;
  const float ks = p.k_scale[i], vs = p.v_scale[i];
  const bool fine = isfinite(vs);
  const float lv = fminf(fmaxf(log2f(vs) + log_factor, -kMaxLogScale), kMaxLogScale);
  // A non-finite scale marks a block that was written with non-finite values:
  // the queries that see it come out as NaN.
  return make_float3(ks * p.scale, fine ? lv : __int_as_float(0x7fffffff), fine ? exp2f(-lv) : 1.f);
}

// Grid (row tiles, kv_heads, requests), 4 warps.  A CTA owns 16 * MT rows of
// one (request, KV head); its warps take every fourth tile of 32 tokens and
// their sums are joined in shared memory at the end.
//
// Matrix operand layout: in m16n8k16 a lane (g = lane / 4, t = lane % 4) feeds
// B[k = 2t, 2t+1, 2t+8, 2t+9][n = g].  The order of the summed index is free,
// so for the scores (k = dim, n = token) lane t takes 32 consecutive dims of
// token g: two 16-byte loads.  For the output (k = token, n = dim) lane g
// takes 16 consecutive dims of tokens 2t, 2t+1, 2t+8, 2t+9.
template <int HD, int F, int MT>
__global__ void __launch_bounds__(kAttWarps * 32) attend_simple_kernel(const AttendArgs p) {
  constexpr int kParts = HD >= 128 ? HD / 128 : 1;  // 128-dim parts
  constexpr int kPart = HD >= 128 ? 128 : 64;
  constexpr int kWords = kPart / 16;   // 32-bit words of K per lane, token and part (= k16 steps)
  constexpr int kSteps = HD / 16;      // k16 steps of the scores
  constexpr int kTiles = HD / 8;       // n8 tiles of the output
  constexpr int kVWords = kPart / 32;  // 32-bit words of V per lane, token and part
  constexpr int kRows = 16 * MT;
  extern __shared__ __align__(16) unsigned char smem[];
  uint4* qf = reinterpret_cast<uint4*>(smem);                               // [MT][kSteps][32]
  float* qexp = reinterpret_cast<float*>(smem + MT * kSteps * 512);         // [kRows]
  int* qlim = reinterpret_cast<int*>(qexp + kRows);                         // [kRows] last visible position
  float* joined = reinterpret_cast<float*>(qlim + kRows);                   // [warps][kRows][HD]
  float* jm = joined + kAttWarps * kRows * HD;                              // [warps][kRows]
  float* jl = jm + kAttWarps * kRows;                                       // [warps][kRows]

  const int r = blockIdx.z, h = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  pdl_wait_primary();
  const int start = p.starts[r];
  const int n = min(p.starts[r + 1], p.tokens) - start;
  const int len = p.seq_lens[r];
  const int rows = n * p.group;
  const int row0 = blockIdx.x * kRows;
  if (start < 0 || row0 >= rows) return;

  // Q rows: power-of-two scale, fp16, in operand order.
  for (int i = warp; i < kRows; i += kAttWarps) {
    const int row = row0 + i;
    const int qi = row / p.group, gq = row % p.group;
    float v[HD / 32];
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) {
      const long long at = (long long)(start + qi) * p.q_token_stride +
                           (long long)(h * p.group + gq) * p.q_head_stride + lane * (HD / 32) + e;
      v[e] = row < rows ? load_q(p, at) : 0.f;
      most = fmaxf(most, fabsf(v[e]));
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m));
    int ex = (int)(__float_as_uint(most) >> 23) - 126;  // most < 2^ex
    ex = isfinite(most) ? min(max(ex, -100), 100) : 0;
    const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
    if (lane == 0) {
      qexp[i] = __uint_as_float((uint32_t)(127 + ex) << 23);
      qlim[i] = row < rows ? len - n + qi : -1;
    }
    // dim d: part, lane t = (d % kPart) / (2 kWords) ... see the layout above
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) {
      const int d = lane * (HD / 32) + e;
      const int part = d / kPart, dd = d % kPart;
      const int tt = dd / (4 * kWords), w = (dd / 4) % kWords, b = dd & 3;
      const int step = part * kWords + w;
      // a0: row g, k 2t,2t+1; a1: row g + 8; a2: row g, k 2t+8,2t+9; a3: row g + 8
      const int reg = ((i & 15) >> 3) + 2 * (b >> 1);
      const int ln = (i & 7) * 4 + tt;
      reinterpret_cast<__half*>(qf + ((i >> 4) * kSteps + step) * 32 + ln)[reg * 2 + (b & 1)] =
          __float2half_rn(v[e] * down);
    }
  }
  __syncthreads();

  float o[MT][kTiles][4];
  float m[MT][2], l[MT][2], qe[MT][2];
  int lim[MT][2];
  int last = -1;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][j][e] = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      m[mt][x] = -INFINITY;
      l[mt][x] = 0.f;
      qe[mt][x] = qexp[mt * 16 + x * 8 + g];
      lim[mt][x] = min(qlim[mt * 16 + x * 8 + g], len - 1);
    }
  }
  for (int i = 0; i < kRows; ++i) last = max(last, min(qlim[i], len - 1));
  const int kv_len = last + 1;
  const int bs_mask = (1 << p.block_shift) - 1;

  for (int j0 = warp * 32; j0 < kv_len; j0 += kAttWarps * 32) {
    size_t base[2];
    float3 pc[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int pos = min(j0 + 16 * hh, (kv_len - 1) & ~15);
      const int col = pos >> p.block_shift;
      int page = col < p.table_width ? p.table[(size_t)r * p.table_width + col] : -1;
      if ((unsigned)page >= (unsigned)p.num_blocks) {
        record_device_error(kDevErrBadIndex);
        page = 0;
      }
      base[hh] = ((((size_t)page * p.kv_heads + h) << p.block_shift) + (pos & bs_mask)) * HD;
      pc[hh] = page_constants(p, page, h, Code<F>::kLogFactor);
    }
    // scores of 32 tokens: 4 n8 tiles
    float s[MT][4][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][j][e] = 0.f;
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      uint32_t kw[4][kWords];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t* src = p.k_cache + base[j >> 1] + (size_t)((j & 1) * 8 + g) * HD + part * 128 + t * (4 * kWords);
#pragma unroll
        for (int w = 0; w < kWords; w += 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(src + 4 * w);
          kw[j][w] = x.x; kw[j][w + 1] = x.y; kw[j][w + 2] = x.z; kw[j][w + 3] = x.w;
        }
      }
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        uint4 a[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) a[mt] = qf[(mt * kSteps + part * kWords + w) * 32 + lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t b0, b1;
          Code<F>::unpack(kw[j][w], b0, b1);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) mma_16816(s[mt][j], a[mt], b0, b1);
        }
      }
    }
    // weights; s[.][j][2x + y]: row g + 8x, token 8 j + 2 t + y
    uint4 pa[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float top[2] = {m[mt][0], m[mt][1]};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int x = e >> 1;
          const int pos = j0 + 8 * j + 2 * t + (e & 1);
          const float v = pos <= lim[mt][x] ? fmaf(s[mt][j][e], pc[j >> 1].x * qe[mt][x], pc[j >> 1].y) : -INFINITY;
          s[mt][j][e] = v;
          top[x] = fmaxf(top[x], v);
        }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
        const float ref = top[x] == -INFINITY ? 0.f : top[x];
        const float fade = exp2_approx(m[mt][x] - ref);  // 0 while m is -inf
        m[mt][x] = top[x];
        l[mt][x] *= fade;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          o[mt][j][2 * x] *= fade;
          o[mt][j][2 * x + 1] *= fade;
        }
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float sum = 0.f;
#pragma unroll
          for (int j = 2 * hh; j < 2 * hh + 2; ++j) {
            s[mt][j][2 * x] = exp2_approx(s[mt][j][2 * x] - ref);
            s[mt][j][2 * x + 1] = exp2_approx(s[mt][j][2 * x + 1] - ref);
            sum += s[mt][j][2 * x] + s[mt][j][2 * x + 1];
          }
          l[mt][x] = fmaf(sum, pc[hh].z, l[mt][x]);
        }
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        pa[mt][hh].x = h2_as_u32(__floats2half2_rn(s[mt][2 * hh][0], s[mt][2 * hh][1]));
        pa[mt][hh].y = h2_as_u32(__floats2half2_rn(s[mt][2 * hh][2], s[mt][2 * hh][3]));
        pa[mt][hh].z = h2_as_u32(__floats2half2_rn(s[mt][2 * hh + 1][0], s[mt][2 * hh + 1][1]));
        pa[mt][hh].w = h2_as_u32(__floats2half2_rn(s[mt][2 * hh + 1][2], s[mt][2 * hh + 1][3]));
      }
    }
    // output += weights x V
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        uint32_t vw[4][kVWords];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tok = 2 * t + (i & 1) + 8 * (i >> 1);
          const uint8_t* src = p.v_cache + base[hh] + (size_t)tok * HD + part * 128 + g * (4 * kVWords);
          if constexpr (kVWords == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(src);
            vw[i][0] = x.x; vw[i][1] = x.y; vw[i][2] = x.z; vw[i][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(src);
            vw[i][0] = x.x; vw[i][1] = x.y;
          }
        }
#pragma unroll
        for (int w = 0; w < kVWords; ++w) {
          uint32_t b[4][2];  // [dim of the word][k half]
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t a01 = __byte_perm(vw[2 * i][w], vw[2 * i + 1][w], 0x5140);
            const uint32_t a23 = __byte_perm(vw[2 * i][w], vw[2 * i + 1][w], 0x7362);
            Code<F>::unpack(a01, b[0][i], b[1][i]);
            Code<F>::unpack(a23, b[2][i], b[3][i]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              mma_16816(o[mt][part * (kPart / 8) + 4 * w + e], pa[mt][hh], b[e][0], b[e][1]);
        }
      }
  }

  // Join the warps.  o[.][j][2x + y]: row g + 8x, dim of n = 2t + y in tile j.
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = mt * 16 + x * 8 + g;
      float sum = l[mt][x];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == 0) {
        jm[warp * kRows + row] = m[mt][x];
        jl[warp * kRows + row] = sum;
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int part = j / (kPart / 8), jj = j % (kPart / 8);
          joined[(warp * kRows + row) * HD + part * kPart + (2 * t + y) * (kPart / 8) + jj] = o[mt][j][2 * x + y];
        }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * HD; i += kAttWarps * 32) {
    const int row = i / HD, d = i % HD;
    if (row0 + row >= rows) break;
    float top = -INFINITY;
    for (int w = 0; w < kAttWarps; ++w) top = fmaxf(top, jm[w * kRows + row]);
    const float ref = top == -INFINITY ? 0.f : top;
    float num = 0.f, den = 0.f;
    for (int w = 0; w < kAttWarps; ++w) {
      const float f = exp2_approx(jm[w * kRows + row] - ref);
      num = fmaf(joined[(w * kRows + row) * HD + d], f, num);
      den = fmaf(jl[w * kRows + row], f, den);
    }
    const float v = den == 0.f ? 0.f : num / den;
    const int qi = (row0 + row) / p.group, gq = (row0 + row) % p.group;
    const long long at = (long long)(start + qi) * p.out_token_stride +
                         (long long)(h * p.group + gq) * p.out_head_stride + d;
    if (p.bf16)
      static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
    else
      static_cast<__half*>(p.out)[at] = __float2half_rn(v);
  }
}

template <int HD, int F>
int launch_attend(AttendArgs& a, int max_query_len, const DeviceInfo& dev, cudaStream_t stream) {
  const long long rows = (long long)max_query_len * a.group;
  constexpr int kBig = HD == 256 ? 1 : 2;
  const bool big = rows > 16 && kBig == 2;
  const int mt = big ? 2 : 1;
  const int kr = 16 * mt;
  const size_t smem = (size_t)mt * (HD / 16) * 512 + kr * 8 + (size_t)kAttWarps * kr * (HD + 2) * 4;
  auto kernel = big ? attend_simple_kernel<HD, F, kBig> : attend_simple_kernel<HD, F, 1>;
  cudaError_t e = ensure_smem(kernel, (int)smem, dev.ordinal);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(attend)");
  const dim3 grid((unsigned)((rows + kr - 1) / kr), a.kv_heads, a.requests);
  e = launch(kernel, grid, dim3(kAttWarps * 32), smem, stream, g_pdl_enabled != 0, a);
  return e == cudaSuccess ? GDSQ_OK : cuda_fail(e, "attend launch");
}

}  // namespace

cudaError_t attend_error_bits(bool clear, int* bits) {
  int own = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&own, g_device_error, sizeof(int));
  if (e == cudaSuccess) *bits |= own;
  const int zero = 0;
  if (e == cudaSuccess && clear) e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
  return e;
}

}  // namespace gdsq

using namespace gdsq;

extern "C" size_t gdsq_attend_kv8_workspace(int num_requests, int max_query_len, int num_heads, int num_kv_heads,
                                            int head_dim) {
  (void)num_requests; (void)max_query_len; (void)num_heads; (void)num_kv_heads; (void)head_dim;
  return 0;
}

extern "C" int gdsq_attend_kv8(const void* q, int elem_type, long long q_token_stride, long long q_head_stride,
                               const void* k_cache, const void* v_cache, int cache_type, const float* k_scale,
                               const float* v_scale, int num_blocks, int block_size, const int32_t* block_table,
                               int table_width, const int32_t* seq_lens, const int32_t* query_starts,
                               int num_requests, int num_tokens, int max_query_len, int max_seq_len, int num_heads,
                               int num_kv_heads, int head_dim, float softmax_scale, void* out, void* workspace,
                               size_t workspace_bytes, void* stream_v) {
  t_last_error.clear();
  if (elem_type != GDSQ_ELEM_F16 && elem_type != GDSQ_ELEM_BF16)
    return fail(GDSQ_ERR_INVALID_VALUE, "attend_kv8: elem_type %d is not fp16 or bf16", elem_type);
  if (cache_type != GDSQ_CACHE_INT8 && cache_type != GDSQ_CACHE_E4M3)
    return fail(GDSQ_ERR_INVALID_VALUE, "attend_kv8: cache_type %d is not int8 or e4m3", cache_type);
  if (num_heads < 1 || num_kv_heads < 1 || num_heads % num_kv_heads != 0 || num_kv_heads > 65535)
    return fail(GDSQ_ERR_INVALID_VALUE, "attend_kv8: heads %d must be a multiple of kv heads %d", num_heads,
                num_kv_heads);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(GDSQ_ERR_UNSUPPORTED, "attend_kv8: head_dim %d is not 64, 128 or 256", head_dim);
  if (block_size != 16 && block_size != 32 && block_size != 64 && block_size != 128)
    return fail(GDSQ_ERR_UNSUPPORTED, "attend_kv8: block_size %d is not 16, 32, 64 or 128", block_size);
  if (num_requests < 0 || num_requests > 65535 || num_tokens < 0 || num_blocks < 0 || table_width < 0 ||
      max_query_len < 0 || max_seq_len < 0)
    return fail(GDSQ_ERR_INVALID_VALUE, "attend_kv8: requests %d (0..65535), tokens %d, blocks %d, table width %d, "
                "longest query %d and sequence %d must not be negative", num_requests, num_tokens, num_blocks,
                table_width, max_query_len, max_seq_len);
  if (num_requests == 0 || num_tokens == 0 || max_query_len == 0) return GDSQ_OK;
  if (!q || !k_cache || !v_cache || !k_scale || !v_scale || !block_table || !seq_lens || !query_starts || !out)
    return fail(GDSQ_ERR_INVALID_VALUE, "attend_kv8: null pointer");
  if (!aligned(q, 16) || !aligned(out, 16) || q_token_stride % 8 != 0 || q_head_stride % 8 != 0)
    return fail(GDSQ_ERR_MISALIGNED, "attend_kv8: q and out 16-byte alignment, q strides multiples of 8 elements");
  if (!aligned(k_cache, 128) || !aligned(v_cache, 128) || !aligned(k_scale, 4) || !aligned(v_scale, 4) ||
      !aligned(block_table, 4) || !aligned(seq_lens, 4) || !aligned(query_starts, 4))
    return fail(GDSQ_ERR_MISALIGNED, "attend_kv8: caches 128-byte, scales, table and lengths 4-byte alignment");
  (void)workspace;
  (void)workspace_bytes;
  const DeviceInfo* dev = nullptr;
  int st = device_info(&dev);
  if (st != GDSQ_OK) return st;
  AttendArgs a = {};
  a.q = q;
  a.k_cache = static_cast<const uint8_t*>(k_cache);
  a.v_cache = static_cast<const uint8_t*>(v_cache);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.table = block_table;
  a.seq_lens = seq_lens;
  a.starts = query_starts;
  a.out = out;
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.out_token_stride = (long long)num_heads * head_dim;
  a.out_head_stride = head_dim;
  a.requests = num_requests;
  a.num_blocks = num_blocks;
  a.table_width = table_width;
  a.kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.block_shift = __builtin_ctz(block_size);
  a.tokens = num_tokens;
  a.bf16 = elem_type == GDSQ_ELEM_BF16;
  const float factor = cache_type == GDSQ_CACHE_INT8 ? Code<GDSQ_CACHE_INT8>::kFactor : Code<GDSQ_CACHE_E4M3>::kFactor;
  a.scale = softmax_scale * kLog2e * factor;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (cache_type == GDSQ_CACHE_INT8) {
    if (head_dim == 64) return launch_attend<64, GDSQ_CACHE_INT8>(a, max_query_len, *dev, stream);
    if (head_dim == 128) return launch_attend<128, GDSQ_CACHE_INT8>(a, max_query_len, *dev, stream);
    return launch_attend<256, GDSQ_CACHE_INT8>(a, max_query_len, *dev, stream);
  }
  if (head_dim == 64) return launch_attend<64, GDSQ_CACHE_E4M3>(a, max_query_len, *dev, stream);
  if (head_dim == 128) return launch_attend<128, GDSQ_CACHE_E4M3>(a, max_query_len, *dev, stream);
  return launch_attend<256, GDSQ_CACHE_E4M3>(a, max_query_len, *dev, stream);
}
