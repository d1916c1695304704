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
// exact in fp16.  A query row is scaled by a power of two to just under 2^15, the
// top of fp16's range, so that all elements down to 2^-29 of its largest keep the
// bits they came with, and a smaller one is off by 2^-40 of the largest at most.
// So what is rounded is the softmax weight, to the 11 bits that an fp16 output has.
//
// One pass with a running reference point: with lv = log2(vs[page]), a weight is
// p_j = 2^(s_j log2(e) + lv - r).  r is set kUnder below the largest s_j log2(e)
// + lv seen, and moved only when a weight would pass 2^kMostWeight, so the largest
// weight is between 2^kUnder and 2^kMostWeight whatever the scales are: near
// the top of fp16's range, so that a weight keeps its 11 bits down to 2^-21 of the
// largest, and a smaller one is off by 2^-32 of the largest at most.  (With the largest
// at 1, 131072 tokens at 2^-25.2 of one other token, 0.3 % of the softmax, came
// out as nothing.)  sum p_j vq_j needs no scale of its own, and the softmax's
// denominator is sum p_j 2^-lv, kept from the fp32 weights before they are rounded
// (2^-kUnder of it, so that 2^100 from the smallest value scales leaves room for 2^20 tokens).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gdsq.h"
#include "host.h"
#include "common.cuh"

namespace gdsq {
namespace {

constexpr int kAttWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;
// Positions of a table row: positions, and those of the 16 tiles of 128 tokens that a lane looks up ahead, stay below 2^31.
constexpr long long kMostPositions = (1ll << 31) - 4096;
constexpr float kNoMax = -1e30f;       // the reference point before any score
constexpr float kUnder = 7.f, kMostWeight = 15.f;  // log2
constexpr float kWeightUnit = 1.f / 128.f;         // 2^-kUnder
constexpr int kQTop = 15;                          // a query row's elements are below 2^kQTop as fp16
// log2 of a value scale is held to these.  The cache write stores a scale below 2^-100 as zero, and none above 2^122.
constexpr float kLeastLogScale = -100.f, kMostLogScale = 126.f;

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
  float scale;  // softmax scale * log2(e)
};

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// Lane (g, t) holds elements (g, 2t), (g, 2t + 1) of an 8 x 8 matrix and gets (2t, g), (2t + 1, g).
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes of global memory to shared memory, or zeros.
__device__ __forceinline__ void copy16_async(uint32_t to, const void* from, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// 8-bit codes to fp16 pairs, exactly.
template <int F>
struct Code;

template <>
struct Code<GDSQ_CACHE_INT8> {
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
  static __device__ __forceinline__ uint32_t widen(uint16_t x) {
    uint32_t d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(x));
    return d;
  }
  static __device__ __forceinline__ void unpack(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = widen((uint16_t)w);
    hi = widen((uint16_t)(w >> 16));
  }
};

__device__ __forceinline__ float2 unpack_q(bool bf16, uint32_t w) {
  return bf16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)) : __half22float2(u32_as_h2(w));
}

// The power of two that a q row with this largest magnitude is below; a row with inf or NaN keeps its values.
__device__ __forceinline__ int q_exponent(float most) {
  return isfinite(most) ? max((int)(__float_as_uint(most) >> 23) - 126, -100) : kQTop;
}

// N pairs of one q row, from element i (aligned to N pairs).
template <int N>
__device__ __forceinline__ void load_q(const AttendArgs& p, long long i, uint32_t (&w)[N]) {
  const uint16_t* src = static_cast<const uint16_t*>(p.q) + i;
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(src);
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(src);
    w[0] = x.x; w[1] = x.y;
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(src);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  }
}

// The cache is read once where one tile of rows covers a request's queries.
__device__ __forceinline__ uint64_t l2_policy_normal() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// Four dims of one output row.
__device__ __forceinline__ void store_out(const AttendArgs& p, int start, int h, int row, int d, const float (&num)[4],
                                          float den) {
  const float inv = den == 0.f ? 0.f : kWeightUnit / den;
  const long long at = (long long)(start + row / p.group) * p.out_token_stride +
                       (long long)(h * p.group + row % p.group) * p.out_head_stride + d;
  uint2 v;
  if (p.bf16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(num[0] * inv, num[1] * inv);
    const __nv_bfloat162 b = __floats2bfloat162_rn(num[2] * inv, num[3] * inv);
    v = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    v = make_uint2(h2_as_u32(__floats2half2_rn(num[0] * inv, num[1] * inv)),
                   h2_as_u32(__floats2half2_rn(num[2] * inv, num[3] * inv)));
  }
  *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + at) = v;
}

// Tokens behind the last request's (a step padded to a fixed size) belong to none: zeros.
// `thread` of the `threads` in every CTA that share the work.
__device__ __forceinline__ void zero_padding(const AttendArgs& p, int thread, int threads) {
  const long long first = max(min(p.starts[p.requests], p.tokens), 0) * p.out_token_stride / 8, last = p.tokens * p.out_token_stride / 8;
  for (long long i = first + (long long)blockIdx.x * threads + thread; i < last; i += (long long)gridDim.x * threads)
    static_cast<uint4*>(p.out)[i] = make_uint4(0, 0, 0, 0);
}

// Eight dims of one output row, from `to`.
__device__ __forceinline__ void store_out8(void* to, bool bf16, const float (&num)[8], float inv) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = num[2 * i] * inv, y = num[2 * i + 1] * inv;
    const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
    w[i] = bf16 ? *reinterpret_cast<const uint32_t*>(&b) : h2_as_u32(__floats2half2_rn(x, y));
  }
  *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Per-page constants of the softmax: x = kscale factor, y = lv, z = 2^(-lv - kUnder).
__device__ __forceinline__ float3 page_constants(const AttendArgs& p, int page, int h) {
  const size_t i = (size_t)page * p.kv_heads + h;
  const float ks = p.k_scale[i], vs = p.v_scale[i];
  const bool fine = isfinite(vs);
  const float lv = fminf(fmaxf(log2f(vs), kLeastLogScale), kMostLogScale);
  // A non-finite scale marks a block that was written with non-finite values:
  // the queries that see it come out as NaN.
  return make_float3(ks * p.scale, fine ? lv : __int_as_float(0x7fffffff), fine ? exp2f(-lv - kUnder) : 1.f);
}

// ---------------------------------------------------------------------------
// Few rows per (request, KV head): single tokens, drafts, short chunks.
//
// Bound by reading the cache, so the work is cut by cache tokens, evenly: an
// item is (request, KV head, tile of 8 * NT rows) and counts kItemCost steps
// plus one for each 128 tokens; CTA c of C takes the steps [c S / C, (c + 1) S
// / C) of all items in order.  An item that ends in the CTA it began in is
// written out; the others leave partial sums, and the CTA that arrives last at
// an item's counter adds them in CTA order.  So neither ragged lengths nor few
// requests leave SMs idle, and the result does not depend on who finishes
// first: two requests of 131072 tokens, 64 heads on 8 of 128, took 2146 us with
// one CTA for each (request, KV head).
//
// Measured, on the GPU alone: those two requests 100 us, 5.4 TB/s (82 % of a
// copy's rate); 64 requests of 1 to 16384 tokens, the same heads, e4m3, 47.4 us,
// 69 %, the rest being the cut, the filling of the rings and the joins; one
// request of 513 tokens with 32 heads 10.2 us, bound by the latency of a chain:
// lengths, table and scales, copies, a step, the warps' join, partial sums out, the
// counter, partial sums back.
//
// In a step, warp w takes the 32 tokens from 32 w, through its own ring of
// TMA boxes of 16 tokens (one block holds at least 16).  A lane looks up the
// block, scales and constants of one half tile for 16 tiles at a time.
//
// The products are taken transposed, tokens (scores) and dims (output) as the
// 16 rows of m16n8k16 and 8 query rows as its columns, so that eight queries
// of a group waste nothing.  A lane (g = lane / 4, t = lane % 4) feeds A[rows
// g, g + 8][k = 2t, 2t+1, 2t+8, 2t+9].  The order of the summed index is free:
// for the scores lane t takes 32 consecutive dims of tokens g and g + 8, two
// 16-byte loads each; for the output lane g takes 16 consecutive dims of
// tokens 2t, 2t+1, 2t+8, 2t+9.  With the 128-byte TMA swizzle both are free of
// bank conflicts.  The weights come out as [token][query] and are fed back as
// [query][token], one 8 x 8 transpose per 8 tokens.

constexpr int kStepTokens = kAttWarps * 32;
constexpr int kRing = 2;      // stages per warp
// What beginning and ending an item costs, in steps: the 64 ragged requests take
// 55.3 us with 1, 47.9 with 2, 46.8 with 3 and 46.3 with 4, which leaves the
// smallest calls more uneven.
constexpr int kItemCost = 3;

template <int HD, int NT>
struct StreamLayout {
  static constexpr int kStage = 2 * 32 * HD;  // K and V of 32 tokens
  static constexpr int kRingBytes = kAttWarps * kRing * kStage;
  static constexpr int kRows = 8 * NT;
  static constexpr int kPitch = HD + 4;  // floats of a row in the join
  static constexpr int kQ = NT * (HD / 16) * 256;
  static constexpr int kJoin = kRingBytes + kQ;  // eight rows
  static constexpr int kBars = kJoin + 8 * kPitch * 4;
  static constexpr int kRowInfo = kBars + 128;
  static constexpr int kMl = kRowInfo + kRows * 8;                 // [warps][kRows] m, l
  static constexpr int kTotal = kMl + kAttWarps * kRows * 8 + 64 + 1024;  // + alignment
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// CTAs per SM that registers and shared memory allow, which the grid is sized for.
template <int HD, int NT>
constexpr int stream_per_sm() {
  constexpr int by_smem = 227 * 1024 / (StreamLayout<HD, NT>::kTotal + 1024);
  constexpr int by_regs = HD * NT <= 256 ? 3 : 2;
  return by_smem < by_regs ? by_smem : by_regs;
}

template <int HD, int F, int NT>
__global__ void __launch_bounds__(kAttWarps * 32, (stream_per_sm<HD, NT>()))
    attend_stream_kernel(const AttendArgs p, const __grid_constant__ CUtensorMap kmap,
                         const __grid_constant__ CUtensorMap vmap, float* parts, int* counters) {
  using L = StreamLayout<HD, NT>;
  constexpr int kParts = HD >= 128 ? HD / 128 : 1;  // 128-dim parts
  constexpr int kPart = HD >= 128 ? 128 : 64;
  constexpr int kWords = kPart / 16;   // 32-bit words of K per lane, token and part (= k16 steps)
  constexpr int kSteps = HD / 16;      // k16 steps of the scores
  constexpr int kTiles = HD / 16;      // m16 tiles of the output
  constexpr int kVWords = kPart / 32;  // 32-bit words of V per lane, token and part
  constexpr int kRows = L::kRows;
  constexpr int kHalfBytes = 16 * HD;  // K (or V) of 16 tokens
  constexpr int kBox = 16 * kPart;     // one TMA box
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  uint4* qf = reinterpret_cast<uint4*>(smem + L::kRingBytes);  // [NT][kSteps / 2][32]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  float* qexp = reinterpret_cast<float*>(smem + L::kRowInfo);  // [kRows]
  int* qlim = reinterpret_cast<int*>(qexp + kRows);            // [kRows] last visible position
  float* jm = reinterpret_cast<float*>(smem + L::kMl);         // [warps][kRows]
  float* jl = jm + kAttWarps * kRows;
  int* shared_int = reinterpret_cast<int*>(jl + kAttWarps * kRows);  // [4]
  long long* shared_ll = reinterpret_cast<long long*>(shared_int + 4);  // [5]
  float* joined = reinterpret_cast<float*>(smem + L::kJoin);   // [8][kPitch]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  unsigned char* ring = smem + warp * kRing * L::kStage;
  uint64_t* full = bars + warp * kRing;
  if (lane == 0) {
    for (int s = 0; s < kRing; ++s) mbar_init(full + s, 1);
    fence_barrier_init();
    prefetch_tensor_map(&kmap);
    prefetch_tensor_map(&vmap);
  }
  pdl_launch_dependents();
  pdl_wait_primary();

  // The schedule: every CTA adds up all requests' steps and finds its first.
  const int most_len = p.table_width << p.block_shift;
  auto rows_of = [&](int r) { return max(min(p.starts[r + 1], p.tokens) - max(p.starts[r], 0), 0) * p.group; };
  auto steps_of = [&](int r) { return max(ceil_div(min(p.seq_lens[r], most_len), kStepTokens), 1); };
  const int per = ceil_div(p.requests, kAttWarps * 32);
  const int ra = min((int)threadIdx.x * per, p.requests), rb = min(ra + per, p.requests);
  long long mine = 0;
  auto cost_of = [&](int r) {
    return (long long)ceil_div(rows_of(r), kRows) * p.kv_heads * (steps_of(r) + kItemCost);
  };
  for (int r = ra; r < rb; ++r) mine += cost_of(r);
  long long upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += x;
  }
  if (lane == 31) shared_ll[warp] = upto;
  if (threadIdx.x == 0) shared_int[0] = -1;
  __syncthreads();
  long long all = 0, before = upto - mine;
#pragma unroll
  for (int w = 0; w < kAttWarps; ++w) {
    if (w < warp) before += shared_ll[w];
    all += shared_ll[w];
  }
  zero_padding(p, threadIdx.x, kAttWarps * 32);
  const long long C = min((long long)gridDim.x, all);  // every CTA in use has a step
  if (blockIdx.x >= C) return;
  long long s0 = all * blockIdx.x / C;
  const long long s1 = all * (blockIdx.x + 1) / C;
  if (before <= s0 && s0 < before + mine) {
    int r = ra;
    long long at = before;
    for (; r < rb; ++r) {
      const long long n = cost_of(r);
      if (s0 < at + n) break;
      at += n;
    }
    shared_int[0] = r;
    shared_ll[4] = at;
  }
  __syncthreads();
  int r = shared_int[0];
  long long request_at = shared_ll[4];  // first step of request r
  uint32_t used = 0;                    // tiles that this warp's ring has delivered
  bool dead = false;                    // a copy never arrived

  // The steps of one item that this CTA takes.
  struct Segment {
    int r, h, row0, rows, start, lim0;  // row i of the item sees positions up to lim0 + (row0 + i) / group
    int t0, t1, count;                  // this warp's first token, the end, and its tiles
    int kv_len, steps;
    long long first_step;  // of the item, among all steps
    bool opens, whole, once;
  };
  auto next_segment = [&](Segment& a) {
    while (s0 < s1) {
      const int start = max(p.starts[r], 0);
      const int n = max(min(p.starts[r + 1], p.tokens) - start, 0);
      const int rows = n * p.group;
      const int row_tiles = ceil_div(rows, kRows);
      const int len = min(p.seq_lens[r], most_len);
      if (len < p.seq_lens[r]) record_device_error(kDevErrBadIndex);
      const int steps = max(ceil_div(len, kStepTokens), 1), cost = steps + kItemCost;
      const long long request_cost = (long long)row_tiles * p.kv_heads * cost;
      if (s0 >= request_at + request_cost) {
        request_at += request_cost;
        ++r;
        continue;
      }
      const int item = (int)((s0 - request_at) / cost);
      const long long first_step = request_at + (long long)item * cost + kItemCost;
      const int step = (int)max(s0 - first_step, 0ll);
      s0 = first_step + step;
      if (s0 >= s1) return false;
      const int step_end = (int)min((long long)steps, step + (s1 - s0));
      s0 += step_end - step;
      a.r = r;
      a.h = item / row_tiles;
      a.row0 = (item % row_tiles) * kRows;
      a.rows = rows;
      a.start = start;
      a.lim0 = len - n;
      a.kv_len = max(min(len, a.lim0 + (min(rows, a.row0 + kRows) - 1) / p.group + 1), 0);
      a.t0 = step * kStepTokens + warp * 32;
      a.t1 = min(a.kv_len, step_end * kStepTokens);
      a.count = a.t0 < a.t1 ? (a.t1 - a.t0 + kStepTokens - 1) / kStepTokens : 0;
      a.steps = steps;
      a.first_step = first_step;
      a.opens = step == 0;
      a.whole = step == 0 && step_end == steps;
      a.once = row_tiles == 1;
      return true;
    }
    return false;
  };
  // Lane's half tile of the batch of 16 tiles from tile i: its block and row in the cache.
  auto half_row = [&](const Segment& a, int i) {
    const int pos = min(a.t0 + (i + (lane >> 1)) * kStepTokens + (lane & 1) * 16, (a.t1 - 1) & ~15);
    const int col = pos >> p.block_shift;
    int page = col < p.table_width ? p.table[(size_t)a.r * p.table_width + col] : -1;
    if ((unsigned)page >= (unsigned)p.num_blocks) {
      record_device_error(kDevErrBadIndex);
      page = 0;
    }
    return make_int2(page, (int)((((long long)page * p.kv_heads + a.h) << p.block_shift) + (pos & ((1 << p.block_shift) - 1))));
  };
  auto issue = [&](uint32_t tile, bool once, int row_lo, int row_hi) {  // one lane: the boxes of the warp's tile-th tile
    unsigned char* st = ring + (tile % kRing) * L::kStage;
    uint64_t* bar = full + tile % kRing;
    mbar_arrive_expect_tx(bar, L::kStage);
    const uint64_t policy = once ? l2_policy_evict_first() : l2_policy_normal();
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      tma_load_2d(st + part * kBox, &kmap, part * 128, row_lo, bar, policy);
      tma_load_2d(st + kHalfBytes + part * kBox, &kmap, part * 128, row_hi, bar, policy);
      tma_load_2d(st + 2 * kHalfBytes + part * kBox, &vmap, part * 128, row_lo, bar, policy);
      tma_load_2d(st + 3 * kHalfBytes + part * kBox, &vmap, part * 128, row_hi, bar, policy);
    }
  };
  constexpr int kMine = kRows / kAttWarps, kPairs = HD / 64;  // q rows per warp, pairs per lane
  // A segment's first copies and its q rows, asked for while the one before it is being joined.
  auto begin = [&](const Segment& a, int2& at, uint32_t(&raw)[kMine][kPairs]) {
    if (a.count > 0) {
      at = half_row(a, 0);
      // The warp has read the stages' last tiles (the __syncwarp that ends a step); the copies come after those reads.
      if (lane == 0) fence_proxy_async_smem();
#pragma unroll
      for (int i = 0; i < kRing; ++i) {
        const int lo = __shfl_sync(0xffffffffu, at.y, 2 * i), hi = __shfl_sync(0xffffffffu, at.y, 2 * i + 1);
        if (lane == 0 && i < a.count && !dead) issue(used + i, a.once, lo, hi);
      }
    }
    // lane i finds where the warp's row i is
    const int mine_row = a.row0 + warp + (lane % kMine) * kAttWarps;
    const long long mine_at = (long long)(a.start + mine_row / p.group) * p.q_token_stride +
                              (long long)(a.h * p.group + mine_row % p.group) * p.q_head_stride;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const long long at = __shfl_sync(0xffffffffu, mine_at, i);
#pragma unroll
      for (int e = 0; e < kPairs; ++e) raw[i][e] = 0;
      if (a.row0 + warp + i * kAttWarps < a.rows) load_q<kPairs>(p, at + lane * (HD / 32), raw[i]);
    }
  };

  Segment now, after;
  int2 cur = make_int2(0, 0);
  uint32_t raw[kMine][kPairs];
  bool more = next_segment(now);
  if (more) begin(now, cur, raw);
  while (more) {
    const int h = now.h, row0 = now.row0, rows = now.rows, t0 = now.t0, t1 = now.t1, count = now.count;
    const int first_lim = now.lim0 + row0 / p.group;
    int2 nxt = make_int2(0, 0);
    // Q rows: power-of-two scale, fp16, in operand order.
    if (lane < kMine) {
      const int i = warp + lane * kAttWarps, row = row0 + i;
      qlim[i] = row < rows ? now.lim0 + row / p.group : now.kv_len - 1;  // rows past the end are not written
    }
#pragma unroll
    for (int ii = 0; ii < kMine; ++ii) {
      const int i = warp + ii * kAttWarps;
      float v[HD / 32];
      float most = 0.f;
#pragma unroll
      for (int e = 0; e < kPairs; ++e) {
        const float2 x = unpack_q(p.bf16, raw[ii][e]);
        v[2 * e] = x.x;
        v[2 * e + 1] = x.y;
        most = fmaxf(most, fmaxf(fabsf(x.x), fabsf(x.y)));
      }
      most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
      const int ex = q_exponent(most);
      const float by = __uint_as_float((uint32_t)(127 + kQTop - ex) << 23);
      if (lane == 0) qexp[i] = __uint_as_float((uint32_t)(127 - kQTop + ex) << 23);
#pragma unroll
      for (int e = 0; e < HD / 32; e += 2) {
        const int d = lane * (HD / 32) + e;
        const int part = d / kPart, dd = d % kPart;
        const int tt = dd / (4 * kWords), w = (dd / 4) % kWords, b = dd & 3;
        // b0: dims 0,1 of the word, b1: dims 2,3; two steps side by side
        const int reg = (w & 1) * 2 + (b >> 1);
        const int ln = (i & 7) * 4 + tt;
        reinterpret_cast<uint32_t*>(qf + (((i >> 3) * kSteps + part * kWords + w) >> 1) * 32 + ln)[reg] =
            h2_as_u32(__floats2half2_rn(v[e] * by, v[e + 1] * by));
      }
    }
    float3 cc = make_float3(0.f, 0.f, 0.f), nc = cc;
    if (count > 0) cc = page_constants(p, cur.x, h);
    __syncthreads();

    float o[kTiles][NT][4];
    float m[NT][2], l[NT][2], qe[NT][2];  // of rows 8 nt + 2 t + y
    int lim[NT][2];
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][nt][e] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        m[nt][y] = kNoMax;
        l[nt][y] = 0.f;
        qe[nt][y] = qexp[nt * 8 + 2 * t + y];
        lim[nt][y] = min(qlim[nt * 8 + 2 * t + y], t1 - 1);
      }

    for (int i = 0; i < count; ++i) {
      const int j0 = t0 + i * kStepTokens;
      const int u = i & 15;
      if (u == 0 && i > 0) {
        cur = nxt;
        cc = nc;
      }
      if (u == 0 && i + 16 < count) nxt = half_row(now, i + 16);
      if (u == 8 && i + 8 < count) nc = page_constants(p, nxt.x, h);
      float3 pc[2];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
        pc[hh] = make_float3(__shfl_sync(0xffffffffu, cc.x, 2 * u + hh), __shfl_sync(0xffffffffu, cc.y, 2 * u + hh),
                             __shfl_sync(0xffffffffu, cc.z, 2 * u + hh));
      const uint32_t stage = (used + i) % kRing;
      const uint32_t kb = smem_addr(ring + stage * L::kStage), vb = kb + 2 * kHalfBytes;
      if (!dead && !mbar_wait(full + stage, ((used + i) / kRing) & 1)) {
        record_device_error(kDevErrBarrierTimeout);
        dead = true;
      }
      dead = __any_sync(0xffffffffu, dead);

      // scores; s[hh][nt][2 x + y]: token 16 hh + 8 x + g, row 8 nt + 2 t + y
      float s[2][NT][4];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[hh][nt][e] = 0.f;
#pragma unroll
      for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          uint32_t kw[2][kWords];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t row = kb + hh * kHalfBytes + part * kBox + (x * 8 + g) * kPart;
            if constexpr (kWords == 8) {
              const uint4 a = lds128(row + (((2 * t) ^ g) << 4)), b = lds128(row + (((2 * t + 1) ^ g) << 4));
              kw[x][0] = a.x; kw[x][1] = a.y; kw[x][2] = a.z; kw[x][3] = a.w;
              kw[x][4] = b.x; kw[x][5] = b.y; kw[x][6] = b.z; kw[x][7] = b.w;
            } else {
              const uint4 a = lds128(row + ((t ^ (g >> 1)) << 4));
              kw[x][0] = a.x; kw[x][1] = a.y; kw[x][2] = a.z; kw[x][3] = a.w;
            }
          }
#pragma unroll
          for (int w = 0; w < kWords; w += 2) {
            uint4 a0, a1;
            Code<F>::unpack(kw[0][w], a0.x, a0.z);
            Code<F>::unpack(kw[1][w], a0.y, a0.w);
            Code<F>::unpack(kw[0][w + 1], a1.x, a1.z);
            Code<F>::unpack(kw[1][w + 1], a1.y, a1.w);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint4 b = qf[((nt * kSteps + part * kWords + w) >> 1) * 32 + lane];
              mma_16816(s[hh][nt], a0, b.x, b.y);
              mma_16816(s[hh][nt], a1, b.z, b.w);
            }
          }
        }
      // weights
      const bool cut = j0 + 31 > min(first_lim, t1 - 1);
      uint32_t pb[2][NT][2];  // [hh][nt][x]: operand registers of tokens 8 x + 2 t, + 1, row g
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float v[2][4];
        float most[2] = {kNoMax, kNoMax};
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float c = pc[hh].x * qe[nt][y], b = pc[hh].y - m[nt][y];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float z = fmaf(s[hh][nt][2 * x + y], c, b);
              if (cut && j0 + 16 * hh + 8 * x + g > lim[nt][y]) z = -INFINITY;
              v[hh][2 * x + y] = z;
              most[y] = fmaxf(most[y], z);
            }
          }
        if (__any_sync(0xffffffffu, fmaxf(most[0], most[1]) > kMostWeight)) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float top = most[y];  // relative to m
            if (m[nt][y] == kNoMax) {
              top = -INFINITY;
#pragma unroll
              for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                  const bool in = !cut || j0 + 16 * hh + 8 * x + g <= lim[nt][y];
                  const float z = fmaf(s[hh][nt][2 * x + y], pc[hh].x * qe[nt][y], pc[hh].y);
                  if (in) top = fmaxf(top, z);
                }
            }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            float up;  // how far m rises
            if (m[nt][y] == kNoMax) {
              up = top == -INFINITY ? 0.f : INFINITY;
              if (top != -INFINITY) m[nt][y] = top - kUnder;
            } else {
              up = fmaxf(top - kUnder, 0.f);
              m[nt][y] += up;
            }
            const float fade = exp2_approx(-up);
            l[nt][y] *= fade;
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
              o[j][nt][y] *= fade;
              o[j][nt][2 + y] *= fade;
            }
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                float z = fmaf(s[hh][nt][2 * x + y], pc[hh].x * qe[nt][y], pc[hh].y - m[nt][y]);
                if (cut && j0 + 16 * hh + 8 * x + g > lim[nt][y]) z = -INFINITY;
                v[hh][2 * x + y] = z;
              }
          }
        }
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[hh][e] = exp2_approx(v[hh][e]);
#pragma unroll
          for (int y = 0; y < 2; ++y) l[nt][y] = fmaf(v[hh][y] + v[hh][2 + y], pc[hh].z, l[nt][y]);
#pragma unroll
          for (int x = 0; x < 2; ++x)
            pb[hh][nt][x] = transpose_8x8(h2_as_u32(__floats2half2_rn(v[hh][2 * x], v[hh][2 * x + 1])));
        }
      }
      // output += V^T x weights; o[.][nt][2 x + y]: dim 16 g + 2 tile + x, row 8 nt + 2 t + y
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          uint32_t vw[4][kVWords];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int tok = 2 * t + (c & 1) + 8 * (c >> 1);
            const bool past = F == GDSQ_CACHE_E4M3 && cut && j0 + 16 * hh + tok >= t1;  // may hold NaN codes
            const uint32_t row = vb + hh * kHalfBytes + part * kBox + tok * kPart;
            if constexpr (kVWords == 4) {
              const uint4 x = lds128(row + ((g ^ (tok & 7)) << 4));
              vw[c][0] = x.x; vw[c][1] = x.y; vw[c][2] = x.z; vw[c][3] = x.w;
            } else {
              const uint32_t at = row + (((g >> 1) ^ ((tok >> 1) & 3)) << 4) + (g & 1) * 8;
              vw[c][0] = lds32(at);
              vw[c][1] = lds32(at + 4);
            }
            if (past)
#pragma unroll
              for (int w = 0; w < kVWords; ++w) vw[c][w] = 0;
          }
#pragma unroll
          for (int w = 0; w < kVWords; ++w) {
            uint32_t b[4][2];  // [dim of the word][token half]
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t a01 = __byte_perm(vw[2 * c][w], vw[2 * c + 1][w], 0x5140);
              const uint32_t a23 = __byte_perm(vw[2 * c][w], vw[2 * c + 1][w], 0x7362);
              Code<F>::unpack(a01, b[0][c], b[1][c]);
              Code<F>::unpack(a23, b[2][c], b[3][c]);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint4 a = make_uint4(b[2 * e][0], b[2 * e + 1][0], b[2 * e][1], b[2 * e + 1][1]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_16816(o[part * (kPart / 16) + 2 * w + e][nt], a, pb[hh][nt][0], pb[hh][nt][1]);
            }
          }
        }
      // the stage is free: fetch tile i + kRing into it
      const int v2 = (u + kRing) & 15;
      const int src = u + kRing < 16 ? cur.y : nxt.y;
      const int lo = __shfl_sync(0xffffffffu, src, 2 * v2), hi = __shfl_sync(0xffffffffu, src, 2 * v2 + 1);
      if (lane == 0 && i + kRing < count && !dead) {
        fence_proxy_async_smem();
        issue(used + i + kRing, now.once, lo, hi);
      }
      __syncwarp();
    }
    used += count;

    more = next_segment(after);
    if (more) begin(after, cur, raw);

    // Join the warps: each adds its sums, scaled to the largest maximum, in turn; eight rows at a time.
    const bool whole = now.whole;
    const int slot = (int)blockIdx.x * 2 + (now.opens ? 1 : 0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float sum = l[nt][y];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (g == 0) {
          jm[warp * kRows + nt * 8 + 2 * t + y] = m[nt][y];
          jl[warp * kRows + nt * 8 + 2 * t + y] = sum;
        }
      }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (row0 + nt * 8 >= rows) break;
      float fade[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float top = kNoMax;
#pragma unroll
        for (int w = 0; w < kAttWarps; ++w) top = fmaxf(top, jm[w * kRows + nt * 8 + 2 * t + y]);
        fade[y] = exp2_approx(m[nt][y] - top);
      }
      for (int w = 0; w < kAttWarps; ++w) {
        if (w == warp) {
#pragma unroll
          for (int y = 0; y < 2; ++y)
            if (row0 + nt * 8 + 2 * t + y < rows) {
#pragma unroll
              for (int part = 0; part < kParts; ++part)
#pragma unroll
                for (int j = 0; j < kPart / 16; j += 2) {
                  float4* dst = reinterpret_cast<float4*>(joined + (2 * t + y) * L::kPitch + part * kPart + g * (kPart / 8) + 2 * j);
                  const int jj = part * (kPart / 16) + j;
                  float4 x = w ? *dst : make_float4(0.f, 0.f, 0.f, 0.f);
                  x.x = fmaf(o[jj][nt][y], fade[y], x.x);
                  x.y = fmaf(o[jj][nt][2 + y], fade[y], x.y);
                  x.z = fmaf(o[jj + 1][nt][y], fade[y], x.z);
                  x.w = fmaf(o[jj + 1][nt][2 + y], fade[y], x.w);
                  *dst = x;
                }
            }
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < 8 * HD / 4; i += kAttWarps * 32) {
        const int row = i / (HD / 4), d = (i % (HD / 4)) * 4;
        const int tr = nt * 8 + row;
        if (row0 + tr >= rows) break;
        float top = kNoMax, den = 0.f;
#pragma unroll
        for (int w = 0; w < kAttWarps; ++w) top = fmaxf(top, jm[w * kRows + tr]);
#pragma unroll
        for (int w = 0; w < kAttWarps; ++w) den = fmaf(jl[w * kRows + tr], exp2_approx(jm[w * kRows + tr] - top), den);
        const float4 x = *reinterpret_cast<const float4*>(joined + row * L::kPitch + d);
        const float num[4] = {x.x, x.y, x.z, x.w};
        if (whole) {
          store_out(p, now.start, h, row0 + tr, d, num, den);
        } else {
          float* part = parts + (size_t)slot * kRows * (HD + 2);
          *reinterpret_cast<float4*>(part + (size_t)tr * HD + d) = make_float4(num[0], num[1], num[2], num[3]);
          if (d == 0) *reinterpret_cast<float2*>(part + kRows * HD + 2 * tr) = make_float2(top, den);
        }
      }
      __syncthreads();
    }
    if (!whole) {
      // the CTAs that hold the item's first and last step
      const int c0 = (int)(((now.first_step + 1) * C - 1) / all), c1 = (int)(((now.first_step + now.steps) * C - 1) / all);
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) shared_int[1] = atomicAdd(counters + c0, 1) == c1 - c0;
      __syncthreads();
      if (shared_int[1]) {
        __threadfence();
        const int live = min(rows - row0, kRows);
        for (int i = threadIdx.x; i < live * (HD / 4); i += kAttWarps * 32) {
          const int tr = i / (HD / 4), d = (i % (HD / 4)) * 4;
          float top = kNoMax;
          for (int c = c0; c <= c1; ++c) {
            const float* part = parts + (size_t)(2 * c + (c == c0)) * kRows * (HD + 2);
            top = fmaxf(top, __ldcg(part + kRows * HD + 2 * tr));
          }
          float num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
          for (int c = c0; c <= c1; ++c) {
            const float* part = parts + (size_t)(2 * c + (c == c0)) * kRows * (HD + 2);
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(part + kRows * HD + 2 * tr));
            const float4 x = __ldcg(reinterpret_cast<const float4*>(part + (size_t)tr * HD + d));
            const float f = exp2_approx(ml.x - top);
            num[0] = fmaf(x.x, f, num[0]);
            num[1] = fmaf(x.y, f, num[1]);
            num[2] = fmaf(x.z, f, num[2]);
            num[3] = fmaf(x.w, f, num[3]);
            den = fmaf(ml.y, f, den);
          }
          store_out(p, now.start, h, row0 + tr, d, num, den);
        }
        if (threadIdx.x == 0) counters[c0] = 0;
      }
    }
    now = after;
  }
}

// One counter per CTA, then partial sums of two items per CTA.  The counters
// are where they are for every variant, since they must stay zero between calls.
constexpr size_t kCounterBytes = 16384;

template <int HD, int NT>
size_t stream_workspace(int sms) {
  return kCounterBytes + (size_t)sms * stream_per_sm<HD, NT>() * 2 * (8 * NT) * (HD + 2) * 4;
}

// ---------------------------------------------------------------------------
// Many rows per (request, KV head): prompts and long chunks.
//
// Bound by the tensor cores and the exponentials, so the products run on
// tcgen05: an item is QT tiles of 128 rows, a step is BN tokens.  The cut into
// steps and the joining of partial sums are those of the kernel above, with one
// CTA per SM.
//
//   warps 0-7   softmax: warp group t owns the rows of tile t, a thread a row.  Q
//               row to fp16 in shared memory; then per step the scores from
//               TMEM, weights back to TMEM over them, in the end the output.
//   warps 8-11  widen the 8-bit tiles to fp16
//   warp 12     issues the products
//   warp 13     TMA of the 8-bit tiles, and the blocks' scales (14 and 15: zeros for the step's padding)
//
// K and V are widened to the same layout, [64 dims][token][128 bytes], 128-byte
// swizzled: K major for the scores (a row of B is a token) and N major for the
// output (a column of B is a dim).  With two tiles the order of products is
// O0(i) S0(i+1) O1(i) S1(i+1), so that one tile's softmax runs beside the other's
// products; the weights take the scores' place in TMEM.  Widened K needs no second
// buffer: scores i are done long before K i+1 is needed; V has two.  With one tile
// (heads of 256) the scores alternate between two places, S(i+1) O(i), so that the
// softmax runs beside the products all the same.
//
// Measured: three prompts of up to 2048 tokens over up to 6000 cached, 64 heads on
// 8 of 128, e4m3: 539 us, 905 TFLOP/s counting the visible positions (55 % of the
// measured matrix rate), where one tile with mma.sync took 3220; the same with 32
// heads on 8 of 64: 260 us, 470 TFLOP/s; 33 requests with five tokens each, 32 heads on
// 2 of 256, over up to 2047: 30 to 33 us, bound by latency (the schedule 3 k cycles, Q 8 k,
// a step 2 k, the output 2 k, a join 10 k).  A step of two tiles took about 4600 cycles
// when the prompts took 566 us: 2048 are the exponential unit's (32768 weights,
// 16 a cycle), 2600 the products', at 80 to 90 cycles where alone they take 64,
// since the widening and the Q tiles use the same shared memory, and the two
// overlap in part.  A polynomial for some of the exponentials was slower (936
// us then to 1070), as was a fixed turn between the tiles (741 to 814).

template <int HD>
struct TileLayout {
  static constexpr int QT = HD == 256 ? 1 : 2;   // tiles of 128 rows
  static constexpr int BN = HD == 256 ? 64 : 128;  // tokens per step
  static constexpr int kRows = 128 * QT;
  static constexpr int kQ = 128 * HD * 2;        // one tile of Q
  static constexpr int kWide = BN * HD * 2;      // K or V of a step in fp16
  static constexpr int kRaw = BN * HD;           // in 8 bits
  static constexpr int kKOff = QT * kQ, kVOff = kKOff + kWide, kRawOff = kVOff + 2 * kWide;  // V twice
  static constexpr int kConst = kRawOff + 4 * kRaw;  // [2][BN / 16] float4
  static constexpr int kBars = kConst + 2 * (BN / 16) * 16;
  static constexpr int kNeed = kBars + 512 + 1024;
  static constexpr int kTotal = kNeed > 116 * 1024 ? kNeed : 116 * 1024;  // one CTA (512 TMEM columns) per SM
};
constexpr int kTileThreads = 16 * 32;
// Tokens that are added up in tensor memory before the sum is taken out.  The tensor cores cut off what does not fit when they add,
// always toward zero: over 131072 tokens of about equal weight a sum came out 1.0e-3 of itself too small, over 16384 at a time as
// exact as fp16 shows (1.8e-4, the rounding of the output).
constexpr int kChain = 16384;
// What beginning and ending an item costs, in tokens: the three prompts above
// take 539 us with 896, 555 with 768 and 543 with 1024, and with heads of 64 260 with
// 896, 279 with 448 and 268 with 1792 (33 requests of ten tokens on them 36, 30 and 44);
// for heads of 256 the 33 requests with five tokens take 33.0 us with 320, 33.5 with 448.
template <int HD>
__host__ __device__ constexpr int item_tokens() { return HD == 256 ? 320 : 896; }
// Registers per thread of the softmax, widening and other warp groups: together the launch's 4 x 128.
constexpr int kSoftmaxRegs = 176, kWidenRegs = 80, kOtherRegs = 80;

// The whole warp calls these and the lane with leader != 0 issues, so that the
// code around them is not divergent and their operands stay in uniform
// registers: issued from a branch of one lane, a product took 110 cycles to
// issue, twice its own time.  Descriptors are given by their low word.
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t a_hi, uint32_t b_hi,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 e, %0, 0;\n\tsetp.ne.b32 p, %7, 0;\n\t"
      "mov.b64 a, {%2, %4};\n\tmov.b64 b, {%3, %5};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%1], a, b, %6, p;\n\t}" ::"r"(leader),
      "r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(a_hi), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 e, %0, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 b, {%3, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], b, %5, p;\n\t}" ::"r"(leader),
      "r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_by(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %0, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(leader),
      "r"(smem_addr(bar))
      : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle: 8 rows of 128 bytes per
// 1024-byte atom.  K major: `sbo` bytes between groups of 8 rows.  N major:
// `sbo` bytes between groups of 8 K rows, `lbo` between blocks of 64 columns.
// Low word (the start and `lbo`) and high word of the descriptor.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return ((saddr >> 4) & 0x3FFFu) | ((lbo >> 4) & 0x3FFFu) << 16; }
__host__ __device__ constexpr uint32_t desc_hi(uint32_t sbo) {
  return ((sbo >> 4) & 0x3FFFu) | 1u << 14 | 2u << 29;  // version for sm_100, 128-byte swizzle
}

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {  // does not block
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2f(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
template <int HD, int F>
__global__ void __launch_bounds__(kTileThreads, 1)
    attend_tile_kernel(const AttendArgs p, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, float* parts, int* counters) {
  using L = TileLayout<HD>;
  constexpr int QT = L::QT, BN = L::BN, kRows = L::kRows;
  constexpr int kParts = HD >= 128 ? HD / 128 : 1, kPart = HD >= 128 ? 128 : 64;
  constexpr uint32_t kOCol = 2 * BN;  // after the scores: of two tiles, or of one tile in two places
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  const uint32_t sbase = smem_addr(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* raw_full = bars;        // [2][K, V]
  uint64_t* raw_empty = bars + 4;   // [2][K, V]
  uint64_t* wide_full = bars + 8;   // [K, V even, V odd]
  uint64_t* wide_empty = bars + 44; // [K, V even, V odd]
  uint64_t* s_full = bars + 12;     // [QT]
  uint64_t* p_full = bars + 14;     // [QT]
  uint64_t* o_full = bars + 16;
  uint64_t* q_full = bars + 17;
  uint64_t* const_full = bars + 18;  // [2]
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(bars + 20);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_at + 1);  // a wait ran out
  int* last_one = reinterpret_cast<int*>(tmem_at + 2);
  // The schedule: a sum from each warp, and apart from them what one thread finds while the sums are still being read.
  constexpr int kWarps = kTileThreads / 32, kSumsAt = 24, kFoundAt = 47;
  static_assert(kSumsAt + kWarps <= 40 && kFoundAt >= 47 && (kFoundAt + 1) * 8 <= 512, "the schedule's words overlap others");
  long long* warp_sums = reinterpret_cast<long long*>(bars + kSumsAt);  // [kWarps]
  int* shared_r = reinterpret_cast<int*>(bars + 40);                    // the CTA's first request ..
  long long* shared_at = reinterpret_cast<long long*>(bars + kFoundAt);  // .. and where it begins
  uint64_t* const_empty = bars + 42;  // [2]
  const float4* consts = reinterpret_cast<const float4*>(smem + L::kConst);  // [2][BN / 16]

  // From one lane, so that the compiler knows the roles' branches to be uniform.
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int kMmaWarp = 12, kTmaWarp = 13;
  if (warp == kTmaWarp && lane == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(raw_full + i, 1);
      mbar_init(raw_empty + i, 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 4);
      mbar_init(const_full + i, 1);
      mbar_init(const_empty + i, 4 * QT);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(wide_full + i, 4);
      mbar_init(wide_empty + i, 1);
    }
    mbar_init(o_full, 1);
    mbar_init(q_full, 4 * QT);
    *dead = 0;
    fence_barrier_init();
    prefetch_tensor_map(&kmap);
    prefetch_tensor_map(&vmap);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_at, 512);
    tmem_relinquish();
  }
  pdl_launch_dependents();
  pdl_wait_primary();

  // The schedule, in tokens: tile j of a request's rows counts an item's fixed cost
  // and about the tokens that it sees, `first` + j * `rise`, whose running sum is
  // quadratic in j.  A step belongs to the CTA whose share its first token falls in.
  const int most_len = p.table_width << p.block_shift;
  const int rise = ceil_div(kRows, p.group);
  auto rows_of = [&](int r) { return max(min(p.starts[r + 1], p.tokens) - max(p.starts[r], 0), 0) * p.group; };
  auto first_of = [&](int r) {  // cost of the first row tile
    const int n = max(min(p.starts[r + 1], p.tokens) - max(p.starts[r], 0), 0);
    return (long long)item_tokens<HD>() + max(min(p.seq_lens[r], most_len) - n, 0) + rise + 1;
  };
  auto upto_tile = [&](long long first, long long j) { return j * first + j * (j - 1) / 2 * rise; };
  auto cost_of = [&](int r) { return upto_tile(first_of(r), ceil_div(rows_of(r), kRows)) * p.kv_heads; };
  long long all, s0, s1, request_at;
  const int per = ceil_div(p.requests, kTileThreads);
  const int ra = min((int)threadIdx.x * per, p.requests), rb = min(ra + per, p.requests);
  long long mine = 0;
  for (int r = ra; r < rb; ++r) mine += cost_of(r);
  long long upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += x;
  }
  if (lane == 31) warp_sums[warp] = upto;
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_at;
  long long before = upto - mine;
  all = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_sums[w];
    all += warp_sums[w];
  }
  const long long C = max(min((long long)gridDim.x, all / BN), 1ll);  // a share holds a step at least
  const bool works = blockIdx.x < C && all > 0;
  s0 = works ? all * blockIdx.x / C : 0;
  s1 = works ? all * (blockIdx.x + 1) / C : 0;
  if (works && before <= s0 && s0 < before + mine) {
    int r = ra;
    long long at = before;
    for (; r < rb; ++r) {
      const long long n = cost_of(r);
      if (s0 < at + n) break;
      at += n;
    }
    *shared_r = r;
    *shared_at = at;
  }
  __syncthreads();
  int r = works ? *shared_r : 0;
  request_at = works ? *shared_at : 0;

  // What a CTA takes of an item is its run; a segment is up to kChain tokens of a run.
  struct Segment {
    int r, h, row0, rows, start, lim0;  // row i of the item sees positions up to lim0 + (row0 + i) / group
    int t0, t1, count;                  // first token, the end, and the steps
    int steps;              // of the item
    long long first_token;  // of the item, in the schedule
    bool opens, whole;      // the run begins the item; it is all of the item
    bool goes_on, last;     // not the run's first segment; its last
  };
  const long long cta_s0 = s0;
  auto next_segment = [&](Segment& a) {
    while (s0 < s1) {
      const int start = max(p.starts[r], 0);
      const int n = max(min(p.starts[r + 1], p.tokens) - start, 0);
      const int rows = n * p.group;
      const int row_tiles = ceil_div(rows, kRows);
      const int len = min(p.seq_lens[r], most_len);
      if (len < p.seq_lens[r]) record_device_error(kDevErrBadIndex);
      const long long first = first_of(r), head_cost = upto_tile(first, row_tiles);
      if (s0 >= request_at + head_cost * p.kv_heads) {
        request_at += head_cost * p.kv_heads;
        ++r;
        continue;
      }
      const int h = (int)((s0 - request_at) / head_cost);
      const long long in_head = s0 - request_at - h * head_cost;
      int tile = 0;
      for (int end = row_tiles; end - tile > 1;) {  // the last tile that begins at or before it
        const int mid = (tile + end) >> 1;
        if (upto_tile(first, mid) <= in_head) tile = mid;
        else end = mid;
      }
      const long long item_at = request_at + h * head_cost + upto_tile(first, tile);
      const long long item_end = item_at + first + (long long)tile * rise;
      a.first_token = item_at + item_tokens<HD>();
      a.r = r;
      a.h = h;
      a.row0 = tile * kRows;
      a.rows = rows;
      a.start = start;
      a.lim0 = len - n;
      const int kv_len = max(min(len, a.lim0 + (min(rows, a.row0 + kRows) - 1) / p.group + 1), 0);
      a.steps = max(ceil_div(kv_len, BN), 1);
      // steps whose first token is at a share's start or after it, and before its end
      auto step_from = [&](long long at) { return (int)min(max((at - a.first_token + BN - 1) / BN, 0ll), (long long)a.steps); };
      const int step = step_from(s0), run_begin = step_from(cta_s0), run_end = step_from(s1);
      const int step_end = min(run_end, step + kChain / BN);
      a.last = step_end == run_end;
      s0 = a.last ? item_end : a.first_token + (long long)step_end * BN;
      if (step >= step_end) continue;
      a.t0 = step * BN;
      a.t1 = min(kv_len, step_end * BN);
      a.count = a.t0 < a.t1 ? (a.t1 - a.t0 + BN - 1) / BN : 0;
      a.opens = run_begin == 0;
      a.whole = run_begin == 0 && run_end == a.steps;
      a.goes_on = step > run_begin;
      return true;
    }
    return false;
  };
  // Waits of one warp; once one has run out nobody waits any more.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_test_wait(bar, parity) || *dead) return;
    if (!mbar_wait(bar, parity)) {
      record_device_error(kDevErrBarrierTimeout);
      *dead = 1;
    }
  };

  Segment a;
  if (warp >= 12) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp == kTmaWarp) {
    uint32_t i = 0;  // steps so far
    while (next_segment(a))
      for (int step = 0; step < a.count; ++step, ++i) {
        const int j0 = a.t0 + step * BN, stage = i & 1;
        // lane's group of 16 tokens
        int page = 0, row = 0;
        if (lane < BN / 16) {
          const int pos = min(j0 + 16 * lane, (a.t1 - 1) & ~15);
          const int col = pos >> p.block_shift;
          page = col < p.table_width ? p.table[(size_t)a.r * p.table_width + col] : -1;
          if ((unsigned)page >= (unsigned)p.num_blocks) {
            record_device_error(kDevErrBadIndex);
            page = 0;
          }
          row = (int)((((long long)page * p.kv_heads + a.h) << p.block_shift) + (pos & ((1 << p.block_shift) - 1)));
        }
        const float3 c = lane < BN / 16 ? page_constants(p, page, a.h) : make_float3(0.f, 0.f, 0.f);
        if (i >= 2) wait(const_empty + stage, ((i >> 1) - 1) & 1);
        if (lane < BN / 16) reinterpret_cast<float4*>(smem + L::kConst)[stage * (BN / 16) + lane] = make_float4(c.x, c.y, c.z, 0.f);
        __syncwarp();
        if (lane == 0) mbar_arrive(const_full + stage);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          uint64_t* bar = raw_full + 2 * stage + kv;
          if (i >= 2) wait(raw_empty + 2 * stage + kv, ((i >> 1) - 1) & 1);
          if (lane == 0 && !*dead) mbar_arrive_expect_tx(bar, L::kRaw);
          __syncwarp();
          if (lane < BN / 16 && !*dead) {
            const uint64_t policy = l2_policy_normal();
            unsigned char* dst = smem + L::kRawOff + (2 * stage + kv) * L::kRaw + lane * 16 * kPart;
#pragma unroll
            for (int part = 0; part < kParts; ++part)
              tma_load_2d(dst + part * BN * kPart, kv ? &vmap : &kmap, part * 128, row, bar, policy);
          }
          __syncwarp();
        }
      }
  } else if (warp == kMmaWarp) {
    constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | (8u << 24);
    constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);  // B is N major
    uint32_t i = 0, seg = 0;
    const uint32_t leader = lane == 0;
    uint32_t phase0 = 0, phase1 = 0;  // parity of the next p_full of each tile
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t q_lo = desc_lo(sbase, 16), k_lo = desc_lo(sbase + L::kKOff, 16), v_lo = desc_lo(sbase + L::kVOff, BN * 128);
    constexpr uint32_t kHi = desc_hi(1024);
    auto scores = [&](int t, int tile) {
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
        mma_ss(leader, tm + t * BN, q_lo + ((tile * L::kQ + (k / 4) * (128 * 128) + (k % 4) * 32) >> 4),
               k_lo + (((k / 4) * (BN * 128) + (k % 4) * 32) >> 4), kHi, kHi, kIdescS, k > 0);
      commit_by(leader, s_full + t);
    };
    auto output = [&](int t, int tile, bool first, uint32_t buffer) {
#pragma unroll
      for (int k = 0; k < BN / 16; ++k)
        mma_ts(leader, tm + kOCol + tile * HD, tm + t * BN + k * 8, v_lo + buffer * (L::kWide >> 4) + k * (2048 >> 4), kHi, kIdescO,
               !(first && k == 0));
    };
    auto commit = [&](uint64_t* bar) { commit_by(leader, bar); };
    while (__shfl_sync(0xffffffffu, (int)next_segment(a), 0)) {
      const int count = __shfl_sync(0xffffffffu, a.count, 0);
      const bool two = QT == 2 && __shfl_sync(0xffffffffu, a.rows - a.row0, 0) > 128;  // the second tile has rows
      if (count == 0) continue;
      wait(q_full, seg & 1);
      ++seg;
      tc_fence_after_sync();
      wait(wide_full + 0, i & 1);
      tc_fence_after_sync();
      auto products = [&](auto tiles) {
        constexpr int kTiles = decltype(tiles)::value;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) scores(t, t);
        commit(wide_empty + 0);
        for (int step = 0; step < count; ++step, ++i) {
          const bool more = step + 1 < count;
          wait(wide_full + 1 + (i & 1), (i >> 1) & 1);
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            wait(p_full + t, t ? phase1 : phase0);
            tc_fence_after_sync();
            output(t, t, step == 0, i & 1);
            if (t == kTiles - 1) commit(wide_empty + 1 + (i & 1));
            if (more) {
              if (t == 0) wait(wide_full + 0, (i + 1) & 1);
              tc_fence_after_sync();
              scores(t, t);
              if (t == kTiles - 1) commit(wide_empty + 0);
            }
          }
          phase0 ^= 1;
          if (kTiles == 2) phase1 ^= 1;
        }
      };
      if constexpr (QT == 1) {
        // one tile: the next scores go to another place, ahead of this step's weights
        scores(i & 1, 0);
        commit(wide_empty + 0);
        for (int step = 0; step < count; ++step, ++i) {
          if (step + 1 < count) {
            wait(wide_full + 0, (i + 1) & 1);
            tc_fence_after_sync();
            scores((i + 1) & 1, 0);
            commit(wide_empty + 0);
          }
          wait(wide_full + 1 + (i & 1), (i >> 1) & 1);
          wait(p_full + (i & 1), (i >> 1) & 1);
          tc_fence_after_sync();
          output(i & 1, 0, step == 0, i & 1);
          commit(wide_empty + 1 + (i & 1));
        }
      } else if (two) products(std::integral_constant<int, QT>{});
      else products(std::integral_constant<int, 1>{});
      commit(o_full);
    }
  } else {
    zero_padding(p, threadIdx.x - (kTmaWarp + 1) * 32, kTileThreads - (kTmaWarp + 1) * 32);
  }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWidenRegs));
    // widen: 16 codes of one token at a time
    const int tid = threadIdx.x - 256;
    uint32_t i = 0;
    while (next_segment(a))
      for (int step = 0; step < a.count; ++step, ++i) {
        const int stage = i & 1, left = a.t1 - (a.t0 + step * BN);  // tokens from here on hold nothing
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          wait(raw_full + 2 * stage + kv, (i >> 1) & 1);
          // K has one buffer, V two
          if (kv == 0 && i >= 1) wait(wide_empty, (i - 1) & 1);
          if (kv == 1 && i >= 2) wait(wide_empty + 1 + (i & 1), ((i >> 1) - 1) & 1);
          const uint32_t raw = sbase + L::kRawOff + (2 * stage + kv) * L::kRaw;
          const uint32_t wide = sbase + (kv ? L::kVOff + (i & 1) * L::kWide : L::kKOff);
#pragma unroll 4
          for (int j = 0; j < BN * (HD / 16) / 128; ++j) {
            const int unit = tid + j * 128, tok = unit % BN, c = unit / BN;  // chunk of 16 dims
            uint32_t at;
            if constexpr (kPart == 128)
              at = raw + (c / 8) * (BN * 128) + tok * 128 + (((c % 8) ^ (tok & 7)) << 4);
            else
              at = raw + tok * 64 + ((c ^ ((tok >> 1) & 3)) << 4);
            uint4 x = lds128(at);
            if (F == GDSQ_CACHE_E4M3 && kv && tok >= left) x = make_uint4(0, 0, 0, 0);  // may hold NaN codes
            uint32_t o[8];
            Code<F>::unpack(x.x, o[0], o[1]);
            Code<F>::unpack(x.y, o[2], o[3]);
            Code<F>::unpack(x.z, o[4], o[5]);
            Code<F>::unpack(x.w, o[6], o[7]);
            const uint32_t row = wide + (c / 4) * (BN * 128) + tok * 128;
            const uint32_t c0 = (c % 4) * 2;
            sts128(row + ((c0 ^ (tok & 7)) << 4), o[0], o[1], o[2], o[3]);
            sts128(row + (((c0 + 1) ^ (tok & 7)) << 4), o[4], o[5], o[6], o[7]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(raw_empty + 2 * stage + kv);
            mbar_arrive(wide_full + (kv ? 1 + (i & 1) : 0));
          }
        }
      }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = QT == 1 ? 0 : warp >> 2;         // tile
    const bool helps = QT == 1 && warp >= 4;       // with the joining of partial sums only
    const int local = t * 128 + (threadIdx.x & 127);  // row of the item
    const uint32_t quarter = (uint32_t)(warp & 3) << 21;  // TMEM lane (warp % 4) * 32 in the address
    const uint32_t s_at0 = tmem + quarter + t * BN, o_at = tmem + quarter + kOCol + t * HD;
    uint32_t i = 0, seg = 0;
    [[maybe_unused]] uint32_t s_phase = 0;
    while (next_segment(a)) {
      const int row = a.row0 + local;
      const bool live = row < a.rows;
      float m = kNoMax, l = 0.f;
      const int slot = (int)blockIdx.x * 2 + (a.opens ? 1 : 0);
      float* part = parts + (size_t)slot * kRows * (HD + 2);
      __half* const out_row = static_cast<__half*>(p.out) + (long long)(a.start + row / p.group) * p.out_token_stride +
                    (long long)(a.h * p.group + row % p.group) * p.out_head_stride;  // 16 bits of either type
      if (!helps) {
        float qe = 1.f;
        int lim = a.t1 - 1;
        if (a.count > 0) {
          // The warp's 32 Q rows, kLanes lanes to a row: power-of-two scale, fp16.  Copied as
          // it is, then scaled in place in a short loop: with all rows side by side in
          // registers the fetching of the instructions took most of 20000 cycles.
          constexpr int kLanes = HD / 8, kAtOnce = 32 / kLanes;  // 16-byte vectors
          constexpr int kBatch = 4;                              // of a lane at a time
          const int sub = lane / kLanes, vec = lane % kLanes;
          const float sign = copysignf(1.f, p.scale);
          const long long from = live ? (long long)(a.start + row / p.group) * p.q_token_stride +
                                            (long long)(a.h * p.group + row % p.group) * p.q_head_stride
                                      : -1;
          auto place_of = [&](int at) {
            return sbase + t * L::kQ + (vec / 8) * (128 * 128) + ((warp & 3) * 32 + at) * 128 + (((vec % 8) ^ (at & 7)) << 4);
          };
#pragma unroll 4
          for (int r0 = 0; r0 < 32; r0 += kAtOnce) {
            const long long at = __shfl_sync(0xffffffffu, from, r0 + sub);
            copy16_async(place_of(r0 + sub), static_cast<const uint16_t*>(p.q) + max(at, 0ll) + vec * 8, at >= 0);
          }
          copy_async_wait();
          auto scale_rows = [&](auto bf16) {
            constexpr bool kBf16 = decltype(bf16)::value;
#pragma unroll 1
            for (int r0 = 0; r0 < 32; r0 += kAtOnce * kBatch) {
              uint4 w[kBatch];
              float most[kBatch];
#pragma unroll
              for (int c = 0; c < kBatch; ++c) w[c] = lds128(place_of(r0 + c * kAtOnce + sub));
#pragma unroll
              for (int c = 0; c < kBatch; ++c) {
                const uint32_t ww[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
                most[c] = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 f = unpack_q(kBf16, ww[e]);
                  most[c] = fmaxf(most[c], fmaxf(fabsf(f.x), fabsf(f.y)));
                }
              }
            // level by level, so that the rows' shuffles do not wait for one another
#pragma unroll
              for (int d = 1; d < kLanes; d <<= 1)
#pragma unroll
                for (int c = 0; c < kBatch; ++c) most[c] = fmaxf(most[c], __shfl_xor_sync(0xffffffffu, most[c], d));
#pragma unroll
              for (int c = 0; c < kBatch; ++c) {
                const int ex = q_exponent(most[c]);
                const float by = sign * __uint_as_float((uint32_t)(127 + kQTop - ex) << 23);
                const int at = r0 + c * kAtOnce + sub;
                // the row's own thread keeps its scale
#pragma unroll
                for (int s = 0; s < kAtOnce; ++s) {
                  const int theirs = __shfl_sync(0xffffffffu, ex, s * kLanes);
                  if (lane == r0 + c * kAtOnce + s) qe = __uint_as_float((uint32_t)(127 - kQTop + theirs) << 23);
                }
                const uint32_t ww[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 f = unpack_q(kBf16, ww[e]);
                  o[e] = h2_as_u32(__floats2half2_rn(f.x * by, f.y * by));
                }
                sts128(place_of(at), o[0], o[1], o[2], o[3]);
              }
            }
          };
          if (p.bf16) scale_rows(std::true_type{});
          else scale_rows(std::false_type{});
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(q_full);
          if (live) lim = min(a.lim0 + row / p.group, a.t1 - 1);
        }
        const bool idle = a.row0 + t * 128 >= a.rows;  // no row of this tile: only the barriers that count both
        for (int step = 0; step < a.count; ++step, ++i) {
          const int j0 = a.t0 + step * BN, stage = i & 1;
          wait(const_full + stage, (i >> 1) & 1);
          if (idle) {
            __syncwarp();
            if (lane == 0) mbar_arrive(const_empty + stage);
            continue;
          }
          const uint32_t place = QT == 1 ? i & 1 : 0;  // of the scores and the weights
          const uint32_t s_at = s_at0 + place * BN;
          if constexpr (QT == 1) {
            wait(s_full + place, (i >> 1) & 1);
          } else {
            wait(s_full + t, s_phase);
            s_phase ^= 1;
          }
          tc_fence_after_sync();
          const float4* cs = consts + stage * (BN / 16);
          const int seen = lim - j0;  // columns up to here count
          const bool cut = __any_sync(0xffffffffu, seen < BN - 1);
          // Weights against the reference point m, in one pass; `over`: one has passed 2^kMostWeight, which is not stored.
          uint32_t w[BN / 2];
          float more = 0.f;
          bool over = false;
          auto weights = [&](auto masked) {
            constexpr bool kCut = decltype(masked)::value;
            __half2 high = __float2half2_rn(0.f);
            more = 0.f;
            uint32_t ahead[2][32];  // the next 32 scores are on their way while these are worked on
            tmem_ld32(s_at, ahead[0]);
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) {
              tmem_wait_ld();
              if (c + 1 < BN / 32) tmem_ld32(s_at + (c + 1) * 32, ahead[(c + 1) & 1]);
              const uint32_t(&s)[32] = ahead[c & 1];
#pragma unroll
              for (int g = 0; g < 2; ++g) {
                const float4 k = cs[2 * c + g];
                const float mul = fabsf(k.x) * qe, add = k.y - m;
                const float2 mul2 = make_float2(mul, mul), add2 = make_float2(add, add);
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                  const float2 z = fma2(make_float2(__uint_as_float(s[16 * g + e]), __uint_as_float(s[16 * g + e + 1])), mul2, add2);
                  float2 x = make_float2(exp2_approx(z.x), exp2_approx(z.y));
                  if (kCut) {
                    if (32 * c + 16 * g + e > seen) x.x = 0.f;
                    if (32 * c + 16 * g + e + 1 > seen) x.y = 0.f;
                  }
                  sum = add2f(sum, x);
                  const __half2 h = __floats2half2_rn(x.x, x.y);
                  high = __hmax2(high, h);
                  w[16 * c + 8 * g + e / 2] = h2_as_u32(h);
                }
                more = fmaf(sum.x + sum.y, k.z, more);
              }
            }
            over = __half2float(__hmax(__low2half(high), __high2half(high))) > 32768.f;
          };
          auto both = [&](auto f) {
            if (cut) f(std::true_type{});
            else f(std::false_type{});
          };
          // The reference point moves in a segment's first step and when a weight has passed the limit.
          bool move = step == 0;
#pragma unroll 1
          for (;;) {
            if (move) {
              float top = -INFINITY;
              both([&](auto masked) {
                constexpr bool kCut = decltype(masked)::value;
#pragma unroll 1
                for (int c = 0; c < BN / 16; ++c) {
                  uint32_t s[16];
                  tmem_ld16(s_at + c * 16, s);
                  tmem_wait_ld();
                  const float4 k = cs[c];
                  float high = -INFINITY;
#pragma unroll
                  for (int e = 0; e < 16; ++e)
                    if (!kCut || 16 * c + e <= seen) high = fmaxf(high, __uint_as_float(s[e]));
                  if (high > -INFINITY) top = fmaxf(top, fmaf(high, fabsf(k.x) * qe, k.y));
                }
              });
              float fade = 1.f;
              const float to = top - kUnder;
              if (top > -INFINITY && (to > m || m == kNoMax)) {
                fade = m == kNoMax ? 0.f : exp2_approx(m - to);
                m = to;
                l *= fade;
              }
              if (step > 0) {
                if (QT == 1) {  // the output of the step before may still be on its way
                  wait(wide_empty + 1 + ((i - 1) & 1), ((i - 1) >> 1) & 1);
                  tc_fence_after_sync();
                }
#pragma unroll 1
                for (int c = 0; c < HD / 16; ++c) {
                  uint32_t o[16];
                  tmem_ld16(o_at + c * 16, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fade);
                  tmem_st16(o_at + c * 16, o);
                }
              }
            }
            both(weights);
            if (move || !__any_sync(0xffffffffu, over || m == kNoMax)) break;
            move = true;
          }
          l += more;
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) {
            uint32_t out[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) out[e] = w[16 * c + e];
            tmem_st16(s_at + c * 16, out);
          }
          tmem_wait_st();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(const_empty + stage);
            mbar_arrive(p_full + (QT == 1 ? place : t));
          }
        }
        if (a.count > 0) {
          wait(o_full, seg & 1);
          ++seg;
          tc_fence_after_sync();
        }
        // The run's earlier segments, left by this thread in the CTA's place for partial sums.
        float by = 1.f, by_before = 0.f;
        if (a.goes_on && live) {
          const float2 ml = *reinterpret_cast<const float2*>(part + kRows * HD + 2 * local);
          const float top = fmaxf(m, ml.x);
          by = exp2_approx(m - top);
          by_before = exp2_approx(ml.x - top);
          l = fmaf(l, by, ml.y * by_before);
          m = top;
        }
        const bool writes_out = a.whole && a.last;
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          if (a.count > 0 && !idle) {
            tmem_ld32(o_at + c * 32, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0;
          }
          // partial sums: [4 dims][row], so that a warp writes 32 rows side by side
          const float inv = l == 0.f ? 0.f : kWeightUnit / l;
          if (!live) continue;
          if (a.goes_on) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 x = *reinterpret_cast<const float4*>(part + ((size_t)((c * 32 + e) / 4) * kRows + local) * 4);
              o[e] = __float_as_uint(fmaf(__uint_as_float(o[e]), by, x.x * by_before));
              o[e + 1] = __float_as_uint(fmaf(__uint_as_float(o[e + 1]), by, x.y * by_before));
              o[e + 2] = __float_as_uint(fmaf(__uint_as_float(o[e + 2]), by, x.z * by_before));
              o[e + 3] = __float_as_uint(fmaf(__uint_as_float(o[e + 3]), by, x.w * by_before));
            }
          }
          if (writes_out) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              float num[8];
#pragma unroll
              for (int y = 0; y < 8; ++y) num[y] = __uint_as_float(o[e + y]);
              store_out8(out_row + c * 32 + e, p.bf16, num, inv);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4*>(part + ((size_t)((c * 32 + e) / 4) * kRows + local) * 4) =
                  make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        tc_fence_before_sync();  // the next segment's products overwrite the output
      }
      if (live && !helps && !(a.whole && a.last)) *reinterpret_cast<float2*>(part + kRows * HD + 2 * local) = make_float2(m, l);
      if (!a.whole && a.last) {
        const int c0 = (int)(((a.first_token + 1) * C - 1) / all);
        const int c1 = (int)(((a.first_token + (long long)(a.steps - 1) * BN + 1) * C - 1) / all);
        __threadfence();
        named_barrier_sync(1, 256);
        if (threadIdx.x == 0) *last_one = atomicAdd(counters + c0, 1) == c1 - c0;
        named_barrier_sync(1, 256);
        if (*last_one) {
          __threadfence();
          if (live) {
            auto from = [&](int c) { return parts + ((size_t)(2 * c + (c == c0)) * kRows) * (HD + 2); };
            float top = kNoMax, den = 0.f;
#pragma unroll 4
            for (int c = c0; c <= c1; ++c) {
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(from(c) + kRows * HD + 2 * local));
              const float high = fmaxf(top, ml.x);
              den = fmaf(ml.y, exp2_approx(ml.x - high), den * exp2_approx(top - high));
              top = high;
            }
            const float inv = den == 0.f ? 0.f : kWeightUnit / den;
#pragma unroll 1
            for (int d = helps ? HD / 2 : 0; d < (QT == 1 && !helps ? HD / 2 : HD); d += 32) {
              float num[32];
#pragma unroll
              for (int y = 0; y < 32; ++y) num[y] = 0.f;
              // two partial sums on their way at a time
              for (int c = c0; c <= c1; c += 2) {
                float f[2];
                float4 x[2][8];
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                  const float* part = from(min(c + z, c1));
                  f[z] = __ldcg(part + kRows * HD + 2 * local);
#pragma unroll
                  for (int y = 0; y < 8; ++y) x[z][y] = __ldcg(reinterpret_cast<const float4*>(part + ((size_t)(d / 4 + y) * kRows + local) * 4));
                }
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                  if (c + z > c1) break;
                  const float by = exp2_approx(f[z] - top);
#pragma unroll
                  for (int y = 0; y < 8; ++y) {
                    num[4 * y] = fmaf(x[z][y].x, by, num[4 * y]);
                    num[4 * y + 1] = fmaf(x[z][y].y, by, num[4 * y + 1]);
                    num[4 * y + 2] = fmaf(x[z][y].z, by, num[4 * y + 2]);
                    num[4 * y + 3] = fmaf(x[z][y].w, by, num[4 * y + 3]);
                  }
                }
              }
#pragma unroll
              for (int y = 0; y < 32; y += 8) {
                float out[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) out[e] = num[y + e];
                store_out8(out_row + d + y, p.bf16, out, inv);
              }
            }
          }
          if (threadIdx.x == 0) counters[c0] = 0;
        }
        named_barrier_sync(1, 256);  // *last_one is read before it is written again
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// Counters, then partial sums of two items per CTA.
template <int HD>
size_t tile_workspace(int sms) {
  return kCounterBytes + (size_t)sms * 2 * TileLayout<HD>::kRows * (HD + 2) * 4;
}

// The cache as a 2-D tensor of bytes [blocks * kv_heads * block_size][dim]; one
// box is 16 tokens of one head (a 128-dim part of them), swizzled.
int cache_map(const void* cache, long long rows, int dim, CUtensorMap* out) {
  PFN_cuTensorMapEncodeTiled_v12000 encode;
  int st = get_encoder(&encode);
  if (st != GDSQ_OK) return st;
  const cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)dim};
  const cuuint32_t box[2] = {(cuuint32_t)std::min(dim, 128), 16};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(cache), dims, strides, box, estr,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(GDSQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for a cache of %lld x %d bytes", (int)r, rows, dim);
  return GDSQ_OK;
}

template <int HD, int F, int NT>
int launch_stream(const AttendArgs& a, const DeviceInfo& dev, void* workspace, size_t bytes, cudaStream_t stream) {
  const size_t need = stream_workspace<HD, NT>(dev.sms);
  if (bytes < need)
    return fail(GDSQ_ERR_INVALID_VALUE, "attend_kv8: workspace of %zu bytes, %zu needed", bytes, need);
  const long long rows = ((long long)a.num_blocks * a.kv_heads) << a.block_shift;
  CUtensorMap kmap, vmap;
  int st = cache_map(a.k_cache, rows, HD, &kmap);
  if (st == GDSQ_OK) st = cache_map(a.v_cache, rows, HD, &vmap);
  if (st != GDSQ_OK) return st;
  auto kernel = attend_stream_kernel<HD, F, NT>;
  constexpr int smem = StreamLayout<HD, NT>::kTotal;
  cudaError_t e = ensure_smem(kernel, smem, dev.ordinal);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(attend)");
  const int ctas = dev.sms * stream_per_sm<HD, NT>();
  if ((size_t)ctas * sizeof(int) > kCounterBytes) return fail(GDSQ_ERR_UNSUPPORTED, "attend_kv8: %d SMs", dev.sms);
  int* counters = static_cast<int*>(workspace);
  float* parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
  e = launch(kernel, dim3(ctas), dim3(kAttWarps * 32), smem, stream, g_pdl_enabled != 0, a, kmap, vmap, parts, counters);
  return e == cudaSuccess ? GDSQ_OK : cuda_fail(e, "attend launch");
}

// Rows per (request, KV head) up to which the stream kernel is taken; a tile's 128
// rows are a whole product however few are filled.  Stream against tile, heads of
// 128: 20 rows of 32 requests of 2000 tokens 70 and 84 us, 24 rows of 64 of 4000
// 187 and 251, 32 rows of 16 of 2000 (32 KV heads) 126 and 160.  From 33 rows on the stream
// kernel reads the cache twice: 40 rows of those requests 127 and 89, 367 and 260, 222
// and 164; 64 rows 136 and 88, 381 and 262, 239 and 176; with heads of 64 (32 requests
// of 2000 tokens, 8 KV heads) 72 and 73 with 40 rows, 77 and 73 with 64.  Heads of 256 leave
// the stream kernel registers for 16 rows only: 32 rows of 16 requests of 1000
// tokens would take it two readings of the cache, 33 us, and take the tile kernel 26.
template <int HD>
constexpr int stream_rows() { return HD == 256 ? 16 : 32; }

template <int HD, int F>
int launch_tile(const AttendArgs& a, const DeviceInfo& dev, void* workspace, size_t bytes, cudaStream_t stream) {
  const size_t need = tile_workspace<HD>(dev.sms);
  if (bytes < need)
    return fail(GDSQ_ERR_INVALID_VALUE, "attend_kv8: workspace of %zu bytes, %zu needed", bytes, need);
  if ((size_t)dev.sms * sizeof(int) > kCounterBytes) return fail(GDSQ_ERR_UNSUPPORTED, "attend_kv8: %d SMs", dev.sms);
  const long long rows = ((long long)a.num_blocks * a.kv_heads) << a.block_shift;
  CUtensorMap kmap, vmap;
  int st = cache_map(a.k_cache, rows, HD, &kmap);
  if (st == GDSQ_OK) st = cache_map(a.v_cache, rows, HD, &vmap);
  if (st != GDSQ_OK) return st;
  auto kernel = attend_tile_kernel<HD, F>;
  constexpr int smem = TileLayout<HD>::kTotal;
  cudaError_t e = ensure_smem(kernel, smem, dev.ordinal);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(attend)");
  int* counters = static_cast<int*>(workspace);
  float* parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
  e = launch(kernel, dim3(dev.sms), dim3(kTileThreads), smem, stream, g_pdl_enabled != 0, a, kmap, vmap, parts, counters);
  return e == cudaSuccess ? GDSQ_OK : cuda_fail(e, "attend launch");
}

template <int HD, int F>
int launch_attend(const AttendArgs& a, int max_query_len, const DeviceInfo& dev, void* workspace, size_t bytes,
                  cudaStream_t stream) {
  const long long rows = (long long)max_query_len * a.group;
  if (rows <= 8) return launch_stream<HD, F, 1>(a, dev, workspace, bytes, stream);
  if (rows <= 16) return launch_stream<HD, F, 2>(a, dev, workspace, bytes, stream);
  if constexpr (HD != 256)
    if (rows <= stream_rows<HD>()) return launch_stream<HD, F, 4>(a, dev, workspace, bytes, stream);
  return launch_tile<HD, F>(a, dev, workspace, bytes, stream);
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
  if (num_requests <= 0 || max_query_len <= 0 || num_heads <= 0 || num_kv_heads <= 0) return 0;
  const DeviceInfo* dev = nullptr;
  if (device_info(&dev) != GDSQ_OK) return 0;
  const long long rows = (long long)max_query_len * (num_heads / num_kv_heads);
  // the largest of the variants that up to this many rows can take
  const int n = dev->sms;
  auto most = [&](size_t one, size_t two, size_t four, int upto, size_t tile) {
    return std::max(std::max(one, rows > 8 ? two : 0), std::max(rows > 16 ? four : 0, rows > upto ? tile : 0));
  };
  if (head_dim == 64)
    return most(stream_workspace<64, 1>(n), stream_workspace<64, 2>(n), stream_workspace<64, 4>(n), stream_rows<64>(), tile_workspace<64>(n));
  if (head_dim == 128)
    return most(stream_workspace<128, 1>(n), stream_workspace<128, 2>(n), stream_workspace<128, 4>(n), stream_rows<128>(), tile_workspace<128>(n));
  return most(stream_workspace<256, 1>(n), stream_workspace<256, 2>(n), 0, stream_rows<256>(), tile_workspace<256>(n));
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
  if (!workspace || !aligned(workspace, 16))
    return fail(GDSQ_ERR_MISALIGNED, "attend_kv8: a 16-byte aligned workspace is needed");
  if ((((long long)num_blocks * num_kv_heads * block_size) >> 31) != 0 || num_blocks < 1)
    return fail(GDSQ_ERR_UNSUPPORTED, "attend_kv8: %d blocks of %d heads x %d tokens, not 1 to 2^31 - 1 rows", num_blocks,
                num_kv_heads, block_size);
  if ((long long)table_width * block_size > kMostPositions)
    return fail(GDSQ_ERR_UNSUPPORTED, "attend_kv8: table rows of %d blocks of %d tokens, more than 2^31 - 4096 positions", table_width,
                block_size);
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
  a.scale = softmax_scale * kLog2e;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (cache_type == GDSQ_CACHE_INT8) {
    if (head_dim == 64) return launch_attend<64, GDSQ_CACHE_INT8>(a, max_query_len, *dev, workspace, workspace_bytes, stream);
    if (head_dim == 128) return launch_attend<128, GDSQ_CACHE_INT8>(a, max_query_len, *dev, workspace, workspace_bytes, stream);
    return launch_attend<256, GDSQ_CACHE_INT8>(a, max_query_len, *dev, workspace, workspace_bytes, stream);
  }
  if (head_dim == 64) return launch_attend<64, GDSQ_CACHE_E4M3>(a, max_query_len, *dev, workspace, workspace_bytes, stream);
  if (head_dim == 128) return launch_attend<128, GDSQ_CACHE_E4M3>(a, max_query_len, *dev, workspace, workspace_bytes, stream);
  return launch_attend<256, GDSQ_CACHE_E4M3>(a, max_query_len, *dev, workspace, workspace_bytes, stream);
}
