// Sampling (gdsq_sample).
//
// e_i = exp((l_i - max) / T) and the whole-number weight w_i = floor(2^31 e_i):
// sums of weights are exact, so neither the order of additions nor the number
// of threads can change the token.  A NaN logit counts as -inf; one equal to
// the maximum has e = 1 (so +inf logits share the choice).  In the order
// (logit descending, index ascending) the kept tokens are the longest prefix
// inside the first top_k, with the weight before it below top_p of the
// top_k's, and with e >= min_p; the first is always kept.  The token is the
// first kept index, in index order, whose running sum exceeds floor(u * sum).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
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

// A row is streamed by one cluster, each warp a stretch of it, in blocks of 256
// logits; passes after the first come from L1 and L2.
//
//   1  the maximum of the row, and of each thread's logits
//   2  no cut:    the weight of every block
//      top_k:     the logits that can be among the top k, into a list.  Each CTA
//                 finds a value that ceil(k / CTAs) of its threads' maxima reach; k
//                 logits of the row reach the lowest of these values.
//      top_p:     the weights by 2048 bins of equal width in the logit; then the
//                 logits of the bin where the cut falls, into a list
//   3  the weight of every block that is kept
//   4  the block that holds the target, logit by logit
//
// A list of at most 256 of the top_k goes to one CTA, where every entry is
// compared with every other, which gives its place, the weight before it and
// with that the token; the other CTAs leave.  In longer lists a cut is found by
// histograms over the distance of a logit's ordered bit pattern from the
// maximum's, 2048 bins at a time until a bin is one logit value; ties then
// follow from counts alone.  Where a list overflows, the row itself is counted.
//
// Bound by the passes over a row where top_p stands alone (its bins are shared
// atomics), else by latency: 256 rows of 131072 fp16 logits with all mixes of
// filters take 106 us (10.3 for reading them once), with top_k in each row 39,
// with top_p alone in each 156, without filters 49; one row of 32000 with top_k and top_p 8.9 us; 48
// rows of 50001 fp32 logits without filters 13 us (1.5 for reading).  Counting all
// logits by bins, without lists, the 256 mixed rows took 3270 us and the one row 445.

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBlock = 256;        // logits: 8 per lane
constexpr int kMaxBlocks = 1024;   // per CTA
constexpr int kMaxBinned = 511;    // with top_p: a CTA's weights in units of 2^16, at most 2^15 each, add up below 2^32
constexpr int kBins = 2048;
constexpr int kPerThread = kBins / kThreads;  // a 16-byte vector
static_assert(kPerThread == 4, "bins are read by vectors");
constexpr int kList = 2048;
constexpr int kShort = 256;
constexpr float kWeightCut = -21.6f;  // floor(2^31 exp(z)) = 0 below (ln 2^-31 = -21.49)
constexpr float kOne = 2147483648.f;  // the weight of the largest logit

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

template <typename T>
__device__ __forceinline__ float widen(uint32_t bits) {  // low 16 bits
  if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)bits));
  return __uint_as_float(bits << 16);
}

// The warp's stretch of a row.
template <typename T>
struct Stretch {
  static constexpr int kWords = 8 * sizeof(T) / 4;  // of 8 logits
  static constexpr int kDrop = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16;  // fp32 bits that say nothing
  static constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  const T* row;
  int vocab, skew;  // skew: logits between the 16-byte boundary below the row and its start
  int begin, end;   // blocks

  // Index of this lane's first logit of block b; negative before the row.
  __device__ __forceinline__ int first(int b) const { return b * kBlock + (threadIdx.x & 31) * 8 - skew; }

  __device__ __forceinline__ void load(int b, int to, uint32_t (&w)[kWords]) const {
    const int i = first(b);
#pragma unroll
    for (int j = 0; j < kWords; ++j) w[j] = kNone;
    if (b >= to) return;
    if (i >= 0 && i + 8 <= vocab) {
#pragma unroll
      for (int j = 0; j < kWords; j += 4) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(row + i) + j / 4);
        w[j] = x.x; w[j + 1] = x.y; w[j + 2] = x.z; w[j + 3] = x.w;
      }
    } else if (i + 8 > 0 && i < vocab) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e >= 0 && i + e < vocab) {
          if constexpr (sizeof(T) == 4) {
            w[e] = __float_as_uint(row[i + e]);
          } else {
            const uint32_t x = reinterpret_cast<const unsigned short*>(row)[i + e];
            w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | x << 16 : (w[e / 2] & 0xffff0000u) | x;
          }
        }
    }
  }
  static __device__ __forceinline__ float get(const uint32_t (&w)[kWords], int e) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
    else return widen<T>(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu);
  }

  // fn(b, w) for the warp's blocks, the next ones on their way.
  template <typename Fn>
  __device__ __forceinline__ void each(Fn fn) const {
    uint32_t w0[kWords], w1[kWords], w2[kWords];
    load(begin, end, w0);
    load(begin + 1, end, w1);
#pragma unroll 1
    for (int b = begin; b < end; ++b) {
      load(b + 2, end, w2);
      fn(b, w0);
#pragma unroll
      for (int j = 0; j < kWords; ++j) {
        w0[j] = w1[j];
        w1[j] = w2[j];
      }
    }
  }
};

struct SampleShared {
  alignas(16) uint32_t lo[kBins];  // counts, or low halves of weights
  alignas(16) uint32_t hi[kBins];  // high halves of weights
  uint32_t value[kList];
  int index[kList];
  unsigned long long block[kMaxBlocks];
  uint32_t block_ties[kMaxBlocks];
  unsigned long long sum[kWarps];
  uint32_t num[kWarps];
  // by cluster rank, each written once per launch
  uint32_t rank_top[16], rank_bound[16], rank_count[16], rank_ties[16];
  unsigned long long rank_sum[16], rank_part[16];
  // a scan's answer
  uint32_t bin, found;
  unsigned long long before, at, all;
  int count;  // the list's length
};

// Grid: one cluster of `ranks` CTAs per row.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs p, const int ranks) {
  using Row = Stretch<T>;
  constexpr int kDrop = Row::kDrop, kWords = Row::kWords;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = ranks > 1 ? (int)(blockIdx.x % ranks) : 0;
  const int b = blockIdx.x / ranks;
  const int V = p.vocab;
  auto everyone = [&] {
    if (ranks > 1) cluster_sync_all();
    else __syncthreads();
  };
  // Stores `v` to *slot in every CTA of the cluster; one warp calls it.
  auto tell_u64 = [&](unsigned long long* slot, unsigned long long v) {
    if (ranks == 1) {
      if (lane == 0) *slot = v;
    } else if (lane < ranks) {
      st_cluster_u64(map_to_rank(slot, lane), v);
    }
  };
  auto tell_u32 = [&](uint32_t* slot, uint32_t v) {
    if (ranks == 1) {
      if (lane == 0) *slot = v;
    } else if (lane < ranks) {
      st_cluster_u32(map_to_rank(slot, lane), v);
    }
  };

  if (ranks > 1) cluster_arrive_relaxed();  // waited for before the first store to a peer
  pdl_launch_dependents();
  pdl_wait_primary();
  Row x;
  x.row = static_cast<const T*>(p.logits) + (long long)b * p.row_stride;
  x.vocab = V;
  x.skew = (int)((reinterpret_cast<uintptr_t>(x.row) & 15) / sizeof(T));
  const int blocks = (V + x.skew + kBlock - 1) / kBlock, per_cta = (blocks + ranks - 1) / ranks;
  const int cta_begin = min(rank * per_cta, blocks), cta_end = min(cta_begin + per_cta, blocks);
  const int per_warp = (cta_end - cta_begin + kWarps - 1) / kWarps;
  x.begin = min(cta_begin + warp * per_warp, cta_end);
  x.end = min(x.begin + per_warp, cta_end);

  const float temp = p.temperature ? p.temperature[b] : 1.f;
  const bool greedy = !(temp > 0.f);
  const float inv = greedy ? 1.f : __frcp_rn(temp);
  const float mp = p.min_p ? p.min_p[b] : 0.f;
  const float tp = p.top_p ? p.top_p[b] : 1.f;
  const float u = p.uniforms[b];
  int k = p.top_k ? p.top_k[b] : 0;
  if (greedy || mp > 1.f || !(mp == mp)) k = 1;  // min_p above 1: nothing but the first passes
  if (k <= 0 || k > V) k = V;
  const bool by_count = k > 1 && k < V;
  const bool by_weight = k > 1 && (tp < 1.f || !(tp == tp));
  const int share = (k + ranks - 1) / ranks;
  const bool bounded = by_count && share <= kThreads;

  // 1: the maximum, and a value that `share` of this CTA's threads' maxima reach.
  float own_most = -INFINITY;
  x.each([&](int, const uint32_t(&w)[kWords]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) own_most = fmaxf(own_most, Row::get(w, e));
  });
  {
    const uint32_t w = __reduce_max_sync(0xffffffffu, order_key(own_most));
    if (lane == 0) sh.num[warp] = w;
    for (int i = tid; i < kBins; i += kThreads) {
      sh.lo[i] = 0;
      sh.hi[i] = 0;
    }
    if (tid == 0) {
      sh.found = 0;
      sh.count = 0;
    }
    __syncthreads();
    const uint32_t cta_top = __reduce_max_sync(0xffffffffu, lane < kWarps ? sh.num[lane] : 0);
    float bound = -INFINITY;
    if (bounded) {
      // bins of equal width in the logit, down to where weights vanish
      const float high = key_value(cta_top), width = -kWeightCut / inv / kBins;
      const float d = (high - own_most) / width;
      if (d < (float)kBins) atomicAdd(&sh.lo[(int)d], 1u);
      __syncthreads();
      const uint4 n = *reinterpret_cast<const uint4*>(&sh.lo[tid * kPerThread]);
      const uint32_t nn[4] = {n.x, n.y, n.z, n.w}, sum = n.x + n.y + n.z + n.w;
      uint32_t upto = sum;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, upto, s);
        if (lane >= s) upto += a;
      }
      if (lane == 31) sh.num[warp] = upto;
      __syncthreads();
      uint32_t at = upto - sum;
      for (int i = 0; i < warp; ++i) at += sh.num[i];
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        if (at < (uint32_t)share && at + nn[j] >= (uint32_t)share) {
          sh.bin = tid * kPerThread + j;
          sh.found = 1;
        }
        at += nn[j];
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
  const uint32_t top_key = top >> kDrop;
  // Where the maximum and 1 / T are finite, exp(z) is 1 at the maximum and 0 for -inf by itself, and the weight of a NaN converts
  // to 0.
  const bool regular = isfinite(most) && isfinite(inv);
  auto z_of = [&](float v) { return __fmul_rn(v - most, inv); };
  auto e_of = [&](float v) {
    float e = expf(z_of(v));
    if (!regular) e = v == most ? 1.f : v < most ? e : 0.f;
    return e;
  };
  auto w_of = [&](float v) { return (uint32_t)(e_of(v) * kOne); };
  auto near = [&](float v, float cut) { return v == most || z_of(v) >= cut; };
  auto target_of = [&](unsigned long long whole) {
    const double d = (double)u * (double)whole;
    return min(d > 0.0 ? (unsigned long long)d : 0ull, whole - 1);
  };
  auto limit_of = [&](unsigned long long all) {
    const double d = (double)tp * (double)all;
    return d > 1.0 ? (unsigned long long)ceil(d) : 1ull;
  };
  auto say = [&](int token, uint32_t weight, unsigned long long whole) {
    p.tokens[b] = token;
    if (p.logprobs) p.logprobs[b] = logf((float)((double)weight / (double)whole));
  };
  // Not above any logit with z >= cut, and not below any with z <= cut.
  auto low_of = [&](float cut) {
    const float far = cut / inv;
    return isfinite(most) ? most + far - 1e-5f * (fabsf(most) + fabsf(far)) : -INFINITY;
  };
  auto high_of = [&](float cut) {
    const float far = cut / inv;
    return isfinite(most) && isfinite(far) ? fminf(most, most + far + 1e-5f * (fabsf(most) + fabsf(far))) : most;
  };
  auto distance = [&](float v) { return top_key - min(order_key(v) >> kDrop, top_key); };

  // Adds up the bins over the cluster, in order, from `before` on: sh.bin is the one
  // where the sum reaches want(all) (sh.found), sh.before the sum ahead of it, sh.at
  // its own and sh.all the whole.  fix(bin) is taken off a bin.
  auto scan = [&](bool weights, unsigned long long before, auto want, auto fix) {
    everyone();
    if (rank == 0) {
      unsigned long long mine[kPerThread], sum = 0;
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        mine[j] = sh.lo[tid * kPerThread + j];
        if (weights) mine[j] += (unsigned long long)sh.hi[tid * kPerThread + j] << 16;
      }
      // two peers' bins on their way at a time
#pragma unroll 1
      for (int r = 1; r < ranks; r += 2) {
        uint4 lo[2], hi[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
          if (r + i < ranks) {
            lo[i] = ld_cluster_v4(map_to_rank(&sh.lo[tid * kPerThread], r + i));
            if (weights) hi[i] = ld_cluster_v4(map_to_rank(&sh.hi[tid * kPerThread], r + i));
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          mine[0] += lo[i].x + ((unsigned long long)hi[i].x << 16);
          mine[1] += lo[i].y + ((unsigned long long)hi[i].y << 16);
          mine[2] += lo[i].z + ((unsigned long long)hi[i].z << 16);
          mine[3] += lo[i].w + ((unsigned long long)hi[i].w << 16);
        }
      }
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        mine[j] -= fix(tid * kPerThread + j);
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
      unsigned long long at = before + upto - sum, all = before;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) at += sh.sum[i];
        all += sh.sum[i];
      }
      const unsigned long long goal = want(all);
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        if (at < goal && at + mine[j] >= goal) {
          sh.bin = tid * kPerThread + j;
          sh.before = at;
          sh.at = mine[j];
          sh.found = 1;
        }
        at += mine[j];
      }
      if (tid == 0) sh.all = all;
      __syncthreads();
      if (warp == 0 && ranks > 1) {
        const uint32_t bin = sh.bin, found = sh.found;
        const unsigned long long ahead = sh.before, in = sh.at, whole = sh.all;
        __syncwarp();
        tell_u32(&sh.bin, bin);
        tell_u32(&sh.found, found);
        tell_u64(&sh.before, ahead);
        tell_u64(&sh.at, in);
        tell_u64(&sh.all, whole);
      }
    }
    everyone();
  };
  auto clear = [&] {
    for (int i = tid; i < kBins; i += kThreads) {
      sh.lo[i] = 0;
      sh.hi[i] = 0;
    }
    __syncthreads();
  };
  const bool carries = per_cta * kBlock > 65536;  // the low halves of this many weights can pass 2^32
  auto put = [&](bool weights, uint32_t bin, uint32_t w) {
    if (weights) {
      const uint32_t low = w & 0xffffu;
      uint32_t high = w >> 16;
      if (carries) high += atomicAdd(&sh.lo[bin], low) + low < low ? 65536u : 0u;
      else atomicAdd(&sh.lo[bin], low);
      atomicAdd(&sh.hi[bin], high);
    } else {
      atomicAdd(&sh.lo[bin], 1u);
    }
  };

  // The value where the running sum over falling logits reaches `want`: its distance
  // `first` from the maximum, `before` the sum over nearer ones, `at` the value's own.
  // each(f) calls f(logit) for the candidates, at distances [first, first + span).
  struct Cut {
    uint32_t first;
    unsigned long long before, at;
    bool found;
  };
  auto histogram = [&](unsigned long long want, uint32_t first, uint32_t span, unsigned long long before, bool weights, auto each,
                       auto fix) {
    Cut c{first, before, 0, true};
    for (;;) {
      const int shift = max(0, 21 - __clz(span - 1));  // span <= 2048 << shift
      clear();
      each([&](float v) {
        const uint32_t d = top_key - (order_key(v) >> kDrop) - c.first;
        if (d < span) put(weights, d >> shift, weights ? w_of(v) : 1u);
      });
      scan(weights, c.before, [&](unsigned long long) { return want; },
           [&](uint32_t bin) { return fix(c.first + (bin << shift), c.first + ((bin + 1) << shift)); });
      c.found = sh.found != 0;
      if (!c.found) return c;
      c.before = sh.before;
      c.at = sh.at;
      c.first += sh.bin << shift;
      if (shift == 0) return c;
      span = 1u << shift;
    }
  };
  // Puts the logits with in(v) into the CTAs' lists; the longest list and the number of all.
  int longest = 0, listed = 0;
  auto gather = [&](auto in) {
    x.each([&](int blk, const uint32_t(&w)[kWords]) {
      uint32_t mask = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) mask |= (uint32_t)in(Row::get(w, e)) << e;
      if (mask) {
        int at = atomicAdd(&sh.count, __popc(mask));
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (mask >> e & 1) {
            if (at < kList) {
              sh.value[at] = __float_as_uint(Row::get(w, e));
              sh.index[at] = x.first(blk) + e;
            }
            ++at;
          }
      }
    });
    __syncthreads();
    if (warp == 0) tell_u32(&sh.rank_count[rank], sh.count);
    everyone();
    for (int r = 0; r < ranks; ++r) {
      longest = max(longest, (int)sh.rank_count[r]);
      listed += sh.rank_count[r];
    }
  };
  // f(logit) for this CTA's candidates: its list, or the row where a list has overflowed.
  auto candidates = [&](auto in, auto f) {
    if (longest <= kList) {
      for (int i = tid; i < sh.count; i += kThreads) f(__uint_as_float(sh.value[i]));
    } else {
      x.each([&](int, const uint32_t(&w)[kWords]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = Row::get(w, e);
          if (in(v)) f(v);
        }
      });
    }
  };

  // 2: kept are keys above `thr`, and the first `ties` (in index order) of those equal to it
  uint32_t thr = 0, ties = 0xffffffffu;
  const float min_cut = mp > 0.f ? fmaxf(kWeightCut, logf(mp) - 1e-3f) : kWeightCut;
  auto value_of = [&](uint32_t key) {  // the logit with this key
    const uint32_t full = key << kDrop;
    return key_value(full & 0x80000000u ? full : full | ((1u << kDrop) - 1));
  };
  auto cut_at = [&](const Cut& c, unsigned long long limit, bool again) {  // a weight's cut
    const uint32_t key = top_key - c.first;
    const unsigned long long w = w_of(value_of(key));
    const uint32_t n = (uint32_t)min((limit - c.before + w - 1) / w, 0xffffffffull);
    ties = again && key == thr ? min(ties, n) : n;
    thr = key;
  };
  auto no_fix = [](uint32_t, uint32_t) { return 0ull; };
  if (k == 1) {
    thr = top_key;
    ties = 1;
  } else if (by_count) {
    uint32_t bound = 0xffffffffu;
    for (int r = 0; r < ranks; ++r) bound = min(bound, sh.rank_bound[r]);
    const float low = fmaxf(key_value(bound), low_of(by_weight ? kWeightCut : min_cut));
    auto in = [&](float v) { return v >= low; };
    gather(in);
    if (listed <= kShort) {
      // to the first CTA; its own entries are in place
      if (ranks > 1) {
        int at = 0;
        for (int r = 0; r < rank; ++r) at += sh.rank_count[r];
        if (rank > 0 && tid < sh.count) {
          st_cluster_u32(map_to_rank(&sh.value[at + tid], 0), sh.value[tid]);
          st_cluster_u32(map_to_rank(&sh.index[at + tid], 0), (uint32_t)sh.index[tid]);
        }
        everyone();
        if (rank != 0) return;
      }
      if (tid >= kShort) return;
      auto sync = [] { named_barrier_sync(1, kShort); };
      const bool live = tid < listed;
      const float v = live ? __uint_as_float(sh.value[tid]) : -INFINITY;
      const int index = live ? sh.index[tid] : 0x7fffffff;
      const uint32_t key = order_key(v);
      const float e = live ? e_of(v) : 0.f;
      const uint32_t w = (uint32_t)(e * kOne);
      sh.lo[tid] = live ? key : 0;
      sh.hi[tid] = w;
      sh.lo[kShort + tid] = index;
      sync();
      const uint32_t keys = smem_addr(sh.lo), weights = smem_addr(sh.hi), order = keys + 4 * kShort;
      uint32_t place = 0;
      unsigned long long ahead = 0;
      if (warp * 32 < listed)
        for (int j = 0; j < listed; j += 4) {
          const uint4 kj = lds128(keys + 4 * j), wj = lds128(weights + 4 * j), ij = lds128(order + 4 * j);
          const uint32_t kk[4] = {kj.x, kj.y, kj.z, kj.w}, ww[4] = {wj.x, wj.y, wj.z, wj.w};
          const int ii[4] = {(int)ij.x, (int)ij.y, (int)ij.z, (int)ij.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const bool first = kk[y] > key || (kk[y] == key && ii[y] < index);
            place += first;
            ahead += first ? ww[y] : 0;
          }
        }
      auto sum_of = [&](unsigned long long s) {
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        if (lane == 0) sh.sum[warp] = s;
        sync();
        s = 0;
        for (int i = 0; i < kShort / 32; ++i) s += sh.sum[i];
        sync();
        return s;
      };
      bool keep = live && place < (uint32_t)k;
      if (by_weight) {
        const unsigned long long limit = limit_of(sum_of(keep ? w : 0));
        keep = keep && ahead < limit;
      }
      keep = keep && (e >= mp || place == 0);
      sync();
      sh.hi[tid] = keep ? w : 0;
      sync();
      unsigned long long upto = 0, whole = 0;
      if (warp * 32 < listed)
        for (int j = 0; j < listed; j += 4) {
          const uint4 wj = lds128(weights + 4 * j), ij = lds128(order + 4 * j);
          const uint32_t ww[4] = {wj.x, wj.y, wj.z, wj.w};
          const int ii[4] = {(int)ij.x, (int)ij.y, (int)ij.z, (int)ij.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            whole += ww[y];
            upto += ii[y] < index ? ww[y] : 0;
          }
        }
      if (keep) {
        const unsigned long long target = target_of(whole);
        if (upto <= target && target < upto + w) say(index, w, whole);
      }
      return;
    }
    uint32_t span = distance(low) + 2;
    const Cut c = histogram(k, 0, span, 0, false, [&](auto f) {
      candidates(in, [&](float v) {
        if (near(v, kWeightCut)) f(v);
      });
    }, no_fix);
    if (c.found) {
      thr = top_key - c.first;
      ties = k - (uint32_t)c.before;
      span = c.first + 1;
    }
    if (by_weight) {
      const float at_thr = value_of(thr);
      const unsigned long long w_thr = c.found ? w_of(at_thr) : 0;
      unsigned long long own = 0;
      candidates(in, [&](float v) {
        if ((order_key(v) >> kDrop) > thr && near(v, kWeightCut)) own += w_of(v);
      });
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) own += __shfl_xor_sync(0xffffffffu, own, m);
      if (lane == 0) sh.sum[warp] = own;
      __syncthreads();
      if (warp == 0) {
        own = lane < kWarps ? sh.sum[lane] : 0;
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) own += __shfl_xor_sync(0xffffffffu, own, m);
        tell_u64(&sh.rank_part[rank], own);
      }
      everyone();
      unsigned long long all = c.found ? ties * w_thr : 0;
      for (int r = 0; r < ranks; ++r) all += sh.rank_part[r];
      const unsigned long long limit = limit_of(all);
      const uint32_t at = top_key - thr;
      const unsigned long long extra = c.found && near(at_thr, kWeightCut) ? (c.at - ties) * w_thr : 0;
      const Cut d = histogram(limit, 0, span, 0, true, [&](auto f) {
        candidates(in, [&](float v) {
          if (near(v, kWeightCut)) f(v);
        });
      }, [&](uint32_t lo, uint32_t hi) { return extra && lo <= at && at < hi ? extra : 0ull; });
      if (d.found) cut_at(d, limit, c.found);
    }
  } else if (by_weight) {
    const float per_bin = kBins / -kWeightCut;
    auto bin_of = [&](float v) { return v == most ? 0 : min((int)(-z_of(v) * per_bin), kBins - 1); };
    x.each([&](int, const uint32_t(&w)[kWords]) {
      uint32_t weight[8];
      int at[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        weight[e] = w_of(Row::get(w, e));
        at[e] = bin_of(Row::get(w, e));
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (weight[e]) put(true, at[e], weight[e]);
    });
    scan(true, 0, limit_of, [](uint32_t) { return 0ull; });
    if (sh.found) {
      const unsigned long long limit = limit_of(sh.all), before = sh.before;
      const int bin = sh.bin;
      const float low = low_of(-(float)(bin + 1) / per_bin), high = high_of(-(float)bin / per_bin);
      auto in = [&](float v) { return (v >= low) & (v <= high) && bin_of(v) == bin; };
      gather(in);
      const uint32_t first = distance(high);
      const Cut c = histogram(limit, first, distance(low) + 2 - first, before, true, [&](auto f) { candidates(in, f); }, no_fix);
      if (c.found) cut_at(c, limit, false);
    }
  }

  // 3: the kept weight of every block, apart from that of ties, and of the warp's stretch
  const float edge = thr ? value_of(thr) : low_of(min_cut);  // no filter but min_p: below every kept logit, so equal to none
  const bool all_of = thr == 0 && !(mp > 0.f);
  // Kept weights of 8 logits, and which of them are ties.
  auto kept = [&](const uint32_t(&w)[kWords], uint32_t(&weight)[8]) {
    uint32_t tie = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = Row::get(w, e);
      const float x1 = e_of(v);
      const bool keep = v >= edge && (x1 >= mp || v == most);
      weight[e] = keep ? (uint32_t)(x1 * kOne) : 0;
      tie |= (uint32_t)(keep && v == edge) << e;
    }
    return thr ? tie : 0;
  };
  unsigned long long own = 0, own_ties = 0;
  x.each([&](int blk, const uint32_t(&w)[kWords]) {
    float high = Row::get(w, 0);
#pragma unroll
    for (int e = 1; e < 8; ++e) high = fmaxf(high, Row::get(w, e));
    unsigned long long sum = 0;
    uint32_t tied = 0;
    if (__any_sync(0xffffffffu, high >= edge)) {
      uint32_t tie = 0;
      if (all_of) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += w_of(Row::get(w, e));
      } else {
        uint32_t weight[8];
        tie = kept(w, weight);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += tie >> e & 1 ? 0 : weight[e];
      }
      // 8 x 2^31 at most: two sums of 32 lanes in 32 bits
      const uint32_t a = __reduce_add_sync(0xffffffffu, (uint32_t)sum & 0xffffu), c = __reduce_add_sync(0xffffffffu, (uint32_t)(sum >> 16));
      sum = a + ((unsigned long long)c << 16);
      tied = thr ? __reduce_add_sync(0xffffffffu, __popc(tie)) : 0;
    }
    if (lane == 0) {
      sh.block[blk - cta_begin] = sum;
      sh.block_ties[blk - cta_begin] = tied;
    }
    own += sum;
    own_ties += tied;
  });
  if (lane == 0) {
    sh.sum[warp] = own;
    sh.num[warp] = (uint32_t)own_ties;
  }
  __syncthreads();
  if (warp == 0) {
    unsigned long long a = lane < kWarps ? sh.sum[lane] : 0;
    const uint32_t c = __reduce_add_sync(0xffffffffu, lane < kWarps ? sh.num[lane] : 0);
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) a += __shfl_xor_sync(0xffffffffu, a, m);
    tell_u64(&sh.rank_sum[rank], a);
    tell_u32(&sh.rank_ties[rank], c);
  }
  everyone();
  // Sums ahead of this warp: of its CTA's warps (lanes 0 to 15) and of the CTAs (from lane 16 on).
  unsigned long long before = 0, whole = 0;
  uint32_t ties_before = 0, ties_all = 0;
  if (lane < kWarps && lane < warp) {
    before = sh.sum[lane];
    ties_before = sh.num[lane];
  } else if (lane >= 16 && lane - 16 < ranks) {
    whole = sh.rank_sum[lane - 16];
    ties_all = sh.rank_ties[lane - 16];
    if (lane - 16 < rank) {
      before = whole;
      ties_before = ties_all;
    }
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, m);
    whole += __shfl_xor_sync(0xffffffffu, whole, m);
  }
  ties_before = __reduce_add_sync(0xffffffffu, ties_before);
  ties_all = __reduce_add_sync(0xffffffffu, ties_all);
  const uint32_t w_thr = ties_all ? w_of(edge) : 0;
  auto with_ties = [&](unsigned long long sum, uint32_t n) { return sum + (unsigned long long)min(n, ties) * w_thr; };
  whole = with_ties(whole, ties_all);
  const unsigned long long target = target_of(whole);
  if (!(with_ties(before, ties_before) <= target && target < with_ties(before + own, ties_before + (uint32_t)own_ties))) return;

  // 4: this warp's stretch holds the target: the block, then the logit
  int blk = x.begin;
  for (int at = x.begin; at < x.end; at += 32) {
    const unsigned long long sum = at + lane < x.end ? sh.block[at + lane - cta_begin] : 0;
    const uint32_t tied = at + lane < x.end ? sh.block_ties[at + lane - cta_begin] : 0;
    unsigned long long upto = sum;
    uint32_t upto_ties = tied;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned long long a = __shfl_up_sync(0xffffffffu, upto, d);
      const uint32_t c = __shfl_up_sync(0xffffffffu, upto_ties, d);
      if (lane >= d) {
        upto += a;
        upto_ties += c;
      }
    }
    const unsigned hits = __ballot_sync(0xffffffffu, target < with_ties(before + upto, ties_before + upto_ties));
    const int hit = hits ? __ffs(hits) - 1 : 31;
    if (hits) {
      upto -= sum;
      upto_ties -= tied;
    }
    before += __shfl_sync(0xffffffffu, upto, hit);
    ties_before += __shfl_sync(0xffffffffu, upto_ties, hit);
    if (hits) {
      blk = at + hit;
      break;
    }
  }
  uint32_t w[kWords], weight[8];
  x.load(blk, x.end, w);
  const uint32_t tie = kept(w, weight);
  unsigned long long sum = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum += tie >> e & 1 ? 0 : weight[e];
  unsigned long long upto = sum;
  uint32_t upto_ties = __popc(tie);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned long long a = __shfl_up_sync(0xffffffffu, upto, d);
    const uint32_t c = __shfl_up_sync(0xffffffffu, upto_ties, d);
    if (lane >= d) {
      upto += a;
      upto_ties += c;
    }
  }
  before += upto - sum;
  ties_before += upto_ties - __popc(tie);
  const bool here = with_ties(before, ties_before) <= target &&
                    target < with_ties(before + sum, ties_before + __popc(tie));
  if (!here) return;
  int chosen = 0;
  uint32_t share_of = 0;
  bool found = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (tie >> e & 1) ++ties_before;
    else before += weight[e];
    if (!found && target < with_ties(before, ties_before)) {
      found = true;
      chosen = e;
      share_of = weight[e];
    }
  }
  say(x.first(blk) + chosen, share_of, whole);
}

// CTAs per row: enough to fill the GPU, two to an SM, with 16 blocks (4096 logits)
// each at least, and at most 8; at least as many as hold a row's block sums.  With
// top_p, which makes some rows several times as long as others, up to twice as
// many CTAs as run at a time: 256 rows of 131072, one in four with top_p alone,
// take 134 us with one CTA each, 107 with two, 127 with four (all with top_k:
// 30, 40 and 54).
template <typename T>
int launch_sample(const SampleArgs& a, int rows, cudaStream_t stream) {
  const DeviceInfo* dev = nullptr;
  const int st = device_info(&dev);
  if (st != GDSQ_OK) return st;
  const int blocks = (a.vocab + 8 + kBlock - 1) / kBlock;
  int ranks = 1;
  while (ranks < 8 && (blocks > ranks * (a.top_p ? kMaxBinned : kMaxBlocks) || (ranks * rows <= dev->sms * (a.top_p ? 2 : 1) && blocks >= 32 * ranks))) ranks *= 2;
  auto kernel = sample_kernel<T>;
  cudaError_t e = ensure_smem(kernel, (int)sizeof(SampleShared), dev->ordinal);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(sample)");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * ranks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(SampleShared);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (ranks > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = ranks;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (g_pdl_enabled) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  e = cudaLaunchKernelEx(&cfg, kernel, a, ranks);
  return e == cudaSuccess ? GDSQ_OK : cuda_fail(e, "sample launch");
}

}  // namespace
}  // namespace gdsq

using namespace gdsq;

extern "C" int gdsq_sample(int elem_type, const void* logits, long long row_stride, int num_rows, int vocab,
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
