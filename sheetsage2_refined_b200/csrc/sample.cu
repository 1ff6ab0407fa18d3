// Token sampling from given uniforms: s2r_sample.
//
// The grammar-masked selection of select.cuh / noalloc.cu picks the largest
// allowed logit; this draws from the allowed tokens instead.  With
// x_i = float(logit_i) + bias_i over the allowed tokens, M = max x and
// w_i = exp((x_i - M) / T), tokens ordered by value (descending), then index:
//   top-k   the first k;
//   top-p   of those the shortest prefix whose weights reach p of their sum;
//   min-p   of those the ones with w_i >= min_p;
//   token   the lowest index whose running sum of kept weights exceeds
//           u * (their sum);
//   logprob x_t - M - log sum_allowed exp(x - M): the token's log-probability
//           before temperature and filters, to rank readings by.
//
// Every filter keeps a prefix of one order, so what is kept is "values above a
// threshold, and the first few of the threshold's ties".  Most draws keep few
// tokens, and those are found by a sieve: where k lanes hold a value of at least
// L, so do k tokens, so the k-th largest of what each lane holds at most bounds
// the k-th largest token from below, and little more than k tokens pass it.
// Top-p alone starts from a histogram of the weights over 1024 bins linear in
// M - x: the bin in which the sum crosses its share bounds what is kept.  Up to
// 2048 tokens from the bound on are gathered and finished by one CTA.  Where
// there are more, the threshold is searched among all: a histogram of counts or
// weights, then the tokens of the crossing bin, gathered and sorted; and when
// that bin holds too many (masses of equal values), radix rounds over the images.
//
// Weights are fixed-point integers, rint(exp(.) * 2^(61 - bits(vocab))), with
// the exponential in 64 bits: which token is drawn depends on which side of a
// border a running sum falls, integer sums do not depend on the order in
// which threads add, and the rounding (2^-46 of the largest weight at 32,576
// tokens) is far below what a 32-bit sum could resolve.  Tokens whose weight
// rounds to 0 cannot be drawn.  With top-k only what passed the sieve needs the
// exponential.
//
// A row is one thread-block cluster of C CTAs, each holding a contiguous
// share of the vocabulary as images in shared memory; sums cross the cluster
// through distributed shared memory, one cluster barrier per exchange, so a
// call needs no scratch memory, no atomics on global memory and one launch.
//
// What bounds it: a few rows, the chain of exchanges (one row of 32,576 tokens,
// top-k 50 and top-p: 12 us, of it 2 loading; 16 rows of 2,048: 5.3 us); many
// rows, instruction issue and the barriers, not memory (1,024 rows of 32,576
// float32 logits with mask, bias, top-k 200 and top-p: 136 us, 1.2 TB/s, half
// of the issue slots; without the top-k sieve, so with every token's weight in
// 64 bits, 245 us).
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdio>
#include <mutex>

#include "../../include/s2r.h"
#include "common.cuh"
#include "sample.cuh"

namespace s2r {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 1024;  // of either histogram
constexpr int kSampleBinBits = 10;
constexpr int kSampleMaxSplits = 16;
constexpr uint32_t kImgNegInf = 0x007fffffu;  // image of -inf: tokens at or below it are never drawn
constexpr uint32_t kImgPosInf = 0xff800000u;

// Tokens of a list that is gathered: past the sieve, or of the crossing bin.  (Few splits come with
// large shares of the vocabulary and many rows: half the lists let two CTAs fit an SM.)
__host__ __device__ constexpr int list_max(int splits) { return splits >= 4 ? 2048 : 1024; }

template <int C>
struct alignas(16) SampleShared {  // (the images behind it are stored four at a time)
  u64 hist[2][kSampleBins];             // by parity of the exchange, so one cluster barrier each suffices
  u64 list[list_max(C)];                // this CTA's tokens past the sieve, or of the crossing bin
  u64 sorted[list_max(C)];              // the cluster's
  u64 inbox[2][kSampleMaxSplits][2];    // what the peers sent, by parity of the exchange
  u64 part[kSampleWarps];               // per-warp values of a block reduction
  u64 scan[kSampleWarps];
  double pow2[64];                      // 2^(j / 64)
  u64 found[2];
  unsigned listed, counts[kSampleWarps];
};

// Order-preserving image of a float (select.cuh): -0 as +0, every NaN on top.  The addition makes +0 of
// -0 and the canonical (positive) NaN of every NaN.
__device__ __forceinline__ uint32_t value_image(float v) {
  const uint32_t u = __float_as_uint(__fadd_rn(v, 0.f));
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float image_value(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// What a lane knows of its tokens after loading them: the largest image, the lowest drawable one less
// kImgNegInf + 1 (those that cannot be drawn wrap to the top), and z = sum exp(x - m) over the allowed with m
// the largest value (kept up as the sum of a running softmax).
struct LaneStats {
  uint32_t top = 0, bottom = 0xffffffffu;
  float m = -INFINITY, z = 0.f;
};

__device__ __forceinline__ float exp_approx(float x) { return exp2_approx(x * 1.4426950408889634f); }

// This warp's images [w0, w1) (masked tokens as -inf) into shared memory.  VEC: the row's
// logits, mask and bias allow four tokens a load.
template <typename T, bool VEC>
__device__ __forceinline__ void load_images(const T* __restrict__ logits, const float* __restrict__ bias,
                                            const uint8_t* __restrict__ allowed, uint32_t* img, int w0, int w1,
                                            LaneStats& st) {
  constexpr int kEach = VEC ? 4 : 1, kBatch = VEC ? 4 : 2;  // loads in flight a lane: kBatch of each kind
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int i0 = w0 + lane * kEach; i0 < w1; i0 += 32 * kEach * kBatch) {
    alignas(16) T raw[kBatch][kEach];
    float4 b[VEC ? kBatch : 1];
    float b1[kBatch];
    uint32_t mask[kBatch];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int i = i0 + q * 32 * kEach;
      mask[q] = 0;
      if (i >= w1) continue;
      if constexpr (VEC) {
        if constexpr (sizeof(T) == 4)
          *reinterpret_cast<uint4*>(raw[q]) = __ldg(reinterpret_cast<const uint4*>(logits + i));
        else
          *reinterpret_cast<uint2*>(raw[q]) = __ldg(reinterpret_cast<const uint2*>(logits + i));
        mask[q] = allowed ? __ldg(reinterpret_cast<const uint32_t*>(allowed + i)) : 0xffffffffu;
        b[q] = bias ? __ldg(reinterpret_cast<const float4*>(bias + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
      } else {
        raw[q][0] = logits[i];
        mask[q] = allowed ? allowed[i] : 1u;
        b1[q] = bias ? bias[i] : 0.f;
      }
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int i = i0 + q * 32 * kEach;
      if (i >= w1) break;
      float x[kEach];
      uint32_t u[kEach];
      float m = st.m;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const float add = VEC ? (j == 0 ? b[q].x : j == 1 ? b[q].y : j == 2 ? b[q].z : b[q].w) : b1[q];
        const bool ok = ((mask[q] >> (8 * j)) & 0xffu) != 0;
        x[j] = bias ? __fadd_rn(to_float(raw[q][j]), add) : to_float(raw[q][j]);
        x[j] = ok ? x[j] : -INFINITY;
        u[j] = value_image(x[j]);
        st.top = max(st.top, u[j]);
        st.bottom = min(st.bottom, u[j] - (kImgNegInf + 1));
        m = fmaxf(m, x[j]);
      }
      if (m != -INFINITY) {
        float z = st.z * exp_approx(st.m - m);
#pragma unroll
        for (int j = 0; j < kEach; ++j) z += exp_approx(x[j] - m);
        st.z = z;
        st.m = m;
      }
      if constexpr (VEC)
        *reinterpret_cast<uint4*>(img + i) = make_uint4(u[0], u[1], u[2], u[3]);
      else
        img[i] = u[0];
    }
  }
}

template <typename T>
__device__ __forceinline__ void load_images(const SampleArgs& a, int r, int first, uint32_t* img, int w0, int w1,
                                            LaneStats& st) {
  const T* logits = static_cast<const T*>(a.logits) + (size_t)r * a.logits_stride + first;
  const uint8_t* allowed = a.allowed ? a.allowed + (size_t)r * a.allowed_stride + first : nullptr;
  const float* bias = a.bias ? a.bias + first : nullptr;
  // w0 and first are multiples of 4; only a row's last tokens can be fewer
  const bool vec = reinterpret_cast<uintptr_t>(logits) % (4 * sizeof(T)) == 0 &&
                   reinterpret_cast<uintptr_t>(allowed) % 4 == 0 && reinterpret_cast<uintptr_t>(bias) % 16 == 0;
  int from = w0;
  if (vec) {
    from = w0 + (w1 - w0) / 4 * 4;
    load_images<T, true>(logits, bias, allowed, img, w0, from, st);
  }
  load_images<T, false>(logits, bias, allowed, img, from, w1, st);
}

// The warps' partials, one a lane (twice over a warp), added up by every warp for itself.
__device__ __forceinline__ u64 sum_partials(u64 v) {
#pragma unroll
  for (int o = kSampleWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One row's search state; every thread of the cluster (of C CTAs) holds the same values.
template <int C>
struct RowSampler {
  SampleShared<C>& sh;
  const uint32_t* img;  // this CTA's images
  int first;            // its share of the vocabulary
  int rank;
  int w0, w1;           // this warp's part of the share
  int turn = 0;         // exchanges done (parity of the buffers)
  float best;
  double inv_t;  // 1 / (T ln 2)
  int scale_bits;

  __device__ void barrier() {
    if (C > 1)
      cg::this_cluster().sync();
    else
      __syncthreads();
  }
  template <typename T>
  __device__ T* peer(T* p, int r) {
    return C > 1 ? cg::this_cluster().map_shared_rank(p, r) : p;
  }

  // Sum of `v` over the block, on every thread.
  __device__ u64 block_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = v;
    __syncthreads();
    return sum_partials(sh.part[threadIdx.x & (kSampleWarps - 1)]);
  }
  // Send a block-uniform pair to every CTA of the cluster; behind the barrier inbox[r] holds rank
  // r's.  Senders write into the peers' memory, so what follows reads only this CTA's own.
  __device__ const u64 (*exchange(u64 a, u64 b))[2] {
    u64(*box)[2] = sh.inbox[turn & 1];
    ++turn;
    if (threadIdx.x < C) {
      u64* dst = peer(box[rank], (int)threadIdx.x);
      dst[0] = a;
      dst[1] = b;
    }
    barrier();
    return box;
  }

  // Bins of best - x, `per_unit` to a unit, the largest values in bin 0.
  float per_unit;
  __device__ int bin_of(uint32_t u) const { return min(kSampleBins - 1, (int)((best - image_value(u)) * per_unit)); }
  // The lowest image whose bin is at most `b` (the bins fall as the images rise): 32 probes a round,
  // by every warp for itself.
  __device__ uint32_t bin_floor(int b) const {
    uint32_t lo = kImgNegInf + 1, n = value_image(best) - kImgNegInf;  // candidates lo .. lo + n - 1; the last one is in
    while (n > 1) {
      const uint32_t step = (n + 31) / 32, at = lo + min((uint32_t)(threadIdx.x & 31) * step + step - 1, n - 1);
      const unsigned in = __ballot_sync(0xffffffffu, bin_of(at) <= b);
      const uint32_t skip = (uint32_t)(__ffs(in) - 1) * step;  // the first group whose last candidate is in
      lo += skip;
      n = min(step, n - skip);
    }
    return lo;
  }

  // rint(exp((x - best) / T) * 2^scale_bits): y = (x - best) / (T ln 2) = k / 64 + f, 2^y =
  // 2^(k >> 6) * pow2[k & 63] * 2^f with |f| <= 1/128 (the table-driven exponential of Tang, 1989),
  // 2^f by its series: the first term left out is (ln2 / 128)^6 / 720 = 4e-17.
  __device__ u64 weight(uint32_t u) {
    const double y = ((double)image_value(u) - (double)best) * inv_t;  // (T's factor holds 1 / ln 2)
    if (!(y > -62.0 - 1.0)) return 0;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer in the low word
    const double shifted = fma(y, 64.0, magic);
    const int k = __double2loint(shifted);
    const double f = fma(shifted - magic, -0.015625, y);
    double q = fma(f, 0x1.5d87fe78a6730p-10, 0x1.3b2ab6fba4e77p-7);
    q = fma(f, q, 0x1.c6b08d704a0bfp-5);
    q = fma(f, q, 0x1.ebfbdff82c58ep-3);
    q = fma(f, q, 0x1.62e42fefa39efp-1);
    const double m = sh.pow2[k & 63] * fma(f, q, 1.0);
    return __double2ull_rn(m * __hiloint2double(((k >> 6) + scale_bits + 1023) << 20, 0));
  }
};

// What a row keeps: images above `lo`, and of those equal to it the indices up to `last`.
struct Kept {
  uint32_t lo = kImgNegInf;  // exclusive below kImgNegInf + 1: every drawable token
  int last = -1;
  __device__ bool has(uint32_t u, int i) const { return u > lo || (u == lo && i <= last); }
};

// The shortest prefix of `kept` whose sum of value(token) reaches `target` (1 <= target <= the sum
// over `kept`), by radix rounds over the images.  COUNT: value = 1, else the weight.
// Out of line and by value: rare, and the common path's state stays in registers.
struct RadixResult {
  Kept kept;
  int turn;
};
template <bool COUNT, int C>
__device__ __noinline__ RadixResult shrink_radix(RowSampler<C> row, Kept kept, u64 target) {
  SampleShared<C>& sh = row.sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t lo = kept.lo + (kept.last < 0 ? 1u : 0u), hi = value_image(row.best);  // open range, both inclusive
  u64 above = 0;                                                                    // sum over images > hi
  u64 group = 0;                                                                    // sum over the last bin
  for (;;) {
    const uint32_t range = hi - lo;
    const int bits = 32 - __clz(range);
    const int shift = bits > kSampleBinBits ? bits - kSampleBinBits : 0;
    u64* hist = sh.hist[row.turn & 1];
    ++row.turn;
    __syncthreads();
    for (int b = threadIdx.x; b < kSampleBins; b += kSampleThreads) hist[b] = 0;
    __syncthreads();
    for (int i = row.w0 + lane; i < row.w1; i += 32) {
      const uint32_t u = row.img[i];
      if (u >= lo && u <= hi && kept.has(u, row.first + i)) atomicAdd(&hist[(u - lo) >> shift], COUNT ? 1ull : row.weight(u));
    }
    row.barrier();
    // each thread: 4 bins summed over the cluster, top bin first
    constexpr int kPer = kSampleBins / kSampleThreads;
    const int b1 = kSampleBins - 1 - (int)threadIdx.x * kPer;  // bins b1, b1 - 1, ...
    u64 v[kPer], sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = 0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      const u64* h = row.peer(hist, r);
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] += h[b1 - j];
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum += v[j];
    u64 incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) sh.scan[warp] = incl;
    __syncthreads();
    u64 run = above + incl - sum;
    for (int w = 0; w < warp; ++w) run += sh.scan[w];
    // the bin in which the running sum reaches the target
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (run < target && run + v[j] >= target) {
        sh.found[0] = ((u64)(b1 - j) << 1);
        sh.part[0] = run;
        sh.part[1] = v[j];
      }
      run += v[j];
    }
    __syncthreads();
    const uint32_t bin = (uint32_t)(sh.found[0] >> 1);
    above = sh.part[0];
    group = sh.part[1];
    const uint32_t base = lo + (bin << shift);
    if (shift == 0) {
      lo = base;
      break;
    }
    const uint32_t top = base + ((1u << shift) - 1u);
    hi = top < hi ? top : hi;
    lo = base;
    if (COUNT && above + group == target) {  // the whole bin: everything at or above its lower edge
      if (lo > kept.lo) {
        kept.lo = lo - 1;
        kept.last = -1;
      }
      return RadixResult{kept, row.turn};
    }
  }
  // one value is left: its ties are taken in index order
  const u64 each = COUNT ? 1ull : row.weight(lo);
  const u64 need = each ? (target - above + each - 1) / each : 0;
  if (each == 0 || need * each >= group) {  // all of them
    if (lo > kept.lo) {
      kept.lo = lo - 1;
      kept.last = -1;
    }
    return RadixResult{kept, row.turn};
  }
  u64 mine = 0;
  for (int i = row.w0 + lane; i < row.w1; i += 32) mine += row.img[i] == lo && kept.has(lo, row.first + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  const u64 block = row.block_sum(lane == 0 ? mine : 0ull);  // leaves the warps' counts in sh.part
  u64 before = 0;
  for (int w = 0; w < warp; ++w) before += sh.part[w];
  const u64(*blocks)[2] = row.exchange(block, 0);
  for (int r = 0; r < row.rank; ++r) before += blocks[r][0];
  __syncthreads();
  if (threadIdx.x == 0) sh.found[1] = 0;
  __syncthreads();
  if (before < need && before + mine >= need) {  // the need-th tie is in this warp's part
    u64 seen = before;
    for (int i0 = row.w0; i0 < row.w1; i0 += 32) {
      const int i = i0 + lane;
      const bool tie = i < row.w1 && row.img[i] == lo && kept.has(lo, row.first + i);
      const unsigned m = __ballot_sync(0xffffffffu, tie);
      const int c = __popc(m);
      if (seen + c >= need) {
        const int pick = __fns(m, 0, (int)(need - seen));
        if (lane == 0) sh.found[1] = (u64)(row.first + i0 + pick) + 1;
        break;
      }
      seen += c;
    }
  }
  __syncthreads();
  const u64(*all)[2] = row.exchange(sh.found[1], 0);
  u64 last = 0;
#pragma unroll
  for (int r = 0; r < C; ++r) last += all[r][0];
  kept.lo = lo;
  kept.last = (int)last - 1;
  return RadixResult{kept, row.turn};
}

// Sort sh.sorted[0, padded) (a power of two), largest first.
__device__ __forceinline__ void sort_descending(u64* v, int padded) {
  for (int size = 2; size <= padded; size *= 2)  // bitonic
    for (int step = size / 2; step > 0; step /= 2) {
      for (int i = threadIdx.x; i < padded / 2; i += kSampleThreads) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const u64 x = v[lo], y = v[hi];
        if ((x < y) == ((lo & size) == 0)) {
          v[lo] = y;
          v[hi] = x;
        }
      }
      // pairs within 32 entries belong to one warp from step 16 down
      if (step > 32)
        __syncthreads();
      else
        __syncwarp();
      if (step == 1 || step == 64) __syncthreads();
    }
}

// The cluster's lists one after the other into sh.sorted, filled up with zeros to a power of two.
template <int C>
__device__ __forceinline__ int gather(RowSampler<C>& row, const u64* list, const unsigned (&count)[C], unsigned n) {
  int padded = 32;
  while (padded < (int)n) padded *= 2;
  unsigned from = 0;
#pragma unroll
  for (int r = 0; r < C; ++r) {
    const u64* theirs = row.peer(list, r);
    for (unsigned i = threadIdx.x; i < count[r]; i += kSampleThreads) row.sh.sorted[from + i] = theirs[i];
    from += count[r];
  }
  for (unsigned i = n + threadIdx.x; i < (unsigned)padded; i += kSampleThreads) row.sh.sorted[i] = 0;
  __syncthreads();
  return padded;
}

// Inclusive sums over the block's threads.
template <int C>
__device__ __forceinline__ u64 block_scan(SampleShared<C>& sh, u64 v, u64* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  if (lane == 31) sh.scan[warp] = v;
  __syncthreads();
  u64 w = sh.scan[lane & (kSampleWarps - 1)];  // the warps' sums, scanned by every warp for itself
#pragma unroll
  for (int o = 1; o < kSampleWarps; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, w, o, kSampleWarps);
    if ((lane & (kSampleWarps - 1)) >= o) w += x;
  }
  *all = __shfl_sync(0xffffffffu, w, kSampleWarps - 1);
  const u64 below = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
  return warp ? v + below : v;
}

__device__ __forceinline__ u64 share_of(float share, u64 all) {  // the least sum that holds a share
  const double goal = ceil((double)share * (double)all);
  return goal < 1.0 ? 1ull : goal >= (double)all ? all : (u64)goal;
}

// This CTA's sum of the threads' parts, in a fixed order.
template <int C>
__device__ __forceinline__ float block_sum_f32(SampleShared<C>& sh, float z) {
  z = warp_sum(z);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = __float_as_uint(z);
  __syncthreads();
  z = __uint_as_float((uint32_t)sh.part[threadIdx.x & (kSampleWarps - 1)]);
#pragma unroll
  for (int o = kSampleWarps / 2; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
  return z;
}

struct DrawArgs {  // a row's filters and its uniform
  int k;
  float p, uniform;
  u64 floor_w;
};

// The integer target of the running sums: the token's sum is the first above it.
__device__ __forceinline__ u64 draw_target(float uniform, u64 total) {
  const u64 goal = uniform > 0.f ? (u64)((double)uniform * (double)total) : 0ull;
  return goal >= total ? total - 1 : goal;
}

// The key in bin `bin` of the n gathered tokens at which a filter's running sum (COUNT: of tokens, `above`
// before the bin; else of weights, `above_w` before it) reaches `target`: the bin's tokens are listed and
// each adds up what lies above it among them.  `through`: the weight up to and with that key.
template <bool COUNT, int C>
__device__ u64 cross_key(RowSampler<C>& row, int n, int bin, u64 above, u64 above_w, u64 target, uint16_t* places,
                         u64* through) {
  SampleShared<C>& sh = row.sh;
  const u64* weight = sh.list;
  if (threadIdx.x == 0) sh.listed = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kSampleThreads)
    if (row.bin_of((uint32_t)(sh.sorted[i] >> 32)) == bin) places[atomicAdd(&sh.listed, 1u)] = (uint16_t)i;
  __syncthreads();
  const int c = (int)sh.listed;
  for (int x = threadIdx.x; x < c; x += kSampleThreads) {
    const int i = places[x];
    const u64 key = sh.sorted[i];
    u64 rank = 0, w = 0;
    for (int y = 0; y < c; ++y) {
      const int j = places[y];
      if (sh.sorted[j] > key) {
        ++rank;
        w += weight[j];
      }
    }
    const u64 before = COUNT ? above + rank : above_w + w;
    if (before < target && before + (COUNT ? 1ull : weight[i]) >= target) {
      sh.found[0] = key;
      sh.found[1] = above_w + w + weight[i];
    }
  }
  __syncthreads();
  *through = sh.found[1];
  const u64 key = sh.found[0];
  __syncthreads();
  return key;
}

// All filters and the draw on the n gathered tokens of sh.sorted, in index order (rank 0's CTA alone).  They
// hold the k largest (COUNT), or all that the prefix which reaches `target` takes.  Leaves the drawn
// token's key in sh.found[0].  The thresholds come from one histogram of the gathered tokens, counts and weights.
template <bool COUNT, int C>
__device__ __noinline__ void finish(RowSampler<C> row, int n, uint32_t lowest, u64 target, const DrawArgs& d) {
  SampleShared<C>& sh = row.sh;
  constexpr int kEach = list_max(C) / kSampleThreads;
  // the histograms' memory is free here: counts, low and high words of the weights, places of a bin's tokens
  uint32_t* hist = reinterpret_cast<uint32_t*>(sh.hist[0]);
  uint16_t* places = reinterpret_cast<uint16_t*>(hist + 3 * kSampleBins);
  static_assert(3 * kSampleBins * sizeof(uint32_t) + list_max(C) * sizeof(uint16_t) <= sizeof(sh.hist), "fits");
  u64* weight = sh.list;  // by place
  row.per_unit = fminf((float)kSampleBins / (row.best - image_value(lowest)), 3e38f);
  for (int b = threadIdx.x; b < 3 * kSampleBins; b += kSampleThreads) hist[b] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kSampleThreads) {
    const uint32_t u = (uint32_t)(sh.sorted[i] >> 32);
    const u64 w = row.weight(u);
    uint32_t* bin = hist + row.bin_of(u);
    weight[i] = w;
    atomicAdd(bin, 1u);
    const uint32_t low = (uint32_t)w, old = atomicAdd(bin + kSampleBins, low);
    const uint32_t high = (uint32_t)(w >> 32) + (old + low < old ? 1u : 0u);
    if (high) atomicAdd(bin + 2 * kSampleBins, high);
  }
  __syncthreads();
  const int b0 = 2 * (int)threadIdx.x;
  const u64 c0 = hist[b0], c1 = hist[b0 + 1];
  const u64 v0 = hist[kSampleBins + b0] | (u64)hist[2 * kSampleBins + b0] << 32;
  const u64 v1 = hist[kSampleBins + b0 + 1] | (u64)hist[2 * kSampleBins + b0 + 1] << 32;
  u64 all = 0, total = 0;
  const u64 run_c = block_scan(sh, c0 + c1, &all) - c0 - c1;
  __syncthreads();
  const u64 run_w = block_scan(sh, v0 + v1, &total) - v0 - v1;
  u64 least = 0;  // tokens with a key from here on are kept
  if (COUNT && n > d.k) {
    const u64 k = (u64)d.k;
    if (run_c < k && run_c + c0 + c1 >= k) {
      const bool second = run_c + c0 < k;
      sh.part[0] = b0 + second;
      sh.part[1] = second ? run_c + c0 : run_c;
      sh.part[2] = second ? run_w + v0 : run_w;
    }
    __syncthreads();
    least = cross_key<true>(row, n, (int)sh.part[0], sh.part[1], sh.part[2], k, places, &total);
  }
  if (!COUNT || d.p < 1.f) {
    if (COUNT) target = share_of(d.p, total);
    if (run_w < target && run_w + v0 + v1 >= target) {
      const bool second = run_w + v0 < target;
      sh.part[0] = b0 + second;
      sh.part[2] = second ? run_w + v0 : run_w;
    }
    __syncthreads();
    const u64 key = cross_key<false>(row, n, (int)sh.part[0], 0, sh.part[2], target, places, &total);
    least = key > least ? key : least;
  }
  // running sums in index order
  const int i0 = kEach * (int)threadIdx.x;
  u64 w[kEach], mine = 0, sum = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    w[e] = i0 + e < n && sh.sorted[i0 + e] >= least ? weight[i0 + e] : 0ull;
    if (w[e] < d.floor_w) w[e] = 0;
    mine += w[e];
  }
  u64 begin = block_scan(sh, mine, &sum) - mine;
  const u64 goal = draw_target(d.uniform, sum);
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (w[e] && begin <= goal && begin + w[e] > goal) sh.found[0] = sh.sorted[i0 + e];
    begin += w[e];
  }
  __syncthreads();
}

// The CTA's tokens from image `lowest` on into sh.list, in index order; how many, or more than
// list_max(C) where they do not fit.
template <int C>
__device__ unsigned collect(RowSampler<C>& row, uint32_t lowest) {
  SampleShared<C>& sh = row.sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned count = 0;
  const int whole = row.w0 + (row.w1 - row.w0) / 4 * 4;
#pragma unroll 4
  for (int i = row.w0 + 4 * lane; i < whole; i += 128) {
    const uint4 u = *reinterpret_cast<const uint4*>(row.img + i);
    count += (unsigned)(u.x >= lowest) + (u.y >= lowest) + (u.z >= lowest) + (u.w >= lowest);
  }
  if (whole + lane < row.w1) count += row.img[whole + lane] >= lowest;
  count = __reduce_add_sync(0xffffffffu, count);
  if (lane == 0) sh.counts[warp] = count;
  __syncthreads();
  const unsigned c = lane < kSampleWarps ? sh.counts[lane] : 0u;
  unsigned from = __reduce_add_sync(0xffffffffu, lane < warp ? c : 0u);
  const unsigned all = __reduce_add_sync(0xffffffffu, c);
  if (all > (unsigned)list_max(C)) return list_max(C) + 1;
  for (int i0 = row.w0; count && i0 < row.w1; i0 += 128) {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = i0 + lane + 32 * e < row.w1 ? row.img[i0 + lane + 32 * e] : 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned in = __ballot_sync(0xffffffffu, u[e] >= lowest);
      if (in >> lane & 1)
        sh.list[from + __popc(in & ((1u << lane) - 1))] =
            ((u64)u[e] << 32) | (uint32_t)~(uint32_t)(row.first + i0 + lane + 32 * e);
      from += __popc(in);
    }
  }
  return all;  // (published by the exchange's barrier)
}

// Gather the tokens from image `lowest` on, if they fit, and have rank 0 apply the filters to them and
// draw (finish's COUNT and target).  z: in this CTA's sum of exponentials, out the row's.
template <bool COUNT, int C>
__device__ bool try_finish(RowSampler<C>& row, const SampleArgs& a, int r, uint32_t lowest, u64 target, const DrawArgs& d,
                           float& z) {
  SampleShared<C>& sh = row.sh;
  const unsigned mine = collect(row, lowest);
  const u64(*box)[2] = row.exchange(mine, __float_as_uint(z));
  unsigned total = 0, count[C];
  z = 0.f;
#pragma unroll
  for (int p = 0; p < C; ++p) {
    total += count[p] = (unsigned)box[p][0];
    z += __uint_as_float((uint32_t)box[p][1]);
  }
  if (total > (unsigned)list_max(C)) return false;
  // into rank 0's memory, where they are in index order; the peers are then done
  unsigned from = 0;
#pragma unroll
  for (int p = 0; p < C; ++p) from += p < row.rank ? count[p] : 0u;
  u64* to = row.peer(sh.sorted, 0) + from;
  for (unsigned i = threadIdx.x; i < mine; i += kSampleThreads) to[i] = sh.list[i];
  row.barrier();
  if (row.rank != 0) return true;
  finish<COUNT, C>(row, (int)total, lowest, target, d);
  if (threadIdx.x == 0) {
    const u64 key = sh.found[0];
    a.tokens[r] = (int64_t)~(uint32_t)key;
    if (a.logprobs) a.logprobs[r] = (image_value((uint32_t)(key >> 32)) - row.best) - logf(z);
  }
  return true;
}

// Cuts `kept` to its first k tokens (COUNT) or to the shortest prefix that holds a share p of its
// weight, from the histogram that fill_histogram left in sh.hist[buffer] behind a barrier.
template <bool COUNT, int C>
__device__ void shrink(RowSampler<C>& row, Kept& kept, const DrawArgs& d, int buffer) {
  SampleShared<C>& sh = row.sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64* hist = sh.hist[buffer];
  constexpr int kPer = kSampleBins / kSampleThreads;  // bin 0 holds the largest values
  static_assert(kPer == 2, "two bins a thread");
  const int b0 = (int)threadIdx.x * kPer;
  u64 v0 = 0, v1 = 0;
#pragma unroll
  for (int r = 0; r < C; ++r) {
    if (COUNT) {
      const uint2 x = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint32_t*>(row.peer(hist, r)) + b0);
      v0 += x.x;
      v1 += x.y;
    } else {
      const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(row.peer(hist, r) + b0);
      v0 += x.x;
      v1 += x.y;
    }
  }
  if (threadIdx.x == 0) sh.listed = 0;
  u64 all = 0;
  const u64 incl = block_scan(sh, v0 + v1, &all);
  const u64 target = COUNT ? (u64)d.k : share_of(d.p, all);
  if (target > all) return;  // nothing to leave out (counts only)
  const u64 run = incl - v0 - v1;
  if (run < target && incl >= target) {
    const bool second = run + v0 < target;
    sh.found[0] = (u64)(b0 + second);
    sh.found[1] = second ? run + v0 : run;
  }
  __syncthreads();
  const int bin = (int)sh.found[0];
  const u64 above = sh.found[1];
  const uint32_t lowest = row.bin_floor(bin);
  // ---- the tokens of the crossing bin
  for (int i = row.w0 + lane; i < row.w1; i += 32) {
    const uint32_t u = row.img[i];
    if (u >= lowest && row.bin_of(u) == bin && kept.has(u, row.first + i)) {
      const unsigned at = atomicAdd(&sh.listed, 1u);
      if (at < (unsigned)list_max(C)) sh.list[at] = ((u64)u << 32) | (uint32_t)~(uint32_t)(row.first + i);
    }
  }
  __syncthreads();
  const u64(*box)[2] = row.exchange(sh.listed, 0);
  unsigned n = 0, count[C];
#pragma unroll
  for (int r = 0; r < C; ++r) n += count[r] = (unsigned)box[r][0];
  if (n > (unsigned)list_max(C)) {
    const RadixResult res = shrink_radix<COUNT, C>(row, kept, target);
    kept = res.kept;
    row.turn = res.turn;
    return;
  }
  const int padded = gather(row, sh.list, count, n);
  sort_descending(sh.sorted, padded);
  if (warp == 0) {  // the entry at which the running sum reaches the target
    u64 before = above;
    for (int i0 = 0; i0 < (int)n; i0 += 32) {
      const u64 key = i0 + lane < (int)n ? sh.sorted[i0 + lane] : 0ull;
      u64 s = key ? (COUNT ? 1ull : row.weight((uint32_t)(key >> 32))) : 0ull;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + s >= target);
      if (hit) {
        if (lane == __ffs(hit) - 1) sh.found[0] = key;
        break;
      }
      before += __shfl_sync(0xffffffffu, s, 31);
    }
  }
  __syncthreads();
  kept.lo = (uint32_t)(sh.found[0] >> 32);
  kept.last = (int)~(uint32_t)sh.found[0];
}

// Histogram of the row's kept tokens, of counts or weights, behind a barrier.
template <bool COUNT, int C>
__device__ void fill_histogram(RowSampler<C>& row, const Kept& kept) {
  u64* hist = row.sh.hist[row.turn & 1];
  constexpr int kWords = kSampleBins * (COUNT ? 1 : 2);
  __syncthreads();
  for (int b = threadIdx.x; b < kWords; b += kSampleThreads) reinterpret_cast<uint32_t*>(hist)[b] = 0;
  __syncthreads();
  for (int i = row.w0 + (int)(threadIdx.x & 31); i < row.w1; i += 128) {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = i + 32 * e < row.w1 ? row.img[i + 32 * e] : 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (u[e] <= kImgNegInf || !kept.has(u[e], row.first + i + 32 * e)) continue;
      uint32_t* bin = reinterpret_cast<uint32_t*>(hist) + row.bin_of(u[e]) * (COUNT ? 1 : 2);
      if (COUNT) {
        atomicAdd(bin, 1u);
      } else {  // 64-bit sum from 32-bit atomics: exactly the add that wraps the low word carries
        const u64 w = row.weight(u[e]);
        const uint32_t low = (uint32_t)w, old = atomicAdd(bin, low);
        const uint32_t high = (uint32_t)(w >> 32) + (old + low < old ? 1u : 0u);
        if (high) atomicAdd(bin + 1, high);
      }
    }
  }
  ++row.turn;
  row.barrier();
}

// Top-p alone, on the same histogram: the bin in which the sum crosses its share bounds what is kept, and the
// tokens from it on are finished, if they fit; true if they did.  z: in this CTA's sum of exponentials, out
// the row's.
template <int C>
__device__ bool nucleus(RowSampler<C>& row, const SampleArgs& a, int r, const DrawArgs& d, float& z) {
  SampleShared<C>& sh = row.sh;
  const u64* hist = sh.hist[(row.turn - 1) & 1];
  u64 v0 = 0, v1 = 0, all = 0;
#pragma unroll
  for (int p = 0; p < C; ++p) {
    const ulonglong2 x = reinterpret_cast<const ulonglong2*>(row.peer(hist, p))[threadIdx.x];
    v0 += x.x;
    v1 += x.y;
  }
  const u64 incl = block_scan(sh, v0 + v1, &all), run = incl - v0 - v1, target = share_of(d.p, all);
  if (run < target && incl >= target) sh.found[0] = 2 * threadIdx.x + (run + v0 < target);
  __syncthreads();
  return try_finish<false>(row, a, r, row.bin_floor((int)sh.found[0]), target, d, z);
}

// A bound below the row's k-th largest value from what each lane holds at most: where k lanes reach a
// bin, so do k tokens.  The lowest drawable value if fewer lanes hold any.
template <int C>
__device__ uint32_t sieve(RowSampler<C>& row, uint32_t lane_top, uint32_t bottom, int k) {
  SampleShared<C>& sh = row.sh;
  uint32_t* hist = reinterpret_cast<uint32_t*>(sh.hist[row.turn & 1]);
  ++row.turn;
  hist[threadIdx.x] = hist[threadIdx.x + kSampleThreads] = 0;
  static_assert(kSampleBins == 2 * kSampleThreads, "two bins a thread");
  if (threadIdx.x == 0) sh.found[0] = kSampleBins;
  __syncthreads();
  if (lane_top > kImgNegInf) atomicAdd(hist + row.bin_of(lane_top), 1u);
  row.barrier();
  uint32_t v0 = 0, v1 = 0;
#pragma unroll
  for (int r = 0; r < C; ++r) {
    const uint2 x = reinterpret_cast<const uint2*>(row.peer(hist, r))[threadIdx.x];
    v0 += x.x;
    v1 += x.y;
  }
  u64 all = 0;
  const u64 incl = block_scan(sh, (u64)(v0 + v1), &all), run = incl - v0 - v1;
  if (run < (u64)k && incl >= (u64)k) sh.found[0] = 2 * threadIdx.x + (run + v0 < (u64)k);
  __syncthreads();
  const int bin = (int)sh.found[0];
  if (bin >= kSampleBins) return bottom;
  // the bin's lower edge, or a little below it: more than the roundings of bin_of, 2^-23 each of the
  // gap, of its product and of the edge
  const float gap = (float)(bin + 1) / row.per_unit, edge = row.best - gap * 1.000001f;
  return max(value_image(edge - (fabsf(edge) + fabsf(row.best)) * 1e-6f), bottom);
}

template <int C>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) unsigned char sample_smem[];
  SampleShared<C>& sh = *reinterpret_cast<SampleShared<C>*>(sample_smem);
  uint32_t* img = reinterpret_cast<uint32_t*>(sample_smem + sizeof(SampleShared<C>));
  const int rank = (int)(blockIdx.x % C), r = (int)(blockIdx.x / C);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = min(a.vocab, rank * a.chunk), n = min(a.vocab - first, a.chunk);
  const int per_warp = a.chunk / kSampleWarps;
  const int w0 = min(n, warp * per_warp), w1 = min(n, w0 + per_warp);
  if (threadIdx.x < 64) sh.pow2[threadIdx.x] = exp2((double)threadIdx.x * 0.015625);
  pdl_wait();
  const float t = a.temperature ? a.temperature[r] : a.temperature_all;
  const double inv_t = 1.4426950408889634 / (double)t;  // (a long chain: under the loads)
  // ---- images of the allowed tokens; the largest and the lowest drawable value
  LaneStats st;
  if (a.dtype == S2R_F32)
    load_images<float>(a, r, first, img, w0, w1, st);
  else if (a.dtype == S2R_BF16)
    load_images<bf16>(a, r, first, img, w0, w1, st);
  else
    load_images<__half>(a, r, first, img, w0, w1, st);
  DrawArgs d;
  d.k = a.top_k ? a.top_k[r] : a.top_k_all;
  d.p = a.top_p ? a.top_p[r] : a.top_p_all;
  d.uniform = a.uniforms[r];
  const float m = a.min_p ? a.min_p[r] : a.min_p_all;
  RowSampler<C> row{sh, img, first, rank, w0, w1};
  uint32_t top = __reduce_max_sync(0xffffffffu, st.top);
  uint32_t bottom = __reduce_min_sync(0xffffffffu, st.bottom);
  {
    if (lane == 0) sh.part[warp] = ((u64)top << 32) | bottom;
    __syncthreads();
    const u64 x = sh.part[lane & (kSampleWarps - 1)];
    top = __reduce_max_sync(0xffffffffu, (uint32_t)(x >> 32));
    bottom = __reduce_min_sync(0xffffffffu, (uint32_t)x);
    const u64(*box)[2] = row.exchange(((u64)top << 32) | bottom, 0);
#pragma unroll
    for (int p = 0; p < C; ++p) {
      top = max(top, (uint32_t)(box[p][0] >> 32));
      bottom = min(bottom, (uint32_t)box[p][0]);
    }
    bottom += kImgNegInf + 1;
  }
  const bool finite = top > kImgNegInf && top < kImgPosInf;
  row.best = finite ? image_value(top) : 0.f;
  row.inv_t = inv_t;
  row.scale_bits = a.scale_bits;
  const bool greedy = !finite || !(t > 0.f);
  d.floor_w = m > 0.f ? (u64)ceil((double)fminf(m, 1.f) * (double)(1ull << a.scale_bits)) : 0ull;
  // this CTA's sum of exp(x - best) over the allowed tokens
  float z = block_sum_f32(sh, finite && st.m != -INFINITY ? st.z * exp_approx(st.m - row.best) : 0.f);

  if (greedy) {
    uint32_t lowest = 0xffffffffu;
    for (int i = w0 + lane; i < w1; i += 32)
      if (img[i] == top) lowest = min(lowest, (uint32_t)(first + i));
    lowest = __reduce_min_sync(0xffffffffu, lowest);
    if (lane == 0) sh.scan[warp] = lowest;
    __syncthreads();
    lowest = __reduce_min_sync(0xffffffffu, (uint32_t)sh.scan[lane & (kSampleWarps - 1)]);
    const u64(*box)[2] = row.exchange(lowest, __float_as_uint(z));
    z = 0.f;
#pragma unroll
    for (int p = 0; p < C; ++p) {
      lowest = min(lowest, (uint32_t)box[p][0]);
      z += __uint_as_float((uint32_t)box[p][1]);
    }
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[r] = top > kImgNegInf ? (int64_t)lowest : 0;
      if (a.logprobs)
        a.logprobs[r] = finite ? -logf(z)
                        : top <= kImgNegInf ? -INFINITY
                        : top == kImgPosInf ? 0.f
                                            : __uint_as_float(0x7fc00000u);
    }
    return;  // (nothing reads a peer's memory: what was sent landed before the barrier)
  }

  // ---- the filters
  const bool by_count = d.k > 0 && d.k < a.vocab, by_share = d.p < 1.f;
  // tokens a.cut temperatures below the best weigh nothing
  row.per_unit = fminf((float)kSampleBins / fminf(a.cut * t, row.best - image_value(bottom)), 3e38f);
  Kept kept;
  if (by_count) {
    if (try_finish<true>(row, a, r, sieve(row, st.top, bottom, d.k), 0, d, z)) return;
    fill_histogram<true>(row, kept);
    shrink<true>(row, kept, d, (row.turn - 1) & 1);
    if (kept.lo > kImgNegInf)
      row.per_unit = fminf((float)kSampleBins / (row.best - image_value(kept.lo)), 3e38f);
  }
  if (by_share) {
    fill_histogram<false>(row, kept);
    const int buffer = (row.turn - 1) & 1;
    if (!by_count && nucleus(row, a, r, d, z)) return;
    shrink<false>(row, kept, d, buffer);
  }
  const bool summed = by_count || by_share;  // z is the row's

  // ---- the token: running sums in index order
  auto kept_weight = [&](int i, uint32_t u) -> u64 {
    if (u <= kImgNegInf || !kept.has(u, first + i)) return 0;
    const u64 w = row.weight(u);
    return w >= d.floor_w ? w : 0ull;
  };
  u64 sum = 0, before = 0;
#pragma unroll 2
  for (int i = w0 + lane; i < w1; i += 32) sum += kept_weight(i, img[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const u64 mine = sum;
  const u64 block = row.block_sum(lane == 0 ? mine : 0ull);
  u64 run = sum_partials((lane & (kSampleWarps - 1)) < warp ? sh.part[lane & (kSampleWarps - 1)] : 0ull);
  u64 total = 0;
  {
    const u64(*box)[2] = row.exchange(block, __float_as_uint(z));
    float sum_z = 0.f;
#pragma unroll
    for (int q = 0; q < C; ++q) {
      if (q < rank) before += box[q][0];
      total += box[q][0];
      sum_z += __uint_as_float((uint32_t)box[q][1]);
    }
    if (!summed) z = sum_z;
  }
  run += before;
  const u64 target = draw_target(d.uniform, total);
  if (run <= target && target < run + mine) {
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t u = i < w1 ? img[i] : 0u;
      u64 s = kept_weight(i, u);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, run + s > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          a.tokens[r] = first + i;
          if (a.logprobs) a.logprobs[r] = (image_value(u) - row.best) - logf(z);
        }
        break;
      }
      run += __shfl_sync(0xffffffffu, s, 31);
    }
  }
}

static_assert(sizeof(SampleShared<1>) % 16 == 0 && sizeof(SampleShared<4>) % 16 == 0, "images start 16-byte aligned");

constexpr int kSampleMaxChunk = 40960;  // tokens of one CTA: 160 KB of images

typedef void (*SampleFn)(const SampleArgs);

SampleFn sample_fn(int splits) {
  switch (splits) {
    case 1: return sample_kernel<1>;
    case 2: return sample_kernel<2>;
    case 4: return sample_kernel<4>;
    case 8: return sample_kernel<8>;
    default: return sample_kernel<16>;
  }
}

size_t shared_bytes(int splits) {
  return splits == 1 ? sizeof(SampleShared<1>) : splits == 2 ? sizeof(SampleShared<2>) : sizeof(SampleShared<4>);
}

int sample_chunk(int vocab, int splits) {  // a multiple of 32 tokens a warp
  const int per = (vocab + splits - 1) / splits;
  return (per + kSampleWarps * 32 - 1) / (kSampleWarps * 32) * (kSampleWarps * 32);
}

// CTAs per row: enough that two of them fit an SM (1,024 rows of 32,576 tokens: one CTA a row took 188 us,
// two 152 us, four 228 us, more of it in barriers), then more while the rows leave SMs idle and a
// share is worth splitting.
int sample_splits(int rows, int vocab, int sms) {
  int c = 1;
  while (c < kSampleMaxSplits && shared_bytes(c) + sample_chunk(vocab, c) * sizeof(uint32_t) > 112 * 1024) c *= 2;
  while (c < 8 && (long long)rows * c * 2 <= 2 * sms && vocab / (2 * c) >= 2048) c *= 2;
  return c;
}

// Per device, once: SMs, and every instantiation allowed its shared memory and cluster size.
struct SampleDevice {
  int sms = 0;
  cudaError_t error = cudaSuccess;
};

const SampleDevice& sample_device(int device) {
  static std::mutex mu;
  static SampleDevice devices[64];
  static std::atomic<bool> ready[64];
  SampleDevice& dev = devices[device];
  if (ready[device].load(std::memory_order_acquire)) return dev;
  std::lock_guard<std::mutex> lock(mu);
  if (ready[device].load(std::memory_order_relaxed)) return dev;
  dev.error = cudaDeviceGetAttribute(&dev.sms, cudaDevAttrMultiProcessorCount, device);
  for (int c = 1; c <= kSampleMaxSplits && dev.error == cudaSuccess; c *= 2) {
    const int smem = (int)(shared_bytes(c) + kSampleMaxChunk * sizeof(uint32_t));
    dev.error = cudaFuncSetAttribute(sample_fn(c), cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (dev.error == cudaSuccess && c > 8)
      dev.error = cudaFuncSetAttribute(sample_fn(c), cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (dev.error == cudaSuccess)
      dev.error = cudaFuncSetAttribute(sample_fn(c), cudaFuncAttributePreferredSharedMemoryCarveout,
                                       (int)cudaSharedmemCarveoutMaxShared);
  }
  if (dev.error == cudaSuccess) ready[device].store(true, std::memory_order_release);
  return dev;
}

}  // namespace

int launch_sample(SampleArgs a, cudaStream_t stream, const char** why) {
  int device = 0;
  *why = "no usable current device";
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return S2R_ECUDA;
  const SampleDevice& dev = sample_device(device);
  if (dev.error != cudaSuccess) return S2R_ECUDA;
  const int splits = sample_splits(a.rows, a.vocab, dev.sms);
  a.chunk = sample_chunk(a.vocab, splits);
  int bits = 0;
  while ((1ll << bits) <= a.vocab) ++bits;
  a.scale_bits = 61 - bits;
  a.cut = (float)(a.scale_bits + 2) * 0.69315f;  // exp(-cut) * 2^scale_bits < 1/2
  *why = "launch failed";
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * splits);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = shared_bytes(splits) + (size_t)a.chunk * sizeof(uint32_t);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = splits;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, sample_fn(splits), a) == cudaSuccess ? S2R_OK : S2R_ECUDA;
}

}  // namespace s2r

// Records `msg` as s2r_last_error() of this thread (defined with the engine).
__attribute__((visibility("hidden"))) int s2r_record_error(int code, const char* msg);

extern "C" int32_t s2r_sample(const s2r_sample_args* in, void* stream) {
  auto bad = [](const char* msg) { return s2r_record_error(S2R_EINVAL, msg); };
  if (!in || !in->logits || !in->uniforms || !in->tokens) return bad("s2r_sample: NULL pointer");
  if (in->rows < 1 || in->vocab < 1) return bad("s2r_sample: rows and vocab must be >= 1");
  if (in->rows > S2R_SAMPLE_MAX_ROWS || in->vocab > S2R_SAMPLE_MAX_VOCAB)
    return bad("s2r_sample: at most 65536 rows and 524288 tokens a call");
  if (in->logits_dtype != S2R_F32 && in->logits_dtype != S2R_BF16 && in->logits_dtype != S2R_F16)
    return bad("s2r_sample: logits must be float32, bfloat16 or float16");
  if (in->logits_stride < 0 || in->allowed_stride < 0) return bad("s2r_sample: negative row stride");
  if (!in->temperature && !(in->temperature_all >= 0.f)) return bad("s2r_sample: temperature must be >= 0");
  if (!in->top_p && !(in->top_p_all >= 0.f && in->top_p_all <= 1.f)) return bad("s2r_sample: top_p must be in [0, 1]");
  if (!in->min_p && !(in->min_p_all >= 0.f && in->min_p_all <= 1.f)) return bad("s2r_sample: min_p must be in [0, 1]");
  if (!in->top_k && in->top_k_all < 0) return bad("s2r_sample: top_k must be >= 0");
  auto off = [](const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; };
  if (off(in->logits, in->logits_dtype == S2R_F32 ? 4 : 2) || off(in->bias, 4) || off(in->uniforms, 4) ||
      off(in->temperature, 4) || off(in->top_k, 4) || off(in->top_p, 4) || off(in->min_p, 4) || off(in->tokens, 8) ||
      off(in->logprobs, 4))
    return bad("s2r_sample: a pointer is not aligned to its type");
  s2r::SampleArgs a{};
  a.logits = in->logits;
  a.dtype = in->logits_dtype;
  a.logits_stride = in->logits_stride;
  a.rows = in->rows;
  a.vocab = in->vocab;
  a.bias = in->bias;
  a.allowed = in->allowed;
  a.allowed_stride = in->allowed_stride;
  a.uniforms = in->uniforms;
  a.temperature = in->temperature;
  a.top_k = in->top_k;
  a.top_p = in->top_p;
  a.min_p = in->min_p;
  a.temperature_all = in->temperature_all;
  a.top_k_all = in->top_k_all;
  a.top_p_all = in->top_p_all;
  a.min_p_all = in->min_p_all;
  a.tokens = in->tokens;
  a.logprobs = in->logprobs;
  const char* why = "";
  const int rc = s2r::launch_sample(a, static_cast<cudaStream_t>(stream), &why);
  if (rc != S2R_OK) {
    char msg[96];
    snprintf(msg, sizeof(msg), "s2r_sample: %s (%s)", why, cudaGetErrorString(cudaGetLastError()));
    return s2r_record_error(rc, msg);
  }
  return S2R_OK;
}
