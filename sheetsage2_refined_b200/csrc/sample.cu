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
// threshold, and the first few of the threshold's ties".  The threshold is
// found in two exchanges: a histogram of counts (top-k) or weights (top-p) over
// 1024 bins linear in M - x, which a decoder's logits fill evenly, then the
// tokens of the bin in which the sum crosses its target, gathered and sorted.
// When that bin holds more than 2048 tokens (masses of equal values) a radix
// search over the 32-bit images of the values takes over.
//
// Weights are fixed-point integers, rint(exp(.) * 2^(61 - bits(vocab))), with
// the exponential in 64 bits: which token is drawn depends on which side of a
// border a running sum falls, integer sums do not depend on the order in
// which threads add, and the rounding (2^-46 of the largest weight at 32,576
// tokens) is far below what a 32-bit sum could resolve.  Tokens whose weight
// rounds to 0 cannot be drawn and are left out from the start.  With top-k the
// counts come first, so that only the k survivors need the exponential.
//
// A row is one thread-block cluster of C CTAs, each holding a contiguous
// share of the vocabulary as images in shared memory; sums cross the cluster
// through distributed shared memory, one cluster barrier per exchange, so a
// call needs no scratch memory, no atomics on global memory and one launch.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdio>

#include "../../include/s2r.h"
#include "common.cuh"
#include "sample.cuh"

namespace s2r {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048;
constexpr int kSampleBinBits = 11;
constexpr int kSampleMaxSplits = 16;
constexpr int kSampleLinear = 1024;  // bins of the first histogram
constexpr int kSampleListMax = 2048;  // tokens of its crossing bin that are gathered and sorted
constexpr uint32_t kImgNegInf = 0x007fffffu;  // image of -inf: tokens at or below it are never drawn
constexpr uint32_t kImgPosInf = 0xff800000u;

struct SampleShared {
  u64 hist[2][kSampleBins];  // by parity of the exchange, so one cluster barrier each suffices; also the lists
  u64 sorted[kSampleListMax];
  double pow2[64];           // 2^(j / 64)
  unsigned listed;
  u64 part[kSampleWarps];    // per-warp values of a block reduction
  u64 cta[2][2];             // this CTA's values of an exchange, by parity
  u64 scan[kSampleWarps];
  u64 found[2];
};

// Order-preserving image of a float (select.cuh): -0 as +0, every NaN on top.
__device__ __forceinline__ uint32_t value_image(float v) {
  uint32_t u = __float_as_uint(v);
  if (u == 0x80000000u) u = 0u;
  if (v != v) u = 0x7fffffffu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float image_value(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

__device__ __forceinline__ float load_logit(const void* p, int dtype, size_t i) {
  if (dtype == S2R_F32) return static_cast<const float*>(p)[i];
  if (dtype == S2R_BF16) return __bfloat162float(static_cast<const bf16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// One row's search state; every thread of the cluster holds the same values.
struct RowSampler {
  SampleShared& sh;
  const uint32_t* img;  // this CTA's images
  int first, n;         // its share of the vocabulary
  int C, rank;
  int w0, w1;           // this warp's part of the share
  int turn = 0;         // exchanges done (parity of the buffers)
  float best;
  float cut;     // tokens with best - x >= cut weigh nothing
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
    u64 s = 0;
#pragma unroll
    for (int w = 0; w < kSampleWarps; ++w) s += sh.part[w];
    return s;
  }
  __device__ u64 block_max(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 x = __shfl_xor_sync(0xffffffffu, v, o);
      v = x > v ? x : v;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 s = 0;
#pragma unroll
    for (int w = 0; w < kSampleWarps; ++w) s = sh.part[w] > s ? sh.part[w] : s;
    return s;
  }
  // Publish a block-uniform pair to the cluster; afterwards peer(sh.cta[t & 1], r) holds rank r's.
  __device__ const u64* exchange(u64 a, u64 b) {
    u64* mine = sh.cta[turn & 1];
    ++turn;
    if (threadIdx.x == 0) {
      mine[0] = a;
      mine[1] = b;
    }
    barrier();
    return mine;
  }
  // Sums over the cluster and over the ranks below this one.
  __device__ u64 cluster_sum(u64 block_value, u64* before) {
    const u64* mine = exchange(block_value, 0);
    u64 s = 0, lo = 0;
    for (int r = 0; r < C; ++r) {
      const u64 x = peer(mine, r)[0];
      if (r < rank) lo += x;
      s += x;
    }
    if (before) *before = lo;
    return s;
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
template <bool COUNT>
__device__ __noinline__ RadixResult shrink_radix(RowSampler row, Kept kept, u64 target) {
  SampleShared& sh = row.sh;
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
    for (int r = 0; r < row.C; ++r) {
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
  u64 in_block = 0;
  for (int w = 0; w < warp; ++w) in_block += sh.part[w];
  row.cluster_sum(block, &before);
  before += in_block;
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
  const u64* all = row.exchange(sh.found[1], 0);
  u64 last = 0;
  for (int r = 0; r < row.C; ++r) last += row.peer(all, r)[0];
  kept.lo = lo;
  kept.last = (int)last - 1;
  return RadixResult{kept, row.turn};
}

// The same through the histogram that fill_histogram left in sh.hist[(turn - 1) & 1], one barrier
// after it was filled: `per_unit` bins per unit of best - x.  `total`, if given, receives the sum over
// `kept` and `share` of it is the target.
template <bool COUNT>
__device__ void shrink(RowSampler& row, Kept& kept, float per_unit, u64 target, const float* share) {
  SampleShared& sh = row.sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64* hist = sh.hist[(row.turn - 1) & 1];
  constexpr int kPer = kSampleLinear / kSampleThreads;  // bin 0 holds the largest values
  const int b0 = (int)threadIdx.x * kPer;
  u64 v[kPer], sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) v[j] = 0;
  if (COUNT) {
    for (int r = 0; r < row.C; ++r) {
      const uint2 x = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint32_t*>(row.peer(hist, r)) + b0);
      v[0] += x.x;
      v[1] += x.y;
    }
  } else {
    for (int r = 0; r < row.C; ++r) {
      const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(row.peer(hist, r) + b0);
      v[0] += x.x;
      v[1] += x.y;
    }
  }
  static_assert(kPer == 2, "two bins a thread");
#pragma unroll
  for (int j = 0; j < kPer; ++j) sum += v[j];
  u64 incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) sh.scan[warp] = incl;
  if (threadIdx.x == 0) sh.listed = 0;
  __syncthreads();
  u64 run = incl - sum, all = 0;
  for (int w = 0; w < kSampleWarps; ++w) {
    if (w < warp) run += sh.scan[w];
    all += sh.scan[w];
  }
  if (share) {  // a share of the whole sum
    const double goal = ceil((double)*share * (double)all);
    target = goal < 1.0 ? 1ull : (u64)goal;
  }
  if (target >= all && COUNT) return;  // nothing to leave out
  target = target > all ? all : target;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (run < target && run + v[j] >= target) {
      sh.found[0] = (u64)(b0 + j);
      sh.part[0] = run;
    }
    run += v[j];
  }
  __syncthreads();
  const int bin = (int)sh.found[0];
  const u64 above = sh.part[0];
  // ---- the tokens of the crossing bin
  u64* list = sh.hist[row.turn & 1];
  for (int i = row.w0 + lane; i < row.w1; i += 32) {
    const uint32_t u = row.img[i];
    if (u <= kImgNegInf) continue;
    const float d = row.best - image_value(u);
    if (d < row.cut && min(kSampleLinear - 1, (int)(d * per_unit)) == bin && kept.has(u, row.first + i)) {
      const unsigned at = atomicAdd(&sh.listed, 1u);
      if (at < (unsigned)kSampleListMax) list[at] = ((u64)u << 32) | (uint32_t)~(uint32_t)(row.first + i);
    }
  }
  __syncthreads();
  const u64* counts = row.exchange(sh.listed, 0);
  unsigned n = 0;
  for (int r = 0; r < row.C; ++r) n += (unsigned)row.peer(counts, r)[0];
  if (n > (unsigned)kSampleListMax) {
    const RadixResult res = shrink_radix<COUNT>(row, kept, target);
    kept = res.kept;
    row.turn = res.turn;
    return;
  }
  int padded = 32;
  while (padded < (int)n) padded *= 2;
  unsigned from = 0;
  for (int r = 0; r < row.C; ++r) {
    const unsigned c = (unsigned)row.peer(counts, r)[0];
    const u64* theirs = row.peer(list, r);
    for (unsigned i = threadIdx.x; i < c; i += kSampleThreads) sh.sorted[from + i] = theirs[i];
    from += c;
  }
  for (unsigned i = n + threadIdx.x; i < (unsigned)padded; i += kSampleThreads) sh.sorted[i] = 0;
  __syncthreads();
  for (int size = 2; size <= padded; size *= 2)  // bitonic, descending
    for (int step = size / 2; step > 0; step /= 2) {
      for (int i = threadIdx.x; i < padded / 2; i += kSampleThreads) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const u64 x = sh.sorted[lo], y = sh.sorted[hi];
        if ((x < y) == ((lo & size) == 0)) {
          sh.sorted[lo] = y;
          sh.sorted[hi] = x;
        }
      }
      __syncthreads();
    }
  // ---- the entry at which the running sum reaches the target (warp 0)
  if (warp == 0) {
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

// Bins of best - x over the row's kept tokens, of counts or weights, behind one cluster barrier.
template <bool COUNT>
__device__ void fill_histogram(RowSampler& row, const Kept& kept, float per_unit) {
  u64* hist = row.sh.hist[row.turn & 1];
  ++row.turn;
  __syncthreads();
  constexpr int kWords = kSampleLinear * (COUNT ? 1 : 2);
  for (int b = threadIdx.x; b < kWords; b += kSampleThreads) reinterpret_cast<uint32_t*>(hist)[b] = 0;
  __syncthreads();
  for (int i = row.w0 + (int)(threadIdx.x & 31); i < row.w1; i += 32) {
    const uint32_t u = row.img[i];
    if (u <= kImgNegInf) continue;
    const float d = row.best - image_value(u);
    if (!(d < row.cut) || !kept.has(u, row.first + i)) continue;
    uint32_t* bin = reinterpret_cast<uint32_t*>(hist) + min(kSampleLinear - 1, (int)(d * per_unit)) * (COUNT ? 1 : 2);
    if (COUNT) {
      atomicAdd(bin, 1u);
    } else {  // 64-bit sum from 32-bit atomics: exactly the add that wraps the low word carries
      const u64 w = row.weight(u);
      const uint32_t low = (uint32_t)w, old = atomicAdd(bin, low);
      const uint32_t high = (uint32_t)(w >> 32) + (old + low < old ? 1u : 0u);
      if (high) atomicAdd(bin + 1, high);
    }
  }
  row.barrier();
}

__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) unsigned char sample_smem[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(sample_smem);
  uint32_t* img = reinterpret_cast<uint32_t*>(sample_smem + sizeof(SampleShared));
  const int C = a.splits, rank = blockIdx.x % C, r = blockIdx.x / C;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = min(a.vocab, rank * a.chunk), n = min(a.vocab - first, a.chunk);
  const int per_warp = ((a.chunk + kSampleWarps - 1) / kSampleWarps + 31) / 32 * 32;
  const int w0 = min(n, warp * per_warp), w1 = min(n, w0 + per_warp);
  if (threadIdx.x < 64) sh.pow2[threadIdx.x] = exp2((double)threadIdx.x * 0.015625);
  pdl_wait();

  // ---- images of the allowed tokens; the largest
  const size_t at = (size_t)r * a.logits_stride + first;
  const uint8_t* allowed = a.allowed ? a.allowed + (size_t)r * a.allowed_stride + first : nullptr;
  uint32_t top = 0, bottom = 0xffffffffu;  // bottom: the lowest drawable value
#pragma unroll 4
  for (int i = w0 + lane; i < w1; i += 32) {
    float x = load_logit(a.logits, a.dtype, at + i);
    if (a.bias) x = __fadd_rn(x, a.bias[first + i]);
    const uint32_t u = (!allowed || allowed[i]) ? value_image(x) : 0u;
    img[i] = u;
    top = u > top ? u : top;
    if (u > kImgNegInf) bottom = u < bottom ? u : bottom;
  }
  RowSampler row{sh, img, first, n, C, rank, w0, w1};
  {
    top = __reduce_max_sync(0xffffffffu, top);
    bottom = __reduce_min_sync(0xffffffffu, bottom);
    if (lane == 0) sh.part[warp] = ((u64)top << 32) | bottom;
    __syncthreads();
    for (int w = 0; w < kSampleWarps; ++w) {
      top = max(top, (uint32_t)(sh.part[w] >> 32));
      bottom = min(bottom, (uint32_t)sh.part[w]);
    }
    const u64* all = row.exchange(((u64)top << 32) | bottom, 0);
    for (int p = 0; p < C; ++p) {
      const u64 x = row.peer(all, p)[0];
      top = max(top, (uint32_t)(x >> 32));
      bottom = min(bottom, (uint32_t)x);
    }
  }
  const float t = a.temperature ? a.temperature[r] : a.temperature_all;
  const bool finite = top > kImgNegInf && top < kImgPosInf;
  const float best = finite ? image_value(top) : 0.f;
  row.best = best;
  row.inv_t = 1.4426950408889634 / (double)t;
  row.scale_bits = a.scale_bits;
  row.cut = a.cut * t;
  const bool greedy = !finite || !(t > 0.f);

  // ---- sum of exp(x - best) for the log-probability, and the greedy index
  float z = 0.f;
  int lowest = INT_MAX;
  for (int i = w0 + lane; i < w1; i += 32) {
    const uint32_t u = img[i];
    if (greedy && u == top) lowest = min(lowest, i);
    if (finite && u > kImgNegInf) z += __expf(image_value(u) - best);
  }
  z = warp_sum(z);
  // the float sums cross the block and the cluster in a fixed order
  __syncthreads();
  if (lane == 0) sh.part[warp] = __float_as_uint(z);
  __syncthreads();
  z = 0.f;
  for (int w = 0; w < kSampleWarps; ++w) z += __uint_as_float((uint32_t)sh.part[w]);
  if (greedy) {
    const u64 low = ~row.block_max(~(u64)(lowest == INT_MAX ? 0xffffffffu : (uint32_t)(first + lowest)));
    const u64* all = row.exchange(low, __float_as_uint(z));
    z = 0.f;
    u64 lowest_all = 0xffffffffu;
    for (int p = 0; p < C; ++p) {
      const u64* x = row.peer(all, p);
      lowest_all = x[0] < lowest_all ? x[0] : lowest_all;
      z += __uint_as_float((uint32_t)x[1]);
    }
    if (rank == 0 && threadIdx.x == 0) {
      a.tokens[r] = top > kImgNegInf ? (int64_t)lowest_all : 0;
      if (a.logprobs)
        a.logprobs[r] = finite ? -logf(z)
                        : top <= kImgNegInf ? -INFINITY
                        : top == kImgPosInf ? 0.f
                                            : __uint_as_float(0x7fc00000u);
    }
    row.barrier();  // peers have read this CTA's values
    return;
  }

  // ---- the filters
  Kept kept;
  const int k = a.top_k ? a.top_k[r] : a.top_k_all;
  const float p = a.top_p ? a.top_p[r] : a.top_p_all;
  const float m = a.min_p ? a.min_p[r] : a.min_p_all;
  float per_unit = fminf((float)kSampleLinear / fminf(row.cut, best - image_value(bottom)), 3e38f);
  if (k > 0 && k < a.vocab) {
    fill_histogram<true>(row, kept, per_unit);
    shrink<true>(row, kept, per_unit, (u64)k, nullptr);
    if (kept.lo > kImgNegInf) per_unit = fminf((float)kSampleLinear / (best - image_value(kept.lo)), 3e38f);
  }
  if (p < 1.f) {
    fill_histogram<false>(row, kept, per_unit);
    shrink<false>(row, kept, per_unit, 0, &p);
  }
  const u64 floor_w = m > 0.f ? (u64)ceil((double)fminf(m, 1.f) * (double)(1ull << a.scale_bits)) : 0ull;
  auto kept_weight = [&](int i) -> u64 {
    const uint32_t u = img[i];
    if (!kept.has(u, first + i) || u <= kImgNegInf) return 0;
    const u64 w = row.weight(u);
    return w >= floor_w ? w : 0ull;
  };

  // ---- the token: running sums in index order
  u64 sum = 0, before = 0;
  for (int i = w0 + lane; i < w1; i += 32) sum += kept_weight(i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const u64 mine = sum;
  const u64 block = row.block_sum(lane == 0 ? mine : 0ull);
  u64 run = 0;
  for (int w = 0; w < warp; ++w) run += sh.part[w];
  u64 total = 0;
  {
    const u64* all = row.exchange(block, __float_as_uint(z));
    z = 0.f;
    for (int q = 0; q < C; ++q) {
      const u64* x = row.peer(all, q);
      if (q < rank) before += x[0];
      total += x[0];
      z += __uint_as_float((uint32_t)x[1]);
    }
  }
  run += before;
  const float uniform = a.uniforms[r];
  u64 target = uniform > 0.f ? (u64)((double)uniform * (double)total) : 0ull;
  target = target >= total ? total - 1 : target;
  if (run <= target && target < run + mine) {
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      u64 s = i < w1 ? kept_weight(i) : 0ull;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += x;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, run + s > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          a.tokens[r] = first + i;
          if (a.logprobs) a.logprobs[r] = (image_value(img[i]) - best) - logf(z);
        }
        break;
      }
      run += __shfl_sync(0xffffffffu, s, 31);
    }
  }
  row.barrier();  // peers have read this CTA's values
}

constexpr int kSampleMaxChunk = 40960;  // tokens of one CTA: 160 KB of images

}  // namespace

// CTAs per row: enough that a CTA's share fits its shared memory, then more while the rows leave
// SMs idle and a share is worth splitting.
static int sample_splits(int rows, int vocab, int sms) {
  int c = 1;
  while (c < kSampleMaxSplits && (vocab + c - 1) / c > kSampleMaxChunk) c *= 2;
  while (c < 8 && (long long)rows * c * 2 <= sms && vocab / (2 * c) >= 2048) c *= 2;
  return c;
}

int launch_sample(SampleArgs a, cudaStream_t stream, const char** why) {
  int device = 0, sms = 0;
  *why = "no usable current device";
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return S2R_ECUDA;
  a.splits = sample_splits(a.rows, a.vocab, sms);
  a.chunk = (a.vocab + a.splits - 1) / a.splits;
  int bits = 0;
  while ((1ll << bits) <= a.vocab) ++bits;
  a.scale_bits = 61 - bits;
  a.cut = (float)(a.scale_bits + 2) * 0.69315f;  // exp(-cut) * 2^scale_bits < 1/2
  const size_t smem = sizeof(SampleShared) + (size_t)a.chunk * sizeof(uint32_t);
  *why = "launch failed";
  if (cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
      (a.splits > 8 &&
       cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess))
    return S2R_ECUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * a.splits);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.splits;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = a.splits > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, sample_kernel, a) == cudaSuccess ? S2R_OK : S2R_ECUDA;
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
