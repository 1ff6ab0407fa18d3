// Attention of many rows over one shared K/V and each row's own pages:
// s2r_shared_attention.
//
// Row r, query head h of kv head g = h / (heads / kv_heads) attends to the
// keys [shared 0 .. S) ++ [own 0 .. n_r): s_j = scale * q . k_j,
// out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), lse = m + log sum.
// Readings of one window share its cross K/V, readings behind one prompt the
// prompt's K/V: that part is read once for all rows, where attention row by
// row reads it once per row.
//
// The keys of a (row, head) are cut into parts; every part gives (m, l, o)
// with o = sum exp(s - m) v in float32, and the parts are joined in a fixed
// order: M = max m, out = sum_p o_p 2^(m_p - M) / sum_p l_p 2^(m_p - M), with
// m in units of log2.  Shared parts come from shared_tile_kernel (tensor
// cores), own parts from own_attn_kernel, which runs beside it.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdio>
#include <mutex>
#include <type_traits>
#include <utility>

#include "../../include/s2r.h"
#include "common.cuh"
#include "mbarrier.cuh"
#include "shared_attn.cuh"
#include "tensor_core.cuh"

namespace s2r {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---- the rows' own parts
//
// The unit of work is one part of one (row, kv head); a warp takes one unit or,
// of short rows, several in turn, and reads their K and V in 16 KB chunks (64
// tokens at dim 64, 32 at dim 128; a page is a contiguous 64 x dim block per
// head) through a ring of two chunks that one lane fills by TMA with the
// 128-byte swizzle.  The ring runs on from unit to unit, so rows of a page or
// two cost no start of their own (a CTA per row and head reached 3.3 TB/s on
// such rows).  Memory bounds this part (a key is read for heads / kv_heads
// queries), so what counts is bytes in flight, 192 KB an SM, and there is no
// barrier beyond the warp (5.6 TB/s on rows of up to 2,500 tokens, 8 heads of
// dim 128; 4.9 TB/s on rows of up to 200, 16 heads of dim 64).  The products are mma.sync m16n8k16, rows = the
// group's queries (8, or 16 with WIDE): a 128-row tcgen05 tile would hold at
// most 16 live rows and its round trip through tensor memory would sit in the
// chain of every chunk.
constexpr int kOwnThreads = 32;
constexpr int kOwnWarps = kOwnThreads / 32;
constexpr int kOwnStages = 2;
constexpr int kOwnPiece = 16;     // tokens of a box of a row's last chunk
constexpr int kOwnStage = 16384;  // bytes of a chunk, K then V (8 KB: rows of up to 200 tokens 3% faster, 1,500 10% slower)
constexpr int kOwnSmem = kOwnWarps * kOwnStages * kOwnStage + 1024;  // + alignment slack

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void mma16816(bf16, float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(__half, float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int D, bool WIDE>
__global__ void __launch_bounds__(kOwnThreads)
    own_attn_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ CUtensorMap map_k_piece, const __grid_constant__ CUtensorMap map_v_piece,
                    const __grid_constant__ SharedAttnArgs a, bool q_pairs, float* part_o, float2* part_ml, int first_part) {
  constexpr int kTokens = kOwnStage / (4 * D);  // of a chunk: 64 or 32
  constexpr int kBoxes = D / 64, kBox = kTokens * 128;
  constexpr int kHalves = WIDE ? 2 : 1;  // live halves of the MMA's 16 rows
  constexpr int kQueries = 8 * kHalves;
  extern __shared__ __align__(1024) unsigned char own_smem[];
  __shared__ __align__(8) uint64_t full[kOwnWarps][kOwnStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* base =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(own_smem) + 1023) & ~uintptr_t(1023));
  unsigned char* ring = base + warp * kOwnStages * kOwnStage;
  const int group = a.heads / a.kv_heads, sets = (group + kQueries - 1) / kQueries, splits = a.own_splits;
  const int per_row = a.kv_heads * sets * splits;
  const int stride = gridDim.x * kOwnWarps;  // (rows x heads <= 2^24, splits <= 32: units stay below 2^31)
  // Unit u is (row, place in the row); steps of `stride` need no division.
  struct Unit {
    int r, place;
  };
  const int step_r = stride / per_row, step_place = stride % per_row;
  auto next = [&](Unit u) {
    u.r += step_r;
    u.place += step_place;
    if (u.place >= per_row) {
      u.place -= per_row;
      ++u.r;
    }
    return u;
  };
  auto part_of = [&](Unit u) { return splits == 1 ? 0 : u.place % splits; };
  auto set_of = [&](Unit u) { return sets == 1 ? 0 : u.place / splits % sets; };
  auto kv_head_of = [&](Unit u) { return splits * sets == 1 ? u.place : u.place / (splits * sets); };

  if (lane == 0) {
    for (int i = 0; i < kOwnStages; ++i) mbar_init(&full[warp][i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  __syncwarp();

  // Chunks [c0, c1) of unit u, given its row's length; a length past the page table counts as 0.
  auto range = [&](Unit u, int n, int& c0, int& c1) {
    const int chunks = ((n < 0 || n > a.pages_per_row * kPageTokens ? 0 : n) + kTokens - 1) / kTokens;
    if (splits == 1) {
      c0 = 0;
      c1 = chunks;
      return;
    }
    const int per = (chunks + splits - 1) / splits;
    c0 = min(chunks, part_of(u) * per);
    c1 = min(chunks, c0 + per);
  };
  auto length = [&](Unit u) { return u.r < a.rows ? a.own_len[u.r] : 0; };

  // ---- the loader: walks the warp's units and their chunks up to kOwnStages chunks ahead.  A unit's
  // length is requested two units ahead and its first page numbers (32 chunks, one a lane) one unit
  // ahead, so that no unit starts with a wait for them.
  const int first = blockIdx.x * kOwnWarps + warp;
  const Unit start{first / per_row, first % per_row};
  Unit lu = start, lu1 = next(lu);  // the unit loaded and the one behind it
  int lc, lc1, base_c, n0, n1, n2, pages, pages1;
  auto first_pages = [&](Unit u, int n) {
    int c0, c1;
    range(u, n, c0, c1);
    const int c = c0 + lane;
    return u.r < a.rows && c < c1 ? a.page_table[u.r * a.page_stride + c * kTokens / kPageTokens] : 0;
  };
  {
    n0 = length(lu);
    n1 = length(lu1);
    n2 = length(next(lu1));
    range(lu, n0, lc, lc1);
    base_c = lc;
    pages = first_pages(lu, n0);
    pages1 = first_pages(lu1, n1);
  }
  int loaded = 0;         // chunks requested
  unsigned bad_stage = 0;  // stages whose page was broken (nothing was loaded)
  auto load_next = [&]() {  // one more chunk into stage loaded % kOwnStages, if there is one
    while (lc >= lc1) {
      if (lu.r >= a.rows) return;
      lu = lu1;
      lu1 = next(lu1);
      range(lu, n1, lc, lc1);
      if (lu.r >= a.rows) {
        lc = lc1 = 0;
        return;
      }
      base_c = lc;
      pages = pages1;
      n0 = n1;
      n1 = n2;
      n2 = length(next(lu1));
      pages1 = first_pages(lu1, n1);
    }
    if (lc >= base_c + 32) {
      base_c = lc;
      const int c = lc + lane;
      pages = c < lc1 ? a.page_table[lu.r * a.page_stride + c * kTokens / kPageTokens] : 0;
    }
    const int page = __shfl_sync(0xffffffffu, pages, lc - base_c), st = loaded % kOwnStages;
    const bool ok = page >= 0 && page < a.own_pages;
    bad_stage = ok ? bad_stage & ~(1u << st) : bad_stage | 1u << st;
    if (lane == 0) {
      unsigned char* stage = ring + st * kOwnStage;
      uint64_t* bar = &full[warp][st];
      if (ok) {
        const int g = kv_head_of(lu);
        const int token = (page * a.kv_heads + g) * kPageTokens + lc * kTokens % kPageTokens;
        const int live = n0 - lc * kTokens;
        if (live > kTokens - kOwnPiece) {
          mbar_expect_tx(bar, kOwnStage);
#pragma unroll
          for (int b = 0; b < kBoxes; ++b) tma_load_2d(stage + b * kBox, &map_k, b * 64, token, bar);
#pragma unroll
          for (int b = 0; b < kBoxes; ++b) tma_load_2d(stage + kOwnStage / 2 + b * kBox, &map_v, b * 64, token, bar);
        } else {  // a row's last chunk: only the pieces that hold tokens
          const int n = (live + kOwnPiece - 1) / kOwnPiece;
          mbar_expect_tx(bar, n * kOwnPiece * D * 4);
          for (int x = 0; x < n; ++x)
#pragma unroll
            for (int b = 0; b < kBoxes; ++b) {
              unsigned char* dst = stage + b * kBox + x * (kOwnPiece * 128);
              tma_load_2d(dst, &map_k_piece, b * 64, token + x * kOwnPiece, bar);
              tma_load_2d(dst + kOwnStage / 2, &map_v_piece, b * 64, token + x * kOwnPiece, bar);
            }
        }
      } else {
        mbar_arrive(bar);
        if (a.error) atomicExch(a.error, kErrOwnPage);
      }
    }
    ++lc;
    ++loaded;
  };
#pragma unroll
  for (int i = 0; i < kOwnStages; ++i) load_next();

  // A unit's queries: the A operand of rows lane / 4 (and 8 more), 16 channels a step.
  auto load_queries = [&](Unit u, uint32_t (&qa)[D / 16][4]) {
    const int g = kv_head_of(u), h0 = g * group + set_of(u) * kQueries;
    const int heads = u.r < a.rows ? min(kQueries, (g + 1) * group - h0) : 0;
    const T* q = static_cast<const T*>(a.q) + u.r * a.q_row + h0 * a.q_head;
#pragma unroll
    for (int e = 0; e < D / 16; ++e)
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int row = lane / 4 + (f & 1) * 8, at = e * 16 + (f >> 1) * 8 + (lane & 3) * 2;
        qa[e][f] = 0;
        if ((f & 1) < kHalves && row < heads) {
          const unsigned short* src = reinterpret_cast<const unsigned short*>(q + row * a.q_head + at);
          qa[e][f] = q_pairs ? *reinterpret_cast<const uint32_t*>(src) : src[0] | (uint32_t)src[1] << 16;
        }
      }
  };
  const float c = a.scale * kLog2e;
  uint32_t qa[D / 16][4], qn[D / 16][4];
  Unit u = start;
  int n_unit = length(u);
  load_queries(u, qa);
  int used = 0;  // chunks consumed
  bool timeout = false;
  for (; u.r < a.rows && !timeout; u = next(u)) {
    int c0, c1;
    const int n = n_unit;
    range(u, n, c0, c1);
    n_unit = length(next(u));
    load_queries(next(u), qn);  // in flight under this unit
    bool broken = n > a.pages_per_row * kPageTokens;
    if (broken && lane == 0 && a.error) atomicExch(a.error, kErrOwnLength);
    float o[D / 8][4], m[kHalves], l[kHalves];
#pragma unroll
    for (int e = 0; e < D / 8; ++e) o[e][0] = o[e][1] = o[e][2] = o[e][3] = 0.f;
#pragma unroll
    for (int f = 0; f < kHalves; ++f) m[f] = -INFINITY, l[f] = 0.f;

    for (int k = c0; k < c1; ++k, ++used) {
      const int st = used % kOwnStages;
      unsigned char* stage = ring + st * kOwnStage;
      const uint32_t k_at = smem_u32(stage), v_at = k_at + kOwnStage / 2;
      if (!__all_sync(0xffffffffu, mbar_wait_fast(&full[warp][st], (used / kOwnStages) & 1))) {
        timeout = true;
        break;
      }
      if (bad_stage >> st & 1) {
        broken = true;
        load_next();
        continue;
      }
      const int live = n - k * kTokens;  // tokens of the chunk, if fewer
      if (live < kTokens) {  // V rows behind the last token may hold anything: zero for the product
        for (int x = live * 8 + lane; x < kTokens * 8; x += 32)
#pragma unroll
          for (int b = 0; b < kBoxes; ++b)
            *reinterpret_cast<uint4*>(stage + kOwnStage / 2 + b * kBox + x * 16) = make_uint4(0, 0, 0, 0);
        fence_async_smem();  // (the stage is filled again by TMA)
        __syncwarp();
      }
      // S = Q K^T, 8 keys a tile
      float s[kTokens / 8][4];
#pragma unroll
      for (int j = 0; j < kTokens / 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int e = 0; e < D / 16; ++e)
#pragma unroll
        for (int j = 0; j < kTokens / 8; j += 2) {
          const int key = j * 8 + (lane & 7) + (lane >> 4) * 8, piece = e * 2 + ((lane >> 3) & 1);
          uint32_t b[4];
          ldmatrix4(b, k_at + (piece / 8) * kBox + sw128_off(key, piece % 8));
          mma16816(T(), s[j], qa[e], b[0], b[1]);
          mma16816(T(), s[j + 1], qa[e], b[2], b[3]);
        }
      if (live < kTokens) {
#pragma unroll
        for (int j = 0; j < kTokens / 8; ++j)
#pragma unroll
          for (int f = 0; f < 4; ++f)
            if (j * 8 + (lane & 3) * 2 + (f & 1) >= live) s[j][f] = -INFINITY;
      }
      // online softmax of each row (4 lanes hold it)
      uint32_t pa[kTokens / 16][4];
#pragma unroll
      for (int f = 0; f < kHalves; ++f) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kTokens / 8; ++j) top = fmaxf(top, fmaxf(s[j][2 * f], s[j][2 * f + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        top = fmaxf(top * c, m[f]);
        if (__any_sync(0xffffffffu, top > m[f])) {
          const float keep = m[f] == -INFINITY ? 1.f : exp2_approx(m[f] - top);
          l[f] *= keep;
#pragma unroll
          for (int e = 0; e < D / 8; ++e) o[e][2 * f] *= keep, o[e][2 * f + 1] *= keep;
          m[f] = top;
        }
        const float shift = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int j = 0; j < kTokens / 8; ++j) {
          const float p0 = exp2_approx(fmaf(s[j][2 * f], c, -shift)), p1 = exp2_approx(fmaf(s[j][2 * f + 1], c, -shift));
          l[f] += p0 + p1;  // (this lane's keys; the row's lanes are added at the end)
          pa[j / 2][(j & 1) * 2 + f] = pack_pair(T(), p0, p1);
        }
      }
      if (!WIDE) {
#pragma unroll
        for (int j = 0; j < kTokens / 16; ++j) pa[j][1] = pa[j][3] = 0;
      }
      // O += P V, 8 channels a tile
#pragma unroll
      for (int j = 0; j < kTokens / 16; ++j)
#pragma unroll
        for (int e = 0; e < D / 8; e += 2) {
          const int key = j * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, piece = e + (lane >> 4);
          uint32_t b[4];
          ldmatrix4_trans(b, v_at + (piece / 8) * kBox + sw128_off(key, piece % 8));
          mma16816(T(), o[e], pa[j], b[0], b[1]);
          mma16816(T(), o[e + 1], pa[j], b[2], b[3]);
        }
      __syncwarp();  // every lane has read the stage
      load_next();
    }
    // ---- the unit's sums
    const int g = kv_head_of(u), h0 = g * group + set_of(u) * kQueries;
    const int heads = min(kQueries, (g + 1) * group - h0);
#pragma unroll
    for (int f = 0; f < kHalves; ++f) {
      l[f] += __shfl_xor_sync(0xffffffffu, l[f], 1);
      l[f] += __shfl_xor_sync(0xffffffffu, l[f], 2);
      if (broken || timeout) l[f] = __uint_as_float(0x7fc00000u);  // a row with broken pages comes out as NaN
      const int row = lane / 4 + 8 * f;
      if (row >= heads) continue;
      const size_t dst = ((size_t)(first_part + part_of(u)) * a.rows + u.r) * a.heads + h0 + row;
      if ((lane & 3) == 0) part_ml[dst] = make_float2(m[f], l[f]);
      if (m[f] == -INFINITY) continue;
#pragma unroll
      for (int e = 0; e < D / 8; ++e)
        *reinterpret_cast<float2*>(part_o + dst * D + e * 8 + (lane & 3) * 2) = make_float2(o[e][2 * f], o[e][2 * f + 1]);
    }
#pragma unroll
    for (int e = 0; e < D / 16; ++e)
#pragma unroll
      for (int f = 0; f < 4; ++f) qa[e][f] = qn[e][f];
  }
  if (timeout) {  // mark what is left, let the copies in flight land before the CTA exits (bounded)
    if (lane == 0 && a.error) atomicExch(a.error, kErrSharedWait);
    for (int i = used; i < loaded; ++i) mbar_wait(&full[warp][i % kOwnStages], (i / kOwnStages) & 1);
    for (; u.r < a.rows; u = next(u))
      for (int row = lane; row < kQueries; row += 32) {
        const int g = kv_head_of(u), h0 = g * group + set_of(u) * kQueries;
        if (h0 + row < (g + 1) * group)
          part_ml[((size_t)(first_part + part_of(u)) * a.rows + u.r) * a.heads + h0 + row] =
              make_float2(-INFINITY, __uint_as_float(0x7fc00000u));
      }
  }
  pdl_launch_dependents();
  pdl_wait();  // this kernel runs beside the shared part; the join waits for both
}

// out and lse of one (row, head) from its joined sums, `n` channels from `d`.
template <typename T, int N>
__device__ __forceinline__ void store_out(const SharedAttnArgs& a, int r, int h, int d, const float (&o)[N], float sum,
                                          float top, bool first) {
  const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no key at all: 0
  T* dst = static_cast<T*>(a.out) + r * a.out_row + h * a.out_head + d;
  if (a.out_vector) {
    if constexpr (N >= 8) {
#pragma unroll
      for (int e = 0; e < N; e += 8)
        *reinterpret_cast<uint4*>(dst + e) =
            make_uint4(pack_pair(T(), o[e] * inv, o[e + 1] * inv), pack_pair(T(), o[e + 2] * inv, o[e + 3] * inv),
                       pack_pair(T(), o[e + 4] * inv, o[e + 5] * inv), pack_pair(T(), o[e + 6] * inv, o[e + 7] * inv));
    } else {
#pragma unroll
      for (int e = 0; e < N; e += 2)
        *reinterpret_cast<uint32_t*>(dst + e) = pack_pair(T(), o[e] * inv, o[e + 1] * inv);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) dst[e] = T(o[e] * inv);
  }
  if (a.lse && first) a.lse[(size_t)r * a.heads + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// Joins the parts of every (row, head): a warp each.  The lanes fetch the parts' (m, l) at once, then
// the parts' sums come eight in flight (one after the other, 30 parts took 9 us).
constexpr int kJoinAhead = 8;

template <typename T, int D>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ SharedAttnArgs a, const float* part_o,
                                                   const float2* part_ml, int parts) {
  constexpr int kEach = D / 32, kRounds = (kMaxSharedSplits + kMaxOwnSplits + 31) / 32;
  const int lane = threadIdx.x & 31;
  const int64_t pair = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), pairs = (int64_t)a.rows * a.heads;
  pdl_launch_dependents();
  pdl_wait();
  if (pair >= pairs) return;
  float2 ml[kRounds];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int p = i * 32 + lane;
    ml[i] = p < parts ? part_ml[p * pairs + pair] : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, ml[i].x);
  }
  top = warp_max(top);
  float sum = 0.f, weight[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    // an empty part (its o is not written): l is 0, or NaN where something broke
    weight[i] = ml[i].x == -INFINITY ? 0.f : exp2f(ml[i].x - top);
    sum += ml[i].x == -INFINITY ? ml[i].y : ml[i].y * weight[i];
  }
  sum = warp_sum(sum);
  float acc[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) acc[e] = 0.f;
  const float* src = part_o + (size_t)pair * D + lane * kEach;
  for (int p0 = 0; p0 < parts; p0 += kJoinAhead) {
    float w[kJoinAhead], x[kJoinAhead][kEach];
    const float mine = p0 < 32 ? weight[0] : p0 < 64 ? weight[1] : weight[kRounds - 1];
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      w[u] = __shfl_sync(0xffffffffu, mine, (p0 + u) & 31);
#pragma unroll
      for (int e = 0; e < kEach; ++e) x[u][e] = 0.f;
      if (w[u] != 0.f) {  // (parts behind the last weigh 0)
        const float* at = src + (size_t)(p0 + u) * pairs * D;
        if constexpr (kEach == 2) {
          const float2 v = *reinterpret_cast<const float2*>(at);
          x[u][0] = v.x, x[u][1] = v.y;
        } else {
          const float4 v = *reinterpret_cast<const float4*>(at);
          x[u][0] = v.x, x[u][1] = v.y, x[u][2] = v.z, x[u][3] = v.w;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u)
#pragma unroll
      for (int e = 0; e < kEach; ++e) acc[e] = fmaf(x[u][e], w[u], acc[e]);
  }
  store_out<T>(a, (int)(pair / a.heads), (int)(pair % a.heads), lane * kEach, acc, sum, top, lane == 0);
}

// ---- the shared part on tensor cores
//
// The queries of one kv head, (row, group member) pairs in order, are tiles of
// 128: the MMA's M, one tensor-memory lane and one softmax thread each.  A CTA
// walks its part of the keys in tiles of 64, with two streams in flight, each
// with a score tile S, a weight tile P, an output accumulator O and a warpgroup
// of its own:
//
//   one query tile (PAIR = false): the streams take the even and the odd key
//     tiles and are joined at the end;
//   two query tiles (PAIR = true): stream s is query tile s, both walk every
//     key tile, which is then read once for 256 queries.
//
//   S = Q K^T      tcgen05.mma M128 N64 K=dim, float32 in tensor memory
//   p = 2^(c s - m) c = scale log2(e); m trails the running maximum by at most
//                  2^8, so that O is rescaled only when the maximum moves far
//                  (Milakov and Gimelshein's online softmax, with slack)
//   O += P V       P packed to 16 bits in tensor memory: the A operand; V as
//                  it lies in memory (token rows): the B operand with the
//                  channel axis contiguous
//
// Rounding: P is rounded to the tensors' 16-bit type for the product, as in
// every 16-bit attention (half a step of each weight); l sums the unrounded
// float32 values; O is float32 throughout.
//
// Warp 0 loads K and V tiles by TMA into a ring, warp 1 (at dim 128 warps 1 and 2,
// one per stream) issues the MMAs, warps 4-7 and 8-11 are the softmax warpgroups.
// What bounds a large call is the chain of one stream, S -> weights -> O (about
// half of a tile's time passes in its barriers and the tensor memory's round
// trips; the exponentials' unit is busy 54% of the time at dim 64), so as many
// streams as fit run on an SM (1,024 rows of 16 heads over 16,384 tokens: 120 us,
// 575 TFLOP/s):
//
//   dim 64: P lies in S's columns, 256 columns and 98 KB a CTA, two CTAs an SM,
//     four streams.  The next S of a stream follows the product that reads P;
//     both accumulators are 128 x 64, and MMAs of one accumulator shape execute in
//     order, so S complete also means the last product complete.
//   dim 128: O alone fills half the tensor memory; one CTA an SM.  S is handed
//     back as soon as the softmax has it in registers, P has columns of its own,
//     and S of the next tile is computed under this tile's exponentials.  With an
//     issuing warp per stream neither waits for the other's softmax (124 -> 102 us
//     at 1,024 rows of 16 heads over 8,192 tokens; at dim 64, where S follows PV
//     anyway, one warp is faster, 126 against 135 us over 16,384).
//
// Every mbarrier wait is bounded; on a timeout the CTA marks its rows NaN, drains
// its copies and MMAs (bounded), frees its tensor memory and returns.
constexpr int kTileThreads = 384;
constexpr int kTileRows = 128;  // queries of a tile
constexpr int KT = 64;          // keys of a tile
constexpr float kMaxSlack = 8.f;

template <int D, bool PAIR>
struct Tile {
  static constexpr bool kShareS = D == 64;            // P in S's columns, two CTAs an SM
  static constexpr int kPerSm = kShareS ? 2 : 1;
  static constexpr int kIssuers = kShareS ? 1 : 2;    // warps that issue MMAs
  static constexpr int kCols = kShareS ? 256 : 512;   // tensor memory: S0 S1 O0 O1 (P0 P1)
  static constexpr uint32_t kAtS = 0, kAtO = 2 * KT, kAtP = kShareS ? kAtS : kAtO + 2 * D;
  static constexpr uint32_t kStepP = kShareS ? KT : KT / 2;
  static_assert(kAtO + 2 * D <= kCols && kAtP + KT <= kCols, "fits the tensor memory");
  // registers: the block's at launch, for the issuing warps and for the softmax warps
  static constexpr int kRegs = kShareS ? 80 : 168, kRegsIssue = kShareS ? 32 : 40, kRegsSoftmax = kShareS ? 104 : 232;
  static_assert(kRegsIssue + 2 * kRegsSoftmax <= 3 * kRegs, "within what the block was launched with");
  static constexpr int kBox = KT * 128;        // bytes of 64 channels of a tile
  static constexpr int kTile = KT * D * 2;     // a K or V tile
  static constexpr int kSlot = 2 * kTile;      // K and V of a key tile
  static constexpr int kQueries = (PAIR ? 2 : 1) * kTileRows * D * 2;
  static constexpr int kSlots = 4;
  static constexpr int kBytes = kQueries + kSlots * kSlot + 1024;  // + alignment slack
  static_assert(kPerSm * (kBytes + 2048) <= 228 * 1024, "fits an SM");
  static_assert(kTileRows * (D + 4) * 4 <= kSlots * kSlot, "a stream's partial fits the ring");
};

struct TileArgs {
  SharedAttnArgs a;
  float* part_o;    // null: the part is the whole answer
  float2* part_ml;
  bool token_last;  // the tensor maps' axes are (channel, head, token) instead of (channel, token, head)
  bool q_vector;    // q can be read 16 bytes at a time
};

template <typename T, int D, bool PAIR>
__global__ void __launch_bounds__(kTileThreads, Tile<D, PAIR>::kPerSm)
    shared_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ TileArgs t) {
  using Shape = Tile<D, PAIR>;
  constexpr int kSlots = Shape::kSlots, kSlot = Shape::kSlot, kTile = Shape::kTile, kBox = Shape::kBox, kBoxes = D / 64;
  constexpr int kQueryBox = kTileRows * 128;
  constexpr bool kShareS = Shape::kShareS;
  const SharedAttnArgs& a = t.a;
  extern __shared__ __align__(1024) unsigned char tile_smem[];
  unsigned char* base =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tile_smem) + 1023) & ~uintptr_t(1023));
  unsigned char* sq = base;                    // query tiles: [tile][box][128 rows][128 bytes]
  unsigned char* ring = base + Shape::kQueries;  // slot k % kSlots: K, then V of the CTA's key tile k
  __shared__ __align__(8) uint64_t full[kSlots], empty[kSlots], s_full[2], s_empty[2], p_full[2], pv_done[2], done;
  __shared__ uint32_t tmem_base;
  __shared__ int aborted;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x, g = blockIdx.y, part = blockIdx.z;  // (the parts' short last ones start last)
  const int group = a.heads / a.kv_heads, queries = a.rows * group;
  const int tile0 = tile * (PAIR ? 2 : 1);  // first query tile

  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], PAIR ? Shape::kIssuers : 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 4);  // one arrival per warp of the stream
      mbar_init(&p_full[s], 4);
      mbar_init(&pv_done[s], 1);
    }
    mbar_init(&done, Shape::kIssuers);
    aborted = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();  // this thread starts copies on them ahead of the block's barrier
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "r"(Shape::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
  }
  pdl_wait();  // the queries come from the kernel before
  const int tokens = a.shared_len ? min(max(*a.shared_len, 0), a.shared_tokens) : a.shared_tokens;
  // every part `per` of the live tiles, in the proportion planned for all of them, the last what is left
  const int tiles = (tokens + KT - 1) / KT, planned = (a.shared_tokens + KT - 1) / KT;
  const int per = tiles == planned ? a.part_tiles : (int)(((long long)tiles * a.part_tiles + planned - 1) / planned);
  const int t0 = min(tiles, part * per), nt = min(tiles, t0 + per) - t0;

  auto fail = [&]() {
    if (a.error) atomicExch(a.error, kErrSharedWait);
    *(volatile int*)&aborted = 1;
  };
  auto stopped = [&]() { return *(volatile int*)&aborted != 0; };
  auto load_tile = [&](int k) {
    const int token = (t0 + k) * KT;
    unsigned char* slot = ring + k % kSlots * kSlot;
    uint64_t* bar = &full[k % kSlots];
    mbar_expect_tx(bar, kSlot);
#pragma unroll
    for (int b = 0; b < kBoxes; ++b)
      tma_load_3d(slot + b * kBox, &map_k, b * 64, t.token_last ? g : token, t.token_last ? token : g, bar);
#pragma unroll
    for (int b = 0; b < kBoxes; ++b)
      tma_load_3d(slot + kTile + b * kBox, &map_v, b * 64, t.token_last ? g : token, t.token_last ? token : g, bar);
  };
  const int ahead = min(nt, kSlots);  // tiles requested before the queries are staged
  if (threadIdx.x == 0)
    for (int k = 0; k < ahead; ++k) load_tile(k);

  // ---- the queries, in the 128-byte-swizzled rows the MMA reads (by the softmax warps, four
  // pieces in flight each)
  if (warp >= 4) {
    constexpr int kPieces = (PAIR ? 2 : 1) * kTileRows * (D / 8), kThreads = kTileThreads - 128;
    static_assert(kPieces % (4 * kThreads) == 0, "whole batches");
#pragma unroll 1
    for (int i0 = threadIdx.x - 128; i0 < kPieces; i0 += 4 * kThreads) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * kThreads, x = tile0 * kTileRows + i / (D / 8), c = i % (D / 8);
        v[u] = make_uint4(0, 0, 0, 0);
        if (x < queries) {
          const int r = group == 1 ? x : x / group;
          const T* src = static_cast<const T*>(a.q) + r * a.q_row + (g * group + x - r * group) * a.q_head + c * 8;
          if (t.q_vector) {
            v[u] = *reinterpret_cast<const uint4*>(src);
          } else {
            const unsigned short* e = reinterpret_cast<const unsigned short*>(src);
            v[u] = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                              e[6] | (uint32_t)e[7] << 16);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * kThreads, row = i / (D / 8), c = i % (D / 8);
        unsigned char* tile = sq + row / kTileRows * (kTileRows * D * 2) + c / 8 * kQueryBox;
        *reinterpret_cast<uint4*>(tile + sw128_off(row % kTileRows, c % 8)) = v[u];
      }
    }
  }
  fence_async_smem();
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  // Dependents may start only now: one that needs tensor memory must not take it ahead of this CTA.
  pdl_launch_dependents();
  const uint32_t tmem = tmem_base;

  // The issuing warps give most of their registers to the softmax warps.
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Shape::kRegsIssue));
  if (warp == 0) {
    if (lane == 0) {
      // ---- producer
      int issued = ahead;
      for (int k = ahead; k < nt; ++k) {
        if (!mbar_wait_fast(&empty[k % kSlots], (k / kSlots - 1) & 1) || stopped()) {
          fail();
          break;
        }
        load_tile(k);
        issued = k + 1;
      }
      // every copy has landed before the ring is reused or the CTA exits (bounded)
      for (int k = max(0, issued - kSlots); k < issued; ++k) mbar_wait(&full[k % kSlots], (k / kSlots) & 1);
    }
  } else if (warp <= Shape::kIssuers) {
    // ---- MMA issuers: the warp stays converged (what describes an MMA is then warp-uniform), one lane
    // issues
    constexpr uint32_t kFormat = std::is_same<T, bf16>::value ? 1u : 0u;
    constexpr uint32_t kIdescS = umma_idesc(kFormat, kTileRows, KT, false);
    constexpr uint32_t kIdescO = umma_idesc(kFormat, kTileRows, D, true);
    bool ok = true;
    auto issue_s = [&](int s, int k, int nth) {  // S_s = Q K_k^T, the stream's nth
      ok = ok && mbar_wait_fast(&full[k % kSlots], (k / kSlots) & 1);
      if (!kShareS && nth > 0) ok = ok && mbar_wait_fast(&s_empty[s], (nth - 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        return;
      }
      tmem_fence_after();
      const uint64_t da = umma_desc_sw128(sq + (PAIR ? s * (kTileRows * D * 2) : 0));
      const uint64_t db = umma_desc_sw128(ring + k % kSlots * kSlot);
      if (elect_one()) {
#pragma unroll
        for (int e = 0; e < D / 16; ++e)  // 16 channels: 32 bytes of a row, a box every 64
          umma_f16(tmem + Shape::kAtS + s * KT, da + (uint64_t)((e / 4) * (kQueryBox >> 4) + (e % 4) * 2),
                   db + (uint64_t)((e / 4) * (kBox >> 4) + (e % 4) * 2), kIdescS, e > 0);
        umma_commit(&s_full[s]);
      }
      __syncwarp();
    };
    auto issue_pv = [&](int s, int k, int nth) {  // O_s += P_s V_k, the stream's nth product
      ok = ok && mbar_wait_fast(&p_full[s], nth & 1);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        return;
      }
      tmem_fence_after();
      const uint64_t db = umma_desc_mn_sw128(ring + k % kSlots * kSlot + kTile, kBox);
      if (elect_one()) {
#pragma unroll
        for (int e = 0; e < KT / 16; ++e)  // 16 keys: 8 columns of packed P, 16 rows of V
          umma_f16_ta(tmem + Shape::kAtO + s * D, tmem + Shape::kAtP + s * Shape::kStepP + e * 8,
                      db + (uint64_t)(e * (16 * 128 >> 4)), kIdescO, nth > 0 || e > 0);
        if (!kShareS) umma_commit(&pv_done[s]);
        if (!PAIR || Shape::kIssuers == 2 || s == 1) umma_commit(&empty[k % kSlots]);
      }
      __syncwarp();
    };
    const int step = PAIR ? 1 : 2;  // between a stream's key tiles
    if (Shape::kIssuers == 2) {  // a warp per stream
      const int s = warp - 1, k0 = PAIR ? 0 : s;
      if (k0 < nt) issue_s(s, k0, 0);
      for (int k = k0, n = 0; k < nt; k += step, ++n) {
        if (k + step < nt) issue_s(s, k + step, n + 1);  // S runs one tile ahead
        issue_pv(s, k, n);
      }
    } else {
      for (int s = 0; s < 2; ++s)
        if ((PAIR ? 0 : s) < nt) issue_s(s, PAIR ? 0 : s, 0);
      for (int k = 0; k < nt; ++k)
        for (int s = PAIR ? 0 : k & 1; s <= (PAIR ? 1 : k & 1); ++s) {
          const int n = PAIR ? k : k >> 1;
          issue_pv(s, k, n);
          if (k + step < nt) issue_s(s, k + step, n + 1);
        }
    }
    if (!ok && lane == 0) fail();
    if (elect_one()) umma_commit(&done);  // arrives once every MMA issued has completed
    __syncwarp();
  }

  __syncthreads();
  if (threadIdx.x == 0) {
    if (!mbar_wait(&done, 0)) fail();  // every MMA has completed
  }
  __syncthreads();
  __syncthreads();  // the softmax warps have read O
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Shape::kCols) : "memory");
  if (!PAIR) __syncthreads();
  return;
  }

  // ---- softmax: thread = query (tensor-memory lane) of stream s
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Shape::kRegsSoftmax));
  const int s = (warp >> 2) - 1;
  const int row = (warp & 3) * 32 + lane;
  const int x = (tile0 + (PAIR ? s : 0)) * kTileRows + row;  // query of the kv head
  float m = -INFINITY, l = 0.f;
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
  const int first = PAIR ? 0 : s, step = PAIR ? 1 : 2;
  const int mine = nt > first ? (nt - first + step - 1) / step : 0;  // tiles of the stream
  bool ok = true;
  {
    const float c = a.scale * kLog2e;
    const uint32_t s_at = tmem + lanes + Shape::kAtS + s * KT, o_at = tmem + lanes + Shape::kAtO + s * D;
    const uint32_t p_at = tmem + lanes + Shape::kAtP + s * Shape::kStepP;
    const bool live_warp = x - lane < queries;  // some query of the warp exists
    for (int j = 0; j < mine; ++j) {
      const int k = first + j * step;
      if (!__all_sync(0xffffffffu, mbar_wait_fast(&s_full[s], j & 1))) {
        ok = false;
        break;
      }
      tmem_fence_after();
      uint32_t v[KT];
      if (live_warp) {
#pragma unroll
        for (int e = 0; e < KT; e += 32) tmem_ld32(s_at + e, *reinterpret_cast<uint32_t(*)[32]>(v + e));
        tmem_wait_ld();
      }
      if (!kShareS) {
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[s]);
      }
      const int live = tokens - (t0 + k) * KT;  // keys of the tile, if fewer
      if (live < KT) {
        // V rows behind the last token may hold anything: zero for the product (P is 0 there)
        if (!__all_sync(0xffffffffu, mbar_wait(&full[k % kSlots], (k / kSlots) & 1))) {
          ok = false;
          break;
        }
        for (int e = live * 8 + row; e < KT * 8; e += kTileRows)
#pragma unroll
          for (int b = 0; b < kBoxes; ++b)
            *reinterpret_cast<uint4*>(ring + k % kSlots * kSlot + kTile + b * kBox + e * 16) = make_uint4(0, 0, 0, 0);
        fence_async_smem();
      }
      float to = m, keep = 1.f;
      bool move = false;
      if (live_warp) {
        if (live < KT) {
#pragma unroll
          for (int e = 0; e < KT; ++e)
            if (e >= live) v[e] = 0xff800000u;
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < KT; e += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            top[q] = max3(top[q], __uint_as_float(v[e + 2 * q]), __uint_as_float(v[e + 2 * q + 1]));
        to = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
        move = __any_sync(0xffffffffu, to > m + kMaxSlack);
        if (move) {
          to = to > m + kMaxSlack ? to : m;
          keep = m == -INFINITY ? 1.f : exp2_approx(m - to);
          m = to;
          l *= keep;
        }
        // the weights 2^(c s - m), in pairs
        const float shift = m == -INFINITY ? 0.f : m;
        const uint64_t c2 = pack2(c, c), shift2 = pack2(-shift, -shift);
        uint64_t sum2[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < KT; e += 2) {
          float p0, p1;
          unpack2(fma2(pack2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), c2, shift2), p0, p1);
          p0 = exp2_approx(p0);
          p1 = exp2_approx(p1);
          sum2[e / 2 & 1] = add2(sum2[e / 2 & 1], pack2(p0, p1));
          v[e / 2] = pack_pair(T(), p0, p1);
        }
        float x0, x1;
        unpack2(add2(sum2[0], sum2[1]), x0, x1);
        l += x0 + x1;
      }
      // P and O are free once the stream's last product has landed (kShareS: it has, before S)
      if (!kShareS && j > 0 && !__all_sync(0xffffffffu, mbar_wait_fast(&pv_done[s], (j - 1) & 1))) {
        ok = false;
        break;
      }
      tmem_fence_after();
      if (live_warp) {
        if (move && j > 0) {
#pragma unroll 1
          for (int e = 0; e < D; e += 32) {
            uint32_t o[32];
            tmem_ld32(o_at + e, o);
            tmem_wait_ld();
#pragma unroll
            for (int q = 0; q < 32; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * keep);
            tmem_st32(o_at + e, o);
          }
        }
#pragma unroll
        for (int e = 0; e < KT / 2; e += 32) tmem_st32(p_at + e, *reinterpret_cast<const uint32_t(*)[32]>(v + e));
        tmem_wait_st();
      }
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[s]);
    }
    if (!ok && lane == 0) fail();
  }
  __syncthreads();
  __syncthreads();  // every MMA has completed
  tmem_fence_after();

  // ---- the part's sums
  const bool good = !stopped();
  float o[D];
  if (mine > 0 && good) {
#pragma unroll
    for (int e = 0; e < D; e += 32) {
      uint32_t v[32];
      tmem_ld32(tmem + lanes + Shape::kAtO + s * D + e, v);
      tmem_wait_ld();
#pragma unroll
      for (int q = 0; q < 32; ++q) o[e + q] = __uint_as_float(v[q]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < D; ++e) o[e] = 0.f;
  }
  if (!good) l = __uint_as_float(0x7fc00000u);
  tmem_fence_before();
  __syncthreads();
  if (!PAIR) {  // stream 1's sums join stream 0's
    float* so = reinterpret_cast<float*>(ring) + row * (D + 4);
    if (s == 1) {
#pragma unroll
      for (int e = 0; e < D; e += 4) *reinterpret_cast<float4*>(so + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      so[D] = m;
      so[D + 1] = l;
    }
    __syncthreads();
    if (s == 0) {
      const float om = so[D], ol = so[D + 1], top = fmaxf(m, om);
      const float f0 = m == -INFINITY ? 0.f : exp2f(m - top), f1 = om == -INFINITY ? 0.f : exp2f(om - top);
      l = (m == -INFINITY ? l : l * f0) + (om == -INFINITY ? ol : ol * f1);
      if (f1 != 0.f) {
#pragma unroll
        for (int e = 0; e < D; ++e) o[e] = fmaf(so[e], f1, o[e] * f0);
      }
      m = top;
    }
    if (s != 0) return;
  }
  if (x >= queries) return;
  const int r = x / group, h = g * group + x % group;
  if (t.part_o == nullptr) {
    store_out<T>(a, r, h, 0, o, l, m, true);
    return;
  }
  const size_t dst = ((size_t)part * a.rows + r) * a.heads + h;
  t.part_ml[dst] = make_float2(m, l);
  if (m != -INFINITY) {
    float4* po = reinterpret_cast<float4*>(t.part_o + dst * D);
#pragma unroll
    for (int e = 0; e < D; e += 4) po[e / 4] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
  }
}

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t s, bool pdl, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// Allow a kernel its dynamic shared memory, once per device.
template <typename Kernel>
cudaError_t allow_smem(Kernel* kernel, int smem, std::atomic<bool> (&done)[64]) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device < 64 && done[device].load(std::memory_order_acquire)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess)  // every kernel of a call wants the same split of an SM's memory
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess && device < 64) done[device].store(true, std::memory_order_release);
  return e;
}

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// Shared K or V as a 3-D tensor of boxes of 64 channels x one tile's tokens x 1 head; tokens past the last
// read as zeros.  The axis with the smaller stride comes first.
bool encode_shared(CUtensorMap* map, const SharedAttnArgs& a, const void* p, int64_t token, int64_t head, bool token_last) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = map_encoder();
  if (!enc) return false;
  const cuuint64_t tokens = (cuuint64_t)a.shared_tokens, heads = (cuuint64_t)a.kv_heads;
  const cuuint64_t row = (cuuint64_t)token * 2, one = (cuuint64_t)(a.kv_heads == 1 ? token : head) * 2;
  cuuint64_t dims[3] = {(cuuint64_t)a.dim, token_last ? heads : tokens, token_last ? tokens : heads};
  cuuint64_t strides[2] = {token_last ? one : row, token_last ? row : one};
  cuuint32_t box[3] = {64, token_last ? 1u : (cuuint32_t)KT, token_last ? (cuuint32_t)KT : 1u};
  cuuint32_t each[3] = {1, 1, 1};
  const CUtensorMapDataType type =
      a.dtype == S2R_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(map, type, 3, const_cast<void*>(p), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A pool of own K or V as rows of `dim` channels, read in boxes of 64 channels x `tokens`.
bool encode_pool(CUtensorMap* map, const SharedAttnArgs& a, const void* p, int tokens) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = map_encoder();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)a.dim, (cuuint64_t)a.own_pages * a.kv_heads * kPageTokens};
  cuuint64_t strides[1] = {(cuuint64_t)a.dim * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)tokens};
  cuuint32_t each[2] = {1, 1};
  const CUtensorMapDataType type =
      a.dtype == S2R_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(map, type, 2, const_cast<void*>(p), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int query_tiles(const SharedAttnArgs& a) { return (a.rows * (a.heads / a.kv_heads) + kTileRows - 1) / kTileRows; }

template <typename T, int D, bool PAIR>
cudaError_t launch_tiles(const SharedAttnArgs& a, float* part_o, float2* part_ml, cudaStream_t s, bool pdl) {
  CUtensorMap map_k, map_v;
  TileArgs t{};
  t.a = a;
  t.part_o = part_o;
  t.part_ml = part_ml;
  t.token_last = a.kv_heads > 1 && a.k_head < a.k_token && a.v_head < a.v_token;
  t.q_vector = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_row % 8 == 0 && a.q_head % 8 == 0;
  if (!encode_shared(&map_k, a, a.shared_k, a.k_token, a.k_head, t.token_last) ||
      !encode_shared(&map_v, a, a.shared_v, a.v_token, a.v_head, t.token_last))
    return cudaErrorInvalidValue;
  auto* kernel = shared_tile_kernel<T, D, PAIR>;
  constexpr int smem = Tile<D, PAIR>::kBytes;
  static std::atomic<bool> done[64];
  const cudaError_t e = allow_smem(kernel, smem, done);
  if (e != cudaSuccess) return e;
  return launch(kernel, dim3(a.query_blocks, a.kv_heads, a.shared_splits), kTileThreads, smem, s, pdl, map_k, map_v, t);
}

template <typename T, int D, bool WIDE>
cudaError_t launch_own(const SharedAttnArgs& a, float* o, float2* ml, cudaStream_t s, bool pdl) {
  CUtensorMap map_k, map_v, map_k_piece, map_v_piece;
  constexpr int kTokens = kOwnStage / (4 * D);
  if (!encode_pool(&map_k, a, a.own_k, kTokens) || !encode_pool(&map_v, a, a.own_v, kTokens) ||
      !encode_pool(&map_k_piece, a, a.own_k, kOwnPiece) || !encode_pool(&map_v_piece, a, a.own_v, kOwnPiece))
    return cudaErrorInvalidValue;
  const bool q_pairs = reinterpret_cast<uintptr_t>(a.q) % 4 == 0 && a.q_row % 2 == 0 && a.q_head % 2 == 0;
  auto* kernel = own_attn_kernel<T, D, WIDE>;
  static std::atomic<bool> done[64];
  const cudaError_t e = allow_smem(kernel, kOwnSmem, done);
  if (e != cudaSuccess) return e;
  const long long group = a.heads / a.kv_heads, queries = WIDE ? 16 : 8;
  const long long units = (long long)a.rows * a.kv_heads * ((group + queries - 1) / queries) * a.own_splits;
  // a warp takes one unit of long rows (the hardware evens out their lengths; a persistent grid with
  // units dealt in turn was a quarter slower), or several of short ones, 16 chunks' room in all, as
  // long as that leaves six warps an SM
  const long long room = std::max<long long>(1, (long long)a.pages_per_row * (kPageTokens / kTokens) / a.own_splits);
  const long long each = std::max<long long>(1, std::min<long long>(16 / room, units / (6 * 148))) * kOwnWarps;
  const dim3 grid((unsigned)((units + each - 1) / each));
  return launch(kernel, grid, kOwnThreads, kOwnSmem, s, pdl, map_k, map_v, map_k_piece, map_v_piece, a, q_pairs, o, ml,
                a.shared_splits);
}

template <typename T, int D>
cudaError_t launch_all(const SharedAttnArgs& a, cudaStream_t s) {
  const int parts = a.shared_splits + a.own_splits;
  const size_t pairs = (size_t)a.rows * a.heads;
  const bool join = parts != 1 || a.own_splits;
  float2* ml = static_cast<float2*>(a.workspace);
  float* o = reinterpret_cast<float*>(ml + (parts * pairs + 1) / 2 * 2);
  cudaError_t e = cudaSuccess;
  if (a.shared_splits)
    e = a.pair ? launch_tiles<T, D, true>(a, join ? o : nullptr, ml, s, a.pdl)
               : launch_tiles<T, D, false>(a, join ? o : nullptr, ml, s, a.pdl);
  // beside the shared part, which reads nothing the own part writes
  if (e == cudaSuccess && a.own_splits)
    e = a.heads / a.kv_heads > 8 ? launch_own<T, D, true>(a, o, ml, s, a.shared_splits > 0)
                                 : launch_own<T, D, false>(a, o, ml, s, a.shared_splits > 0);
  if (e == cudaSuccess && join)
    e = launch(join_kernel<T, D>, dim3((unsigned)((pairs + 3) / 4)), 128, 0, s, parts > 0, a, o, ml, parts);
  return e;
}

}  // namespace

size_t plan_shared_attn(SharedAttnArgs& a, int sms) {
  const size_t pairs = (size_t)a.rows * a.heads;
  a.shared_splits = a.own_splits = 0;
  a.out_vector = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_row % 8 == 0 && a.out_head % 8 == 0;
  if (a.shared_tokens > 0) {
    const int tiles = query_tiles(a), keys = (a.shared_tokens + KT - 1) / KT;
    a.pair = tiles > 1;
    // the split with the fewest key tiles one after the other: waves of CTAs times the tiles of
    // each, plus about 6 tiles' time to start and end it
    a.query_blocks = a.pair ? (tiles + 1) / 2 : tiles;
    const long long ctas = (long long)a.query_blocks * a.kv_heads;
    // Dim 64 runs two CTAs on an SM; a short shared part beside own pages takes one, or at dim 128, whose CTA
    // fills an SM, half of the SMs: the own part's warps have room from the start.  (Dim 64, 64 rows x 16 heads,
    // own rows of up to 1,500: over 2,048 shared tokens 54 -> 50 us, 8,192 57.4 -> 56.3, but 16,384 65.6 -> 67.9.
    // Dim 128, 100 rows x 32/8 heads, own rows of up to 2,500, over 1,111 tokens 123 -> 114 us, 4,000 125 -> 120,
    // 32 rows 61 -> 52, own rows of up to 300 43 -> 40.)
    const bool brief = a.own_k && ctas * keys <= 16ll * sms;
    const long long slots = a.dim == 64 ? (brief ? sms : 2ll * sms) : (brief ? std::max(1, sms / 2) : sms);
    long long best = -1;
    for (int sp = 1; sp <= keys && sp <= kMaxSharedSplits; ++sp) {
      int per = (keys + sp - 1) / sp;
      if ((keys + per - 1) / per != sp) continue;  // the same tiles in fewer parts
      long long cost = (ctas * sp + slots - 1) / slots * (per + 6);
      const long long room = slots - ctas * (sp - 1);
      if (a.dim == 64 && per >= 48 && sp > 1 && room > 0 && room < ctas) {
        // all but the last parts fill most of one wave: shorter last parts, `rounds` of them one after the
        // other in what room is left, so that both end together (dim 64, 1,024 rows x 16 heads over 16,384
        // tokens 126 -> 120 us; dim 128, where a CTA starts on an SM by itself, over 8,192 103 -> 116)
        const long long rounds = (ctas + room - 1) / room;
        const long long last = (keys + 6ll * (sp - 1) * (1 - rounds)) / (rounds * (sp - 1) + 1);
        if (last > 0) {
          const int most = (int)((keys - last + sp - 2) / (sp - 1));
          const long long rest = keys - (long long)most * (sp - 1), even = std::max(most + 6ll, rounds * (rest + 6));
          if (rest > 0 && rest <= most && even < cost) {
            cost = even;
            per = most;
          }
        }
      }
      if (best < 0 || cost < best) {
        best = cost;
        a.shared_splits = sp;
        a.part_tiles = per;
      }
    }
  }
  if (a.own_k) {
    // Six warps an SM, two units for each, of four chunks or more (64 rows x 16 heads of dim 64, own rows of up
    // to 400: one part of 7 pages 25 us, two 28); two pages do while most warps would stay idle (4 rows of
    // 500: 2 pages a part 13.3 us, 4 pages 14.3).
    const int group = a.heads / a.kv_heads, queries = group > 8 ? 16 : 8;
    const long long pieces = (long long)a.rows * a.kv_heads * ((group + queries - 1) / queries);
    const int chunks = a.pages_per_row * (a.dim / 64);
    int sp = 1;
    while (sp < kMaxOwnSplits && pieces * sp < 12ll * sms && chunks / (sp * 2) >= (pieces * sp < 3ll * sms ? a.dim / 32 : 4)) sp *= 2;
    a.own_splits = sp;
  }
  const size_t parts = a.shared_splits + a.own_splits;
  if (parts == 0 || (parts == 1 && !a.own_splits)) return 0;
  return (parts * pairs + 1) / 2 * 16 + parts * pairs * a.dim * sizeof(float);
}

int launch_shared_attn(const SharedAttnArgs& a, cudaStream_t s, const char** why) {
  *why = "launch failed";
  cudaError_t e;
  if (a.dtype == S2R_BF16)
    e = a.dim == 64 ? launch_all<bf16, 64>(a, s) : launch_all<bf16, 128>(a, s);
  else
    e = a.dim == 64 ? launch_all<__half, 64>(a, s) : launch_all<__half, 128>(a, s);
  return e == cudaSuccess ? S2R_OK : S2R_ECUDA;
}

}  // namespace s2r

// Records `msg` as s2r_last_error() of this thread (defined with the engine).
__attribute__((visibility("hidden"))) int s2r_record_error(int code, const char* msg);

namespace {

int shared_fail(int code, const char* what) {
  char msg[160];
  snprintf(msg, sizeof(msg), "s2r_shared_attention: %s", what);
  return s2r_record_error(code, msg);
}

// Check the arguments and turn them into a planned launch; `bytes` is its workspace.
int prepare(const s2r_shared_attention_args* in, s2r::SharedAttnArgs& a, size_t* bytes) {
  auto bad = [](const char* what) { return shared_fail(S2R_EINVAL, what); };
  if (!in) return bad("NULL arguments");
  if (in->dtype != S2R_BF16 && in->dtype != S2R_F16) return bad("tensors must be bfloat16 or float16");
  if (in->head_dim != 64 && in->head_dim != 128) return shared_fail(S2R_ENOTSUP, "head_dim must be 64 or 128");
  if (in->rows < 1 || in->heads < 1 || in->kv_heads < 1 || in->shared_tokens < 0)
    return bad("rows, heads and kv_heads must be >= 1, shared_tokens >= 0");
  if (in->rows > 65535) return bad("at most 65535 rows a call");
  if ((int64_t)in->rows * in->heads > (1 << 24)) return bad("at most 2^24 rows x heads a call");
  if (in->heads % in->kv_heads || in->heads > 4096) return bad("heads must be a multiple of kv_heads, at most 4096");
  if (in->shared_tokens > (1 << 28)) return bad("at most 2^28 shared tokens");
  if (!in->q || !in->out) return bad("q or out is NULL");
  if (!(in->scale > 0.f) || in->scale > 1e30f) return bad("scale must be positive and finite");
  // the stride of an axis of one entry says nothing
  s2r_shared_attention_args given = *in;
  if (given.rows == 1) given.q_row_stride = given.out_row_stride = given.page_table_stride = 0;
  if (given.heads == 1) given.q_head_stride = given.out_head_stride = 0;
  if (given.kv_heads == 1) given.k_head_stride = given.v_head_stride = 0;
  if (given.shared_tokens <= 1) given.k_token_stride = given.v_token_stride = given.head_dim;
  in = &given;
  const int64_t widest = (int64_t)1 << 38;
  const int64_t strides[] = {in->q_row_stride,     in->q_head_stride,   in->k_token_stride, in->k_head_stride,
                             in->v_token_stride,   in->v_head_stride,   in->out_row_stride, in->out_head_stride,
                             in->page_table_stride};
  for (int64_t s : strides)
    if (s < 0 || s > widest) return bad("strides must be between 0 and 2^38 elements");
  // two (row, head) of out share no element if the longer stride steps over all the shorter one spans
  const int64_t rows_apart = (in->heads - 1) * in->out_head_stride + in->head_dim;
  const int64_t heads_apart = (in->rows - 1) * in->out_row_stride + in->head_dim;
  if ((in->rows > 1 && in->out_row_stride < in->head_dim) || (in->heads > 1 && in->out_head_stride < in->head_dim) ||
      (in->rows > 1 && in->heads > 1 && in->out_row_stride < rows_apart && in->out_head_stride < heads_apart))
    return bad("rows or heads of out overlap");
  auto off = [](const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; };
  if (off(in->q, 2) || off(in->out, 2) || off(in->lse, 4) || off(in->shared_len, 4) || off(in->page_table, 4) ||
      off(in->own_len, 4) || off(in->error, 4))
    return bad("a pointer is not aligned to its type");
  if (in->shared_tokens) {
    if (!in->shared_k || !in->shared_v) return bad("shared_k or shared_v is NULL");
    // K and V are fetched in 16-byte pieces
    if (reinterpret_cast<uintptr_t>(in->shared_k) % 16 || reinterpret_cast<uintptr_t>(in->shared_v) % 16 ||
        in->k_token_stride % 8 || in->k_head_stride % 8 || in->v_token_stride % 8 || in->v_head_stride % 8)
      return bad("shared_k and shared_v must be 16-byte aligned with strides that are multiples of 8 elements");
    if (in->shared_tokens > 1 && (in->k_token_stride < in->head_dim || in->v_token_stride < in->head_dim))
      return bad("shared tokens overlap (token stride below head_dim)");
    if (in->kv_heads > 1 && (in->k_head_stride < in->head_dim || in->v_head_stride < in->head_dim))
      return bad("shared heads overlap (head stride below head_dim)");
  }
  const bool own = in->own_k || in->own_v || in->page_table || in->own_len;
  if (own) {
    if (!in->own_k || !in->own_v || !in->page_table || !in->own_len)
      return bad("own_k, own_v, page_table and own_len go together");
    if (in->own_pages < 1 || in->pages_per_row < 1) return bad("own_pages and pages_per_row must be >= 1");
    if (in->pages_per_row > (1 << 22)) return bad("at most 2^22 pages a row");
    if ((int64_t)in->own_pages * in->kv_heads >= (1 << 25)) return bad("own_pages x kv_heads must be below 2^25");
    if (in->rows > 1 && in->page_table_stride < in->pages_per_row && in->page_table_stride != 0)
      return bad("page table rows overlap");
    if (reinterpret_cast<uintptr_t>(in->own_k) % 16 || reinterpret_cast<uintptr_t>(in->own_v) % 16)
      return bad("own_k and own_v must be 16-byte aligned");
  }
  a.dtype = in->dtype;
  a.rows = in->rows;
  a.heads = in->heads;
  a.kv_heads = in->kv_heads;
  a.dim = in->head_dim;
  a.scale = in->scale;
  a.q = in->q;
  a.q_row = in->q_row_stride;
  a.q_head = in->q_head_stride;
  a.shared_k = in->shared_k;
  a.shared_v = in->shared_v;
  a.k_token = in->k_token_stride;
  a.k_head = in->k_head_stride;
  a.v_token = in->v_token_stride;
  a.v_head = in->v_head_stride;
  a.shared_tokens = in->shared_tokens;
  a.shared_len = in->shared_len;
  a.own_k = own ? in->own_k : nullptr;
  a.own_v = in->own_v;
  a.own_pages = in->own_pages;
  a.page_table = in->page_table;
  a.page_stride = in->page_table_stride;
  a.pages_per_row = in->pages_per_row;
  a.own_len = in->own_len;
  a.out = in->out;
  a.out_row = in->out_row_stride;
  a.out_head = in->out_head_stride;
  a.lse = in->lse;
  a.workspace = in->workspace;
  a.error = in->error;
  static std::atomic<int> sms[64];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64)
    return shared_fail(S2R_ECUDA, "no usable current device");
  int n = sms[device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
      return shared_fail(S2R_ECUDA, "no usable current device");
    sms[device].store(n, std::memory_order_relaxed);
  }
  *bytes = s2r::plan_shared_attn(a, n);
  return S2R_OK;
}

}  // namespace

extern "C" int32_t s2r_shared_attention_workspace(const s2r_shared_attention_args* in, int64_t* bytes) {
  s2r::SharedAttnArgs a{};
  size_t need = 0;
  if (!bytes) return shared_fail(S2R_EINVAL, "bytes is NULL");
  const int rc = prepare(in, a, &need);
  if (rc == S2R_OK) *bytes = (int64_t)need;
  return rc;
}

extern "C" int32_t s2r_shared_attention(const s2r_shared_attention_args* in, void* stream) {
  s2r::SharedAttnArgs a{};
  size_t need = 0;
  const int rc = prepare(in, a, &need);
  if (rc != S2R_OK) return rc;
  if (need && (!in->workspace || reinterpret_cast<uintptr_t>(in->workspace) % 16 || in->workspace_bytes < (int64_t)need)) {
    char msg[160];
    snprintf(msg, sizeof(msg), "s2r_shared_attention: needs a 16-byte aligned workspace of %zu bytes, got %lld", need,
             (long long)(in->workspace ? in->workspace_bytes : 0));
    return s2r_record_error(S2R_EINVAL, msg);
  }
  const char* why = "";
  const int code = s2r::launch_shared_attn(a, static_cast<cudaStream_t>(stream), &why);
  if (code != S2R_OK) {
    char msg[160];
    snprintf(msg, sizeof(msg), "s2r_shared_attention: %s (%s)", why, cudaGetErrorString(cudaGetLastError()));
    return s2r_record_error(code, msg);
  }
  return S2R_OK;
}
