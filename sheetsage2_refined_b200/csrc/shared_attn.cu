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
// m in units of log2.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdio>
#include <mutex>

#include "../../include/s2r.h"
#include "common.cuh"
#include "shared_attn.cuh"

namespace s2r {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float2 pair_to_float(bf16, uint32_t v) { return make_float2(bf_lo(v), bf_hi(v)); }
__device__ __forceinline__ float2 pair_to_float(__half, uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
// The 8 elements at p (16-byte aligned) as floats.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 v = ld_stream(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = pair_to_float(T(), w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

constexpr int kOwnThreads = 128;
constexpr int kOwnWarps = kOwnThreads / 32;
constexpr int kOwnUnroll = 4;  // key rows a lane group keeps in flight

// One part of one row's keys for GC query heads of one kv head.  A key row is
// read by D / 8 lanes, 16 bytes each; every such lane group keeps its own
// online softmax over the keys it sees.
template <typename T, int D, int GC, bool PAGED>
__global__ void __launch_bounds__(kOwnThreads) row_attn_kernel(const __grid_constant__ SharedAttnArgs a, float* part_o,
                                                               float2* part_ml, int first_part) {
  constexpr int kLanes = D / 8, kGroups = 32 / kLanes;  // lanes of a key row, key rows of a warp
  const int part = blockIdx.x, splits = gridDim.x;
  const int group = a.heads / a.kv_heads, chunks = (group + GC - 1) / GC;
  const int g = blockIdx.y / chunks, h0 = g * group + (blockIdx.y % chunks) * GC;
  const int heads = min(GC, (g + 1) * group - h0);
  const int r = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / kLanes, at = (lane % kLanes) * 8;
  __shared__ float so[kOwnWarps][GC][D];
  __shared__ float2 sml[kOwnWarps][GC];

  bool broken = false;
  int n;
  if (PAGED) {
    n = a.own_len[r];
    if (n > a.pages_per_row * kPageTokens) {
      broken = true;
      if (threadIdx.x == 0 && a.error) atomicExch(a.error, kErrOwnLength);
    }
    n = broken || n < 0 ? 0 : n;
  } else {
    n = a.shared_len ? min(max(*a.shared_len, 0), a.shared_tokens) : a.shared_tokens;
  }
  const int pages = (n + kPageTokens - 1) / kPageTokens, per = (pages + splits - 1) / splits;
  const int p0 = min(pages, part * per), p1 = min(pages, p0 + per);

  float q[GC][8], o[GC][8], m[GC], l[GC];
#pragma unroll
  for (int i = 0; i < GC; ++i) {
    const T* src = static_cast<const T*>(a.q) + r * a.q_row + (h0 + min(i, heads - 1)) * a.q_head + at;
#pragma unroll
    for (int e = 0; e < 8; ++e) q[i][e] = (float)src[e] * (a.scale * kLog2e);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[i][e] = 0.f;
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
  for (int p = p0 + warp; p < p1; p += kOwnWarps) {
    const T *k, *v;
    int64_t k_step = D, v_step = D;
    if (PAGED) {
      const int page = a.page_table[r * a.page_stride + p];
      if (page < 0 || page >= a.own_pages) {
        broken = true;
        if (lane == 0 && a.error) atomicExch(a.error, kErrOwnPage);
        continue;
      }
      const size_t base = ((size_t)page * a.kv_heads + g) * (kPageTokens * D);
      k = static_cast<const T*>(a.own_k) + base;
      v = static_cast<const T*>(a.own_v) + base;
    } else {
      k_step = a.k_token;
      v_step = a.v_token;
      k = static_cast<const T*>(a.shared_k) + g * a.k_head + (int64_t)p * kPageTokens * k_step;
      v = static_cast<const T*>(a.shared_v) + g * a.v_head + (int64_t)p * kPageTokens * v_step;
    }
    const int live = min(kPageTokens, n - p * kPageTokens);
#pragma unroll 1
    for (int t0 = 0; t0 < live; t0 += kGroups * kOwnUnroll) {
      float kx[kOwnUnroll][8], vx[kOwnUnroll][8];
#pragma unroll
      for (int u = 0; u < kOwnUnroll; ++u) {
        const int t = t0 + u * kGroups + sub;
        if (t < live) {
          load8(k + t * k_step + at, kx[u]);
          load8(v + t * v_step + at, vx[u]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) kx[u][e] = vx[u][e] = 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < GC; ++i) {
        float s[kOwnUnroll], top = m[i];
#pragma unroll
        for (int u = 0; u < kOwnUnroll; ++u) {
          s[u] = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) s[u] = fmaf(q[i][e], kx[u][e], s[u]);
#pragma unroll
          for (int x = kLanes / 2; x > 0; x >>= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], x);
          if (t0 + u * kGroups + sub >= live) s[u] = -INFINITY;
          top = fmaxf(top, s[u]);
        }
        const float keep = top == -INFINITY ? 1.f : exp2f(m[i] - top);
        l[i] *= keep;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[i][e] *= keep;
#pragma unroll
        for (int u = 0; u < kOwnUnroll; ++u) {
          const float w = s[u] == -INFINITY ? 0.f : exp2f(s[u] - top);
          l[i] += w;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[i][e] = fmaf(w, vx[u][e], o[i][e]);
        }
        m[i] = top;
      }
    }
  }
  // ---- join the lane groups, then the warps
#pragma unroll
  for (int i = 0; i < GC; ++i) {
#pragma unroll
    for (int x = kLanes; x < 32; x <<= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m[i], x), ol = __shfl_xor_sync(0xffffffffu, l[i], x);
      const float top = fmaxf(m[i], om);
      const float mine = m[i] == -INFINITY ? 0.f : exp2f(m[i] - top), other = om == -INFINITY ? 0.f : exp2f(om - top);
      l[i] = l[i] * mine + ol * other;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[i][e] = o[i][e] * mine + __shfl_xor_sync(0xffffffffu, o[i][e], x) * other;
      m[i] = top;
    }
    if (broken) l[i] = __uint_as_float(0x7fc00000u);  // a row with broken pages comes out as NaN
    if (sub == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) so[warp][i][at + e] = o[i][e];
    }
    if (lane == 0) sml[warp][i] = make_float2(m[i], l[i]);
  }
  __syncthreads();
  for (int x = threadIdx.x; x < heads * D; x += kOwnThreads) {
    const int i = x / D, e = x % D;
    float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kOwnWarps; ++w) top = fmaxf(top, sml[w][i].x);
#pragma unroll
    for (int w = 0; w < kOwnWarps; ++w) {
      const float2 ml = sml[w][i];
      const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
      sum += ml.x == -INFINITY ? ml.y : ml.y * f;  // (l of an empty part is 0, or NaN where pages are broken)
      acc = fmaf(so[w][i][e], f, acc);
    }
    const size_t dst = ((size_t)(first_part + part) * a.rows + r) * a.heads + h0 + i;
    part_o[dst * D + e] = acc;
    if (e == 0) part_ml[dst] = make_float2(top, sum);
  }
}

// Joins the parts of every (row, head): a warp each.
template <typename T, int D>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ SharedAttnArgs a, const float* part_o,
                                                   const float2* part_ml, int parts) {
  const int lane = threadIdx.x & 31;
  const int64_t pair = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), pairs = (int64_t)a.rows * a.heads;
  if (pair >= pairs) return;
  constexpr int kEach = D / 32;
  float top = -INFINITY;
  for (int p = 0; p < parts; ++p) top = fmaxf(top, part_ml[p * pairs + pair].x);
  float sum = 0.f, acc[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) acc[e] = 0.f;
  for (int p = 0; p < parts; ++p) {
    const float2 ml = part_ml[p * pairs + pair];
    const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
    sum += ml.x == -INFINITY ? ml.y : ml.y * f;
    const float* src = part_o + (size_t)(p * pairs + pair) * D + lane * kEach;
#pragma unroll
    for (int e = 0; e < kEach; ++e) acc[e] = fmaf(src[e], f, acc[e]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no key at all: 0
  const int r = (int)(pair / a.heads), h = (int)(pair % a.heads);
  T* dst = static_cast<T*>(a.out) + r * a.out_row + h * a.out_head + lane * kEach;
#pragma unroll
  for (int e = 0; e < kEach; ++e) dst[e] = T(acc[e] * inv);
  if (a.lse && lane == 0) a.lse[pair] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

template <typename T, int D, int GC>
cudaError_t launch_rows(const SharedAttnArgs& a, cudaStream_t s) {
  const int group = a.heads / a.kv_heads, chunks = (group + GC - 1) / GC, parts = a.shared_splits + a.own_splits;
  const size_t pairs = (size_t)a.rows * a.heads;
  float2* ml = static_cast<float2*>(a.workspace);
  float* o = reinterpret_cast<float*>(ml + (parts * pairs + 1) / 2 * 2);
  if (a.shared_splits)
    row_attn_kernel<T, D, GC, false><<<dim3(a.shared_splits, a.kv_heads * chunks, a.rows), kOwnThreads, 0, s>>>(a, o, ml, 0);
  if (a.own_splits)
    row_attn_kernel<T, D, GC, true><<<dim3(a.own_splits, a.kv_heads * chunks, a.rows), kOwnThreads, 0, s>>>(
        a, o, ml, a.shared_splits);
  join_kernel<T, D><<<(unsigned)((pairs + 3) / 4), 128, 0, s>>>(a, o, ml, parts);
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t launch_group(const SharedAttnArgs& a, cudaStream_t s) {
  const int group = a.heads / a.kv_heads;
  if (group == 1) return launch_rows<T, D, 1>(a, s);
  if (group == 2) return launch_rows<T, D, 2>(a, s);
  return launch_rows<T, D, 4>(a, s);
}

}  // namespace

size_t plan_shared_attn(SharedAttnArgs& a, int sms) {
  auto splits = [&](int tokens) {
    const int pages = (tokens + kPageTokens - 1) / kPageTokens;
    int sp = 1;
    while (sp < 16 && (long long)a.rows * a.kv_heads * sp < 4ll * sms && pages / (sp * 2) >= 2) sp *= 2;
    return tokens > 0 ? sp : 0;
  };
  a.shared_splits = splits(a.shared_tokens);
  a.own_splits = a.own_k ? splits(a.pages_per_row * kPageTokens) : 0;
  const size_t pairs = (size_t)a.rows * a.heads, parts = a.shared_splits + a.own_splits;
  return (parts * pairs + 1) / 2 * 16 + parts * pairs * a.dim * sizeof(float);
}

int launch_shared_attn(const SharedAttnArgs& a, cudaStream_t s, const char** why) {
  *why = "launch failed";
  cudaError_t e;
  if (a.dtype == S2R_BF16)
    e = a.dim == 64 ? launch_group<bf16, 64>(a, s) : launch_group<bf16, 128>(a, s);
  else
    e = a.dim == 64 ? launch_group<__half, 64>(a, s) : launch_group<__half, 128>(a, s);
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
  if ((in->rows > 1 && in->out_row_stride < in->head_dim) || (in->heads > 1 && in->out_head_stride < in->head_dim))
    return bad("rows or heads of out overlap");
  if (in->shared_tokens) {
    if (!in->shared_k || !in->shared_v) return bad("shared_k or shared_v is NULL");
    // K and V are fetched in 16-byte pieces
    if (reinterpret_cast<uintptr_t>(in->shared_k) % 16 || reinterpret_cast<uintptr_t>(in->shared_v) % 16 ||
        in->k_token_stride % 8 || in->k_head_stride % 8 || in->v_token_stride % 8 || in->v_head_stride % 8)
      return bad("shared_k and shared_v must be 16-byte aligned with strides that are multiples of 8 elements");
    if (in->shared_tokens > 1 && (in->k_token_stride < in->head_dim || in->v_token_stride < in->head_dim))
      return bad("shared tokens overlap (token stride below head_dim)");
  }
  const bool own = in->own_k || in->own_v || in->page_table || in->own_len;
  if (own) {
    if (!in->own_k || !in->own_v || !in->page_table || !in->own_len)
      return bad("own_k, own_v, page_table and own_len go together");
    if (in->own_pages < 1 || in->pages_per_row < 1) return bad("own_pages and pages_per_row must be >= 1");
    if (in->pages_per_row > (1 << 22)) return bad("at most 2^22 pages a row");
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
