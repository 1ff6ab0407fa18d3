// Launch interface of the shared-window attention (shared_attn.cu), used by
// the C entry point and by the engine's shared-window cross attention.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace s2r {

constexpr int kErrOwnPage = 11;    // a page of a row's own K/V outside the pool
constexpr int kErrOwnLength = 12;  // a row longer than its page table
constexpr int kErrSharedWait = 13;  // a wait of the shared part timed out
constexpr int kMaxSharedSplits = 64;
constexpr int kMaxOwnSplits = 32;

struct SharedAttnArgs {
  int dtype;  // s2r_dtype: bf16 or f16
  int rows, heads, kv_heads, dim;
  float scale;
  const void* q;  // [rows, heads, dim], strides in elements
  int64_t q_row, q_head;
  const void *shared_k, *shared_v;  // [tokens, kv_heads, dim]
  int64_t k_token, k_head, v_token, v_head;
  int shared_tokens;
  const int32_t* shared_len;  // null, or the device's count of live shared tokens (<= shared_tokens)
  const void *own_k, *own_v;  // [own_pages][kv_heads][64][dim]
  int own_pages;
  const int32_t* page_table;  // [rows, pages_per_row], row stride page_stride
  int64_t page_stride;
  int pages_per_row;
  const int32_t* own_len;  // [rows]
  void* out;               // [rows, heads, dim]
  int64_t out_row, out_head;
  float* lse;  // [rows, heads] or null
  void* workspace;
  int* error;  // null, or set to kErrOwn* when a row's pages are broken
  // set by plan_shared_attn
  int shared_splits, own_splits;  // parts of a (row, head)'s keys
  int part_tiles;                 // key tiles of a shared part (the last has what is left)
  int query_blocks;               // CTAs that a part's queries take
  bool pair;                      // two query tiles a CTA
  bool out_vector;                // out can be written 16 bytes at a time
  bool pdl;                       // the first launch may start while the kernel before it drains (it waits itself)
};

// Choose the splits for `sms` SMs and return the workspace bytes the launch needs.
size_t plan_shared_attn(SharedAttnArgs& a, int sms);
// Queue the kernels of a planned call on `stream` of the current device; an s2r_status, and on failure why.
int launch_shared_attn(const SharedAttnArgs& a, cudaStream_t stream, const char** why);

}  // namespace s2r
