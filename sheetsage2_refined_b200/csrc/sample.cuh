// Launch interface of the sampling kernel (sample.cu), used by the C entry
// point and by the engine's sampled step.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace s2r {

struct SampleArgs {
  const void* logits;  // [rows, vocab], row stride logits_stride (elements)
  int dtype;           // s2r_dtype
  int64_t logits_stride;
  int rows, vocab;
  const float* bias;  // [vocab] or null
  const uint8_t* allowed;
  int64_t allowed_stride;
  const float* uniforms;  // [rows]
  // per row, or null: the values below
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all;
  int top_k_all;
  float top_p_all, min_p_all;
  int64_t* tokens;  // [rows]
  float* logprobs;  // [rows] or null
  // set by launch_sample
  int chunk;       // tokens per CTA
  int scale_bits;  // fixed-point scale of the weights: 2^scale_bits
  float cut;       // tokens this many temperatures below the best weigh nothing
};

// Queue the kernel on `stream` of the current device; an s2r_status, and on failure why.
int launch_sample(SampleArgs a, cudaStream_t stream, const char** why);

}  // namespace s2r
