// Launchers of the operators on vocabulary rows (validated arguments; the
// C entry points are in vocab_api.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace hkb {

struct VocabRows {
  int64_t rows;
  int vocab;
  int dtype;  // hkb_dtype
  const void* logits;
  int64_t row_stride;  // elements
};

struct SampleArgs {
  const float* temperatures;  // [N] or null: temperature
  const int32_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  float temperature;
  int32_t top_k;
  float top_p;
  float min_p;
  const void* uniforms;  // [N] f32 or f64
  int uniforms_f64;
  int32_t* tokens;
  float* log_probs;
  int32_t* kept;
};
cudaError_t launch_sample_tokens(cudaStream_t st, const VocabRows& r, const SampleArgs& a);

struct TopArgs {
  int k;
  double inv_temperature;
  float c;           // log2(e) / temperature
  void* values;      // [N,k], the logits' type
  int32_t* tokens;   // [N,k]
  float* log_norm;   // [N] or null
};
cudaError_t launch_top_logits(cudaStream_t st, const VocabRows& r, const TopArgs& a);

struct DistillArgs {
  int k;
  int teacher_dtype;
  const void* values;    // [N,k]
  const int32_t* tokens; // [N,k]
  const float* log_norm; // [N] or null
  double temperature, inv_temperature;
  float c;               // log2(e) / temperature
  float* loss;           // [N] or null
  void* grad;            // [N, vocab] or null
  int64_t grad_row_stride;
  const float* row_weights;
  int64_t row_weight_stride;
  double* stats;         // [N, HKB_DISTILL_STATS] or null
};
cudaError_t launch_distill(cudaStream_t st, const VocabRows& r, const DistillArgs& a);
cudaError_t launch_distill_backward(cudaStream_t st, const VocabRows& r, const DistillArgs& a);

// Launch shape of the row kernels: CTAs per row, threads and elements per CTA.
struct RowShape {
  int cluster;
  int threads;
  int chunk;       // elements of a slice, a multiple of 16 bytes
  size_t smem;     // bytes of a slice's buffer
};
RowShape row_shape(int64_t rows, int vocab, int elem_bytes);

}  // namespace hkb
