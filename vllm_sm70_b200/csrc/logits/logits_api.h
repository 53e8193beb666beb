// Host API of the kernels over rows of logits: log-probabilities of given
// tokens (token_logprobs.cu) and distillation from a teacher's top values
// (distill.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace b200 {

constexpr int kMaxTopN = 64;       // alternatives a row (token_logprobs)
constexpr int kMaxTeacherK = 128;  // teacher values a row (distill_loss)
constexpr int kMaxVocab = 1 << 22;

// Rows of logits [rows, V], bf16 or fp32, unit inner stride, `ld` elements
// between rows.
struct LogitRows {
  const void* x;
  bool bf16;
  int64_t rows, ld;
  int V;
};

struct TokenLogprobsArgs {
  LogitRows in;
  const void* ids;  // int32 or int64 [rows]; outside [0, V): no token
  bool ids64;
  int top_n;
  float temperature;
  float* logprob;   // [rows]
  int* rank;        // [rows]
  float* entropy;   // [rows]
  float* lse;       // [rows]
  int* top_ids;     // [rows, top_n]
  float* top_lp;    // [rows, top_n]
  float* stats;     // [rows, 4] for the backward pass: m, 1 / s, log2 s, entropy
};
void token_logprobs_launch(const TokenLogprobsArgs& a, cudaStream_t stream);

struct TokenLogprobsBwdArgs {
  LogitRows in;
  const void* ids;
  bool ids64;
  float temperature;
  const float* stats;      // of the forward pass
  const float* g_logprob;  // [rows] or nullptr
  const float* g_entropy;  // [rows] or nullptr
  void* grad;              // [rows, V] contiguous, type of the logits
};
void token_logprobs_bwd_launch(const TokenLogprobsBwdArgs& a, cudaStream_t stream);

struct DistillArgs {
  LogitRows in;
  const int* t_ids;    // [rows, K]; outside [0, V): absent
  const float* t_lp;   // [rows, K]
  int K;
  const float* weights;  // [rows] or nullptr (1)
  float temperature;
  bool tail;
  float grad_scale;    // dL/d(row loss * weight): 1 (sum) or 1 / rows (mean)
  float* row_loss;     // [rows], times weight
  float* stats;        // [rows, 8] for distill_bwd: Numbers of distill.cu
  void* grad;          // [rows, V] contiguous or nullptr (forward only)
  int* counter;        // one int of scratch, with grad
  float* loss;         // scalar: grad_scale * sum(row_loss), or nullptr
};
void distill_launch(const DistillArgs& a, cudaStream_t stream);

struct DistillBwdArgs {
  LogitRows in;
  const int* t_ids;
  const float* t_lp;
  int K;
  const float* weights;   // [rows] or nullptr
  float temperature;
  bool tail;
  const float* stats;     // of the forward pass
  const float* g_rows;    // upstream gradient: [rows], or one value for all rows
  int g_stride;           // 1, or 0 for one value
  float g_scale;          // times the upstream gradient
  bool unless_one;        // one value that is 1: grad stays as it is
  void* grad;
};
void distill_bwd_launch(const DistillBwdArgs& a, cudaStream_t stream);

}  // namespace b200
