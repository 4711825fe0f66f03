// lora_head_core.h — the operators of include/lora_head.h as the other
// translation units of the library call them: the head of a trainer's handle
// has its own layouts of A and B, and takes the gradients in its own.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace lce {

struct HeadCore {
  const __half* W;
  const float* A;  // [d][lda]
  int lda;
  const float* B;  // layout 0: [r][V]; layout 1: pair-interleaved at kernel rank lda
  int layout;
  int d, V, r;
  float scale;
};

struct GradOut {
  float* gA;    // null: the loss alone
  float* gB;
  int layout;   // as HeadCore::layout
  float* tail;  // layout 1: [sum of losses, counted positions]
};

// Sizes already checked; return 0 or a LORA_CE_E* code with the message in *why.
size_t head_score_bytes(const HeadCore& hd, int T, int top_k);
size_t head_distill_bytes(const HeadCore& hd, int T, int K, bool grads);
int head_score_run(const HeadCore& hd, const void* H, int dtype, int T, const int32_t* tokens,
                   int top_k, float* logprob, float* entropy, int32_t* top_ids,
                   float* top_logprobs, void* ws, cudaStream_t st, const char** why);
int head_distill_run(const HeadCore& hd, const void* H, int dtype, int T, int K,
                     const int32_t* ids, const float* teacher, float tau, const float* weight,
                     float* loss, const GradOut& out, void* ws, cudaStream_t st, const char** why);

// After the sums over ranks: lh_tail on a workspace that head_distill_run has used.
int head_step_tail(const void* ws, float* tail, int* err, cudaStream_t st);

// Smallest and largest sizes (a message, or null).
const char* head_score_refuses(const HeadCore& hd, int T, int top_k);
const char* head_distill_refuses(const HeadCore& hd, int T, int K, bool grads, float tau);

}  // namespace lce
