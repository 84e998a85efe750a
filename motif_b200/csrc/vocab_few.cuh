// The vocabulary loss of a few fp32 tokens (vocab_few.cu), as the entry points of vocab_loss.cu call it.
#pragma once

#include "common.cuh"

namespace mb {

struct FewCall {
  const float *x, *w;
  int64_t xs, ws;
  const int64_t* labels;
  int64_t ignore, N, V, d;
  int reduction;
  float* loss;
  unsigned char *state, *work;  // work: the pass's own scratch
  const float* up;              // backward: null for 1
  int64_t up_stride;
  float *dx, *dw;
  cudaStream_t st;
};

// Whether these kernels take a call of these sizes.
bool few_tokens(int64_t N, int64_t d, int dtype);
// Bytes of what the forward pass leaves, and of each pass's scratch.
void few_sizes(int64_t N, int64_t V, int64_t d, int64_t* state, int64_t* forward, int64_t* backward);
int few_forward(const FewCall& c);
int few_backward(const FewCall& c);

}  // namespace mb
