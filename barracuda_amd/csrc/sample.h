// sample.h -- the choice of tokens from rows of logits (sample.hip) as its launcher sees it.
#pragma once
#include "bch_internal.h"

namespace bch {

struct SampleRule {
  float temperature;
  int top_k;
  float top_p, min_p;
};
struct SampleCall {
  int vocab, unit_log;  // unit_log: sample_unit_log(vocab)
  long long stride;
  SampleRule rule;          // every row's, unless
  const SampleRule* rules;  // a rule for each row
  const float *logits, *u;
  int* tokens;
  float* probs;  // or null
};
int sample_unit_log(int vocab);
hipError_t launch_sample(hipStream_t s, const SampleCall& call, int rows, void* ws, size_t ws_bytes);
size_t sample_workspace_bytes(const SampleCall& call, int rows);  // with less it runs slower

}  // namespace bch
