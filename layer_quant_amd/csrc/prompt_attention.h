// What the kernels of prompt_attention.hip and prompt_attention_mfma.hip are launched with.
#pragma once

#include <math.h>

#include "prompt_spans.h"

namespace lq {

constexpr int PROMPT_ATTENTION_MAX_D = 256;

struct PromptAttention {
  View q, k, v, out;  // strides of (batch row, row, head, dim)
  Spans spans;
  int Hkv, nrep, D;
  float scale;  // log2(e) times the caller's
};

}  // namespace lq
