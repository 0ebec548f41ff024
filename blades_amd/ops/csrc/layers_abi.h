// What the kernels of the batch-independent layers (groupnorm_{fwd,bwd}.hip, dropout.hip, rope.hip) and their autograd nodes
// (autograd.cpp, another library, which reaches them by address) agree on: plans and entry points.  Both sides include this,
// so neither compiles against another's idea of them; the sources say what the arguments mean.
#pragma once
#include <hip/hip_runtime_api.h>

namespace groupnorm { struct Layer; }
namespace rope { struct RopePlan; }

// What a dropout layer's shape and key fix.  dtype 0 fp32, 1 bf16, 2 fp16.  kind 0 element, 1 channel, 2 sample.  last:
// channels-last maps, else contiguous [.., C, HW].  inner: [B][Kc][C] instead of [Kc][B][C] in the leading dimensions.  least:
// smallest 24-bit draw that is kept, below 2^24.
struct DropPlan {
  long B, C, HW;
  unsigned long long seed;
  int Kc, kind, inner, last, dtype;
  unsigned c3, least;
  float scale;
};

extern "C" {
long blades_group_norm_plan_size();
int blades_group_norm_plan(groupnorm::Layer* p, long N, long P, int C, int G, float eps, int act, int per_client, long gstride,
                           long bstride, int dtype, int vec, long* ws);
int blades_group_norm_forward(const void* x, const void* res, const float* gamma, const float* beta, void* y, void* gate,
                              float* stats, float* ws, const groupnorm::Layer* p, hipStream_t st);
int blades_group_norm_backward(const void* x, const void* res, const void* gy, const void* gate, const float* gamma,
                               const float* beta, const float* stats, void* dx, void* dres, const float* coef, float* dgamma,
                               float* dbeta, long ld, int accumulate, float* ws, const groupnorm::Layer* p, hipStream_t st);
long blades_client_dropout_plan_size();
int blades_client_dropout(const void* x, void* y, const long* uids, const long* tag, long tag_value, const DropPlan* p,
                          hipStream_t st);
long blades_rope_plan_size();
int blades_rope_plan(rope::RopePlan* p, int pos_float, long psr, long R, long N, int S, int H, int D, long sr, long sn, long ss,
                     long sh, int rot, const int* axes, int A, double base, int dtype, int vec);
int blades_rope_axes(const void* x, void* y, const void* pos, const rope::RopePlan* p, int inverse, hipStream_t st);
}
