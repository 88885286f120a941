// Internal interface of the gradient operators (tk_grads.cu): the norm over
// many tensors, clipping by it and the sum over micro-batches.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "tk_internal.h"

namespace tk {
namespace gr {

// One tensor.  Its elements stand at positions [phase, phase + n) from `g`,
// the gradient's address rounded down to a whole unit of kUnit elements, so
// that unit u (positions kUnit*u .. kUnit*u + 7) is one aligned vector access.
// `out` is the target's address less the same `phase` elements.
constexpr int kUnit = 8;
struct GradDesc {
  const char* g;
  char* out;
  uint64_t n;
  uint64_t u_begin : 44;    // first unit of this tensor in its launch
  uint64_t phase : 4;
  uint64_t g_dtype : 4;
  uint64_t out_dtype : 4;
  uint64_t out_vec : 4;     // out's units are aligned for vector access too
  uint64_t in_place : 4;    // out is the gradient itself
};
static_assert(sizeof(GradDesc) == 32, "one descriptor is 32 bytes of kernel parameters");

// The tensors of one launch travel in the kernel's parameters, as the leaf
// tables of the step do.
constexpr int kMaxGrads = 960;
template <int CAP>
struct GradLaunch {
  uint64_t units;  // of all tensors
  int32_t n;
  int32_t reserved;
  GradDesc d[CAP];
};

struct GradList {  // host side: the descriptors of one launch
  const GradDesc* d;
  int n;
  uint64_t units;
};

// Blocks that the norm of `units` units is split over (0: no device).
int norm_blocks(uint64_t units);

// Sum of powers (or largest magnitude) of every block's share into
// partials[0..blocks); with `slots`, also block b's share of tensor i into
// slots[b + i].
int launch_norm(const GradList& l, int norm, int blocks, double* partials, double* slots,
                cudaStream_t s);
// out = out + alpha g, or alpha g; norm < 0: without the norm.
int launch_sum(const GradList& l, int norm, float alpha, bool overwrite, int blocks,
               double* partials, cudaStream_t s);
// Norm and clip scale of the partials (norm_out, scale_out may be null).
int launch_fold(int norm, const double* partials, int n, float max_norm, float* norm_out,
                float* scale_out, cudaStream_t s);
// Norm of each tensor of one launch from its slots.
int launch_fold_each(const GradList& l, int norm, int blocks, const double* slots, float* each,
                     cudaStream_t s);
// out = scale g with the scale of the partials.
int launch_clip(const GradList& l, int norm, const double* partials, int n, float max_norm,
                float* norm_out, float* scale_out, cudaStream_t s);

}  // namespace gr
}  // namespace tk
