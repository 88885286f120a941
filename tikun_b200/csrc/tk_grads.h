// Internal interface of the gradient operators (tk_grads.cu): the norm over
// many tensors, clipping by it and the sum over micro-batches.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <memory>

#include "tk_internal.h"

namespace tk {
namespace gr {

// Elements are handled in units of kUnit, one vector access each, and the
// units of a tensor in tiles of 32 KB of gradients, one CTA each.
constexpr int kUnit = 8;
template <int G_DTYPE>
constexpr int kTileUnits = G_DTYPE == TK_F32 ? 1024 : 2048;

// One tensor.  Its elements stand at positions [phase, phase + n) from `g`,
// the gradient's address rounded down to a whole unit, so that unit u
// (positions kUnit*u .. kUnit*u + 7) is one aligned access.  `out` is the
// target's address less the same `phase` elements.  t_begin counts the tiles
// over the launch.
struct GradDesc {
  const char* g;
  char* out;
  uint64_t n : 44;
  uint64_t phase : 4;
  uint64_t out_dtype : 4;
  uint64_t out_vec : 4;   // out's units are aligned for vector access too
  uint64_t in_place : 8;  // out is the gradient itself
  uint32_t t_begin;
  uint32_t id;            // its place in the caller's list
};
static_assert(sizeof(GradDesc) == 32, "one descriptor is 32 bytes of kernel parameters");

// The tensors of one launch, all of one type, travel in the kernel's
// parameters, as the leaf tables of the step do: the smallest of three tables
// that holds them, since a launch copies its parameters (host time of a launch
// with 2, 10 and 31 kB of them: 3, 4 and 6 us).
//
// A CTA finds its tile's tensor from `first`: the tensor of every 2^shift-th
// tile, so that one more load or two decide.  (A binary search over all of
// them takes nine loads one after the other, each of which misses the constant
// cache when a launch begins.)
constexpr int kMaxGrads = 960;
template <int CAP>
struct GradLaunch {
  static constexpr int kBuckets = CAP <= 64 ? 64 : 256;
  uint32_t tiles;  // of all tensors
  int32_t n;
  int32_t shift;
  int32_t reserved;
  uint16_t first[kBuckets + 4];
  GradDesc d[CAP];
};
// What folding the tensors' own norms needs of them.
template <int CAP>
struct FoldLaunch {
  uint32_t tiles;
  int32_t n;
  struct {
    uint32_t t_begin, id;
  } d[CAP];
};

struct GradPart {  // host side: one launch
  int g_dtype = TK_F32;
  int n = 0;
  uint32_t tiles = 0;
  uint64_t units = 0;
  bool all_in_place = true;             // so is what clipping writes
  int cap = 0;                          // 64, 320 or kMaxGrads
  std::unique_ptr<uint64_t[]> launch;   // GradLaunch<cap>
  std::unique_ptr<uint64_t[]> fold;     // FoldLaunch<cap>
  int build(int g_dtype, const GradDesc* d, int n, uint32_t tiles);
};

inline uint64_t tiles_of(int g_dtype, uint64_t phase, uint64_t n) {
  const uint64_t per = (uint64_t)kUnit * (g_dtype == TK_F32 ? kTileUnits<TK_F32> : kTileUnits<TK_BF16>);
  return n ? (phase + n + per - 1) / per : 0;
}

// Sum of powers (or largest magnitude) of each tile into partials[0..p.tiles).
// again: launch_clip will read the tiles once more, the last ones first.
int launch_norm(const GradPart& p, int norm, bool again, double* partials, cudaStream_t s);
// out = out + alpha g, or alpha g, and the same of each tile of the new out;
// norm TK_NORM_NONE: without it.
int launch_sum(const GradPart& p, int norm, float alpha, bool overwrite, double* partials,
               cudaStream_t s);

// The norm and its clip scale, each where it is not null.
struct NormOut {
  float max_norm = 0.0f;
  float* norm = nullptr;
  float* scale = nullptr;
  // for launch_clip: the scale again, and behind it a counter per part, set to 0;
  // aligned to 32 bytes, with room to a multiple of them
  float* line = nullptr;
  int n_tickets = 0;
};
// Both from n partials.  Enqueued right behind the launches that write them (of
// none: an ordinary launch, the call's first).
int launch_fold(int norm, const double* partials, int64_t n, const NormOut& out, cudaStream_t s);
// Norm of each tensor of one part from its partials, into each[id]; with out,
// the norm of n partials from `all` too.
int launch_fold_each(const GradPart& p, int norm, const double* partials, float* each,
                     const double* all, int64_t n, const NormOut* out, cudaStream_t s);
// Whether so few partials are folded by every CTA of the scaling itself, in
// place of launch_fold.
bool folds_itself(const GradPart& p);
// out = scale g, with the scale of the partials that the launch before wrote.
int launch_fold_clip(const GradPart& p, int norm, const double* partials, const NormOut& out,
                     cudaStream_t s);
// out = *scale g.  Enqueued right behind the launch that writes *scale and sets
// *ticket to 0.
int launch_clip(const GradPart& p, const float* scale, uint32_t* ticket, cudaStream_t s);

// A whole call in one launch, for a table of one part and few tiles (small).
bool small(const GradPart& p);
enum { SMALL_NORM = 0, SMALL_CLIP = 1, SMALL_SUM = 2, SMALL_FIRST = 3 };
int launch_small(const GradPart& p, int op, int norm, float alpha, const NormOut& out,
                 cudaStream_t s);

}  // namespace gr
}  // namespace tk
