// Gradient operators for sm_100a: the norm over many tensors, clipping by it
// and the sum over micro-batches.  All of them stream memory once per pass and
// compute next to nothing, so HBM bounds them, and latency where there is
// little to read.
//
// Work split: each tensor is cut into tiles of 32 KB of gradients, and every
// tile is one CTA's.  The CTAs of a launch then start in the order of the
// tiles and sweep memory together, and an SM that is done takes the next tile.
// (B200, scaling 436M f32 values: 7.0 TB/s this way, 6.2 with one resident wave
// of CTAs that take the tiles in turn.  Norm of 2.8 GB of bf16: 391 us, 410 in
// turn, 495 with one contiguous slice per CTA.)  A tile's share of a norm goes
// to a slot of its own, which is why the norms of the single tensors come at
// no cost.
//
// Units of 8 elements are one 256-bit access (f32) or one 128-bit access
// (bf16, f16).  A tensor that starts off such a boundary is counted from the
// boundary before it, and only its first and last units are done element by
// element.
//
// Sums are f64.  Squares of f32 values are exact there.  For bf16 and f16 the
// conversions to f64 would take longer than the reading (5.3 of 7.2 TB/s), so
// eight at a time are added in f32 first, where their squares are exact too.
//
// The fold of a norm and the scaling are launched as programmatic dependents of
// the launch before them: their CTAs start when that one has no CTA left to
// start, and wait for its results (griddepcontrol.wait; the first launch of a
// call is an ordinary one and starts after all earlier work).  A call's last
// launch lets nothing start early.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>

#include "tk_grads.h"
#include "tk_internal.h"
#include "tk_pointwise_math.cuh"

namespace tk {
namespace gr {
namespace {

using pw::bf16_to_f32;

constexpr int kThreads = 256;
constexpr int kMaxCluster = 8;  // the largest that every device setting allows

// Calls of at most so many tiles and units are one launch of one cluster
// (small_kernel).  A clip through the Python functions, us a call among others,
// so against in two launches: 32 whole f32 tiles 8.2 and 11.4, 48 of them 12.2
// and 11.1; 96 tensors of 768 elements 8.2 and 11.7, 128 of them 10.3 and 11.7
// (alone, with the wait for it, 20.4 and 19.9, 21.4 and 19.3).  The limits are
// the clips'.  A sum with its norm would take a few more: 32 whole f32 tiles 8.2
// and 11.6, 48 of them 10.3 and 11.7, 64 of them 12.3 and 11.6.  A norm, which
// writes nothing, four times as many: 64 of them 8.2 and 11.6, 128 of them 10.3
// and 11.4 (on the device, in a graph of calls, 5.5 and 3.1, 8.0 and 3.4); 256
// tensors of 768 elements 10.3 and 11.7.
constexpr uint32_t kSmallTiles = 96;
constexpr uint64_t kSmallUnits = 32 * 1024;
constexpr int kSmallThreads = 1024;

// Up to so many tiles every CTA of a clip's scaling folds the norm's partials
// for itself, which saves a launch.  C calls, us, so against with a fold
// between: 96 whole f32 tiles 7.0 and 9.5, 592 of them 14.4 and 16.2, 1200 of
// them 21.4 and 22.7, 2441 of them 42.1 and 41.0.
constexpr uint32_t kSelfFoldTiles = 1200;

// ------------------------------------------------------------------ dependent launches
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// What the launch before wrote while this one may have been resident already:
// not constant during this kernel, and read where all SMs see the same, in L2.
// No pointer to such memory is __restrict__ here.
__device__ __forceinline__ float written(const float* p) {
  float v;
  asm volatile("ld.relaxed.gpu.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
// 0 where `there` is false.  (The predicate keeps several in flight: behind a
// branch each would be waited for.)
__device__ __forceinline__ double written_if(bool there, const double* p) {
  double v;
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\tmov.f64 %0, 0d0000000000000000;\n\t"
      "@q ld.relaxed.gpu.global.f64 %0, [%1];\n\t}"
      : "=&d"(v)
      : "l"(p), "r"((int)there));
  return v;
}

// ------------------------------------------------------------------ memory
// A unit as it lies in memory, so that loads in flight hold no converted values.
template <int DT>
struct Raw {
  uint32_t w[DT == TK_F32 ? 8 : 4];
  // With the L2 policy `keep` (createpolicy).
  __device__ __forceinline__ void load(const char* base, uint32_t u, uint64_t keep) {
    const char* p = base + u * (uint32_t)sizeof(w);
    if constexpr (DT == TK_F32)
      asm volatile("ld.global.L2::cache_hint.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8], %9;"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]),
                     "=r"(w[6]), "=r"(w[7])
                   : "l"(p), "l"(keep));
    else
      asm volatile("ld.global.L2::cache_hint.v4.b32 {%0, %1, %2, %3}, [%4], %5;"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "l"(p), "l"(keep));
  }
  __device__ __forceinline__ void load(const char* base, uint32_t u) {
    const char* p = base + u * (uint32_t)sizeof(w);
    if constexpr (DT == TK_F32)
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]),
                     "=r"(w[6]), "=r"(w[7])
                   : "l"(p));
    else
      asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "l"(p));
  }
  __device__ __forceinline__ void expand(float (&x)[kUnit]) const {
#pragma unroll
    for (int j = 0; j < kUnit; ++j) {
      if constexpr (DT == TK_F32) x[j] = __uint_as_float(w[j]);
      else if constexpr (DT == TK_BF16)
        x[j] = j & 1 ? __uint_as_float(w[j / 2] & 0xffff0000u) : __uint_as_float(w[j / 2] << 16);
      else x[j] = __half2float(__ushort_as_half((unsigned short)(j & 1 ? w[j / 2] >> 16 : w[j / 2])));
    }
  }
};

template <int DT>
constexpr uint64_t unit_bytes = sizeof(Raw<DT>);

template <int DT>
__device__ __forceinline__ float load_one(const char* base, int pos) {
  if constexpr (DT == TK_F32) return reinterpret_cast<const float*>(base)[pos];
  else if constexpr (DT == TK_BF16) return bf16_to_f32(reinterpret_cast<const uint16_t*>(base)[pos]);
  else return __half2float(reinterpret_cast<const __half*>(base)[pos]);
}

template <class Pair>
__device__ __forceinline__ uint32_t bits(const Pair& p) {
  return *reinterpret_cast<const uint32_t*>(&p);
}

// Conversions by the hardware's paired instructions: spelled out in integers
// they made the bf16 clip of a 7M-element table take 18.8 us, not 14.9, most of
// it instruction fetches.
template <int DT>
__device__ __forceinline__ void store_unit(char* base, uint32_t u, const float (&x)[kUnit]) {
  if constexpr (DT == TK_F32) {
    float* p = reinterpret_cast<float*>(base) + u * kUnit;
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]),
                 "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                 : "memory");
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = DT == TK_BF16 ? bits(__floats2bfloat162_rn(x[2 * i], x[2 * i + 1]))
                           : bits(__floats2half2_rn(x[2 * i], x[2 * i + 1]));
    reinterpret_cast<uint4*>(base)[u] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int DT>
__device__ __forceinline__ void store_one(char* base, int pos, float x) {
  if constexpr (DT == TK_F32) reinterpret_cast<float*>(base)[pos] = x;
  else if constexpr (DT == TK_BF16) reinterpret_cast<__nv_bfloat16*>(base)[pos] = __float2bfloat16_rn(x);
  else reinterpret_cast<__half*>(base)[pos] = __float2half_rn(x);
}

// ------------------------------------------------------------------ the running norm
// L2: sum of x^2; L1: sum of |x|; both f64, in two independent chains.  Max:
// the largest magnitude as the bits of an f32, whose order as integers is the
// order of the magnitudes with every NaN above infinity, so that one NaN makes
// the result NaN.
template <int NORM>
struct Acc {
  double s[2] = {0.0, 0.0};
  __device__ __forceinline__ void add(float x, int j) {
    const double d = x;
    if constexpr (NORM == TK_NORM_L2) s[j & 1] = fma(d, d, s[j & 1]);
    else s[j & 1] += fabs(d);
  }
  template <int DT>
  __device__ __forceinline__ void add_unit(const float (&x)[kUnit]) {
    if constexpr (DT == TK_F32) {
#pragma unroll
      for (int j = 0; j < kUnit; ++j) add(x[j], j);
    } else {
      // at most four roundings of f32 on the way of each value
      float a = 0.0f, b = 0.0f;
#pragma unroll
      for (int j = 0; j < kUnit; j += 2) {
        if constexpr (NORM == TK_NORM_L2) {
          a = __fmaf_rn(x[j], x[j], a);
          b = __fmaf_rn(x[j + 1], x[j + 1], b);
        } else {
          a = __fadd_rn(a, fabsf(x[j]));
          b = __fadd_rn(b, fabsf(x[j + 1]));
        }
      }
      const float t = __fadd_rn(a, b);
      // f16 stays far inside f32's range.  bf16 has f32's own: where the sum
      // overflows, or is so small that squares in it may have lost bits below
      // 2^-149, the eight are added in f64 (NaN and infinity come out the same).
      // Eight zeros, as in the gradient of an embedding, need neither.
      constexpr float kLow = NORM == TK_NORM_L2 ? 0x1p-100f : 0.0f;
      if (DT == TK_F16 || (t >= kLow && t <= 0x1.fffffep127f)) {
        s[0] += (double)t;
      } else {
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < kUnit; ++j) bits |= __float_as_uint(x[j]);
        if (bits << 1) {
#pragma unroll
          for (int j = 0; j < kUnit; ++j) add(x[j], 1);
        }
      }
    }
  }
  __device__ __forceinline__ double value() const { return s[0] + s[1]; }
};

template <>
struct Acc<TK_NORM_MAX> {
  uint32_t m = 0;
  __device__ __forceinline__ void add(float x, int) {
    m = max(m, __float_as_uint(x) & 0x7fffffffu);
  }
  template <int DT>
  __device__ __forceinline__ void add_unit(const float (&x)[kUnit]) {
#pragma unroll
    for (int j = 0; j < kUnit; ++j) add(x[j], j);
  }
  __device__ __forceinline__ double value() const { return __longlong_as_double((long long)m); }
};

template <>
struct Acc<TK_NORM_NONE> {
  __device__ __forceinline__ void add(float, int) {}
  template <int DT>
  __device__ __forceinline__ void add_unit(const float (&)[kUnit]) {}
};

// Partial results are f64 sums, or the largest magnitude's bits as an integer.
template <int NORM>
__device__ __forceinline__ double join(double a, double b) {
  if constexpr (NORM == TK_NORM_MAX)
    return __longlong_as_double(max(__double_as_longlong(a), __double_as_longlong(b)));
  else return a + b;
}

template <int NORM>
__device__ __forceinline__ float root(double v) {
  if constexpr (NORM == TK_NORM_L2) return __double2float_rn(sqrt(v));
  else if constexpr (NORM == TK_NORM_L1) return __double2float_rn(v);
  else return __uint_as_float((uint32_t)__double_as_longlong(v));
}

template <int NORM>
__device__ __forceinline__ double warp_join(double x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x = join<NORM>(x, __shfl_down_sync(0xffffffffu, x, off));
  return x;
}

// In a fixed order; valid in thread 0.
template <int NORM, int THREADS>
__device__ __forceinline__ double block_join(double x) {
  constexpr int kWarps = THREADS / 32;
  __shared__ double warp_tot[kWarps];
  x = warp_join<NORM>(x);
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  if (lane == 0) warp_tot[wid] = x;
  __syncthreads();
  return wid == 0 ? warp_join<NORM>(lane < kWarps ? warp_tot[lane] : 0.0) : 0.0;
}

// Each thread of a cluster calls enter_cluster early and cluster_join later:
// no CTA may write another's shared memory before that one runs.
__device__ __forceinline__ void enter_cluster() {
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}

// The join over the CTAs of a cluster, in the order of their ranks: valid in
// every thread of each of them.  x counts in each CTA's thread 0.
template <int NORM>
__device__ __forceinline__ double cluster_join(double x) {
  __shared__ double cta_tot[kMaxCluster];
  asm volatile("barrier.cluster.wait;" ::: "memory");
  cooperative_groups::cluster_group c = cooperative_groups::this_cluster();
  const unsigned n = c.num_blocks();
  if (threadIdx.x == 0)
    for (unsigned r = 0; r < n; ++r) *c.map_shared_rank(&cta_tot[c.block_rank()], r) = x;
  c.sync();
  double t = cta_tot[0];
  for (unsigned r = 1; r < n; ++r) t = join<NORM>(t, cta_tot[r]);
  return t;
}

constexpr int kFoldThreads = 512;
// The join of n partials in one CTA, or this CTA's part of it; valid in
// thread 0.
template <int NORM>
__device__ __forceinline__ double fold(const double* partials, int64_t n, int part = 0,
                                       int parts = 1) {
  constexpr int U = 4;
  const int64_t step = (int64_t)kFoldThreads * parts;
  double t[U] = {};
  for (int64_t i = (int64_t)part * kFoldThreads + threadIdx.x; i < n; i += U * step) {
    double v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) v[k] = written_if(i + k * step < n, partials + i + k * step);
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (i + k * step < n) t[k] = join<NORM>(t[k], v[k]);
  }
  return block_join<NORM, kFoldThreads>(join<NORM>(join<NORM>(t[0], t[1]), join<NORM>(t[2], t[3])));
}

// crates/tikun-cpu/src/lib.rs:117-122: the step's own rule for its clip scale.
__device__ __forceinline__ float clip_scale(float norm, float max_norm) {
  if (norm > max_norm && max_norm > 0.0f) return __fdiv_rn(max_norm, __fadd_rn(norm, 1e-6f));
  return 1.0f;
}

__device__ __forceinline__ void report(const NormOut& out, float norm, float scale) {
  if (out.norm != nullptr) *out.norm = norm;
  if (out.scale != nullptr) *out.scale = scale;
  // whole sectors: a read of one that is written in part waits for DRAM (a GPT-2
  // small clip in place under the limit: 77.5 us so, 76.8 with whole ones)
  if (out.line != nullptr)
    for (int i = 0; i <= out.n_tickets; i += kUnit) {
      const float x[kUnit] = {i == 0 ? scale : 0.0f};
      store_unit<TK_F32>(reinterpret_cast<char*>(out.line), i / kUnit, x);
    }
}

// ------------------------------------------------------------------ walking the tensors
// A tile is the work of kThreads threads; a CTA may have several such groups.
__device__ __forceinline__ int tid() { return threadIdx.x % kThreads; }

// A tile's elements: positions [lo, hi) counted from its first unit, u0.
struct Tile {
  uint64_t u0;
  int lo, hi;
};

// The tensor of a tile: the last one with t_begin <= its number; empty tensors
// come before the one that has it.
template <int CAP>
__device__ __forceinline__ const GradDesc& tensor_of(const GradLaunch<CAP>& t, uint32_t at) {
  const uint32_t k = at >> t.shift;
  int lo = t.first[k], hi = t.first[k + 1];
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.d[mid].t_begin <= at) lo = mid; else hi = mid - 1;
  }
  return t.d[lo];
}

template <int DT>
__device__ __forceinline__ Tile tile_of(const GradDesc& d, uint32_t at) {
  constexpr int kTile = kUnit * kTileUnits<DT>;
  const uint32_t own = at - d.t_begin;
  const uint64_t rest = d.phase + d.n - (uint64_t)own * kTile;
  return Tile{(uint64_t)own * kTileUnits<DT>, own == 0 ? (int)d.phase : 0,
              rest < kTile ? (int)rest : kTile};
}

// load(buffer, u) for each unit of a tile that is whole, U of them in flight
// per thread, then use(buffer, u); one(pos) for the elements of a unit at the
// tensor's start or end that is not.
template <int UNITS, int U, class Buf, class Load, class Use, class One>
__device__ __forceinline__ void each_unit(const Tile& t, Load&& load, Use&& use, One&& one) {
  if (t.lo == 0 && t.hi == UNITS * kUnit) {
#pragma unroll
    for (int u = 0; u < UNITS; u += U * kThreads) {
      Buf b[U];
#pragma unroll
      for (int k = 0; k < U; ++k) load(b[k], u + k * kThreads + tid());
#pragma unroll
      for (int k = 0; k < U; ++k) use(b[k], u + k * kThreads + tid());
    }
    return;
  }
  const int first = t.lo ? 1 : 0, last = t.hi / kUnit;
  for (int u = first + tid(); u < last; u += U * kThreads) {
    Buf b[U];
#pragma unroll
    for (int k = 0; k < U; ++k) load(b[k], min(u + k * kThreads, last - 1));  // all at once
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (k == 0 || u + k * kThreads < last) use(b[k], u + k * kThreads);
  }
  if (tid() < kUnit) {
    const int head = tid(), tail = last * kUnit + tid();
    if (t.lo && head >= t.lo && head < t.hi) one(head);
    if (tail < t.hi && last >= first) one(tail);
  }
}

// A tile whose gradients and targets never are aligned together, element by
// element: eight loads of each kind at a time, then use(pos, a, b).
template <class LoadA, class LoadB, class Use>
__device__ __forceinline__ void each_element(const Tile& t, LoadA&& load_a, LoadB&& load_b,
                                             Use&& use) {
  constexpr int U = 8;
  for (int pos = t.lo + tid(); pos < t.hi; pos += U * kThreads) {
    float a[U], b[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int p = min(pos + k * kThreads, t.hi - 1);
      a[k] = load_a(p);
      b[k] = load_b(p);
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (k == 0 || pos + k * kThreads < t.hi) use(pos + k * kThreads, a[k], b[k]);
  }
}

// f(dtype constant) for a run-time element type.
template <int N>
struct Const {
  static constexpr int value = N;
};
template <class F>
__device__ __forceinline__ void with_dtype(int dt, F&& f) {
  if (dt == TK_F32) f(Const<TK_F32>{});
  else if (dt == TK_BF16) f(Const<TK_BF16>{});
  else f(Const<TK_F16>{});
}

// ------------------------------------------------------------------ one tile
// Units of gradients in flight per thread: 64 bytes of them.  (With 128 bytes,
// or with 4 or 5 CTAs per SM in place of 6, large tables read at the same rate
// within 2 %; 6 CTAs leave fewer idle SMs in the last wave of a 20M-element
// table, 20.7 us against 22.5 with 4.)
template <int DT>
constexpr int kDepth = DT == TK_F32 ? 2 : 4;

__device__ __forceinline__ uint64_t policy(bool stay) {
  uint64_t p;
  if (stay) asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  else asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}

template <int DT, class Norm>
__device__ __forceinline__ void norm_tile(const GradDesc& d, uint32_t at, bool stay, Norm& acc) {
  const Tile tile = tile_of<DT>(d, at);
  const char* g = d.g + tile.u0 * unit_bytes<DT>;
  const uint64_t keep = policy(stay);
  each_unit<kTileUnits<DT>, kDepth<DT>, Raw<DT>>(
      tile, [&](Raw<DT>& r, int u) { r.load(g, u, keep); },
      [&](const Raw<DT>& r, int) {
        float x[kUnit];
        r.expand(x);
        acc.template add_unit<DT>(x);
      },
      [&](int pos) { acc.add(load_one<DT>(g, pos), 0); });
}

// The new out counts in acc.
template <int DT, bool FIRST, int U, class Norm>
__device__ __forceinline__ void sum_tile(const GradDesc& d, uint32_t at, float alpha, Norm& acc) {
  const Tile tile = tile_of<DT>(d, at);
  const char* g = d.g + tile.u0 * unit_bytes<DT>;
  char* out = d.out + tile.u0 * unit_bytes<TK_F32>;
  auto one = [&](int pos) {
    const float x = load_one<DT>(g, pos);
    const float y = FIRST ? __fmul_rn(alpha, x) : __fmaf_rn(alpha, x, load_one<TK_F32>(out, pos));
    store_one<TK_F32>(out, pos, y);
    acc.add(y, 0);
  };
  struct Pair {
    Raw<DT> g;
    Raw<TK_F32> a;
  };
  if (d.out_vec) {
    each_unit<kTileUnits<DT>, U, Pair>(
        tile,
        [&](Pair& r, int u) {
          r.g.load(g, u);
          if constexpr (!FIRST) r.a.load(out, u);
        },
        [&](const Pair& r, int u) {
          float x[kUnit], y[kUnit];
          r.g.expand(x);
          if constexpr (!FIRST) r.a.expand(y);
#pragma unroll
          for (int j = 0; j < kUnit; ++j)
            y[j] = FIRST ? __fmul_rn(alpha, x[j]) : __fmaf_rn(alpha, x[j], y[j]);
          acc.template add_unit<TK_F32>(y);
          store_unit<TK_F32>(out, u, y);
        },
        one);
  } else {
    each_element(tile, [&](int pos) {
      return FIRST ? 0.0f : load_one<TK_F32>(out, pos);
    }, [&](int pos) { return load_one<DT>(g, pos); }, [&](int pos, float a, float x) {
      const float y = FIRST ? __fmul_rn(alpha, x) : __fmaf_rn(alpha, x, a);
      store_one<TK_F32>(out, pos, y);
      acc.add(y, 0);
    });
  }
}

template <int GDT, int ODT, int U>
__device__ __forceinline__ void clip_tile(const GradDesc& d, uint32_t at, float scale) {
  const Tile tile = tile_of<GDT>(d, at);
  const char* g = d.g + tile.u0 * unit_bytes<GDT>;
  char* out = d.out + tile.u0 * unit_bytes<ODT>;
  auto one = [&](int pos) {
    store_one<ODT>(out, pos, __fmul_rn(load_one<GDT>(g, pos), scale));
  };
  if (d.out_vec) {
    each_unit<kTileUnits<GDT>, U, Raw<GDT>>(
        tile, [&](Raw<GDT>& r, int u) { r.load(g, u); },
        [&](const Raw<GDT>& r, int u) {
          float x[kUnit];
          r.expand(x);
#pragma unroll
          for (int j = 0; j < kUnit; ++j) x[j] = __fmul_rn(x[j], scale);
          store_unit<ODT>(out, u, x);
        },
        one);
  } else {
    each_element(tile, [](int) { return 0.0f; }, [&](int pos) { return load_one<GDT>(g, pos); },
                 [&](int pos, float, float x) { store_one<ODT>(out, pos, __fmul_rn(x, scale)); });
  }
}

// ------------------------------------------------------------------ kernels
// Tiles before `stay_from` are the first to leave L2 again: where the scaling
// reads the last ones first, that leaves them more of it.  (GPT-2 small table,
// f32 into f32: 226 -> 220 us for both passes, the scaling reads 455 of its 498
// MB from DRAM; 20M elements 41 -> 38; no change from 400M on.  30 to 90 MB of
// tiles that stay measure the same.)
constexpr uint32_t kStayTiles = 1600;  // 52 MB

template <int CAP, int NORM, int DT>
__global__ void __launch_bounds__(kThreads, 6)
norm_kernel(const __grid_constant__ GradLaunch<CAP> t, uint32_t stay_from,
            double* __restrict__ partials) {
  let_next_start();
  Acc<NORM> acc;
  norm_tile<DT>(tensor_of(t, blockIdx.x), blockIdx.x, blockIdx.x >= stay_from, acc);
  const double v = block_join<NORM, kThreads>(acc.value());
  if (threadIdx.x == 0) partials[blockIdx.x] = v;
}

// Four units in flight per thread.  (GPT-2 small table, bf16 into f32 with the
// norm: 189 us = 6.6 TB/s; two units at 4 CTAs per SM 193, one at 6 CTAs 192.)
template <int CAP, int NORM, bool FIRST, int DT>
__global__ void __launch_bounds__(kThreads, FIRST ? 4 : 3)
sum_kernel(const __grid_constant__ GradLaunch<CAP> t, float alpha, double* __restrict__ partials) {
  if constexpr (NORM != TK_NORM_NONE) let_next_start();
  Acc<NORM> acc;
  sum_tile<DT, FIRST, 4>(tensor_of(t, blockIdx.x), blockIdx.x, alpha, acc);
  if constexpr (NORM != TK_NORM_NONE) {
    const double v = block_join<NORM, kThreads>(acc.value());
    if (threadIdx.x == 0) partials[blockIdx.x] = v;
  }
}

// One CTA, or one cluster.
template <int NORM>
__global__ void __launch_bounds__(kFoldThreads)
fold_kernel(const double* partials, int64_t n, const NormOut out) {
  if (out.line != nullptr) let_next_start();  // clip_kernel follows
  if (gridDim.x > 1) enter_cluster();
  wait_for_previous();
  double v = fold<NORM>(partials, n, blockIdx.x, gridDim.x);
  if (gridDim.x > 1) v = cluster_join<NORM>(v);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    const float norm = root<NORM>(v);
    report(out, norm, clip_scale(norm, out.max_norm));
  }
}

// The tensors' own norms, a CTA each, and in the last CTA (of the last part)
// the norm of all `n` partials from `all`.
template <int CAP, int NORM>
__global__ void __launch_bounds__(kFoldThreads)
fold_each_kernel(const __grid_constant__ FoldLaunch<CAP> t, const double* partials, float* each,
                 const double* all, int64_t n, const NormOut out) {
  const int i = blockIdx.x;
  wait_for_previous();
  if (i == t.n) {
    const double v = fold<NORM>(all, n);
    if (threadIdx.x == 0) {
      const float norm = root<NORM>(v);
      report(out, norm, clip_scale(norm, out.max_norm));
    }
    return;
  }
  const uint32_t begin = t.d[i].t_begin, end = i + 1 < t.n ? t.d[i + 1].t_begin : t.tiles;
  const double v = fold<NORM>(partials + begin, end - begin);
  if (threadIdx.x == 0) each[t.d[i].id] = root<NORM>(v);
}

// The last tile first: what the norm read last is still in L2.
template <int CAP, int GDT>
__global__ void __launch_bounds__(kThreads, 5)
clip_kernel(const __grid_constant__ GradLaunch<CAP> t, const float* scale_dev) {
  wait_for_previous();
  const float scale = written(scale_dev);
  const uint32_t at = t.tiles - 1 - blockIdx.x;
  const GradDesc& d = tensor_of(t, at);
  if (scale == 1.0f && d.in_place) return;  // 1 g = g: nothing to write
  with_dtype(d.out_dtype, [&](auto odt) {
    clip_tile<GDT, decltype(odt)::value, 4>(d, at, scale);
  });
}

// The same behind the norm itself, for few partials; CTA 0 reports them.
template <int CAP, int GDT>
__global__ void __launch_bounds__(kThreads, 5)
fold_clip_kernel(const __grid_constant__ GradLaunch<CAP> t, int norm, const double* partials,
                 const NormOut out) {
  __shared__ float s_scale;
  const uint32_t at = t.tiles - 1 - blockIdx.x;
  const GradDesc& d = tensor_of(t, at);
  wait_for_previous();
  auto scale_of = [&](auto k) {
    constexpr int NORM = decltype(k)::value;
    constexpr int U = 4;
    double v = 0.0;
    for (uint32_t i = threadIdx.x; i < t.tiles; i += U * kThreads) {
      double x[U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        x[k] = written_if(i + k * kThreads < t.tiles, partials + i + k * kThreads);
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (i + k * kThreads < t.tiles) v = join<NORM>(v, x[k]);
    }
    v = block_join<NORM, kThreads>(v);
    if (threadIdx.x == 0) {
      const float n = root<NORM>(v);
      s_scale = clip_scale(n, out.max_norm);
      if (blockIdx.x == 0) report(out, n, s_scale);
    }
  };
  if (norm == TK_NORM_L2) scale_of(Const<TK_NORM_L2>{});
  else if (norm == TK_NORM_L1) scale_of(Const<TK_NORM_L1>{});
  else scale_of(Const<TK_NORM_MAX>{});
  __syncthreads();
  const float scale = s_scale;
  if (scale == 1.0f && d.in_place) return;
  with_dtype(d.out_dtype, [&](auto odt) {
    clip_tile<GDT, decltype(odt)::value, 4>(d, at, scale);
  });
}

// The same where every tensor is in place, so that a scale of 1, which most
// steps of a run have, leaves nothing to do at all: one resident wave of CTAs
// that take tile after tile by a ticket, since 15,000 CTAs that only find that
// out take 8 us.  (GPT-2 small table, under the limit: 84 -> 76 us, over it
// 226 -> 228.)  Which CTA has a tile changes no result.
template <int CAP, int DT>
__global__ void __launch_bounds__(kThreads, 4)
clip_in_place_kernel(const __grid_constant__ GradLaunch<CAP> t, const float* scale_dev,
                     uint32_t* ticket) {
  wait_for_previous();
  const float scale = written(scale_dev);
  if (scale == 1.0f) return;
  __shared__ uint32_t next[2];  // one is read while the other is written
  int turn = 0;
  for (uint32_t k = blockIdx.x; k < t.tiles; turn ^= 1) {
    if (threadIdx.x == 0) next[turn] = gridDim.x + atomicAdd(ticket, 1u);
    const uint32_t at = t.tiles - 1 - k;
    clip_tile<DT, DT, 4>(tensor_of(t, at), at, scale);
    __syncthreads();
    k = next[turn];
  }
}

// A whole call in one cluster: the groups of its CTAs take the tiles in turn,
// join their shares of the norm through shared memory, and scale their own
// tiles.
template <int CAP, int NORM, int OP>
__global__ void __launch_bounds__(kSmallThreads)
small_kernel(const __grid_constant__ GradLaunch<CAP> t, int g_dtype, float alpha,
             const NormOut out) {
  enter_cluster();
  const uint32_t first = threadIdx.x / kThreads * gridDim.x + blockIdx.x;
  const uint32_t step = kSmallThreads / kThreads * gridDim.x;
  Acc<NORM> acc;
  with_dtype(g_dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    for (uint32_t at = first; at < t.tiles; at += step) {
      const GradDesc& d = tensor_of(t, at);
      if constexpr (OP == SMALL_SUM || OP == SMALL_FIRST)
        sum_tile<DT, OP == SMALL_FIRST, 2>(d, at, alpha, acc);
      else norm_tile<DT>(d, at, true, acc);
    }
  });
  const float norm = root<NORM>(cluster_join<NORM>(block_join<NORM, kSmallThreads>(acc.value())));
  const float scale = clip_scale(norm, out.max_norm);
  if (blockIdx.x == 0 && threadIdx.x == 0) report(out, norm, scale);
  if constexpr (OP == SMALL_CLIP) {
    with_dtype(g_dtype, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      for (uint32_t at = first; at < t.tiles; at += step) {
        const GradDesc& d = tensor_of(t, at);
        if (d.in_place && scale == 1.0f) continue;
        with_dtype(d.out_dtype, [&](auto odt) {
          clip_tile<DT, decltype(odt)::value, 2>(d, at, scale);
        });
      }
    });
  }
}

// ------------------------------------------------------------------ launches
template <class F>
int with_norm(int norm, F&& f) {
  switch (norm) {
    case TK_NORM_L2: return f(Const<TK_NORM_L2>{});
    case TK_NORM_L1: return f(Const<TK_NORM_L1>{});
    case TK_NORM_MAX: return f(Const<TK_NORM_MAX>{});
    default: return set_error(TK_ERR_INVALID, "unknown norm %d", norm);
  }
}

template <class F>
int with_g_dtype(int dt, F&& f) {
  if (dt == TK_F32) return f(Const<TK_F32>{});
  return dt == TK_BF16 ? f(Const<TK_BF16>{}) : f(Const<TK_F16>{});
}

template <class F>
int with_cap(int cap, F&& f) {
  if (cap == 64) return f(Const<64>{});
  return cap == 320 ? f(Const<320>{}) : f(Const<kMaxGrads>{});
}

// `args` are the addresses of the kernel's arguments.  after: as a
// programmatic dependent of the kernel before it.
int launch(const void* kernel, uint32_t grid, int threads, int cluster, bool after, void** args,
           cudaStream_t s) {
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(threads);
  c.stream = s;
  cudaLaunchAttribute a[2];
  if (cluster > 1) {
    a[c.numAttrs].id = cudaLaunchAttributeClusterDimension;
    a[c.numAttrs].val.clusterDim.x = (unsigned)cluster;
    a[c.numAttrs].val.clusterDim.y = 1;
    a[c.numAttrs].val.clusterDim.z = 1;
    ++c.numAttrs;
  }
  if (after) {
    a[c.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a[c.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++c.numAttrs;
  }
  c.attrs = a;
  TK_CUDA_TRY(cudaLaunchKernelExC(&c, kernel, args));
  return TK_OK;
}

template <class T>
void* at(const T& x) {
  return const_cast<void*>(static_cast<const void*>(&x));
}

}  // namespace

int GradPart::build(int dt, const GradDesc* d, int count, uint32_t all) {
  g_dtype = dt;
  n = count;
  tiles = all;
  units = 0;
  for (int i = 0; i < n; ++i) units += (d[i].phase + d[i].n + kUnit - 1) / kUnit;
  cap = n <= 64 ? 64 : n <= 320 ? 320 : kMaxGrads;
  return with_cap(cap, [&](auto c) {
    constexpr int CAP = decltype(c)::value;
    static_assert(sizeof(GradLaunch<CAP>) % 8 == 0 && sizeof(FoldLaunch<CAP>) % 8 == 0);
    launch.reset(new uint64_t[sizeof(GradLaunch<CAP>) / 8]());
    fold.reset(new uint64_t[sizeof(FoldLaunch<CAP>) / 8]());
    auto* l = reinterpret_cast<GradLaunch<CAP>*>(launch.get());
    auto* f = reinterpret_cast<FoldLaunch<CAP>*>(fold.get());
    l->tiles = f->tiles = tiles;
    l->n = f->n = n;
    constexpr uint32_t kBuckets = GradLaunch<CAP>::kBuckets;
    while (tiles > 0 && (tiles - 1) >> l->shift >= kBuckets) ++l->shift;
    for (uint32_t k = 0, i = 0; k <= kBuckets; ++k) {
      const uint64_t at = (uint64_t)k << l->shift;
      while (i + 1 < (uint32_t)n && d[i + 1].t_begin <= at) ++i;
      l->first[k] = (uint16_t)i;
    }
    for (int i = 0; i < n; ++i) {
      l->d[i] = d[i];
      if (d[i].n && !d[i].in_place) all_in_place = false;
      f->d[i].t_begin = d[i].t_begin;
      f->d[i].id = d[i].id;
    }
    return TK_OK;
  });
}

int launch_norm(const GradPart& p, int norm, bool again, double* partials, cudaStream_t s) {
  const uint32_t stay_from = again && p.tiles > kStayTiles ? p.tiles - kStayTiles : 0;
  return with_cap(p.cap, [&](auto c) {
    return with_g_dtype(p.g_dtype, [&](auto dt) {
      return with_norm(norm, [&](auto k) {
        void* args[] = {p.launch.get(), at(stay_from), at(partials)};
        return gr::launch(
            (const void*)norm_kernel<decltype(c)::value, decltype(k)::value, decltype(dt)::value>,
            p.tiles, kThreads, 1, false, args, s);
      });
    });
  });
}

int launch_sum(const GradPart& p, int norm, float alpha, bool overwrite, double* partials,
               cudaStream_t s) {
  return with_cap(p.cap, [&](auto c) {
    return with_g_dtype(p.g_dtype, [&](auto dt) {
      auto go = [&](auto k) {
        constexpr int CAP = decltype(c)::value, DT = decltype(dt)::value, NORM = decltype(k)::value;
        void* args[] = {p.launch.get(), at(alpha), at(partials)};
        return gr::launch(overwrite ? (const void*)sum_kernel<CAP, NORM, true, DT>
                                    : (const void*)sum_kernel<CAP, NORM, false, DT>,
                          p.tiles, kThreads, 1, false, args, s);
      };
      return norm == TK_NORM_NONE ? go(Const<TK_NORM_NONE>{}) : with_norm(norm, go);
    });
  });
}

int launch_fold(int norm, const double* partials, int64_t n, const NormOut& out, cudaStream_t s) {
  return with_norm(norm, [&](auto k) {
    // one CTA folds 2048 partials a round; from some rounds on, a cluster does
    const int ctas = n > 8192 ? kMaxCluster : 1;
    void* args[] = {at(partials), at(n), at(out)};
    return gr::launch((const void*)fold_kernel<decltype(k)::value>, ctas, kFoldThreads, ctas, n > 0,
                      args, s);
  });
}

int launch_fold_each(const GradPart& p, int norm, const double* partials, float* each,
                     const double* all, int64_t n, const NormOut* out, cudaStream_t s) {
  return with_cap(p.cap, [&](auto c) {
    return with_norm(norm, [&](auto k) {
      const NormOut none;
      void* args[] = {p.fold.get(), at(partials), at(each), at(all), at(n), at(out ? *out : none)};
      return gr::launch((const void*)fold_each_kernel<decltype(c)::value, decltype(k)::value>,
                        p.n + (out ? 1 : 0), kFoldThreads, 1, n > 0, args, s);
    });
  });
}

int launch_clip(const GradPart& p, const float* scale, uint32_t* ticket, cudaStream_t s) {
  int sms = 0;
  TK_TRY(sm_count(&sms));
  return with_cap(p.cap, [&](auto c) {
    return with_g_dtype(p.g_dtype, [&](auto dt) {
      if (p.all_in_place) {
        void* args[] = {p.launch.get(), at(scale), at(ticket)};
        return gr::launch(
            (const void*)clip_in_place_kernel<decltype(c)::value, decltype(dt)::value>,
            std::min(p.tiles, 4u * (uint32_t)sms), kThreads, 1, true, args, s);
      }
      void* args[] = {p.launch.get(), at(scale)};
      return gr::launch((const void*)clip_kernel<decltype(c)::value, decltype(dt)::value>, p.tiles,
                        kThreads, 1, true, args, s);
    });
  });
}

bool folds_itself(const GradPart& p) {
  return p.tiles <= kSelfFoldTiles;
}

int launch_fold_clip(const GradPart& p, int norm, const double* partials, const NormOut& out,
                     cudaStream_t s) {
  return with_cap(p.cap, [&](auto c) {
    return with_g_dtype(p.g_dtype, [&](auto dt) {
      void* args[] = {p.launch.get(), at(norm), at(partials), at(out)};
      return gr::launch((const void*)fold_clip_kernel<decltype(c)::value, decltype(dt)::value>,
                        p.tiles, kThreads, 1, true, args, s);
    });
  });
}

bool small(const GradPart& p) {
  return p.tiles <= kSmallTiles && p.units <= kSmallUnits && p.cap < kMaxGrads;
}

int launch_small(const GradPart& p, int op, int norm, float alpha, const NormOut& out,
                 cudaStream_t s) {
  auto with_op = [&](auto&& f) {
    switch (op) {
      case SMALL_NORM: return f(Const<SMALL_NORM>{});
      case SMALL_CLIP: return f(Const<SMALL_CLIP>{});
      case SMALL_SUM: return f(Const<SMALL_SUM>{});
      default: return f(Const<SMALL_FIRST>{});
    }
  };
  return with_norm(norm, [&](auto k) {
    return with_op([&](auto o) {
      constexpr int NORM = decltype(k)::value, OP = decltype(o)::value;
      void* args[] = {p.launch.get(), at(p.g_dtype), at(alpha), at(out)};
      const int ctas = p.tiles < kMaxCluster ? std::max(1u, p.tiles) : kMaxCluster;
      return gr::launch(p.cap == 64 ? (const void*)small_kernel<64, NORM, OP>
                                    : (const void*)small_kernel<320, NORM, OP>,
                        ctas, kSmallThreads, ctas, false, args, s);
    });
  });
}

}  // namespace gr
}  // namespace tk
