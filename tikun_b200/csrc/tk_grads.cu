// Gradient operators for sm_100a: the norm over many tensors, clipping by it
// and the sum over micro-batches.  All of them stream memory once per pass and
// compute next to nothing, so HBM bounds them.
//
// Work split: the tensors of one launch form one index space of 8-element
// units, and every CTA takes an equal contiguous slice of it, whatever the
// tensors' sizes.  A unit is one 256-bit access (f32) or one 128-bit access
// (bf16, f16): a tensor that starts off such a boundary is counted from the
// boundary before it, and only its first and last units are done element by
// element.
//
// Sums: f32 values are squared (exactly) and added in f64.  A bf16 or f16
// value squared is exact in f32.
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
using pw::f32_to_bf16;

constexpr int kThreads = 256;

// ------------------------------------------------------------------ memory
template <int DT>
__device__ __forceinline__ void load_unit(const char* base, uint64_t u, float (&x)[kUnit]) {
  if constexpr (DT == TK_F32) {
    const float* p = reinterpret_cast<const float*>(base) + u * kUnit;
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]),
                   "=f"(x[6]), "=f"(x[7])
                 : "l"(p));
  } else {
    const uint4 q = reinterpret_cast<const uint4*>(base)[u];
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == TK_BF16) {
        x[2 * i] = bf16_to_f32(w[i] & 0xffffu);
        x[2 * i + 1] = bf16_to_f32(w[i] >> 16);
      } else {
        const __half2 h = *reinterpret_cast<const __half2*>(&w[i]);
        x[2 * i] = __low2float(h);
        x[2 * i + 1] = __high2float(h);
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ float load_one(const char* base, uint64_t pos) {
  if constexpr (DT == TK_F32) return reinterpret_cast<const float*>(base)[pos];
  else if constexpr (DT == TK_BF16) return bf16_to_f32(reinterpret_cast<const uint16_t*>(base)[pos]);
  else return __half2float(reinterpret_cast<const __half*>(base)[pos]);
}

__device__ __forceinline__ uint32_t f32_to_f16(float x) {
  return __half_as_ushort(__float2half_rn(x));
}

template <int DT>
__device__ __forceinline__ void store_unit(char* base, uint64_t u, const float (&x)[kUnit]) {
  if constexpr (DT == TK_F32) {
    float* p = reinterpret_cast<float*>(base) + u * kUnit;
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]),
                 "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                 : "memory");
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = DT == TK_BF16 ? f32_to_bf16(x[2 * i]) | (f32_to_bf16(x[2 * i + 1]) << 16)
                           : f32_to_f16(x[2 * i]) | (f32_to_f16(x[2 * i + 1]) << 16);
    reinterpret_cast<uint4*>(base)[u] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int DT>
__device__ __forceinline__ void store_one(char* base, uint64_t pos, float x) {
  if constexpr (DT == TK_F32) reinterpret_cast<float*>(base)[pos] = x;
  else reinterpret_cast<uint16_t*>(base)[pos] =
      static_cast<uint16_t>(DT == TK_BF16 ? f32_to_bf16(x) : f32_to_f16(x));
}

// ------------------------------------------------------------------ the running norm
// L2: sum of x^2; L1: sum of |x|; both f64, in four independent chains.  Max:
// the largest magnitude as the bits of an f32, whose order as integers is the
// order of the magnitudes with every NaN above infinity, so that one NaN makes
// the result NaN.
template <int NORM>
struct Acc {
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  __device__ __forceinline__ void add(float x, int j) {
    const double d = x;
    if constexpr (NORM == TK_NORM_L2) s[j & 3] = fma(d, d, s[j & 3]);
    else s[j & 3] += fabs(d);
  }
  __device__ __forceinline__ double value() const { return (s[0] + s[1]) + (s[2] + s[3]); }
};

template <>
struct Acc<TK_NORM_MAX> {
  uint32_t m = 0;
  __device__ __forceinline__ void add(float x, int) {
    m = max(m, __float_as_uint(x) & 0x7fffffffu);
  }
  __device__ __forceinline__ double value() const { return __longlong_as_double((long long)m); }
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
template <int NORM>
__device__ __forceinline__ double block_join(double x) {
  __shared__ double warp_tot[kThreads / 32];
  x = warp_join<NORM>(x);
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  if (lane == 0) warp_tot[wid] = x;
  __syncthreads();
  double t = 0.0;
  if (wid == 0) t = warp_join<NORM>(lane < kThreads / 32 ? warp_tot[lane] : 0.0);
  __syncthreads();
  return t;
}

template <int NORM>
__device__ __forceinline__ double fold(const double* __restrict__ partials, int n) {
  double t = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) t = join<NORM>(t, partials[i]);
  return block_join<NORM>(t);
}

// crates/tikun-cpu/src/lib.rs:117-122: the step's own rule for its clip scale.
__device__ __forceinline__ float clip_scale(float norm, float max_norm) {
  if (norm > max_norm && max_norm > 0.0f) return __fdiv_rn(max_norm, __fadd_rn(norm, 1e-6f));
  return 1.0f;
}

// ------------------------------------------------------------------ walking the tensors
__device__ __forceinline__ uint64_t units_of(const GradDesc& t) {
  return t.n ? (t.phase + t.n + kUnit - 1) / kUnit : 0;
}

template <int CAP>
__device__ __forceinline__ int find(const GradLaunch<CAP>& t, uint64_t u) {
  int lo = 0, hi = t.n - 1;  // last tensor with u_begin <= u; empty ones come before it
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.d[mid].u_begin <= u) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// This CTA's slice, cut at the tensors' ends: body(i, tensor, first unit, end).
template <int CAP, class Body>
__device__ __forceinline__ void walk(const GradLaunch<CAP>& t, Body&& body) {
  uint64_t u = t.units * blockIdx.x / gridDim.x;
  const uint64_t end = t.units * (blockIdx.x + 1) / gridDim.x;
  if (u >= end) return;
  for (int i = find(t, u); u < end; ++i) {
    const GradDesc& d = t.d[i];
    const uint64_t stop = min(end, d.u_begin + units_of(d));
    if (u < stop) body(i, d, u - d.u_begin, stop - d.u_begin);
    u = max(u, stop);
  }
}

// Units [u0, u1) of one tensor: whole(u) for each unit that lies inside it,
// one(pos) for the elements of its first and last unit if those are not whole.
template <class Whole, class One>
__device__ __forceinline__ void each_unit(const GradDesc& d, uint64_t u0, uint64_t u1,
                                          Whole&& whole, One&& one) {
  const uint64_t phase = d.phase, end = phase + d.n, last = end / kUnit;
  const uint64_t f0 = u0 == 0 && phase ? 1 : u0, f1 = min(u1, last);
  for (uint64_t u = f0 + threadIdx.x; u < f1; u += kThreads) whole(u);
  if (threadIdx.x < kUnit) {
    if (u0 == 0 && phase) {
      const uint64_t pos = threadIdx.x;
      if (pos >= phase && pos < end) one(pos);
    }
    if (last < u1 && !(last == 0 && phase)) {
      const uint64_t pos = last * kUnit + threadIdx.x;
      if (pos < end) one(pos);
    }
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

// ------------------------------------------------------------------ kernels
template <int CAP, int NORM, bool EACH>
__global__ void __launch_bounds__(kThreads)
norm_kernel(const __grid_constant__ GradLaunch<CAP> t, double* __restrict__ partials,
            double* __restrict__ slots) {
  Acc<NORM> acc;
  double total = 0.0;
  walk(t, [&](int i, const GradDesc& d, uint64_t u0, uint64_t u1) {
    with_dtype(d.g_dtype, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      const char* g = d.g;
      each_unit(
          d, u0, u1,
          [&](uint64_t u) {
            float x[kUnit];
            load_unit<DT>(g, u, x);
#pragma unroll
            for (int j = 0; j < kUnit; ++j) acc.add(x[j], j);
          },
          [&](uint64_t pos) { acc.add(load_one<DT>(g, pos), 0); });
    });
    if constexpr (EACH) {
      const double s = block_join<NORM>(acc.value());
      if (threadIdx.x == 0) slots[blockIdx.x + i] = s;
      total = join<NORM>(total, s);  // meaningful in thread 0
      acc = Acc<NORM>();
    }
  });
  if constexpr (!EACH) total = block_join<NORM>(acc.value());
  if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

// NORM < 0: without the norm.
template <int CAP, int NORM, bool FIRST>
__global__ void __launch_bounds__(kThreads)
sum_kernel(const __grid_constant__ GradLaunch<CAP> t, float alpha, double* __restrict__ partials) {
  Acc<NORM> acc;
  walk(t, [&](int, const GradDesc& d, uint64_t u0, uint64_t u1) {
    with_dtype(d.g_dtype, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      const char* g = d.g;
      char* out = d.out;
      auto one = [&](uint64_t pos) {
        const float x = load_one<DT>(g, pos);
        const float y = FIRST ? __fmul_rn(alpha, x)
                              : __fmaf_rn(alpha, x, load_one<TK_F32>(out, pos));
        store_one<TK_F32>(out, pos, y);
        if constexpr (NORM >= 0) acc.add(y, 0);
      };
      if (d.out_vec) {
        each_unit(
            d, u0, u1,
            [&](uint64_t u) {
              float x[kUnit], y[kUnit];
              load_unit<DT>(g, u, x);
              if constexpr (!FIRST) load_unit<TK_F32>(out, u, y);
#pragma unroll
              for (int j = 0; j < kUnit; ++j) {
                y[j] = FIRST ? __fmul_rn(alpha, x[j]) : __fmaf_rn(alpha, x[j], y[j]);
                if constexpr (NORM >= 0) acc.add(y[j], j);
              }
              store_unit<TK_F32>(out, u, y);
            },
            one);
      } else {
        const uint64_t lo = max(u0 * kUnit, (uint64_t)d.phase), hi = min(u1 * kUnit, d.phase + d.n);
        for (uint64_t pos = lo + threadIdx.x; pos < hi; pos += kThreads) one(pos);
      }
    });
  });
  if constexpr (NORM >= 0) {
    const double total = block_join<NORM>(acc.value());
    if (threadIdx.x == 0) partials[blockIdx.x] = total;
  }
}

template <int NORM>
__global__ void __launch_bounds__(kThreads)
fold_kernel(const double* __restrict__ partials, int n, float max_norm, float* norm_out,
            float* scale_out) {
  const double v = fold<NORM>(partials, n);
  if (threadIdx.x == 0) {
    const float norm = root<NORM>(v);
    if (norm_out != nullptr) *norm_out = norm;
    if (scale_out != nullptr) *scale_out = clip_scale(norm, max_norm);
  }
}

// One CTA per tensor.  Unit u is in the slice of block ((u + 1) blocks - 1) / units.
template <int CAP, int NORM>
__global__ void __launch_bounds__(kThreads)
fold_each_kernel(const __grid_constant__ GradLaunch<CAP> t, int blocks,
                 const double* __restrict__ slots, float* __restrict__ each) {
  const int i = blockIdx.x;
  const GradDesc& d = t.d[i];
  const uint64_t n = units_of(d);
  double v = 0.0;
  if (n) {
    const uint64_t first = d.u_begin, last = first + n - 1;
    const uint64_t b0 = ((first + 1) * blocks - 1) / t.units, b1 = ((last + 1) * blocks - 1) / t.units;
    v = fold<NORM>(slots + b0 + i, (int)(b1 - b0 + 1));
  }
  if (threadIdx.x == 0) each[i] = root<NORM>(v);
}

template <int CAP, int NORM>
__global__ void __launch_bounds__(kThreads)
clip_kernel(const __grid_constant__ GradLaunch<CAP> t, const double* __restrict__ partials, int n,
            float max_norm, float* norm_out, float* scale_out) {
  __shared__ float s_scale;
  const double v = fold<NORM>(partials, n);
  if (threadIdx.x == 0) {
    const float norm = root<NORM>(v);
    const float scale = clip_scale(norm, max_norm);
    s_scale = scale;
    if (blockIdx.x == 0) {
      if (norm_out != nullptr) *norm_out = norm;
      if (scale_out != nullptr) *scale_out = scale;
    }
  }
  __syncthreads();
  const float scale = s_scale;
  walk(t, [&](int, const GradDesc& d, uint64_t u0, uint64_t u1) {
    if (d.in_place && scale == 1.0f) return;  // 1 g = g: nothing to write
    with_dtype(d.g_dtype, [&](auto gdt) {
      constexpr int GDT = decltype(gdt)::value;
      with_dtype(d.out_dtype, [&](auto odt) {
        constexpr int ODT = decltype(odt)::value;
        const char* g = d.g;
        char* out = d.out;
        auto one = [&](uint64_t pos) {
          store_one<ODT>(out, pos, __fmul_rn(load_one<GDT>(g, pos), scale));
        };
        if (d.out_vec) {
          each_unit(
              d, u0, u1,
              [&](uint64_t u) {
                float x[kUnit];
                load_unit<GDT>(g, u, x);
#pragma unroll
                for (int j = 0; j < kUnit; ++j) x[j] = __fmul_rn(x[j], scale);
                store_unit<ODT>(out, u, x);
              },
              one);
        } else {
          const uint64_t lo = max(u0 * kUnit, (uint64_t)d.phase);
          const uint64_t hi = min(u1 * kUnit, d.phase + d.n);
          for (uint64_t pos = lo + threadIdx.x; pos < hi; pos += kThreads) one(pos);
        }
      });
    });
  });
}

// ------------------------------------------------------------------ launches
int blocks_for(uint64_t units, int per_sm) {
  int sms = 0;
  if (pointwise_sms(&sms) != TK_OK) return 0;
  const uint64_t want = (units + kThreads - 1) / kThreads;
  return (int)std::max<uint64_t>(1, std::min<uint64_t>(want, (uint64_t)sms * per_sm));
}

template <int CAP>
void fill(GradLaunch<CAP>* t, const GradList& l) {
  t->units = l.units;
  t->n = l.n;
  t->reserved = 0;
  std::memcpy(t->d, l.d, sizeof(GradDesc) * l.n);
}

// f(table, norm constant) with the smallest table that holds the list: a
// launch copies its parameters, and 31 kB of them take 6 us of host time where
// 2 kB take 3.
template <class F>
int with_table(const GradList& l, F&& f) {
  if (l.n <= 64) {
    GradLaunch<64> t;
    fill(&t, l);
    return f(t);
  }
  if (l.n <= 224) {
    GradLaunch<224> t;
    fill(&t, l);
    return f(t);
  }
  GradLaunch<kMaxGrads> t;
  fill(&t, l);
  return f(t);
}

template <class F>
int with_norm(int norm, F&& f) {
  switch (norm) {
    case TK_NORM_L2: return f(Const<TK_NORM_L2>{});
    case TK_NORM_L1: return f(Const<TK_NORM_L1>{});
    case TK_NORM_MAX: return f(Const<TK_NORM_MAX>{});
    default: return set_error(TK_ERR_INVALID, "unknown norm %d", norm);
  }
}

int launched() {
  TK_CUDA_TRY(cudaGetLastError());
  return TK_OK;
}

}  // namespace

int norm_blocks(uint64_t units) { return blocks_for(units, 8); }

int launch_norm(const GradList& l, int norm, int blocks, double* partials, double* slots,
                cudaStream_t s) {
  return with_table(l, [&](const auto& t) {
    return with_norm(norm, [&](auto k) {
      constexpr int CAP = sizeof(t.d) / sizeof(GradDesc), NORM = decltype(k)::value;
      if (slots != nullptr) norm_kernel<CAP, NORM, true><<<blocks, kThreads, 0, s>>>(t, partials, slots);
      else norm_kernel<CAP, NORM, false><<<blocks, kThreads, 0, s>>>(t, partials, nullptr);
      return launched();
    });
  });
}

int launch_sum(const GradList& l, int norm, float alpha, bool overwrite, int blocks,
               double* partials, cudaStream_t s) {
  return with_table(l, [&](const auto& t) {
    constexpr int CAP = sizeof(t.d) / sizeof(GradDesc);
    auto go = [&](auto k) {
      constexpr int NORM = decltype(k)::value;
      if (overwrite) sum_kernel<CAP, NORM, true><<<blocks, kThreads, 0, s>>>(t, alpha, partials);
      else sum_kernel<CAP, NORM, false><<<blocks, kThreads, 0, s>>>(t, alpha, partials);
      return launched();
    };
    return norm == TK_NORM_NONE ? go(Const<TK_NORM_NONE>{}) : with_norm(norm, go);
  });
}

int launch_fold(int norm, const double* partials, int n, float max_norm, float* norm_out,
                float* scale_out, cudaStream_t s) {
  return with_norm(norm, [&](auto k) {
    fold_kernel<decltype(k)::value><<<1, kThreads, 0, s>>>(partials, n, max_norm, norm_out, scale_out);
    return launched();
  });
}

int launch_fold_each(const GradList& l, int norm, int blocks, const double* slots, float* each,
                     cudaStream_t s) {
  return with_table(l, [&](const auto& t) {
    return with_norm(norm, [&](auto k) {
      constexpr int CAP = sizeof(t.d) / sizeof(GradDesc);
      fold_each_kernel<CAP, decltype(k)::value><<<l.n, kThreads, 0, s>>>(t, blocks, slots, each);
      return launched();
    });
  });
}

int launch_clip(const GradList& l, int norm, const double* partials, int n, float max_norm,
                float* norm_out, float* scale_out, cudaStream_t s) {
  return with_table(l, [&](const auto& t) {
    return with_norm(norm, [&](auto k) {
      constexpr int CAP = sizeof(t.d) / sizeof(GradDesc);
      clip_kernel<CAP, decltype(k)::value><<<blocks_for(l.units, 8), kThreads, 0, s>>>(
          t, partials, n, max_norm, norm_out, scale_out);
      return launched();
    });
  });
}

}  // namespace gr
}  // namespace tk
