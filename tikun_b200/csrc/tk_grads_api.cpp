// C-ABI entry points of the gradient operators (include/tikun_cuda.h): the
// table and its checks, and the order of the launches of tk_grads.cu.
#include <cuda_runtime.h>

#include <exception>
#include <memory>
#include <vector>

#include "tk_grads.h"
#include "tk_internal.h"

struct tk_grad_table {
  int dev = 0;
  size_t n = 0;
  bool can_clip = false;  // no buffer that clipping writes shares memory with another
  bool can_sum = false;   // every out is f32 and not its own g
  std::vector<tk::gr::GradDesc> d;
  struct Part {
    size_t first;
    int n;
    uint64_t units;
  };
  std::vector<Part> parts;  // one launch each
};

namespace tk {
namespace {

constexpr uint64_t kMaxElems = 1ull << 40;  // units * blocks stays far inside 64 bits

size_t size_of(int dt) { return dt == TK_F32 ? 4 : 2; }
bool known(int dt) { return dt == TK_F32 || dt == TK_BF16 || dt == TK_F16; }

// What the host can see of one buffer of tensor i.
int check_address(size_t i, const char* what, const void* p, int dt) {
  if (p == nullptr) return set_error(TK_ERR_INVALID, "gradient %zu: %s is NULL", i, what);
  if (!known(dt))
    return set_error(TK_ERR_INVALID, "gradient %zu: %s dtype %d is not f32, bf16 or f16", i, what, dt);
  if ((uintptr_t)p % size_of(dt) != 0)
    return set_error(TK_ERR_INVALID, "gradient %zu: %s at %p is not aligned to its element size", i,
                     what, p);
  return TK_OK;
}

int check_device(size_t i, const char* what, const void* p, int dev) {
  Residency r;
  TK_TRY(classify_pointer(p, &r, dev));
  if (r != Residency::kDevice)
    return set_error(TK_ERR_INVALID, "gradient %zu: %s at %p is not device memory", i, what, p);
  return TK_OK;
}

int create(const tk_grad* grads, size_t n, tk_grad_table** out) {
  if (out == nullptr) return set_error(TK_ERR_INVALID, "out is NULL");
  *out = nullptr;
  if (n > 0 && grads == nullptr) return set_error(TK_ERR_INVALID, "grads is NULL with n=%zu", n);
  auto t = std::make_unique<tk_grad_table>();
  t->n = n;
  t->can_sum = true;
  t->d.reserve(n);
  // A gradient in place counts as read only in `ranges`, as written in
  // `clipped`: a norm may be taken of one tensor given twice, but clipping it
  // would scale it twice.
  std::vector<ByteRange> ranges, clipped;
  uint64_t total = 0;
  for (size_t i = 0; i < n; ++i) {
    const tk_grad& g = grads[i];
    gr::GradDesc d = {};
    if (g.n > 0) {
      if (g.n > kMaxElems)
        return set_error(TK_ERR_INVALID, "gradient %zu: %llu elements are too many", i,
                         (unsigned long long)g.n);
      TK_TRY(check_address(i, "g", g.g, g.g_dtype));
      if (g.out != nullptr) TK_TRY(check_address(i, "out", g.out, g.out_dtype));
      const bool same = g.out == nullptr || (g.out == g.g && g.out_dtype == g.g_dtype);
      const uintptr_t ga = (uintptr_t)g.g, oa = same ? ga : (uintptr_t)g.out;
      const int odt = same ? g.g_dtype : g.out_dtype;
      const size_t ge = size_of(g.g_dtype), oe = size_of(odt);
      ranges.push_back({ga, ga + g.n * ge, false});
      clipped.push_back({ga, ga + g.n * ge, same});
      if (!same) {
        ranges.push_back({oa, oa + g.n * oe, true});
        clipped.push_back(ranges.back());
      }
      if (same || odt != TK_F32) t->can_sum = false;
      const uint64_t phase = ga / ge % gr::kUnit;
      d.g = reinterpret_cast<const char*>(ga - phase * ge);
      d.out = reinterpret_cast<char*>(oa - phase * oe);
      d.n = g.n;
      d.phase = phase;
      d.g_dtype = (uint64_t)g.g_dtype;
      d.out_dtype = (uint64_t)odt;
      d.out_vec = oa / oe % gr::kUnit == phase;
      d.in_place = same;
      const uint64_t units = (phase + g.n + gr::kUnit - 1) / gr::kUnit;
      total += units;
      if (total > kMaxElems)
        return set_error(TK_ERR_INVALID, "the gradients have too many elements for one table");
    }
    if (t->parts.empty() || t->parts.back().n == gr::kMaxGrads) t->parts.push_back({i, 0, 0});
    tk_grad_table::Part& p = t->parts.back();
    d.u_begin = p.units;
    p.units += d.n ? (d.phase + d.n + gr::kUnit - 1) / gr::kUnit : 0;
    ++p.n;
    t->d.push_back(d);
  }
  TK_TRY(check_overlaps(ranges.data(), ranges.size()));
  t->can_clip = check_overlaps(clipped.data(), clipped.size()) == TK_OK;
  clear_error();
  TK_CUDA_TRY(cudaGetDevice(&t->dev));
  for (size_t i = 0; i < n; ++i) {
    if (grads[i].n == 0) continue;
    TK_TRY(check_device(i, "g", grads[i].g, t->dev));
    if (grads[i].out != nullptr) TK_TRY(check_device(i, "out", grads[i].out, t->dev));
  }
  *out = t.release();
  return TK_OK;
}

int check_call(const tk_grad_table* t, int norm, bool none_ok) {
  if (t == nullptr) return set_error(TK_ERR_INVALID, "null gradient table");
  if (norm != TK_NORM_L2 && norm != TK_NORM_L1 && norm != TK_NORM_MAX &&
      !(none_ok && norm == TK_NORM_NONE))
    return set_error(TK_ERR_INVALID, "unknown norm %d", norm);
  int dev = 0;
  TK_CUDA_TRY(cudaGetDevice(&dev));
  if (dev != t->dev)
    return set_error(TK_ERR_INVALID, "the gradients live on device %d, the current device is %d",
                     t->dev, dev);
  return TK_OK;
}

gr::GradList list_of(const tk_grad_table& t, const tk_grad_table::Part& p) {
  return {t.d.data() + p.first, p.n, p.units};
}

// Blocks of each part's norm, and of all.
int norm_plan(const tk_grad_table& t, std::vector<int>* blocks, int* total) {
  *total = 0;
  for (const auto& p : t.parts) {
    const int b = p.units ? gr::norm_blocks(p.units) : 0;
    if (p.units && b <= 0) return set_error(TK_ERR_CUDA, "could not size the norm grid");
    blocks->push_back(b);
    *total += b;
  }
  return TK_OK;
}

int grad_norm(const tk_grad_table& t, int norm, float max_norm, float* norm_dev, float* each_dev,
              float* scale_dev, cudaStream_t s) {
  NvtxRange r("tikun/grad_norm");
  std::vector<int> blocks;
  int total = 0;
  TK_TRY(norm_plan(t, &blocks, &total));
  Scratch sc;
  // partials of every part, and behind them each part's blocks + n slots
  TK_TRY(sc.alloc(sizeof(double) * (total + (each_dev ? total + t.n : 0) + 1), s));
  double* partials = static_cast<double*>(sc.get());
  double* slots = partials + total;
  int at = 0;
  for (size_t i = 0; i < t.parts.size(); ++i) {
    const auto& p = t.parts[i];
    const gr::GradList l = list_of(t, p);
    if (p.units) TK_TRY(gr::launch_norm(l, norm, blocks[i], partials + at, each_dev ? slots : nullptr, s));
    if (each_dev) {
      TK_TRY(gr::launch_fold_each(l, norm, blocks[i], slots, each_dev + p.first, s));
      slots += blocks[i] + p.n;
    }
    at += blocks[i];
  }
  if (norm_dev == nullptr && scale_dev == nullptr) return TK_OK;
  return gr::launch_fold(norm, partials, total, max_norm, norm_dev, scale_dev, s);
}

int clip_grad_norm(const tk_grad_table& t, int norm, float max_norm, float* norm_dev,
                   float* scale_dev, cudaStream_t s) {
  NvtxRange r("tikun/clip_grad_norm");
  std::vector<int> blocks;
  int total = 0;
  TK_TRY(norm_plan(t, &blocks, &total));
  if (total == 0) return grad_norm(t, norm, max_norm, norm_dev, nullptr, scale_dev, s);
  Scratch sc;
  TK_TRY(sc.alloc(sizeof(double) * total, s));
  double* partials = static_cast<double*>(sc.get());
  int at = 0;
  for (size_t i = 0; i < t.parts.size(); ++i) {
    if (blocks[i]) TK_TRY(gr::launch_norm(list_of(t, t.parts[i]), norm, blocks[i], partials + at, nullptr, s));
    at += blocks[i];
  }
  bool first = true;
  for (const auto& p : t.parts) {
    if (!p.units) continue;
    TK_TRY(gr::launch_clip(list_of(t, p), norm, partials, total, max_norm,
                           first ? norm_dev : nullptr, first ? scale_dev : nullptr, s));
    first = false;
  }
  return TK_OK;
}

int accumulate(const tk_grad_table& t, float alpha, bool overwrite, int norm, float* norm_dev,
               cudaStream_t s) {
  NvtxRange r("tikun/accumulate_grads");
  std::vector<int> blocks;
  int total = 0;
  TK_TRY(norm_plan(t, &blocks, &total));
  Scratch sc;
  double* partials = nullptr;
  if (norm != TK_NORM_NONE) {
    TK_TRY(sc.alloc(sizeof(double) * (total + 1), s));
    partials = static_cast<double*>(sc.get());
  }
  int at = 0;
  for (size_t i = 0; i < t.parts.size(); ++i) {
    if (blocks[i])
      TK_TRY(gr::launch_sum(list_of(t, t.parts[i]), norm, alpha, overwrite, blocks[i],
                            partials ? partials + at : nullptr, s));
    at += blocks[i];
  }
  if (norm == TK_NORM_NONE) return TK_OK;
  return gr::launch_fold(norm, partials, total, 0.0f, norm_dev, nullptr, s);
}

// No C++ exception leaves a C entry point.
template <class F>
int guarded(F&& f) {
  clear_error();
  try {
    return f();
  } catch (const std::exception& e) {
    return set_error(TK_ERR_ALLOC, "host memory: %s", e.what());
  }
}

}  // namespace
}  // namespace tk

using namespace tk;

extern "C" {

int tk_grad_table_create(const tk_grad* grads, size_t n, tk_grad_table** out) {
  return guarded([&] { return create(grads, n, out); });
}

int tk_grad_table_destroy(tk_grad_table* table) {
  clear_error();
  delete table;
  return TK_OK;
}

int tk_grad_norm(const tk_grad_table* table, int32_t norm, float max_norm, float* norm_dev,
                 float* each_dev, float* scale_dev, void* stream) {
  return guarded([&] {
    TK_TRY(check_call(table, norm, false));
    return grad_norm(*table, norm, max_norm, norm_dev, each_dev, scale_dev,
                     static_cast<cudaStream_t>(stream));
  });
}

int tk_clip_grad_norm(const tk_grad_table* table, int32_t norm, float max_norm, float* norm_dev,
                      float* scale_dev, void* stream) {
  return guarded([&] {
    TK_TRY(check_call(table, norm, false));
    if (!(max_norm > 0.0f))
      return set_error(TK_ERR_INVALID, "max_norm %g is not positive", (double)max_norm);
    if (!table->can_clip)
      return set_error(TK_ERR_INVALID, "a gradient that is clipped in place shares memory with "
                       "another buffer of the table");
    return clip_grad_norm(*table, norm, max_norm, norm_dev, scale_dev,
                          static_cast<cudaStream_t>(stream));
  });
}

int tk_accumulate_grads(const tk_grad_table* table, float alpha, int32_t overwrite, int32_t norm,
                        float* norm_dev, void* stream) {
  return guarded([&] {
    TK_TRY(check_call(table, norm, true));
    if (norm != TK_NORM_NONE && norm_dev == nullptr)
      return set_error(TK_ERR_INVALID, "norm_dev is NULL");
    if (!table->can_sum)
      return set_error(TK_ERR_INVALID, "gradients are summed into f32 out buffers of their own");
    return accumulate(*table, alpha, overwrite != 0, norm, norm_dev,
                      static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
