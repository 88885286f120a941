// C-ABI entry points of the gradient operators (include/tikun_cuda.h): the
// table and its checks, and the order of the launches of tk_grads.cu.
#include <cuda_runtime.h>

#include <exception>
#include <initializer_list>
#include <memory>
#include <vector>

#include "tk_grads.h"
#include "tk_internal.h"

struct tk_grad_table {
  int dev = 0;
  bool can_clip = false;  // no buffer that clipping writes shares memory with another
  bool can_sum = false;   // every out is f32 and not its own g
  std::vector<tk::gr::GradPart> parts;  // one launch each
};

namespace tk {
namespace {

constexpr uint64_t kMaxElems = 1ull << 40;  // of one tensor; a descriptor holds 44 bits
constexpr uint64_t kMaxTiles = 1ull << 28;  // of one table; a tile's number has 32 bits, a grid's 31

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

struct Target {
  uintptr_t at;
  int dtype;
  bool in_place;
};

Target target_of(const tk_grad& g) {
  if (g.out == nullptr || (g.out == g.g && g.out_dtype == g.g_dtype))
    return {(uintptr_t)g.g, g.g_dtype, true};
  return {(uintptr_t)g.out, g.out_dtype, false};
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
  t->can_sum = true;
  // A gradient in place counts as read only in `ranges`, as written in
  // `clipped`: a norm may be taken of one tensor given twice, but clipping it
  // would scale it twice.
  std::vector<ByteRange> ranges, clipped;
  uint64_t total = 0;
  for (size_t i = 0; i < n; ++i) {
    const tk_grad& g = grads[i];
    if (g.n == 0) continue;
    if (g.n > kMaxElems)
      return set_error(TK_ERR_INVALID, "gradient %zu: %llu elements are too many", i,
                       (unsigned long long)g.n);
    TK_TRY(check_address(i, "g", g.g, g.g_dtype));
    if (g.out != nullptr) TK_TRY(check_address(i, "out", g.out, g.out_dtype));
    const Target o = target_of(g);
    const uintptr_t ga = (uintptr_t)g.g;
    ranges.push_back({ga, ga + g.n * size_of(g.g_dtype), false});
    clipped.push_back(ranges.back());
    clipped.back().writable = o.in_place;
    if (!o.in_place) {
      ranges.push_back({o.at, o.at + g.n * size_of(o.dtype), true});
      clipped.push_back(ranges.back());
    }
    if (o.in_place || o.dtype != TK_F32) t->can_sum = false;
    total += gr::tiles_of(g.g_dtype, gr::kUnit, g.n);
    if (total > kMaxTiles)
      return set_error(TK_ERR_INVALID, "the gradients have too many elements for one table");
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
  // One type after the other: a kernel is compiled for each, and a part has
  // one.  Empty gradients go with the first; their own norms are 0.
  for (const int dt : {TK_F32, TK_BF16, TK_F16}) {
    std::vector<gr::GradDesc> d;
    uint32_t tiles = 0;
    auto close = [&] {
      if (d.empty()) return;
      t->parts.emplace_back();
      t->parts.back().build(dt, d.data(), (int)d.size(), tiles);
      d.clear();
      tiles = 0;
    };
    for (size_t i = 0; i < n; ++i) {
      const tk_grad& g = grads[i];
      if (g.n == 0 ? dt != TK_F32 : g.g_dtype != dt) continue;
      gr::GradDesc x = {};
      x.t_begin = tiles;
      x.id = (uint32_t)i;
      if (g.n > 0) {
        const Target o = target_of(g);
        const uintptr_t ga = (uintptr_t)g.g;
        const uint64_t phase = ga / size_of(dt) % gr::kUnit;
        x.g = reinterpret_cast<const char*>(ga - phase * size_of(dt));
        x.out = reinterpret_cast<char*>(o.at - phase * size_of(o.dtype));
        x.n = g.n;
        x.phase = phase;
        x.out_dtype = (uint64_t)o.dtype;
        x.out_vec = o.at / size_of(o.dtype) % gr::kUnit == phase;
        x.in_place = o.in_place;
        tiles += (uint32_t)gr::tiles_of(dt, phase, g.n);
      }
      d.push_back(x);
      if (d.size() == gr::kMaxGrads) close();
    }
    close();
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

size_t tiles_of(const tk_grad_table& t) {
  size_t n = 0;
  for (const auto& p : t.parts) n += p.tiles;
  return n;
}

// f64 words that a clip needs: the partials, and behind them the scale and a
// ticket per part, four bytes each, on 128-byte lines of their own: the scale is
// written while CTAs of the same launch read the last partials, and read by CTAs
// that are resident by then.  No call needs more.
constexpr size_t kLineWords = 16;
size_t clip_words(const tk_grad_table& t) {
  const size_t lines = ((1 + t.parts.size()) * 4 + 127) / 128;
  return tiles_of(t) + kLineWords - 1 + lines * kLineWords;
}
float* scale_line(double* partials, size_t total) {
  const uintptr_t end = reinterpret_cast<uintptr_t>(partials + total);
  return reinterpret_cast<float*>((end + 127) / 128 * 128);
}

// Every part's partials, one after the other.
int norm_parts(const tk_grad_table& t, int norm, bool again, double* partials, cudaStream_t s) {
  for (const auto& p : t.parts) {
    if (p.tiles) TK_TRY(gr::launch_norm(p, norm, again, partials, s));
    partials += p.tiles;
  }
  return TK_OK;
}

// The caller's workspace, or `count` f64 of the pool's.
int scratch(void* workspace, size_t count, Scratch* pool, cudaStream_t s, double** out) {
  if (workspace == nullptr) {
    TK_TRY(pool->alloc(sizeof(double) * count, s));
    workspace = pool->get();
  }
  *out = static_cast<double*>(workspace);
  return TK_OK;
}

bool small(const tk_grad_table& t) { return t.parts.size() == 1 && gr::small(t.parts[0]); }

int grad_norm(const tk_grad_table& t, int norm, const gr::NormOut& out, float* each_dev,
              void* workspace, cudaStream_t s) {
  NvtxRange r("tikun/grad_norm");
  if (each_dev == nullptr && small(t))
    return gr::launch_small(t.parts[0], gr::SMALL_NORM, norm, 0.0f, out, s);
  const size_t total = tiles_of(t);
  Scratch pool;
  double* partials = nullptr;
  TK_TRY(scratch(workspace, total, &pool, s, &partials));
  TK_TRY(norm_parts(t, norm, false, partials, s));
  if (each_dev == nullptr || t.parts.empty())
    return gr::launch_fold(norm, partials, (int64_t)total, out, s);
  const double* at = partials;
  for (const auto& p : t.parts) {  // with the last one, the norm of all
    TK_TRY(gr::launch_fold_each(p, norm, at, each_dev, partials, (int64_t)total,
                                &p == &t.parts.back() ? &out : nullptr, s));
    at += p.tiles;
  }
  return TK_OK;
}

int clip_grad_norm(const tk_grad_table& t, int norm, gr::NormOut out, void* workspace,
                   cudaStream_t s) {
  NvtxRange r("tikun/clip_grad_norm");
  if (small(t)) return gr::launch_small(t.parts[0], gr::SMALL_CLIP, norm, 0.0f, out, s);
  const size_t total = tiles_of(t);
  if (total == 0) return gr::launch_fold(norm, nullptr, 0, out, s);  // nothing to scale
  Scratch pool;
  double* partials = nullptr;
  TK_TRY(scratch(workspace, clip_words(t), &pool, s, &partials));
  if (t.parts.size() == 1 && gr::folds_itself(t.parts[0])) {
    TK_TRY(norm_parts(t, norm, true, partials, s));
    return gr::launch_fold_clip(t.parts[0], norm, partials, out, s);
  }
  out.line = scale_line(partials, total);
  uint32_t* tickets = reinterpret_cast<uint32_t*>(out.line + 1);
  out.n_tickets = (int)t.parts.size();
  TK_TRY(norm_parts(t, norm, true, partials, s));
  TK_TRY(gr::launch_fold(norm, partials, (int64_t)total, out, s));
  for (size_t i = t.parts.size(); i-- > 0;)  // the norm's last part first
    if (t.parts[i].tiles) TK_TRY(gr::launch_clip(t.parts[i], out.line, tickets + i, s));
  return TK_OK;
}

int accumulate(const tk_grad_table& t, float alpha, bool overwrite, int norm, float* norm_dev,
               void* workspace, cudaStream_t s) {
  NvtxRange r("tikun/accumulate_grads");
  gr::NormOut out;
  out.norm = norm_dev;
  const bool with = norm != TK_NORM_NONE;
  if (with && small(t))
    return gr::launch_small(t.parts[0], overwrite ? gr::SMALL_FIRST : gr::SMALL_SUM, norm, alpha,
                            out, s);
  const size_t total = tiles_of(t);
  Scratch pool;
  double* partials = nullptr;
  if (with) TK_TRY(scratch(workspace, total, &pool, s, &partials));
  double* at = partials;
  for (const auto& p : t.parts) {
    if (p.tiles) TK_TRY(gr::launch_sum(p, norm, alpha, overwrite, at, s));
    if (with) at += p.tiles;
  }
  return with ? gr::launch_fold(norm, partials, (int64_t)total, out, s) : TK_OK;
}

// A call's own device buffers, each of which may be null.
int check_outputs(const tk_grad_table* t, std::initializer_list<const void*> four_byte,
                  const void* workspace) {
  for (const void* p : four_byte) {
    if (p == nullptr) continue;
    Residency r;
    TK_TRY(classify_pointer(p, &r, t->dev));
    if (r != Residency::kDevice || (uintptr_t)p % 4 != 0)
      return set_error(TK_ERR_INVALID, "%p is not aligned device memory for a result", p);
  }
  if (workspace == nullptr) return TK_OK;
  Residency r;
  TK_TRY(classify_pointer(workspace, &r, t->dev));
  if (r != Residency::kDevice || (uintptr_t)workspace % 8 != 0)
    return set_error(TK_ERR_INVALID, "%p is not aligned device memory for a workspace", workspace);
  return TK_OK;
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

int tk_grad_workspace(const tk_grad_table* table, uint64_t* bytes, uint64_t* bytes_each) {
  clear_error();
  if (table == nullptr || bytes == nullptr || bytes_each == nullptr)
    return set_error(TK_ERR_INVALID, "null argument");
  *bytes_each = sizeof(double) * tk::clip_words(*table);
  *bytes = tk::small(*table) ? 0 : *bytes_each;
  return TK_OK;
}

int tk_grad_norm(const tk_grad_table* table, int32_t norm, float max_norm, float* norm_dev,
                 float* each_dev, float* scale_dev, void* workspace, void* stream) {
  return guarded([&] {
    TK_TRY(check_call(table, norm, false));
    TK_TRY(check_outputs(table, {norm_dev, each_dev, scale_dev}, workspace));
    return grad_norm(*table, norm, {max_norm, norm_dev, scale_dev, nullptr}, each_dev,
                     workspace, static_cast<cudaStream_t>(stream));
  });
}

int tk_clip_grad_norm(const tk_grad_table* table, int32_t norm, float max_norm, float* norm_dev,
                      float* scale_dev, void* workspace, void* stream) {
  return guarded([&] {
    TK_TRY(check_call(table, norm, false));
    TK_TRY(check_outputs(table, {norm_dev, scale_dev}, workspace));
    if (!(max_norm > 0.0f))
      return set_error(TK_ERR_INVALID, "max_norm %g is not positive", (double)max_norm);
    if (!table->can_clip)
      return set_error(TK_ERR_INVALID, "a gradient that is clipped in place shares memory with "
                       "another buffer of the table");
    return clip_grad_norm(*table, norm, {max_norm, norm_dev, scale_dev, nullptr}, workspace,
                          static_cast<cudaStream_t>(stream));
  });
}

int tk_accumulate_grads(const tk_grad_table* table, float alpha, int32_t overwrite, int32_t norm,
                        float* norm_dev, void* workspace, void* stream) {
  return guarded([&] {
    TK_TRY(check_call(table, norm, true));
    TK_TRY(check_outputs(table, {norm_dev}, workspace));
    if (norm != TK_NORM_NONE && norm_dev == nullptr)
      return set_error(TK_ERR_INVALID, "norm_dev is NULL");
    if (!table->can_sum)
      return set_error(TK_ERR_INVALID, "gradients are summed into f32 out buffers of their own");
    return accumulate(*table, alpha, overwrite != 0, norm, norm_dev, workspace,
                      static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
