// torch_calls.cpp -- what a call of the serving operators does on the host
// between Python and the C ABI: checks the tensors, allocates the outputs,
// finds the device and stream, fills the C arguments.  A Python module of its
// own (fa_b200/_build/fa_b200_calls.so); the kernels stay in libb200fa.so, whose
// entry points bind() receives as addresses, so no torch type crosses the C ABI.
//
// In C++ because these calls are made once per layer and token, where the same
// steps in Python took 20 us around kernels of 4.  A pass with new outputs, host
// included: tables of a step 22 -> 15 us, append 26 -> 16, one request's
// attention 25 -> 15.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <array>
#include <atomic>
#include <cmath>
#include <optional>
#include <string>
#include <vector>

#include "b200fa.h"

namespace py = pybind11;
using at::Tensor;

namespace {

struct Abi {
  decltype(&b200fa_build_tables) build_tables = nullptr;
  decltype(&b200fa_rotary) rotary = nullptr;
  decltype(&b200fa_append) append = nullptr;
  decltype(&b200fa_paged_workspace_size) paged_workspace_size = nullptr;
  decltype(&b200fa_paged_fwd) paged_fwd = nullptr;
  decltype(&b200fa_last_error_string) last_error = nullptr;
  PyObject* error = nullptr;  // B200FAError(where, status, message)
} g;

void bind(const py::dict& addresses, const py::object& error) {
  auto at = [&](const char* name) { return addresses[name].cast<uintptr_t>(); };
  g.build_tables = reinterpret_cast<decltype(g.build_tables)>(at("b200fa_build_tables"));
  g.rotary = reinterpret_cast<decltype(g.rotary)>(at("b200fa_rotary"));
  g.append = reinterpret_cast<decltype(g.append)>(at("b200fa_append"));
  g.paged_workspace_size = reinterpret_cast<decltype(g.paged_workspace_size)>(at("b200fa_paged_workspace_size"));
  g.paged_fwd = reinterpret_cast<decltype(g.paged_fwd)>(at("b200fa_paged_fwd"));
  g.last_error = reinterpret_cast<decltype(g.last_error)>(at("b200fa_last_error_string"));
  Py_XDECREF(g.error);
  g.error = py::object(error).release().ptr();
}

void check(int status, const char* where) {
  if (status == 0) return;
  py::object e = py::handle(g.error)(where, status, g.last_error());
  PyErr_SetObject(g.error, e.ptr());
  throw py::error_already_set();
}

void need(bool ok, const char* message) {
  if (!ok) throw py::value_error(message);
}

void need(bool ok, const std::string& message) {
  if (!ok) throw py::value_error(message);
}

bool int32s(const Tensor& t, c10::Device dev) { return t.scalar_type() == at::kInt && t.device() == dev && t.is_contiguous(); }

void need_int32(const char* name, const Tensor& t, int64_t n, c10::Device dev) {
  if (!int32s(t, dev) || t.dim() != 1 || t.size(0) != n)
    throw py::value_error(std::string(name) + " must be contiguous int32 [" + std::to_string(n) + "] on the same CUDA device");
}

int dtype_of(at::ScalarType t) {
  return t == at::kHalf ? B200FA_DTYPE_FP16 : t == at::kBFloat16 ? B200FA_DTYPE_BF16 : t == at::kFloat ? B200FA_DTYPE_FP32 : -1;
}

void* stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

template <typename T>
T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }

int64_t bytes_of(const Tensor& t) { return t.numel() * int64_t(t.element_size()); }

// A dimension of one element has no stride of its own: torch may report any.
int64_t step_of(const Tensor& t, int64_t i) { return t.size(i) == 1 ? 0 : t.stride(i); }
bool rows_contiguous(const Tensor& table) { return table.size(1) == 1 || table.stride(1) == 1; }
int64_t row_stride(const Tensor& table) { return table.size(0) == 1 ? table.size(1) : table.stride(0); }

// Whether indexes of two tensors of the same strides meet: `d`, the distance of
// their starts, is a sum of (index in a - index in b) * stride.  `dims`: stride,
// elements in a, elements in b, largest stride first and each above all the
// smaller ones together, so that a dimension's difference is one of two values.
bool meet(int64_t d, const std::vector<std::array<int64_t, 3>>& dims, size_t i = 0) {
  if (i == dims.size()) return d == 0;
  const auto [s, na, nb] = dims[i];
  if (s == 0) return meet(d, dims, i + 1);
  const int64_t q = d >= 0 ? d / s : -((-d + s - 1) / s);
  for (int64_t x : {q, q + 1})
    if (x < na && -x < nb && meet(d - x * s, dims, i + 1)) return true;
  return false;
}

std::pair<const char*, const char*> extent(const Tensor& t) {
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  const char* p = static_cast<const char*>(t.data_ptr());
  return {p, t.numel() == 0 ? p : p + (last + 1) * int64_t(t.element_size())};
}

// Whether a (written) and b share elements.  Slices of one buffer may lie
// between each other; where that cannot be told, they are taken to be apart.
bool overlap(const Tensor& a, const Tensor& b) {
  const auto [a0, a1] = extent(a);
  const auto [b0, b1] = extent(b);
  if (a0 >= b1 || b0 >= a1) return false;
  bool alike = a.dim() == b.dim() && a.element_size() == b.element_size();
  std::vector<std::array<int64_t, 3>> dims;
  for (int64_t i = 0; alike && i < a.dim(); ++i) {
    const bool one_a = a.size(i) == 1, one_b = b.size(i) == 1;
    alike = one_a || one_b || a.stride(i) == b.stride(i);
    if (!(one_a && one_b)) dims.push_back({one_a ? b.stride(i) : a.stride(i), a.size(i), b.size(i)});
  }
  if (alike) {
    std::sort(dims.begin(), dims.end(), [](const auto& x, const auto& y) { return x[0] > y[0]; });
    return meet((b0 - a0) / int64_t(a.element_size()), dims);
  }
  const auto s = at::get_overlap_status(a, b);
  return s == at::MemOverlapStatus::Partial || s == at::MemOverlapStatus::Full;
}

// The same elements at the same places: written where they are read.
bool same(const Tensor& a, const Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.sizes() != b.sizes()) return false;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

void need_apart(const Tensor& to, const Tensor& from, const char* message) { need(!overlap(to, from), message); }
void need_same_or_apart(const Tensor& to, const Tensor& from, const char* message) {
  need(same(to, from) || !overlap(to, from), message);
}

// A caller's tensor that a kernel writes: a backward pass that saved it must see
// that it changed, as after torch's own in-place operations.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

using Tables = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;  // slots, positions, cu_q, kv_lens, free_left, status

Tables empty_tables(int64_t requests, int64_t tokens, c10::Device dev) {
  const auto ints = at::TensorOptions().dtype(at::kInt).device(dev);
  // One block of int32; the slots are 64-bit.
  Tensor all = at::empty({2 * requests + 3 + tokens}, ints);
  Tensor slots = at::empty({tokens}, ints.dtype(at::kLong));
  int64_t at0 = 0;
  auto take = [&](int64_t n) {
    Tensor t = all.narrow(0, at0, n);
    at0 += n;
    return t;
  };
  Tensor cu = take(requests + 1), kv = take(requests), left = take(1), status = take(1);
  return {slots, take(tokens), cu, kv, left, status};
}

// Contiguous tensors' memory.
bool ranges_meet(const Tensor& t, const Tensor& u) {
  const char *a = ptr<char>(t), *b = ptr<char>(u);
  return a < b + bytes_of(u) && b < a + bytes_of(t);
}

// A contiguous tensor and the rows of a table.
bool meets_rows(const Tensor& table, const Tensor& u) {
  const char *base = ptr<char>(table), *a = ptr<char>(u), *b = a + bytes_of(u);
  const int64_t pitch = row_stride(table) * 4, row = table.size(1) * 4;
  if (a == b || row == 0 || b <= base || pitch <= 0) return false;
  // The first row that ends behind a's start.
  const int64_t r = a < base + row ? 0 : (a - base - row) / pitch + 1;
  return r < table.size(0) && base + r * pitch < b;
}

Tables build_tables(const Tensor& ctx, const Tensor& add, const Tensor& table, const Tensor& free_pages, const Tensor& count,
                    int64_t page_size, int64_t tokens, const std::optional<Tables>& out) {
  const c10::Device dev = ctx.device();
  need(dev.is_cuda() && ctx.dim() == 1 && table.dim() == 2, "ctx_lens must be [R] and block_table [R, width] on a CUDA device");
  const int64_t R = ctx.size(0);
  need_int32("ctx_lens", ctx, R, dev);
  need_int32("new_lens", add, R, dev);
  need(free_pages.dim() == 1 && int32s(free_pages, dev), "free_pages must be contiguous int32 [n] on the same CUDA device");
  need_int32("free_count", count, 1, dev);
  need(table.scalar_type() == at::kInt && table.device() == dev && table.size(0) == R && rows_contiguous(table),
       "block_table must be int32 [R, width] with contiguous rows on the same CUDA device");
  need(tokens >= 0, "num_tokens must be at least 0");
  need(R <= INT32_MAX && table.size(1) <= INT32_MAX && page_size >= 0 && page_size <= INT32_MAX, "a size is out of range");
  if (out) {
    const auto& [slots, pos, cu, kv, left, status] = *out;
    need(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.size(0) == tokens && slots.device() == dev && slots.is_contiguous(),
         "out.slots must be int64 [num_tokens] on the same CUDA device");
    need_int32("out.positions", pos, tokens, dev);
    need_int32("out.cu_q", cu, R + 1, dev);
    need_int32("out.kv_lens", kv, R, dev);
    need_int32("out.free_left", left, 1, dev);
    need_int32("out.status", status, 1, dev);
    const std::array<const Tensor*, 6> outs = {&slots, &pos, &cu, &kv, &left, &status};
    for (size_t i = 0; i < outs.size(); ++i) {
      for (const Tensor* u : {&ctx, &add, &free_pages, &count})
        need(!ranges_meet(*outs[i], *u), "an output overlaps an input: alternate between two StepTables");
      need(!meets_rows(table, *outs[i]), "an output overlaps block_table");
      for (size_t j = 0; j < i; ++j) need(!ranges_meet(*outs[i], *outs[j]), "two outputs overlap");
    }
  }
  for (const Tensor* u : {&ctx, &add, &free_pages, &count}) need(!meets_rows(table, *u), "block_table overlaps another input");
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const Tables r = out ? *out : empty_tables(R, tokens, dev);
  const auto& [slots, pos, cu, kv, left, status] = r;
  check(g.build_tables(ptr<int32_t>(ctx), ptr<int32_t>(add), int32_t(R), ptr<int32_t>(table), row_stride(table), int32_t(table.size(1)),
                       ptr<int32_t>(free_pages), free_pages.size(0), ptr<int32_t>(count), int32_t(page_size), ptr<int64_t>(slots),
                       ptr<int32_t>(pos), tokens, ptr<int32_t>(cu), ptr<int32_t>(kv), ptr<int32_t>(left), ptr<int32_t>(status),
                       stream_of(dev)),
        "b200fa_build_tables");
  written(table);
  if (out)
    for (const Tensor* t : {&slots, &pos, &cu, &kv, &left, &status}) written(*t);
  return r;
}

int position_bits(const Tensor& p, c10::Device dev) {
  need((p.scalar_type() == at::kInt || p.scalar_type() == at::kLong) && p.device() == dev && p.is_contiguous(),
       "positions must be contiguous int32 or int64 on the same device");
  return p.scalar_type() == at::kLong ? 64 : 32;
}

Tensor rotary(const Tensor& x, const std::optional<Tensor>& positions, const std::optional<Tensor>& out_in, uintptr_t desc) {
  const auto* d = reinterpret_cast<const b200fa_rotary_desc*>(desc);
  need((x.dim() == 3 || x.dim() == 4) && x.size(-1) == d->dim,
       "x must be [B,H,N," + std::to_string(d->dim) + "] or [N,H," + std::to_string(d->dim) + "]");
  const int dtype = dtype_of(x.scalar_type());
  const c10::Device dev = x.device();
  need(dtype >= 0 && dev.is_cuda(), "x must be FP16, BF16 or FP32 on a CUDA device");
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const Tensor out = out_in ? *out_in : at::empty_like(x, x.options(), at::MemoryFormat::Contiguous);
  need(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && out.device() == dev,
       "out must be shaped and typed like x, on its device");
  need(x.stride(-1) == 1 && out.stride(-1) == 1, "the last dimension of x and out must be contiguous");
  if (out_in) need_same_or_apart(out, x, "out must be x or lie apart from it");
  const bool four = x.dim() == 4;
  const int64_t B = four ? x.size(0) : 1, N = x.size(four ? 2 : 0), H = x.size(1);
  const int64_t xs[3] = {four ? step_of(x, 0) : 0, step_of(x, four ? 2 : 0), step_of(x, 1)};
  const int64_t os[3] = {four ? step_of(out, 0) : 0, step_of(out, four ? 2 : 0), step_of(out, 1)};
  int bits = 32;
  int64_t pos_stride = 0;
  if (positions) {
    bits = position_bits(*positions, dev);
    if (positions->dim() == 2 && positions->size(0) == B && positions->size(1) == N) pos_stride = N;
    else need(positions->dim() == 1 && positions->size(0) == N, "positions must be [N] or [B,N]");
  }
  check(g.rotary(x.data_ptr(), out.data_ptr(), B, N, H, xs, os, positions ? positions->data_ptr() : nullptr, bits, pos_stride, d,
                 dtype, stream_of(dev)),
        "b200fa_rotary");
  if (out_in) written(out);
  return out;
}

void need_pages(const Tensor& k, const Tensor& v, int64_t dim) {
  need(k.dim() == 4 && v.sizes() == k.sizes() && (dim == 0 || k.size(3) == dim),
       "k_pages and v_pages must be [num_pages, page_size, Hkv, " + (dim ? std::to_string(dim) : std::string("dim")) + "]");
  need(k.is_cuda() && v.device() == k.device() && v.scalar_type() == k.scalar_type() &&
           (k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16),
       "the cache must be FP16 or BF16, K and V alike, on one CUDA device");
  need(k.stride(3) == 1 && v.stride(3) == 1, "the head dimension of the cache must be contiguous");
  need(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX && k.size(2) <= INT32_MAX, "a size is out of range");
}

// heads < 0: any.
void need_rows(const char* name, const Tensor& t, int64_t tokens, int64_t heads, int64_t dim, const Tensor& like) {
  if (!(t.dim() == 3 && t.size(0) == tokens && (heads < 0 || t.size(1) == heads) && t.size(2) == dim && t.size(1) <= INT32_MAX))
    throw py::value_error(std::string(name) + " must be [" + std::to_string(tokens) + ", " +
                          (heads < 0 ? std::string("heads") : std::to_string(heads)) + ", " + std::to_string(dim) + "]");
  if (!(t.scalar_type() == like.scalar_type() && t.device() == like.device() && t.stride(2) == 1))
    throw py::value_error(std::string(name) + " must have the cache's type and device and a contiguous last dimension");
}

std::optional<Tensor> append(const Tensor& k, const Tensor& v, const Tensor& kp, const Tensor& vp, const Tensor& slots,
                             const std::optional<Tensor>& q, const std::optional<Tensor>& positions, uintptr_t desc,
                             const std::optional<Tensor>& q_out_in) {
  need_pages(kp, vp, 0);
  need(k.dim() == 3, "k must be [T, Hkv, dim]");
  const int64_t T = k.size(0), hkv = kp.size(2), dim = kp.size(3);
  need_rows("k", k, T, hkv, dim, kp);
  need_rows("v", v, T, hkv, dim, kp);
  const c10::Device dev = kp.device();
  need(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.size(0) == T && slots.device() == dev && slots.is_contiguous(),
       "slots must be contiguous int64 [T] on the same CUDA device");
  const auto* d = reinterpret_cast<const b200fa_rotary_desc*>(desc);
  int bits = 32;
  if (d) {
    need(positions && positions->dim() == 1 && positions->size(0) == T, "rotary needs positions [T]");
    if (d->dim != dim)
      throw py::value_error("the rotary's dim is " + std::to_string(d->dim) + ", the cache's " + std::to_string(dim));
    bits = position_bits(*positions, dev);
  }
  for (const Tensor* t : {&k, &v})
    for (const Tensor* u : {&kp, &vp}) need_apart(*u, *t, "k or v overlaps the cache");
  bool expanded = false;  // refused below, by its strides
  for (int i = 0; i < 3; ++i) expanded |= kp.stride(i) == 0 && kp.size(i) > 1;
  if (!expanded) need_apart(kp, vp, "k_pages and v_pages overlap");
  const c10::cuda::OptionalCUDAGuard guard(dev);
  std::optional<Tensor> q_out;
  int64_t qs[2] = {0, 0}, os[2] = {0, 0};
  if (q) {
    need_rows("q", *q, T, -1, dim, kp);
    q_out = q_out_in ? *q_out_in : at::empty_like(*q, q->options(), at::MemoryFormat::Contiguous);
    need(q_out->sizes() == q->sizes(), "q_out must be shaped like q");
    need_rows("q_out", *q_out, T, -1, dim, kp);
    if (q_out_in) {
      need_same_or_apart(*q_out, *q, "q_out must be q or lie apart from it");
      for (const Tensor* t : {&k, &v, &kp, &vp}) need_apart(*q_out, *t, "q_out overlaps k, v or the cache");
    }
    for (const Tensor* t : {&kp, &vp}) need_apart(*t, *q, "q overlaps the cache");
    for (int i = 0; i < 2; ++i) qs[i] = step_of(*q, i), os[i] = step_of(*q_out, i);
  }
  const int64_t ks[2] = {step_of(k, 0), step_of(k, 1)}, vs[2] = {step_of(v, 0), step_of(v, 1)};
  const int64_t kps[3] = {step_of(kp, 0), step_of(kp, 1), step_of(kp, 2)}, vps[3] = {step_of(vp, 0), step_of(vp, 1), step_of(vp, 2)};
  check(g.append(q ? q->data_ptr() : nullptr, q ? qs : nullptr, q ? q_out->data_ptr() : nullptr, q ? os : nullptr, k.data_ptr(), ks,
                 v.data_ptr(), vs, kp.data_ptr(), kps, vp.data_ptr(), vps, T, q ? int32_t(q->size(1)) : 0, int32_t(hkv), int32_t(dim),
                 kp.size(0), int32_t(kp.size(1)), ptr<int64_t>(slots), d ? positions->data_ptr() : nullptr, bits, d,
                 dtype_of(kp.scalar_type()), stream_of(dev)),
        "b200fa_append");
  written(kp);
  written(vp);
  if (q && q_out_in) written(*q_out);
  return q_out;
}

// Bytes of a call's workspace: a constant of the (current) device, asked for once.
int64_t workspace_bytes(c10::Device dev) {
  static std::array<std::atomic<int64_t>, 64> known{};
  auto& n = known.at(size_t(dev.index()));
  if (n.load(std::memory_order_relaxed) == 0) {
    const int64_t bytes = g.paged_workspace_size();
    check(int(bytes < 0 ? bytes : 0), "b200fa_paged_workspace_size");
    n.store(bytes, std::memory_order_relaxed);
  }
  return n.load(std::memory_order_relaxed);
}

Tensor paged(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& table, const Tensor& kv, const Tensor& cu,
             int64_t max_q, double scale, int64_t window, int64_t sinks, const std::optional<Tensor>& out_in, const Tensor& status,
             uint32_t timeout_us, uint32_t flags, const std::optional<Tensor>& tables_status) {
  constexpr int64_t kDim = 128;
  need_pages(kp, vp, kDim);
  need(q.dim() == 3, "q must be [T, Hq, 128]");
  const int64_t T = q.size(0), hq = q.size(1), hkv = kp.size(2);
  need_rows("q", q, T, -1, kDim, kp);
  need(hkv > 0 && hq % hkv == 0, "the query heads must be a multiple of the cache's heads");
  const c10::Device dev = q.device();
  need(kv.dim() == 1, "kv_lens must be [R]");
  const int64_t R = kv.size(0);
  need_int32("kv_lens", kv, R, dev);
  need_int32("cu_q", cu, R + 1, dev);
  need(table.dim() == 2 && table.scalar_type() == at::kInt && table.device() == dev && table.size(0) == R && rows_contiguous(table),
       "block_table must be int32 [R, width] with contiguous rows on the same CUDA device");
  need(R <= INT32_MAX && table.size(1) <= INT32_MAX, "a size is out of range");
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const Tensor out = out_in ? *out_in : at::empty({T, hq, kDim}, q.options());
  if (out_in) {
    need_rows("out", out, T, hq, kDim, kp);
    need_same_or_apart(out, q, "out must be q or lie apart from it");
    for (const Tensor* t : {&kp, &vp}) need_apart(out, *t, "out overlaps the cache");
  }
  // Partial results live for this call: a block of torch's allocator belongs to
  // the call's stream, or to the graph that is being captured, so calls that
  // overlap never share one (the join finds its rows by what is written there).
  const Tensor ws = at::empty({workspace_bytes(dev)}, q.options().dtype(at::kByte));
  b200fa_paged_args a = {};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(q.scalar_type());
  a.q = q.data_ptr();
  a.o = out.data_ptr();
  a.k_pages = kp.data_ptr();
  a.v_pages = vp.data_ptr();
  for (int i = 0; i < 2; ++i) a.q_strides[i] = q.stride(i), a.o_strides[i] = out.stride(i);
  for (int i = 0; i < 3; ++i) a.k_strides[i] = kp.stride(i), a.v_strides[i] = vp.stride(i);
  a.block_table = ptr<int32_t>(table);
  a.table_stride = row_stride(table);
  a.kv_lens = ptr<int32_t>(kv);
  a.cu_q = ptr<int32_t>(cu);
  a.tokens = T;
  a.num_pages = kp.size(0);
  a.requests = int32_t(R);
  a.width = int32_t(table.size(1));
  a.page_size = int32_t(kp.size(1));
  a.heads_q = int32_t(hq);
  a.heads_kv = int32_t(hkv);
  a.max_q = int32_t(max_q < 0 ? 0 : max_q > INT32_MAX ? INT32_MAX : max_q);
  a.scale = float(scale);
  a.window = int32_t(window);
  a.sinks = int32_t(sinks);
  a.timeout_us = timeout_us;
  a.flags = flags;
  a.workspace = ws.data_ptr();
  a.ws_bytes = uint64_t(ws.numel());
  a.status = static_cast<uint32_t*>(status.data_ptr());
  if (tables_status) {
    need_int32("tables_status", *tables_status, 1, dev);
    a.tables_status = ptr<int32_t>(*tables_status);
  }
  check(g.paged_fwd(&a, stream_of(dev)), "b200fa_paged_fwd");
  if (out_in) written(out);
  return out;
}

}  // namespace

PYBIND11_MODULE(fa_b200_calls, m) {
  m.def("bind", &bind);
  m.def("empty_tables", [](int64_t requests, int64_t tokens, const at::Device& dev) { return empty_tables(requests, tokens, dev); });
  m.def("build_tables", &build_tables);
  m.def("rotary", &rotary);
  m.def("append", &append);
  m.def("paged", &paged);
}
