// Launch functions of the hot operators as a CPython extension: shape checks, result allocation and the call into
// libttb200.so.  The same in Python (attribute reads, a ctypes object per argument, a structure field at a time) took 12 us for
// a GEMM, 16 us for a norm and 21 us for its backward, of which a launch is 3 us; a training step of a small model is made of
// hundreds of them.  kernels.py holds the documented Python entry points and keeps the keyword interface.
//
// Every function takes its arguments by position, holds the interpreter lock but for the launch itself, allocates from the
// framework's caching allocator on the current stream, and turns failures into kernels.KernelError (launches) or
// AssertionError (arguments).
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/core/CachingHostAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "entries.h"

#include <atomic>
#include <cmath>
#include <string>

using at::Tensor;
using ttb::GemmArgs;

namespace {

PyObject* g_kernel_error = nullptr;    // kernels.KernelError
PyObject* g_oom_error = nullptr;       // torch.OutOfMemoryError
PyObject* g_gemm_splits = nullptr;     // kernels.gemm_splits: the rule lives there
std::atomic<long long> g_launches{0};

struct Raised {};                      // a Python error is set

[[noreturn]] void fail(PyObject* type, const std::string& text) {
  PyErr_SetString(type, text.c_str());
  throw Raised{};
}
void need(bool ok, const char* what) {
  if (!ok) fail(PyExc_AssertionError, what);
}

// positional arguments
struct Args {
  PyObject* const* a;
  Py_ssize_t n;
  Py_ssize_t i = 0;
  Args(PyObject* const* args, Py_ssize_t count, Py_ssize_t expected) : a(args), n(count) {
    if (count != expected) fail(PyExc_TypeError, "expected " + std::to_string(expected) + " arguments, got " + std::to_string(count));
  }
  const Tensor& tensor() {
    PyObject* o = a[i++];
    if (!THPVariable_Check(o)) fail(PyExc_TypeError, "argument " + std::to_string(i) + " must be a tensor");
    return THPVariable_Unpack(o);
  }
  Tensor optional() {
    if (a[i] == Py_None) { ++i; return Tensor(); }
    return tensor();
  }
  bool flag() {
    const int r = PyObject_IsTrue(a[i++]);
    if (r < 0) throw Raised{};
    return r != 0;
  }
  long long integer() {
    const long long v = PyLong_AsLongLong(a[i++]);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
  }
  double real() {
    const double v = PyFloat_AsDouble(a[i++]);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
  }
};

template <typename F>
PyObject* guarded(F body) {
  try {
    return body();
  } catch (const Raised&) {
  } catch (python_error& e) {
    e.restore();
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(g_oom_error ? g_oom_error : PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

const void* at_(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* to_(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const float* f32(const Tensor& t) { return static_cast<const float*>(at_(t)); }
const int* i32(const Tensor& t) { return static_cast<const int*>(at_(t)); }
float* f32w(const Tensor& t) { return static_cast<float*>(to_(t)); }

bool is_bf16(const Tensor& t) { return t.scalar_type() == at::kBFloat16; }
int sms(const Tensor& t) { return at::cuda::getDeviceProperties(t.get_device())->multiProcessorCount; }
at::TensorOptions plain(const Tensor& like) { return like.options().requires_grad(false); }
Tensor empty(at::IntArrayRef shape, at::ScalarType dt, const Tensor& like) { return at::empty(shape, plain(like).dtype(dt)); }
Tensor empty_rows(const Tensor& like) { return at::empty(like.sizes(), plain(like)); }

void check_device(const Tensor& t) {
  const int cur = c10::cuda::current_device();
  if (!t.is_cuda() || t.get_device() != cur)
    fail(g_kernel_error, "operand lives on " + t.device().str() + " but the current CUDA device is " + std::to_string(cur) +
                             "; call torch.cuda.set_device() for this process before using the ops");
}

// Gives the interpreter lock up for its lifetime.  An object, because a call may leave by an exception (the address of a tensor that has
// no storage, such as the batched gradients of `is_grads_batched`), and whoever turns that into a Python error needs the lock.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// Runs a C entry on the current stream without the interpreter lock.
template <typename F>
void launch(const char* what, int kernels, F call) {
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  int code;
  {
    const Unlocked without_lock;
    code = call(stream);
  }
  if (code != 0) fail(g_kernel_error, std::string(what) + " failed with code " + std::to_string(code));
  g_launches.fetch_add(kernels, std::memory_order_relaxed);
}

PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
template <typename... Ts>
PyObject* wrap_all(const Ts&... ts) {
  PyObject* out = PyTuple_New(sizeof...(Ts));
  if (!out) throw Raised{};
  Py_ssize_t i = 0;
  for (PyObject* o : {wrap(ts)...}) PyTuple_SET_ITEM(out, i++, o);
  return out;
}
// rows x last dimension
Tensor rows2d(const Tensor& t) { return t.dim() == 2 ? t.contiguous() : t.reshape({-1, t.size(-1)}).contiguous(); }
Tensor like_shape(const Tensor& t2, const Tensor& x) { return x.dim() == 2 ? t2 : t2.view(x.sizes()); }
int tail_row_blocks(long long rows, long long cols, int num_sms) { return ttb_tail_row_blocks(rows, static_cast<int>(cols), num_sms); }
int narrow_parts(long long rows, int cols, int features, int num_sms, long long* parts) { return ttb_linear_narrow_parts(rows, cols, features, num_sms, parts); }
int logprobs_slots(const GemmArgs& g, int* tile_cols) { return ttb_logprobs_slots(g.M, g.N, g.K, g.num_sms, tile_cols); }
int kda_gate_row_blocks(long long rows, int heads) { return ttb_kda_gate_row_blocks(rows, heads); }
int row_blocks(long long rows, const Tensor& t) { return static_cast<int>(std::max<long long>(1, std::min<long long>(rows, 2 * sms(t)))); }
at::ScalarType out_type(bool f32out) { return f32out ? at::kFloat : at::kBFloat16; }

// into how many pieces along K a product is cut (kernels.gemm_splits)
long long k_splits(long long M, long long N, long long K, int num_sms) {
  PyObject* r = PyObject_CallFunction(g_gemm_splits, "LLLi", M, N, K, num_sms);
  if (!r) throw Raised{};
  const long long s = PyLong_AsLongLong(r);
  Py_DECREF(r);
  if (s == -1 && PyErr_Occurred()) throw Raised{};
  return s;
}

// ---------------------------------------------------------------------------------------------
// GEMM
// ---------------------------------------------------------------------------------------------
PyObject* gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 17);
    const Tensor &a = in.tensor(), &b = in.tensor();
    const bool a_mn = in.flag(), b_mn = in.flag();
    Tensor out = in.optional();
    const bool want_f32 = in.flag(), accumulate = in.flag();
    const Tensor residual = in.optional(), tile_group = in.optional(), group_rows = in.optional();
    const bool swiglu = in.flag();
    const Tensor row_scale = in.optional(), preact = in.optional();
    const long long ep = in.integer();
    const Tensor alpha = in.optional();
    const long long splits = in.integer();
    const Tensor there = in.optional();
    need(is_bf16(a) && is_bf16(b), "operands must be bf16");
    need(a.stride(-1) == 1 && b.stride(-1) == 1, "operands must be contiguous along their last dimension");
    check_device(a);
    GemmArgs g{};
    long long M, N, K;
    if (group_rows.defined()) {
      need(a_mn && b_mn && a.dim() == 2 && b.dim() == 2, "row groups need both operands as [rows, columns]");
      g.groups_k = static_cast<int>(group_rows.numel() - 1);
      M = a.size(1); N = b.size(1); K = 0;
      g.total_rows = a.size(0);
      need(b.size(0) == a.size(0), "operands differ in rows");
    } else {
      need(a.dim() == 2, "a must be a matrix");
      M = a.size(a_mn ? 1 : 0); K = a.size(a_mn ? 0 : 1);
      const long long Kb = b.size(b_mn ? -2 : -1), Nmem = b.size(b_mn ? -1 : -2);
      need(Kb == K, "operands differ in the contracted dimension");
      N = swiglu ? Nmem / 2 : Nmem;
    }
    g.A = a.const_data_ptr(); g.lda = a.stride(0);
    g.B = b.const_data_ptr(); g.ldb = b.stride(-2);
    if (b.dim() == 3) {
      g.b_groups = static_cast<int>(b.size(0)); g.b_group_stride = b.stride(0);
      need(tile_group.defined(), "a stack of matrices needs the tile map");
    } else {
      g.b_groups = 1;
    }
    if (!out.defined()) {
      out = g.groups_k ? empty({g.groups_k, M, N}, out_type(want_f32), a) : empty({M, N}, out_type(want_f32), a);
      need(!accumulate, "nothing to accumulate into");
    }
    need(out.stride(-1) == 1 && (is_bf16(out) || out.scalar_type() == at::kFloat), "out must be bf16 or fp32 with contiguous rows");
    g.C = out.data_ptr(); g.ldc = out.stride(-2);
    g.c_group_stride = g.groups_k ? out.stride(0) : 0;
    g.M = static_cast<int>(M); g.N = static_cast<int>(N); g.K = static_cast<int>(K);
    g.a_mn = a_mn; g.b_mn = b_mn;
    g.c_fp32 = !is_bf16(out); g.accumulate = accumulate;
    if (residual.defined()) {
      need(is_bf16(residual) && is_bf16(out), "the residual and its result are bf16");
      g.residual = residual.const_data_ptr(); g.ldr = residual.stride(0);
    }
    if (tile_group.defined()) {
      need(tile_group.scalar_type() == at::kInt, "the tile map is int32");
      g.tile_group = i32(tile_group); g.m_tiles_cap = static_cast<int>(tile_group.numel());
      need(M <= tile_group.numel() * 128, "more rows than the tile map covers");
    }
    if (group_rows.defined()) {
      need(group_rows.scalar_type() == at::kInt, "row groups are int32");
      g.group_rows = i32(group_rows);
    }
    g.epi = swiglu; g.F = swiglu ? g.N : 0;
    if (row_scale.defined()) {
      need(row_scale.scalar_type() == at::kFloat, "the row scale is fp32");
      g.row_scale = f32(row_scale);
    }
    if (preact.defined()) {
      need(is_bf16(preact), "pre-activations are bf16");
      g.preact = preact.data_ptr(); g.ld_preact = preact.stride(0);
    }
    g.num_sms = sms(a);
    if (alpha.defined()) {
      need(alpha.scalar_type() == at::kFloat && alpha.numel() == 1 && alpha.device() == a.device() && !swiglu, "alpha is one fp32 value on the device");
      g.alpha = f32(alpha);
    }
    g.ep = reinterpret_cast<const ttb::EpFuseArgs*>(ep);
    if (there.defined()) {
      need(there.scalar_type() == at::kInt && there.numel() == 1 && there.device() == a.device(), "how many rows there are is one int32 value on the device");
      g.part_rows = i32(there); g.part_k = a_mn;
    }
    Tensor ws;
    int kernels = 1;
    if (K >= 4096 && !swiglu && !tile_group.defined() && !ep) {
      const long long s = splits ? splits : k_splits(M, N, K, g.num_sms);
      if (s > 1) {
        ws = empty({s, M, N}, at::kFloat, a);
        g.split_ws = f32w(ws); g.k_splits = static_cast<int>(s);
        kernels = 2;
      }
    }
    launch("ttb_gemm_bf16", kernels, [&](void* st) { return ttb_gemm_bf16(&g, st); });
    return wrap(out);
  });
}

// ---------------------------------------------------------------------------------------------
// products with a tail (gemm_tails.cuh), dropout
// ---------------------------------------------------------------------------------------------
// t, scale, seed or the tensor that holds it, first row
struct Dropout {
  unsigned t;
  float scale;
  unsigned long long seed;
  Tensor seed_dev;
  long long first_row;
  const unsigned long long* dev() const { return static_cast<const unsigned long long*>(at_(seed_dev)); }
};
Dropout dropout_args(Args& in, const Tensor& like) {
  Dropout d;
  d.t = static_cast<unsigned>(in.integer());
  d.scale = static_cast<float>(in.real());
  d.seed = static_cast<unsigned long long>(in.integer());
  d.seed_dev = in.optional();
  d.first_row = in.integer();
  need(!d.seed_dev.defined() || (d.seed_dev.scalar_type() == at::kLong && d.seed_dev.numel() == 1 && d.seed_dev.device() == like.device()),
       "a seed tensor is one int64 value on the device of the rows");
  return d;
}
// A user's mistake in an operator's arguments
void fits(bool ok, const char* what) {
  if (!ok) fail(PyExc_ValueError, what);
}
bool on_16_bytes(const Tensor& t) { return reinterpret_cast<uintptr_t>(at_(t)) % 16 == 0; }
Tensor aligned(const Tensor& t) {
  if (!t.defined()) return t;
  const Tensor c = t.contiguous();
  return on_16_bytes(c) ? c : c.clone();
}
// A matrix as the copy engine can read it: values of a row side by side, rows apart by at least their length and by a multiple of 16
// bytes, from a 16-byte boundary on
Tensor operand(const Tensor& t) {
  if (!t.defined()) return t;
  if (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && on_16_bytes(t)) return t;
  return aligned(t);
}
void need_rows(const Tensor& t, long long rows, long long cols, const Tensor& like, const char* what) {
  need(is_bf16(t) && t.dim() == 2 && t.size(0) == rows && t.size(1) == cols && t.stride(1) == 1 && t.device() == like.device(), what);
}
GemmArgs product(const Tensor& a, const Tensor& b) {
  need(is_bf16(a) && is_bf16(b) && a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(1) && a.device() == b.device(), "operands must be bf16 matrices with equal rows' lengths, on one device");
  need(a.stride(1) == 1 && b.stride(1) == 1, "operands must be contiguous along their last dimension");
  need(a.size(0) < (1ll << 31) && b.size(0) < (1ll << 31) && a.size(1) < (1ll << 31), "fewer than 2^31 rows and columns");
  check_device(a);
  GemmArgs g{};
  g.A = a.const_data_ptr(); g.lda = a.stride(0);
  g.B = b.const_data_ptr(); g.ldb = b.stride(0);
  g.b_groups = 1;
  g.M = static_cast<int>(a.size(0)); g.N = static_cast<int>(b.size(0)); g.K = static_cast<int>(a.size(1));
  g.num_sms = sms(a);
  return g;
}

// Whether a linear layer's rows are so few that streaming the weight past them beats tiles of 128 rows, most of them empty.  Times in us,
// rows kernel and tiles, weights from memory: 1 row 1152 x 1152 3.0 and 8.0, 4096 x 4096 8.0 and 16, 4096 -> 12288 19 and 26; 4 rows 3.5
// and 8.0, 12 and 16, 27 and 26; 8 rows 6.0 and 8.0, 19 and 16, 46 and 26.
bool few_rows(const GemmArgs& g) { return g.M <= 4 || (g.M <= 8 && static_cast<long long>(g.N) * g.K <= (1 << 23)); }

// Whether the rows are walked and not tiled (linear_narrow.cu).  us, walk and tiles, with residual: 2048 x 16 -> 4096 11 and 14, 4096 x 16 -> 4096 20 and 22,
// 6000 x 16 -> 4096 29 and 28, 8190 x 16 -> 4096 39 and 36; with GELU (tanh) and pre-activations 13 and 20,
// 18 and 29, 25 and 38, 34 and 43, and 4096 x 16 -> 12288 48 and 67 (the tiles' figures of 24 features, one k-block like 16).  With 64 features the tiles are as fast from 300 rows on.
bool few_features(const GemmArgs& g) { return g.K <= 16 && (g.tail->act || static_cast<long long>(g.M) * g.N <= 3ll << 23); }

PyObject* linear_tail(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 11);
    const Tensor &x_ = in.tensor(), &w_ = in.tensor();
    const Tensor bias = aligned(in.optional());
    ttb::TailArgs t{};
    t.act = static_cast<int>(in.integer());
    const Tensor residual_ = in.optional();
    const Dropout d = dropout_args(in, x_);
    const bool want_pre = in.flag();
    fits(x_.dim() == 2 && w_.dim() == 2 && x_.size(1) == w_.size(1), "rows do not fit the weight");
    fits(!bias.defined() || (bias.dim() == 1 && bias.size(0) == w_.size(0)), "the bias has one value a column of the result");
    fits(!residual_.defined() || (residual_.dim() == 2 && residual_.size(0) == x_.size(0) && residual_.size(1) == w_.size(0)),
         "the residual must have the shape of the result");
    for (const Tensor& o : {w_, bias, residual_}) fits(!o.defined() || o.device() == x_.device(), "operands live on different devices");
    const Tensor x = operand(x_), w = operand(w_), residual = operand(residual_);
    GemmArgs g = product(x, w);
    const long long M = g.M, N = g.N;
    need(N % 8 == 0 && g.K % 8 == 0 && g.K > 0, "widths are multiples of eight");
    const Tensor y = empty({M, N}, at::kBFloat16, x), pre = want_pre ? empty({M, N}, at::kBFloat16, x) : Tensor();
    if (M == 0 || N == 0) return wrap_all(y, pre);
    if (bias.defined()) {
      need(is_bf16(bias), "the bias is bf16");
      t.bias = bias.const_data_ptr();
    }
    if (residual.defined()) {
      need(is_bf16(residual), "the residual is bf16");
      g.residual = residual.const_data_ptr(); g.ldr = residual.stride(0);
    }
    t.pre = to_(pre);
    t.drop_t = d.t; t.drop_scale = d.scale; t.seed = d.seed; t.seed_dev = d.dev(); t.first_row = d.first_row;
    g.C = y.data_ptr(); g.ldc = N;
    g.epi = 2; g.tail = &t;
    Tensor ws;
    if (few_rows(g)) {
      launch("ttb_linear_rows", 1, [&](void* st) { return ttb_linear_rows(&g, st); });
      return wrap_all(y, pre);
    }
    if (few_features(g)) {
      launch("ttb_linear_narrow", 1, [&](void* st) { return ttb_linear_narrow(&g, st); });
      return wrap_all(y, pre);
    }
    const long long s = g.K >= 4096 ? k_splits(M, N, g.K, g.num_sms) : 1;
    if (s > 1) {
      ws = empty({s, M, N}, at::kFloat, x);
      g.split_ws = f32w(ws); g.k_splits = static_cast<int>(s);
    }
    launch("ttb_gemm_bf16", s > 1 ? 2 : 1, [&](void* st) { return ttb_gemm_bf16(&g, st); });
    return wrap_all(y, pre);
  });
}

// (dz, db): dz = dropout(dy) act'(z), its column sums.  `part`, their parts, has to be kept for as long as what is launched next may overlap
// (GemmArgs.overlap); defined if that may be
void tail_gradient(const Tensor& dy, const Tensor& z, int act, const Dropout& d, bool want_db, bool f32out, Tensor& dz, Tensor& db, Tensor& part) {
  check_device(dy);
  need(dy.dim() == 2 && is_bf16(dy) && dy.is_contiguous() && on_16_bytes(dy), "gradients: bf16 rows without gaps");
  need(!z.defined() || (is_bf16(z) && z.is_contiguous() && z.sizes() == dy.sizes() && z.device() == dy.device()), "pre-activations: bf16 rows without gaps");
  const long long R = dy.size(0), C = dy.size(1);
  const bool own = act != 0 || d.t != 0;
  dz = own ? empty_rows(dy) : dy;
  const int grid = tail_row_blocks(R, C, sms(dy));
  part = want_db && R ? empty({grid, C}, at::kFloat, dy) : Tensor();
  db = !want_db ? Tensor() : R ? empty({C}, out_type(f32out), dy) : at::zeros({C}, plain(dy).dtype(out_type(f32out)));
  if (R && (own || want_db))
    launch("ttb_tail_bwd", want_db ? 2 : 1, [&](void* st) {
      return ttb_tail_bwd(at_(dy), at_(z), own ? to_(dz) : nullptr, f32w(part), to_(db), !f32out, R, static_cast<int>(C), act, d.t, d.scale, d.seed,
                          d.dev(), d.first_row, grid, st);
    });
}

PyObject* tail_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 10);
    const Tensor dy = aligned(in.tensor()), z = in.optional();
    const int act = static_cast<int>(in.integer());
    const Dropout d = dropout_args(in, dy);
    const bool want_db = in.flag(), f32out = in.flag();
    Tensor dz, db, part;
    tail_gradient(dy, z, act, d, want_db, f32out, dz, db, part);
    return wrap_all(dz, db);
  });
}

// plain bf16 product of MN-major operands as the backward of a linear layer has them
Tensor backward_product(const Tensor& a, const Tensor& b, bool a_mn, int& overlap) {
  GemmArgs g{};
  const long long M = a.size(a_mn ? 1 : 0), K = a.size(a_mn ? 0 : 1), N = b.size(1);
  const Tensor out = K ? empty({M, N}, at::kBFloat16, a) : at::zeros({M, N}, plain(a));
  if (M == 0 || N == 0 || K == 0) {
    overlap = 0;
    return out;
  }
  g.A = a.const_data_ptr(); g.lda = a.stride(0);
  g.B = b.const_data_ptr(); g.ldb = b.stride(0); g.b_groups = 1;
  g.C = out.data_ptr(); g.ldc = N;
  g.M = static_cast<int>(M); g.N = static_cast<int>(N); g.K = static_cast<int>(K);
  g.a_mn = a_mn; g.b_mn = 1;
  g.num_sms = sms(a);
  Tensor ws;
  const long long s = K >= 4096 ? k_splits(M, N, K, g.num_sms) : 1;
  if (s > 1) {
    ws = empty({s, M, N}, at::kFloat, a);
    g.split_ws = f32w(ws); g.k_splits = static_cast<int>(s);
  }
  // Of a product in pieces the second launch, their sum, would be what the next product need not wait for; and its pieces' memory is free
  // again as soon as this returns, so that the next one could take it while it is in use.
  if (s > 1) overlap &= ~1;
  g.overlap = overlap;
  launch("ttb_gemm_bf16", s > 1 ? 2 : 1, [&](void* st) { return ttb_gemm_bf16(&g, st); });
  return out;
}

// Whether the backward walks the gradient once for all that is wanted of it (linear_narrow.cu): up to 32 input features, or up to 64 of a
// gradient so small that launches are what its time is.  us, a walk with its sums and separate passes: 8190 x 16 -> 4096 24 and 37, with dropout
// 41 and 63, with GELU (erf) and dropout 67 and 83; 32 features 32 and 34, 49 and 60, 72 and 80; 64 features 61 and 34, but 300 rows 10 and 16,
// with dropout 12 and 19.
bool narrow(const Tensor& dy, long long K) {
  return K > 0 && (K <= 32 || (K <= 64 && dy.numel() <= (1ll << 21))) && dy.numel() > 0 && dy.size(0) < (1ll << 30);
}
PyObject* narrow_bwd(const Tensor& dy, const Tensor& x, const Tensor& w, const Tensor& z, int act, const Dropout& d, bool need_x, bool need_w, bool want_db,
                     bool f32out) {
  check_device(dy);
  need(is_bf16(dy) && dy.dim() == 2 && dy.is_contiguous() && on_16_bytes(dy) && dy.size(1) % 8 == 0 && is_bf16(w) && w.size(1) % 8 == 0 &&
           (!x.defined() || (is_bf16(x) && x.size(1) == w.size(1))),
       "gradients: bf16 rows without gaps, widths are multiples of eight");
  need(!z.defined() || (is_bf16(z) && z.is_contiguous() && z.sizes() == dy.sizes() && z.device() == dy.device()), "pre-activations: bf16 rows without gaps");
  const long long R = dy.size(0);
  const int C = static_cast<int>(dy.size(1)), K = static_cast<int>(w.size(1)), num_sms = sms(dy);
  const Tensor dx = need_x ? empty({R, K}, at::kBFloat16, dy) : Tensor(), dw = need_w ? empty({C, K}, at::kBFloat16, dy) : Tensor(),
               db = want_db ? empty({C}, out_type(f32out), dy) : Tensor();
  long long values = 0;
  narrow_parts(R, C, K, num_sms, &values);
  const Tensor parts = empty({values}, at::kFloat, dy);
  launch("ttb_linear_narrow_bwd", 2, [&](void* st) {
    return ttb_linear_narrow_bwd(at_(dy), at_(z), at_(x), x.defined() ? x.stride(0) : K, at_(w), w.stride(0), to_(dx), to_(dw), to_(db), !f32out, f32w(parts), R, C, K, act, d.t,
                                 d.scale, d.seed, d.dev(), d.first_row, num_sms, st);
  });
  return wrap_all(dx, dw, db);
}

// (dx, dw, db) of linear_tail, in one call: the three are four launches.  x may be missing where dw is not wanted
PyObject* linear_tail_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 14);
    const Tensor dy = aligned(in.tensor()), x = operand(in.optional()), w = operand(in.optional()), z = in.optional();
    const int act = static_cast<int>(in.integer());
    const Dropout d = dropout_args(in, dy);
    const bool need_x = in.flag(), need_w = in.flag(), want_db = in.flag(), f32out = in.flag();
    need((!need_x || (w.defined() && is_bf16(w) && w.dim() == 2 && w.size(0) == dy.size(1) && w.device() == dy.device())) &&
             (!need_w || (x.defined() && is_bf16(x) && x.dim() == 2 && x.size(0) == dy.size(0) && x.device() == dy.device())),
         "operands of the backward: bf16 matrices that fit the gradient");
    if ((need_x || need_w || want_db) && w.defined() && w.dim() == 2 && narrow(dy, w.size(1)))
      return narrow_bwd(dy, x, w, z, act, d, need_x, need_w, want_db, f32out);
    Tensor dz, db, part;
    tail_gradient(dy, z, act, d, want_db, f32out, dz, db, part);
    // Neither product needs the other, nor the bias's sums: tiles begin on SMs that the launch before leaves idle.  3001 x 1152 -> 4304, 60 tiles
    // on 74 pairs of SMs and then 85: 75 us one after the other, 58 so, with GELU (erf) and bias 99 and 81; 300 x 1024 -> 1024 34 and 22, 43 and
    // 28.  Products that fill all SMs for long gain nothing: 8192 x 4096 -> 12288 is bound by power.
    int overlap = part.defined() ? 2 : 0;
    Tensor dx, dw;
    if (need_x) {
      overlap |= need_w ? 1 : 0;
      dx = backward_product(dz, w, false, overlap);
      overlap = overlap & 1 ? 2 : 0;
    }
    if (need_w) dw = backward_product(dz, x, true, overlap);
    return wrap_all(dx, dw, db);
  });
}

PyObject* dropout(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 7);
    const Tensor x = aligned(in.tensor()), residual = aligned(in.optional());
    const Dropout d = dropout_args(in, x);
    check_device(x);
    need(x.dim() == 2 && (is_bf16(x) || x.scalar_type() == at::kFloat), "bf16 or fp32 rows");
    need(!residual.defined() || (residual.scalar_type() == x.scalar_type() && residual.sizes() == x.sizes() && residual.device() == x.device()),
         "the residual has the type and shape of the rows");
    need(x.size(1) < (1ll << 31) - 4096, "rows of fewer than 2^31 - 4096 values");
    const Tensor y = empty_rows(x);
    if (x.numel())
      launch("ttb_dropout", 1, [&](void* st) {
        return ttb_dropout(at_(x), at_(residual), to_(y), !is_bf16(x), x.size(0), static_cast<int>(x.size(1)), d.t, d.scale, d.seed, d.dev(), d.first_row,
                           sms(x), st);
      });
    return wrap(y);
  });
}

// (logp, lse, ent, and with `compact` the rows that have a target: hidden states, targets, places, inverse places, count).  Log-probabilities of
// `targets`, log-sum-exp of every row of logits (of the rows with a target, in their order) and, if wanted, its entropy
PyObject* logprobs_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 5);
    const Tensor h = operand(in.tensor()), w = operand(in.tensor());
    const Tensor& targets = in.tensor();
    const bool want_ent = in.flag(), compact = in.flag();
    GemmArgs g = product(h, w);
    const long long M = g.M, K = g.K;
    need(targets.scalar_type() == at::kLong && targets.dim() == 1 && targets.is_contiguous() && targets.numel() == M && targets.device() == h.device(),
         "targets: one int64 value a row");
    need(g.N > 0 && K > 0, "a vocabulary and hidden states of at least one value");
    need(!compact || (!want_ent && K % 8 == 0), "the entropy is of every row");
    const Tensor logp = empty({M}, at::kFloat, h), lse = empty({M}, at::kFloat, h), ent = want_ent ? empty({M}, at::kFloat, h) : Tensor();
    Tensor hc, tc = targets, rows, place, count;
    if (M == 0) return wrap_all(logp, lse, ent, hc, hc, hc, hc, hc);
    if (compact) {
      hc = empty({(M + 255) / 256 * 256, K}, at::kBFloat16, h);
      tc = empty({M}, at::kLong, h); rows = empty({M}, at::kInt, h); place = empty({M}, at::kInt, h); count = empty({1}, at::kInt, h);
      launch("ttb_rows_with_targets", 1, [&](void* st) {
        return ttb_rows_with_targets(static_cast<const long long*>(at_(targets)), M, g.N, static_cast<int*>(to_(rows)), static_cast<int*>(to_(place)),
                                     static_cast<long long*>(to_(tc)), static_cast<int*>(to_(count)), f32w(logp), st);
      });
      launch("ttb_gather_rows", 1, [&](void* st) { return ttb_gather_rows(at_(h), h.stride(0), i32(rows), i32(count), to_(hc), M, static_cast<int>(K), g.num_sms, st); });
      g.A = hc.const_data_ptr(); g.lda = K;
      g.part_rows = i32(count);
    }
    const Tensor hit = empty({M}, at::kFloat, h);
    ttb::TailArgs t{};
    t.vocab = g.N; t.entropy = want_ent;
    g.epi = 3; g.tail = &t;
    // The statistics of all pieces are 8 or 12 bytes for every 128 logits; rows are taken in shares that keep them below 256 MB
    const int planes = want_ent ? 3 : 2;
    const long long share = std::max<long long>(256, (1ll << 26) / (planes * (2ll * ((g.N + 255) / 256) + 2)) / 256 * 256);
    const void* first = g.A;
    Tensor part;
    for (long long r = 0; r < M; r += share) {
      const long long some = std::min(share, M - r);
      g.A = static_cast<const char*>(first) + r * g.lda * 2;
      g.M = static_cast<int>(some);
      g.row0 = static_cast<int>(r);
      const int slots = logprobs_slots(g, &t.tile_cols);
      if (!part.defined() || part.numel() < planes * slots * some) part = empty({planes * slots * some}, at::kFloat, h);
      t.targets = static_cast<const long long*>(at_(tc)) + r;
      t.part = f32w(part); t.target_logit = f32w(hit) + r;
      launch("ttb_gemm_bf16", 1, [&](void* st) { return ttb_gemm_bf16(&g, st); });
      launch("ttb_logprobs_join", 1, [&](void* st) {
        return ttb_logprobs_join(f32(part), t.target_logit, t.targets, compact ? i32(rows) + r : nullptr, g.part_rows, g.row0, slots, some, g.N,
                                 compact ? f32w(logp) : f32w(logp) + r, f32w(lse) + r, ent.defined() ? f32w(ent) + r : nullptr, st);
      });
    }
    return wrap_all(logp, lse, ent, hc, compact ? tc : Tensor(), rows, place, count);
  });
}

// gradient of the logits of columns first_col .. first_col + w.size(0) - 1 of a vocabulary, into `out`; with `rows` and `count` of the rows
// with a target alone
PyObject* logprobs_dlogits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 12);
    const Tensor &h = in.tensor(), &w = in.tensor(), &targets = in.tensor(), &lse = in.tensor();
    const Tensor ent = in.optional(), dlogp = in.optional(), dent = in.optional();
    ttb::TailArgs t{};
    t.first_col = in.integer();
    t.vocab = in.integer();
    const Tensor& out = in.tensor();
    const Tensor rows = in.optional(), count = in.optional();
    GemmArgs g = product(h, w);
    need(targets.scalar_type() == at::kLong && targets.is_contiguous() && targets.numel() == g.M && targets.device() == h.device(), "targets: one int64 value a row");
    for (const Tensor& r : {lse, ent, dlogp, dent})
      need(!r.defined() || (r.scalar_type() == at::kFloat && r.is_contiguous() && r.numel() == g.M && r.device() == h.device()), "statistics and gradients: one fp32 value a row");
    for (const Tensor& r : {rows, count})
      need(!r.defined() || (r.scalar_type() == at::kInt && r.is_contiguous() && r.device() == h.device()), "places of rows are int32");
    need(rows.defined() == count.defined() && (!rows.defined() || (rows.numel() == g.M && count.numel() == 1)), "a place for each row, and how many there are");
    need(!dent.defined() || ent.defined(), "the entropy's gradient needs the entropy");
    t.rest = out.dim() == 2 && out.size(0) == 2ll * g.M;
    need_rows(out, t.rest ? 2ll * g.M : g.M, g.N, h, "the gradient is bf16, a row or two for each of the hidden states");
    need(out.stride(0) % 8 == 0 && on_16_bytes(out), "rows of the gradient start on 16-byte boundaries");
    if (g.M == 0 || g.N == 0) return wrap(out);
    t.targets = static_cast<const long long*>(at_(targets));
    t.lse = f32(lse); t.ent = f32(ent); t.dlogp = f32(dlogp); t.dent = f32(dent);
    t.rows = i32(rows);
    g.part_rows = i32(count);
    g.C = out.data_ptr(); g.ldc = out.stride(0);
    g.epi = 4; g.tail = &t;
    launch("ttb_gemm_bf16", 1, [&](void* st) { return ttb_gemm_bf16(&g, st); });
    return wrap(out);
  });
}

// [R, cols] bf16: row place[r] of x, or zeros where that is negative
PyObject* scatter_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 2);
    const Tensor &x = in.tensor(), &place = in.tensor();
    check_device(x);
    need(x.dim() == 2 && x.is_contiguous() && (is_bf16(x) || x.scalar_type() == at::kFloat) && x.size(1) % 8 == 0 && on_16_bytes(x), "bf16 or fp32 rows without gaps");
    need(place.scalar_type() == at::kInt && place.is_contiguous() && place.dim() == 1 && place.device() == x.device(), "places of rows are int32");
    const Tensor out = empty({place.numel(), x.size(1)}, at::kBFloat16, x);
    launch("ttb_scatter_rows", 1, [&](void* st) {
      return ttb_scatter_rows(at_(x), !is_bf16(x), i32(place), to_(out), place.numel(), static_cast<int>(x.size(1)), sms(x), st);
    });
    return wrap(out);
  });
}

// ---------------------------------------------------------------------------------------------
// norms, bias + activation
// ---------------------------------------------------------------------------------------------
PyObject* rmsnorm_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 5);
    const Tensor &x = in.tensor(), &w = in.tensor();
    const double eps = in.real();
    const Tensor residual = in.optional();
    const bool plus = in.flag();
    const Tensor x2 = rows2d(x), r2 = residual.defined() ? rows2d(residual) : Tensor();
    const long long T = x2.size(0);
    const Tensor y = empty_rows(x2), rstd = empty({T}, at::kFloat, x), sum = residual.defined() ? empty_rows(x2) : Tensor();
    launch("ttb_rmsnorm_fwd", 1, [&](void* st) {
      return ttb_rmsnorm_fwd(at_(x2), at_(r2), at_(w), to_(y), to_(sum), f32w(rstd), T, static_cast<int>(x2.size(1)), static_cast<float>(eps), plus, st);
    });
    return wrap_all(like_shape(y, x), rstd, sum.defined() ? like_shape(sum, x) : x);
  });
}

PyObject* rmsnorm_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 7);
    const Tensor &dy = in.tensor(), &x = in.tensor(), &w = in.tensor(), &rstd = in.tensor();
    const Tensor dres = in.optional();
    const bool plus = in.flag(), f32out = in.flag();
    const Tensor x2 = rows2d(x), dy2 = rows2d(dy), d2 = dres.defined() ? rows2d(dres) : Tensor();
    const long long T = x2.size(0), H = x2.size(1);
    const int grid = row_blocks(T, x);
    const Tensor dx = empty_rows(x2), part = empty({grid, H}, at::kFloat, x), dw = empty({H}, out_type(f32out), x);
    launch("ttb_rmsnorm_bwd", 2, [&](void* st) {
      return ttb_rmsnorm_bwd(at_(dy2), at_(x2), at_(w), f32(rstd), at_(d2), to_(dx), f32w(part), to_(dw), !f32out, T, static_cast<int>(H), plus, grid, st);
    });
    return wrap_all(like_shape(dx, x), dw);
  });
}

PyObject* layernorm_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 4);
    const Tensor &x = in.tensor(), &w = in.tensor(), &b = in.tensor();
    const double eps = in.real();
    const Tensor x2 = rows2d(x);
    const long long T = x2.size(0);
    const Tensor y = empty_rows(x2), mean = empty({T}, at::kFloat, x), rstd = empty({T}, at::kFloat, x);
    launch("ttb_layernorm_fwd", 1, [&](void* st) {
      return ttb_layernorm_fwd(at_(x2), at_(w), at_(b), to_(y), f32w(mean), f32w(rstd), T, static_cast<int>(x2.size(1)), static_cast<float>(eps), st);
    });
    return wrap_all(like_shape(y, x), mean, rstd);
  });
}

PyObject* layernorm_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 6);
    const Tensor &dy = in.tensor(), &x = in.tensor(), &w = in.tensor(), &mean = in.tensor(), &rstd = in.tensor();
    const bool f32out = in.flag();
    const Tensor x2 = rows2d(x), dy2 = rows2d(dy);
    const long long T = x2.size(0), H = x2.size(1);
    const int grid = row_blocks(T, x);
    const Tensor dx = empty_rows(x2), part = empty({grid, 2 * H}, at::kFloat, x), dwdb = empty({2, H}, out_type(f32out), x);
    launch("ttb_layernorm_bwd", 2, [&](void* st) {
      return ttb_layernorm_bwd(at_(dy2), at_(x2), at_(w), f32(mean), f32(rstd), to_(dx), f32w(part), to_(dwdb), !f32out, T, static_cast<int>(H), grid, st);
    });
    return wrap_all(like_shape(dx, x), dwdb.select(0, 0), dwdb.select(0, 1));
  });
}

PyObject* bias_act_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 4);
    const Tensor &x = in.tensor(), &bias = in.tensor();
    const int act = static_cast<int>(in.integer());
    const Tensor residual = in.optional();
    const Tensor x2 = rows2d(x), r2 = residual.defined() ? rows2d(residual) : Tensor(), y = empty_rows(x2);
    launch("ttb_bias_act_fwd", 1, [&](void* st) {
      return ttb_bias_act_fwd(at_(x2), at_(bias), at_(r2), to_(y), x2.size(0), static_cast<int>(x2.size(1)), act, st);
    });
    return wrap(like_shape(y, x));
  });
}

PyObject* bias_act_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 5);
    const Tensor &dy = in.tensor(), &x = in.tensor(), &bias = in.tensor();
    const int act = static_cast<int>(in.integer());
    const bool f32out = in.flag();
    const Tensor x2 = rows2d(x), dy2 = rows2d(dy);
    const long long R = x2.size(0), C = x2.size(1);
    const int grid = row_blocks(R, x);
    const Tensor dx = act ? empty_rows(x2) : Tensor(), part = empty({grid, C}, at::kFloat, x), db = empty({C}, out_type(f32out), x);
    launch("ttb_bias_act_bwd", 2, [&](void* st) {
      return ttb_bias_act_bwd(at_(dy2), at_(x2), at_(bias), to_(dx), f32w(part), to_(db), !f32out, R, static_cast<int>(C), act, grid, st);
    });
    return wrap_all(act ? like_shape(dx, x) : dy, db);
  });
}

// ---------------------------------------------------------------------------------------------
// rotary embedding, SwiGLU
// ---------------------------------------------------------------------------------------------
PyObject* qknorm_rope_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 10);
    const Tensor& qkv = in.tensor();
    const int nq = static_cast<int>(in.integer()), nkv = static_cast<int>(in.integer()), D = static_cast<int>(in.integer());
    const Tensor wq = in.optional(), wk = in.optional();
    const Tensor &cos = in.tensor(), &sin = in.tensor();
    const double eps = in.real();
    const bool norm = in.flag();
    const long long T = qkv.size(0);
    const auto dt = qkv.scalar_type();
    const Tensor q = empty({T, nq, D}, dt, qkv), k = empty({T, nkv, D}, dt, qkv), rstd = empty({T * (nq + nkv)}, at::kFloat, qkv);
    launch("ttb_qknorm_rope_fwd", 1, [&](void* st) {
      return ttb_qknorm_rope_fwd(at_(qkv), qkv.stride(0), nq, nkv, D, at_(wq), at_(wk), f32(cos), f32(sin), to_(q), to_(k), f32w(rstd), T,
                                 static_cast<float>(eps), norm, st);
    });
    return wrap_all(q, k, rstd);
  });
}

PyObject* qknorm_rope_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 15);
    const Tensor &dq = in.tensor(), &dk = in.tensor();
    const Tensor dv = in.optional();
    const Tensor& qkv = in.tensor();
    const int nq = static_cast<int>(in.integer()), nkv = static_cast<int>(in.integer()), D = static_cast<int>(in.integer());
    const Tensor wq = in.optional(), wk = in.optional();
    const Tensor &cos = in.tensor(), &sin = in.tensor(), &rstd = in.tensor(), &dqkv = in.tensor();
    const bool norm = in.flag(), f32out = in.flag();
    const long long T = qkv.size(0), groups = (nq + nkv * (dv.defined() ? 2 : 1) + 3) / 4;     // a warp takes four heads of a token
    const int grid = static_cast<int>(std::max<long long>(1, std::min<long long>((T * groups + 7) / 8, 4 * sms(qkv))));
    const Tensor dw = norm && T ? empty({2, D}, out_type(f32out), qkv) : at::zeros({2, D}, plain(qkv).dtype(out_type(f32out)));
    const Tensor part = norm ? empty({grid, 2 * D}, at::kFloat, qkv) : Tensor();
    launch("ttb_qknorm_rope_bwd", norm ? 2 : 1, [&](void* st) {
      return ttb_qknorm_rope_bwd(at_(dq), at_(dk), at_(dv), at_(qkv), qkv.stride(0), nq, nkv, D, at_(wq), at_(wk), f32(cos), f32(sin), f32(rstd),
                                 to_(dqkv), dqkv.stride(0), f32w(part), to_(dw), !f32out, T, norm, grid, st);
    });
    return wrap_all(dw.select(0, 0), dw.select(0, 1));
  });
}

PyObject* qkv_rope_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 5);
    const Tensor &x = in.tensor(), &bias = in.tensor();
    const int heads = static_cast<int>(in.integer());
    const Tensor &cos = in.tensor(), &sin = in.tensor();
    const long long T = x.size(0), D = x.size(1) / (3 * heads);
    need(x.dim() == 2 && x.is_contiguous() && bias.is_contiguous() && bias.numel() == x.size(1) && D * 3 * heads == x.size(1), "a row is q, k and v of all heads");
    const auto dt = x.scalar_type();
    const Tensor q = empty({T, heads, D}, dt, x), k = empty({T, heads, D}, dt, x), v = empty({T, heads, D}, dt, x);
    launch("ttb_qkv_rope_fwd", 1, [&](void* st) {
      return ttb_qkv_rope_fwd(at_(x), at_(bias), f32(cos), f32(sin), to_(q), to_(k), to_(v), T, heads, static_cast<int>(D / 2),
                              static_cast<int>(std::max<long long>(1, std::min<long long>(T, 4 * sms(x)))), st);
    });
    return wrap_all(q, k, v);
  });
}

PyObject* qkv_rope_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 6);
    const Tensor &dq = in.tensor(), &dk = in.tensor(), &dv = in.tensor(), &cos = in.tensor(), &sin = in.tensor();
    const bool f32out = in.flag();
    const long long T = dq.size(0), heads = dq.size(1), D = dq.size(2), W = 3 * heads * D;
    need(dq.is_contiguous() && dk.is_contiguous() && dv.is_contiguous() && dk.sizes() == dq.sizes() && dv.sizes() == dq.sizes(), "gradients of one shape");
    const int grid = static_cast<int>(std::max<long long>(1, std::min<long long>(T, 2 * sms(dq))));
    const Tensor dx = empty({T, W}, dq.scalar_type(), dq), part = empty({grid, W}, at::kFloat, dq);
    const Tensor db = T ? empty({W}, out_type(f32out), dq) : at::zeros({W}, plain(dq).dtype(out_type(f32out)));
    launch("ttb_qkv_rope_bwd", 2, [&](void* st) {
      return ttb_qkv_rope_bwd(at_(dq), at_(dk), at_(dv), f32(cos), f32(sin), to_(dx), f32w(part), to_(db), !f32out, T, static_cast<int>(heads),
                              static_cast<int>(D / 2), grid, st);
    });
    return wrap_all(dx, db);
  });
}

PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 4);
    const Tensor &x = in.tensor(), &cos = in.tensor(), &sin = in.tensor();
    const double sign = in.real();
    const long long T = x.size(0), heads = x.size(1), D = x.size(2);
    const Tensor y = empty({T, heads, D}, x.scalar_type(), x);
    launch("ttb_rope", 1, [&](void* st) {
      return ttb_rope(at_(x), x.stride(0), x.stride(1), f32(cos), f32(sin), to_(y), T, static_cast<int>(heads), static_cast<int>(D / 2),
                      static_cast<float>(sign), st);
    });
    return wrap(y);
  });
}

PyObject* swiglu_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 3);
    const Tensor& x = in.tensor();
    const Tensor scale = in.optional(), nrows = in.optional();
    const long long R = x.size(0), F = x.size(1) / 2;
    const Tensor y = empty({R, F}, x.scalar_type(), x);
    launch("ttb_swiglu_fwd", 1, [&](void* st) {
      return ttb_swiglu_fwd(at_(x), x.stride(0), to_(y), y.stride(0), f32(scale), R, static_cast<int>(F), i32(nrows), st);
    });
    return wrap(y);
  });
}

PyObject* swiglu_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 6);
    const Tensor &dy = in.tensor(), &x = in.tensor();
    const Tensor scale = in.optional();
    const bool want = in.flag();
    const Tensor nrows = in.optional(), y = in.optional();
    const long long R = x.size(0), F = x.size(1) / 2;
    const Tensor dx = at::empty_like(x, plain(x)), ds = want ? empty({R}, at::kFloat, x) : Tensor();
    launch("ttb_swiglu_bwd", 1, [&](void* st) {
      return ttb_swiglu_bwd(at_(dy), dy.stride(0), at_(x), x.stride(0), f32(scale), to_(dx), dx.stride(0), f32w(ds), to_(y),
                            y.defined() ? y.stride(0) : 0, R, static_cast<int>(F), i32(nrows), st);
    });
    return wrap_all(dx, ds);
  });
}

// ---------------------------------------------------------------------------------------------
// gates of a gated delta net
// ---------------------------------------------------------------------------------------------
bool plain_type(const Tensor& t) { return is_bf16(t) || t.scalar_type() == at::kFloat; }

PyObject* gdn_gate_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 4);
    const Tensor &a = in.tensor(), &b = in.tensor(), &A = in.tensor(), &dt = in.tensor();
    const long long T = a.size(0), H = a.size(1);
    need(is_bf16(a) && is_bf16(b) && b.sizes() == a.sizes() && (H == 1 || (a.stride(1) == 1 && b.stride(1) == 1)), "projections: bf16 rows of heads");
    need(A.numel() == H && dt.numel() == H && A.is_contiguous() && dt.is_contiguous() && plain_type(A) && plain_type(dt), "one value per head");
    const Tensor g = empty({T, H}, at::kFloat, a), beta = empty({T, H}, at::kFloat, a);
    launch("ttb_gdn_gate_fwd", 1, [&](void* st) {
      return ttb_gdn_gate_fwd(at_(a), a.stride(0), at_(b), b.stride(0), at_(A), is_bf16(A), at_(dt), is_bf16(dt), f32w(g), f32w(beta), T,
                              static_cast<int>(H), st);
    });
    return wrap_all(g, beta);
  });
}

PyObject* gdn_gate_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 7);
    const Tensor &dg = in.tensor(), &dbeta = in.tensor(), &a = in.tensor(), &A = in.tensor(), &dt = in.tensor(), &beta = in.tensor();
    const bool f32out = in.flag();
    const long long T = a.size(0), H = a.size(1);
    need(dg.is_contiguous() && dbeta.is_contiguous() && dg.scalar_type() == at::kFloat && dbeta.scalar_type() == at::kFloat, "gradients: fp32 rows of heads");
    const int blocks = static_cast<int>(std::max<long long>(1, std::min<long long>((T + 7) / 8, 2 * sms(a))));
    const Tensor da = empty({T, H}, at::kBFloat16, a), db = empty({T, H}, at::kBFloat16, a), part = empty({blocks, 2, H}, at::kFloat, a);
    const Tensor sums = T ? empty({2, H}, out_type(f32out), a) : at::zeros({2, H}, plain(a).dtype(out_type(f32out)));
    launch("ttb_gdn_gate_bwd", 2, [&](void* st) {
      return ttb_gdn_gate_bwd(f32(dg), f32(dbeta), at_(a), a.stride(0), at_(A), is_bf16(A), at_(dt), is_bf16(dt), f32(beta), to_(da), to_(db),
                              f32w(part), to_(sums), !f32out, T, static_cast<int>(H), blocks, st);
    });
    return wrap_all(da, db, sums.select(0, 0), sums.select(0, 1));
  });
}

// ---------------------------------------------------------------------------------------------
// a tensor times a factor on the device
// ---------------------------------------------------------------------------------------------
PyObject* scale(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 3);
    const Tensor &x = in.tensor(), &g = in.tensor();
    const bool bf16 = in.flag();
    check_device(x);
    check_device(g);
    need(x.is_contiguous() && (is_bf16(x) || x.scalar_type() == at::kFloat), "scale: a contiguous bf16 or fp32 tensor");
    need(g.numel() == 1 && g.scalar_type() == at::kFloat, "scale: one fp32 factor");
    const Tensor out = empty(x.sizes(), bf16 ? at::kBFloat16 : at::kFloat, x);
    launch("ttb_scale", 1, [&](void* st) { return ttb_scale(at_(x), is_bf16(x), f32(g), to_(out), bf16, x.numel(), sms(x), st); });
    return wrap(out);
  });
}

// ---------------------------------------------------------------------------------------------
// tables between pinned host memory and the device
// ---------------------------------------------------------------------------------------------
PyObject* copy_words(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 2);
    const Tensor &dst = in.tensor(), &src = in.tensor();
    const long long bytes = static_cast<long long>(src.nbytes());
    need(dst.scalar_type() == src.scalar_type() && dst.numel() == src.numel() && dst.is_contiguous() && src.is_contiguous() && bytes % 4 == 0,
         "copy_words: two contiguous tensors of one type and of whole 32-bit words");
    for (const Tensor* t : {&dst, &src})
      if (t->is_cuda()) check_device(*t);
      else need(t->is_pinned(), "copy_words: host memory has to be pinned");
    launch("ttb_copy_words", 1, [&](void* st) { return ttb_copy_words(to_(dst), at_(src), bytes / 4, st); });
    // as a copy by torch does: pinned memory that is freed is not handed out again before the stream is past this launch
    for (const Tensor* t : {&dst, &src})
      if (!t->is_cuda()) {
        const auto& data = t->storage().data_ptr();
        at::getHostAllocator(at::kCUDA)->record_event(t->data_ptr(), data.get_context(), at::cuda::getCurrentCUDAStream().unwrap());
      }
    Py_RETURN_NONE;
  });
}

// ---------------------------------------------------------------------------------------------
// Kimi delta attention gate
// ---------------------------------------------------------------------------------------------
PyObject* kda_gate_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 5);
    const Tensor &g = in.tensor(), &A = in.tensor();
    const Tensor dt = in.optional();
    const bool bounded = in.flag();
    const double bound = in.real();
    const Tensor out = empty(g.sizes(), at::kFloat, g);
    launch("ttb_kda_gate_fwd", 1, [&](void* st) {
      return ttb_kda_gate_fwd(at_(g), at_(A), is_bf16(A), at_(dt), dt.defined() && is_bf16(dt), f32w(out), g.size(0), static_cast<int>(g.size(1)),
                              bounded, static_cast<float>(bound), st);
    });
    return wrap(out);
  });
}

PyObject* kda_gate_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 6);
    const Tensor &dd = in.tensor(), &g = in.tensor(), &A = in.tensor();
    const Tensor dt = in.optional();
    const bool bounded = in.flag();
    const double bound = in.real();
    const long long R = g.size(0), H = g.size(1), D = g.size(2);
    const int blocks = kda_gate_row_blocks(R, static_cast<int>(H));
    const Tensor dg = empty_rows(g), part = empty({std::max(blocks, 1), 2, H * D}, at::kFloat, g);
    const Tensor sums = R ? empty({2, H * D}, at::kFloat, g) : at::zeros({2, H * D}, plain(g).dtype(at::kFloat));
    launch("ttb_kda_gate_bwd", 2, [&](void* st) {
      return ttb_kda_gate_bwd(f32(dd), at_(g), at_(A), is_bf16(A), at_(dt), dt.defined() && is_bf16(dt), to_(dg), f32w(part), f32w(sums), R,
                              static_cast<int>(H), bounded, static_cast<float>(bound), st);
    });
    return wrap_all(dg, sums.select(0, 0), sums.select(0, 1).view({H, D}));
  });
}

// ---------------------------------------------------------------------------------------------
// delta rule
// ---------------------------------------------------------------------------------------------
// q, k, v, g, beta, chunk_rows of a call and what the kernels make of them (kernels.delta_prep)
struct DeltaIn {
  const Tensor &q, &k, &v, &g, &beta, &rows;
  ttb::DeltaChunkIn in{};
  explicit DeltaIn(Args& a) : q(a.tensor()), k(a.tensor()), v(a.tensor()), g(a.tensor()), beta(a.tensor()), rows(a.tensor()) {}
  // l2 and scale are a call's last arguments
  const ttb::DeltaChunkIn* fill(Args& a) {
    const bool l2 = a.flag();
    const double scale = a.real();
    need(v.dim() == 3 && q.dim() == 3 && k.dim() == 3 && rows.dim() == 2, "rows of heads");
    const long long R = v.size(0), H = v.size(1), Hk = q.size(1);
    check_device(q);
    auto heads = [&](const Tensor& t, long long n) { return is_bf16(t) && t.size(0) == R && t.size(1) == n && t.size(2) == 128 && t.stride(2) == 1; };
    need(heads(q, Hk) && heads(k, Hk) && heads(v, H), "q, k, v: bf16 rows of 128-wide heads");
    need(Hk > 0 && H % Hk == 0 && (Hk == H || g.dim() == 2), "key heads");
    need(g.scalar_type() == at::kFloat && g.is_contiguous() && (g.dim() == 2 || (g.dim() == 3 && g.size(2) == 128)) && g.size(0) == R && g.size(1) == H, "log decay");
    need(beta.scalar_type() == at::kFloat && beta.is_contiguous() && beta.dim() == 2 && beta.size(0) == R && beta.size(1) == H, "step size");
    need(rows.scalar_type() == at::kInt && rows.is_contiguous() && rows.size(1) == 3, "chunk table");
    auto bf = [](const Tensor& t) { return static_cast<const __nv_bfloat16*>(at_(t)); };
    in.q = bf(q); in.k = bf(k); in.v = bf(v);
    in.q_t = q.stride(0); in.q_h = q.stride(1);
    in.k_t = k.stride(0); in.k_h = k.stride(1);
    in.v_t = v.stride(0); in.v_h = v.stride(1);
    in.g = f32(g); in.beta = f32(beta); in.chunk_rows = i32(rows);
    in.H = static_cast<int>(H); in.NC = static_cast<int>(rows.size(0)); in.l2 = l2; in.scale = static_cast<float>(scale);
    in.rep = static_cast<int>(H / Hk);
    return &in;
  }
  bool vec() const { return g.dim() == 3; }
};

PyObject* delta_prep(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 8);
    DeltaIn d(in);
    const ttb::DeltaChunkIn* a = d.fill(in);
    const long long H = a->H, NC = a->NC;
    const Tensor tri = empty({2, H, NC, 64, 64}, at::kFloat, d.q), u = empty({H, NC, 64, 128}, at::kFloat, d.q);
    const Tensor wk = empty({2, H, NC, 64, 128}, at::kBFloat16, d.q), decay = d.vec() ? empty({H, NC, 128}, at::kFloat, d.q) : empty({H, NC}, at::kFloat, d.q);
    const Tensor T = tri.select(0, 0), A = tri.select(0, 1), w = wk.select(0, 0), k_out = wk.select(0, 1);
    launch(d.vec() ? "ttb_delta_vec_prep" : "ttb_delta_prep", 1, [&](void* st) {
      if (d.vec()) return ttb_delta_vec_prep(a, f32w(T), f32w(A), f32w(u), to_(w), to_(k_out), f32w(decay), st);
      return ttb_delta_prep(a, f32w(T), f32w(A), f32w(u), to_(w), to_(k_out), f32w(decay), st);
    });
    return wrap_all(T, A, u, w, k_out, decay);
  });
}

PyObject* delta_out(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 11);
    DeltaIn d(in);
    const Tensor &A = in.tensor(), &x = in.tensor(), &states = in.tensor();
    const ttb::DeltaChunkIn* a = d.fill(in);
    const Tensor o = empty(d.v.sizes(), at::kBFloat16, d.q);
    launch(d.vec() ? "ttb_delta_vec_out" : "ttb_delta_out", 1, [&](void* st) {
      if (d.vec()) return ttb_delta_vec_out(a, f32(A), f32(x), f32(states), static_cast<int>(states.size(1)) - a->NC, to_(o), st);
      return ttb_delta_out(a, f32(A), f32(x), f32(states), static_cast<int>(states.size(1)) - a->NC, to_(o), st);
    });
    return wrap(o);
  });
}

PyObject* delta_bwd_pre(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 11);
    DeltaIn d(in);
    const Tensor &dout = in.tensor(), &A = in.tensor();
    const int nseq = static_cast<int>(in.integer());
    const ttb::DeltaChunkIn* a = d.fill(in);
    need(dout.is_contiguous() && is_bf16(dout) && dout.sizes() == d.v.sizes(), "the gradient has v's shape");
    const Tensor gx = empty({a->H, a->NC, 64, 128}, at::kFloat, d.q), gs = empty({a->H, a->NC + nseq, 128, 128}, at::kFloat, d.q);
    launch(d.vec() ? "ttb_delta_vec_bwd_pre" : "ttb_delta_bwd_pre", 1, [&](void* st) {
      if (d.vec()) return ttb_delta_vec_bwd_pre(a, at_(dout), f32(A), nseq, f32w(gx), f32w(gs), st);
      return ttb_delta_bwd_pre(a, at_(dout), f32(A), nseq, f32w(gx), f32w(gs), st);
    });
    return wrap_all(gx, gs);
  });
}

PyObject* delta_state_scan(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 11);
    const Tensor &a = in.tensor(), &b = in.tensor(), &u0 = in.tensor(), &decay0 = in.tensor();
    const Tensor init0 = in.optional(), add0 = in.optional();
    const Tensor& seq0 = in.tensor();
    const int reverse = static_cast<int>(in.integer());
    const double s1 = in.real(), s2 = in.real();
    const int longest = static_cast<int>(in.integer());
    need(u0.dim() == 4 && seq0.dim() == 2 && (decay0.dim() == 2 || decay0.dim() == 3), "chunks of 64 rows");
    const long long H = u0.size(0), NC = u0.size(1), nseq = seq0.size(0);
    need(u0.size(2) == 64 && u0.size(3) == 128 && a.sizes() == u0.sizes() && b.sizes() == u0.sizes(), "chunks of 64 rows");
    need(is_bf16(a) && is_bf16(b) && u0.scalar_type() == at::kFloat && a.is_contiguous() && b.is_contiguous() && u0.is_contiguous(), "operands");
    need(decay0.is_contiguous() && decay0.scalar_type() == at::kFloat && decay0.size(0) == H && decay0.size(1) == NC, "decay");
    need(seq0.scalar_type() == at::kInt && seq0.is_contiguous() && seq0.size(1) == 2, "sequence table");
    check_device(u0);
    // the copy engine moves whole rows: tensors that start between 16-byte boundaries are copied
    auto placed = [](const Tensor& t) {
      if (!t.defined()) return t;
      const Tensor c = t.contiguous();
      return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 ? c.clone() : c;
    };
    const Tensor u = placed(u0), decay = placed(decay0), init = placed(init0), add = placed(add0), seq = placed(seq0);
    auto states_like = [&](const Tensor& t, long long slots) {
      return t.scalar_type() == at::kFloat && t.dim() == 4 && t.size(0) == H && t.size(1) == slots && t.size(2) == 128 && t.size(3) == 128;
    };
    need(!init.defined() || states_like(init, nseq), "first states");
    need(!add.defined() || states_like(add, NC + nseq), "added gradients");
    const Tensor x = empty_rows(u), states = empty({H, NC + nseq, 128, 128}, at::kFloat, u);
    launch("ttb_delta_state_scan", 1, [&](void* st) {
      return ttb_delta_state_scan(at_(a), at_(b), f32(u), f32w(x), f32(decay), decay.dim() == 3, f32(init), f32(add), f32w(states), i32(seq),
                                  static_cast<int>(nseq), static_cast<int>(H), static_cast<int>(NC), longest, reverse, static_cast<float>(s1),
                                  static_cast<float>(s2), st);
    });
    return wrap_all(x, states);
  });
}

// ---------------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------------
// Rows that no sequence covers read as zero; [lo, hi) = covered rows, lo < 0 = unknown.
void zero_outside(const Tensor& t, long long lo, long long hi) {
  const long long rows = t.size(0);
  if (lo < 0) {
    t.zero_();
    return;
  }
  if (lo > 0) t.narrow(0, 0, std::min(lo, rows)).zero_();
  if (hi < rows) t.narrow(0, hi, rows - hi).zero_();
}
bool head_widths(long long D, long long Dv) { return (D <= 128 && Dv <= 128 && D % 8 == 0 && Dv % 8 == 0) || (D == 192 && Dv == 128); }

PyObject* attn_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 11);
    const Tensor &q = in.tensor(), &k = in.tensor(), &v = in.tensor(), &tiles = in.tensor();
    const double scale = in.real();
    const bool causal = in.flag(), want_lse = in.flag(), want_max = in.flag();
    const long long lo = in.integer(), hi = in.integer();
    const int tile_rows = static_cast<int>(in.integer());
    const long long T = q.size(0), Hq = q.size(1), D = q.size(2), Hk = k.size(1), Dv = v.size(2);
    need(k.size(2) == D && head_widths(D, Dv), "head widths");
    need(q.stride(2) == 1 && q.stride(1) == D && k.stride(1) == D && k.stride(2) == 1 && v.stride(1) == Dv && v.stride(2) == 1, "heads must lie in a row");
    const Tensor out = empty({T, Hq, Dv}, q.scalar_type(), q);
    zero_outside(out, lo, hi);
    const auto f = plain(q).dtype(at::kFloat);
    const bool all = lo == 0 && hi == T;             // every row's logsumexp is written
    const Tensor lse = !want_lse ? Tensor() : all ? at::empty({Hq, T}, f) : at::full({Hq, T}, -INFINITY, f);
    const Tensor ml = want_max ? at::full({Hq}, -INFINITY, f) : Tensor();
    launch("ttb_attn_fwd", 1, [&](void* st) {
      return ttb_attn_fwd(at_(q), q.stride(0), at_(k), k.stride(0), at_(v), v.stride(0), to_(out), f32w(lse), f32w(ml), i32(tiles),
                          static_cast<int>(tiles.size(0)), tile_rows, T, static_cast<int>(Hq), static_cast<int>(Hk), static_cast<int>(D),
                          static_cast<int>(Dv), static_cast<float>(scale), causal, st);
    });
    return wrap_all(out, lse, ml);
  });
}

PyObject* attn_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 13);
    const Tensor &dout = in.tensor(), &q = in.tensor(), &k = in.tensor(), &v = in.tensor(), &out = in.tensor(), &lse = in.tensor(), &kv = in.tensor();
    const double scale = in.real();
    const bool causal = in.flag();
    const Tensor q_tiles = in.optional();
    const bool deterministic = in.flag();
    const long long lo = in.integer(), hi = in.integer();
    const long long T = q.size(0), Hq = q.size(1), D = q.size(2), Hk = k.size(1), Dv = v.size(2);
    need(dout.is_contiguous() && out.is_contiguous() && q.is_contiguous(), "rows must be contiguous");
    need(k.stride(1) == D && k.stride(2) == 1 && v.stride(1) == Dv && v.stride(2) == 1, "heads must lie in a row");
    const bool split = deterministic || D > 128;
    if (split && !q_tiles.defined()) fail(PyExc_ValueError, "the query-major dQ pass needs the query tile table");
    const auto dt = plain(q);
    const auto f = dt.dtype(at::kFloat);
    if (kv.size(0) == 0)                             // no sequence covers a row
      return wrap_all(at::zeros(q.sizes(), dt), at::zeros({T, Hk, D}, dt), at::zeros({T, Hk, Dv}, dt));
    const Tensor delta = at::empty({Hq * T}, f);
    Tensor dq_acc, dk_acc, dv_acc, dq, dk, dv;
    const bool grouped = Hq != Hk && !deterministic;
    if (grouped) {
      // query heads of a group add into fp32 accumulators, cleared by the first launch and converted by the last; accumulators and
      // results lie back to back, so that they are converted in one
      const long long nq = split ? 0 : T * Hq * D, nk = T * Hk * D, nv = T * Hk * Dv;
      const Tensor acc = at::empty({nq + nk + nv}, f), res = at::empty({nq + nk + nv}, dt);
      auto part = [T](const Tensor& t, long long first, long long H, long long W) { return t.narrow(0, first, T * H * W).view({T, H, W}); };
      if (split) {
        dq = empty_rows(q);
        zero_outside(dq, lo, hi);
      } else {
        dq_acc = part(acc, 0, Hq, D); dq = part(res, 0, Hq, D);
      }
      dk_acc = part(acc, nq, Hk, D); dk = part(res, nq, Hk, D);
      dv_acc = part(acc, nq + nk, Hk, Dv); dv = part(res, nq + nk, Hk, Dv);
    } else {
      if (!split) dq_acc = at::empty({T, Hq, D}, f);
      dq = empty_rows(q);
      if (split) zero_outside(dq, lo, hi);
      dk = at::empty({T, Hk, D}, dt); zero_outside(dk, lo, hi);
      dv = at::empty({T, Hk, Dv}, dt); zero_outside(dv, lo, hi);
    }
    launch("ttb_attn_bwd", !split || grouped ? 3 : 2, [&](void* st) {
      return ttb_attn_bwd(at_(q), at_(k), k.stride(0), at_(v), v.stride(0), at_(out), at_(dout), f32(lse), f32w(delta), f32w(dq_acc), f32w(dk_acc),
                          f32w(dv_acc), to_(dq), to_(dk), to_(dv), i32(kv), static_cast<int>(kv.size(0)), T, static_cast<int>(Hq),
                          static_cast<int>(Hk), static_cast<int>(D), static_cast<int>(Dv), static_cast<float>(scale), causal,
                          split ? (deterministic ? 2 : 0) : 1, st);
    });
    if (split)
      launch("ttb_attn_bwd_dq", 1, [&](void* st) {
        return ttb_attn_bwd_dq(at_(q), at_(k), k.stride(0), at_(v), v.stride(0), at_(dout), f32(lse), f32(delta), to_(dq), i32(q_tiles),
                               static_cast<int>(q_tiles.size(0)), T, static_cast<int>(Hq), static_cast<int>(Hk), static_cast<int>(D),
                               static_cast<int>(Dv), static_cast<float>(scale), causal, st);
      });
    return wrap_all(dq, dk, dv);
  });
}

PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args in(args, n, 3);
    for (int i = 0; i < 3; ++i) Py_INCREF(args[i]);
    g_kernel_error = args[0];
    g_oom_error = args[1];
    g_gemm_splits = args[2];
    Py_RETURN_NONE;
  });
}
PyObject* launches(PyObject*, PyObject* const*, Py_ssize_t) { return PyLong_FromLongLong(g_launches.load(std::memory_order_relaxed)); }

#define ENTRY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(setup), ENTRY(launches), ENTRY(gemm), ENTRY(linear_tail), ENTRY(tail_bwd), ENTRY(linear_tail_bwd), ENTRY(dropout), ENTRY(logprobs_fwd),
                         ENTRY(logprobs_dlogits), ENTRY(scatter_rows), ENTRY(rmsnorm_fwd), ENTRY(rmsnorm_bwd), ENTRY(layernorm_fwd), ENTRY(layernorm_bwd),
                         ENTRY(bias_act_fwd), ENTRY(bias_act_bwd), ENTRY(qknorm_rope_fwd), ENTRY(qknorm_rope_bwd), ENTRY(qkv_rope_fwd), ENTRY(qkv_rope_bwd), ENTRY(gdn_gate_fwd),
                         ENTRY(gdn_gate_bwd), ENTRY(scale), ENTRY(copy_words), ENTRY(kda_gate_fwd), ENTRY(kda_gate_bwd), ENTRY(delta_prep), ENTRY(delta_out), ENTRY(delta_bwd_pre),
                         ENTRY(delta_state_scan), ENTRY(rope), ENTRY(swiglu_fwd),
                         ENTRY(swiglu_bwd), ENTRY(attn_fwd), ENTRY(attn_bwd), {nullptr, nullptr, 0, nullptr}};
#undef ENTRY
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ttb_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_ttb_host() { return PyModule_Create(&module); }
