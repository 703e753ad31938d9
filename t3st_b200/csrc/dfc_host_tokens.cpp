// Host path of the token-table and dropout operators, part of the CPython
// extension t3st_b200._dfc_host: argument checks, outputs, scratch and autograd
// in C++ around the C ABI of libdfc_b200.so (dfc_dropout, dfc_embedding,
// dfc_embedding_grad, through function pointers handed over by the Python
// side).  A Python autograd.Function around ctypes calls cost 20 us a call,
// most of what a small batch takes.
//
// Every tensor stays on the stream that is current on its device; scratch
// comes from PyTorch's caching allocator on that stream, per call.

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/Event.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <atomic>
#include <cstdint>
#include <cstring>
#include <mutex>
#include <optional>
#include <vector>

#include "dfc_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

decltype(&dfc_dropout) f_dropout = nullptr;
decltype(&dfc_embedding) f_embedding = nullptr;
decltype(&dfc_embedding_grad_scratch_bytes) f_scratch = nullptr;
decltype(&dfc_embedding_grad) f_grad = nullptr;
PyObject* check_status = nullptr;  // _lib.check(name, status): raises

// Before anything else in a call: the addresses are there (set together).
void check_bound() {
  TORCH_CHECK(f_grad, "t3st_b200._dfc_host is not bound to the kernels; use it through t3st_b200._lib.host()");
}

// A non-zero status as the exception of the Python layer.
void check(const char* name, int status) {
  if (status == DFC_OK) return;
  pybind11::gil_scoped_acquire gil;
  PyObject* r = PyObject_CallFunction(check_status, "si", name, status);
  Py_XDECREF(r);
  TORCH_CHECK(r == nullptr, name, " failed with status ", status);
  python_error e;
  e.persist();
  throw e;
}

// A mask's generator: seed and offset, or words on the device.
struct Mask {
  double p = 0.0;
  uint64_t seed = 0, offset = 0;
  Tensor state;  // undefined: seed counts

  void check() const {
    TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "dropout probability must be in [0, 1]");
    TORCH_CHECK_TYPE(!state.defined() || (state.scalar_type() == at::kLong && state.numel() == 2 &&
                                          state.is_contiguous()),
                     "the generator state must be two contiguous int64 values (seed, offset)");
  }

  // The C argument; NULL when nothing is dropped.
  const DfcDropout* arg(const at::Device& dev, DfcDropout* d) const {
    TORCH_CHECK(!state.defined() || state.device() == dev, "all tensors of one call must share a device");
    if (p == 0.0) return nullptr;
    *d = DfcDropout{seed, offset, nullptr, p};
    if (state.defined()) d->state = static_cast<const uint64_t*>(state.const_data_ptr());
    return d;
  }
};

int32_t dtype_code(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return DFC_DTYPE_F32;
    case at::kBFloat16: return DFC_DTYPE_BF16;
    case at::kHalf: return DFC_DTYPE_F16;
    default: TORCH_CHECK_TYPE(false, what, " must be FP32, bf16 or fp16");
  }
}

void check_devices(std::initializer_list<const Tensor*> ts) {
  const at::Device dev = (*ts.begin())->device();
  for (const Tensor* t : ts) {
    TORCH_CHECK(t->is_cuda(), "t3st_b200 kernels take CUDA tensors only");
    TORCH_CHECK(t->device() == dev, "all tensors of one call must share a device");
    TORCH_CHECK_TYPE(t->layout() == at::kStrided, "t3st_b200 kernels take strided tensors");
  }
}

void* stream_of(const at::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// ---- tokens outside the table ------------------------------------------------
// One int per device in pinned host memory that the kernels set and the next
// call reads, without waiting.  Backward passes read it from autograd's threads,
// without the interpreter's lock.
constexpr int kDevices = 64;
std::mutex flag_mutex;
std::array<Tensor, kDevices> flag_memory;  // under the mutex
std::array<std::atomic<int32_t*>, kDevices> flags{};

// Of several threads, one reports.
void check_flag(int device) {
  int32_t* f = device >= 0 && device < kDevices ? flags[device].load(std::memory_order_acquire) : nullptr;
  TORCH_CHECK_INDEX(!(f && __atomic_load_n(f, __ATOMIC_RELAXED) && __atomic_exchange_n(f, 0, __ATOMIC_RELAXED)),
                    "an earlier call was given a token outside [0, vocab): "
                    "its rows are NaN, its gradient lacks those tokens");
}

int32_t* flag_of(const at::Device& dev) {
  const int i = dev.index();
  TORCH_CHECK(i >= 0 && i < kDevices, "device index out of range");
  if (!flags[i].load(std::memory_order_acquire)) {
    std::lock_guard<std::mutex> lock(flag_mutex);
    if (!flags[i].load(std::memory_order_relaxed)) {
      TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None,
                  "call the token-table operators once on this device before capturing them: "
                  "the first call allocates pinned memory");
      flag_memory[i] = at::zeros({1}, at::TensorOptions().dtype(at::kInt)).pin_memory();
      flags[i].store(flag_memory[i].data_ptr<int32_t>(), std::memory_order_release);
    }
  }
  check_flag(i);
  return flags[i].load(std::memory_order_acquire);
}

// ---- the calls -----------------------------------------------------------------
void run_dropout(const Tensor& x, const Tensor& residual, const Tensor& out, const Mask& m) {
  check_bound();
  if (residual.defined()) check_devices({&x, &out, &residual});
  else check_devices({&x, &out});
  const int32_t code = dtype_code(x, "x");
  for (const Tensor* t : {&x, &out, &residual}) {
    if (!t->defined()) continue;
    TORCH_CHECK_TYPE(t->scalar_type() == x.scalar_type(), "x, out and residual must share a dtype");
    TORCH_CHECK_VALUE(t->sizes() == x.sizes(), "shapes differ");
    TORCH_CHECK_VALUE(t->is_contiguous(), "tensors must be contiguous");
  }
  DfcDropout d;
  const DfcDropout* arg = m.arg(x.device(), &d);
  const c10::cuda::CUDAGuard guard(x.device());
  check("dfc_dropout", f_dropout(x.const_data_ptr(), residual.defined() ? residual.const_data_ptr() : nullptr,
                                 out.mutable_data_ptr(), x.numel(), code, arg, stream_of(x.device())));
}

int32_t token_bytes(const Tensor& tokens) {
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kInt || tokens.scalar_type() == at::kLong,
                   "tokens must be int32 or int64");
  TORCH_CHECK_VALUE(tokens.is_contiguous(), "tokens must be contiguous");
  return static_cast<int32_t>(tokens.element_size());
}

// (Without elements any strides will do; contiguous() would not change them.)
bool row_matrix(const Tensor& t) {
  return t.dim() == 2 && (t.numel() == 0 || t.size(1) <= 1 || t.stride(1) == 1);
}

// Elements between the rows of a matrix whose rows are contiguous.
int64_t row_pitch(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(row_matrix(t), what, " must be a matrix with contiguous rows");
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

// A gradient of looked-up rows, of any shape, as one row per token.
Tensor token_rows(const Tensor& dy, int64_t n, int64_t dim) {
  return row_matrix(dy) ? dy : dy.reshape({n, dim}).contiguous();
}

void run_embedding(const Tensor& tokens, const Tensor& table, const Tensor& out, double scale, const Mask& m) {
  check_bound();
  check_devices({&tokens, &table, &out});
  const int32_t wide = token_bytes(tokens);
  const int64_t pitch = row_pitch(table, "table"), vocab = table.size(0), dim = table.size(1);
  TORCH_CHECK_VALUE(out.numel() == tokens.numel() * dim && (out.numel() == 0 || out.size(-1) == dim),
                    "out must hold one row of the table's width per token");
  TORCH_CHECK_VALUE(out.is_contiguous(), "out must be contiguous");
  const int32_t tc = dtype_code(table, "table"), oc = dtype_code(out, "out");
  DfcDropout d;
  const DfcDropout* arg = m.arg(table.device(), &d);
  const c10::cuda::CUDAGuard guard(table.device());
  check("dfc_embedding",
        f_embedding(tokens.const_data_ptr(), wide, tokens.numel(), table.const_data_ptr(), tc, pitch, vocab,
                    dim, static_cast<float>(scale), out.mutable_data_ptr(), oc, arg, flag_of(table.device()),
                    stream_of(table.device())));
}

// -1: none
int64_t padding_row(std::optional<int64_t> padding_idx, int64_t vocab) {
  if (!padding_idx) return -1;
  TORCH_CHECK_VALUE(*padding_idx >= -vocab && *padding_idx < vocab, "padding_idx must be within the table");
  return *padding_idx < 0 ? *padding_idx + vocab : *padding_idx;
}

void run_grad(const Tensor& tokens, const Tensor& dy, const Tensor& grad, double scale, int64_t padding,
              const Mask& m, bool accumulate) {
  check_bound();
  check_devices({&tokens, &dy, &grad});
  const int32_t wide = token_bytes(tokens);
  const int64_t n = tokens.numel();
  const int64_t dy_pitch = row_pitch(dy, "dy"), grad_pitch = row_pitch(grad, "grad");
  const int64_t vocab = grad.size(0), dim = grad.size(1);
  TORCH_CHECK_VALUE(dy.size(0) == n && dy.size(1) == dim, "dy must hold one row of grad's width per token");
  TORCH_CHECK_VALUE(grad_pitch >= dim, "grad's rows overlap");
  const int32_t dc = dtype_code(dy, "dy"), gc = dtype_code(grad, "grad");
  const at::Device dev = grad.device();
  DfcDropout d;
  const DfcDropout* arg = m.arg(dev, &d);
  const c10::cuda::CUDAGuard guard(dev);
  const size_t bytes = f_scratch(n, vocab, dim);
  const Tensor scratch = at::empty({static_cast<int64_t>(bytes < 16 ? 16 : bytes)}, grad.options().dtype(at::kByte));
  check("dfc_embedding_grad",
        f_grad(tokens.const_data_ptr(), wide, n, dy.const_data_ptr(), dc, dy_pitch, grad.mutable_data_ptr(), gc,
               grad_pitch, vocab, dim, static_cast<float>(scale), padding, accumulate, arg, flag_of(dev),
               scratch.mutable_data_ptr(), bytes, stream_of(dev)));
}

// Graphs that saved the caller's buffer learn that it has been written.
// (Tensors of inference mode have no counter.)
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ---- autograd --------------------------------------------------------------------
// Scalars of a call, kept between forward and backward as one list.
struct Call {
  double scale = 1.0;
  int64_t padding = -1;
  Mask mask;

  std::vector<int64_t> save() const {
    std::vector<int64_t> v(5);
    std::memcpy(&v[0], &scale, 8);
    v[1] = padding;
    std::memcpy(&v[2], &mask.p, 8);
    v[3] = static_cast<int64_t>(mask.seed);
    v[4] = static_cast<int64_t>(mask.offset);
    return v;
  }
  static Call load(const std::vector<int64_t>& v, const Tensor& state) {
    Call c;
    std::memcpy(&c.scale, &v[0], 8);
    c.padding = v[1];
    std::memcpy(&c.mask.p, &v[2], 8);
    c.mask.seed = static_cast<uint64_t>(v[3]);
    c.mask.offset = static_cast<uint64_t>(v[4]);
    c.mask.state = state;
    return c;
  }
};

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& residual, Call call) {
    ctx->saved_data["call"] = call.save();
    ctx->saved_data["residual"] = residual.has_value();
    ctx->save_for_backward({call.mask.state});
    Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    run_dropout(x.contiguous(), residual ? residual->contiguous() : Tensor(), y, call.mask);
    return y;
  }
  // Linear in x, with the same mask both ways; the residual's gradient is dy.
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const Call call = Call::load(ctx->saved_data["call"].toIntVector(), ctx->get_saved_variables()[0]);
    Tensor dx;
    if (dy[0].defined() && ctx->needs_input_grad(0)) dx = Dropout::apply(dy[0], std::nullopt, call);
    return {dx, ctx->saved_data["residual"].toBool() ? dy[0] : Tensor(), Tensor()};
  }
};

// This backward pass adds to the leaf's .grad, does not hand the gradient to a
// caller of torch.autograd.grad, and nothing looks at the gradient on its way.
// (Hooks that run after the accumulation find it in .grad.)
bool accumulates(const Tensor& leaf) {
  const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (!accumulator || !accumulator->tensor_pre_hooks().empty() || !accumulator->pre_hooks().empty()) return false;
  const auto* only = torch::autograd::get_current_graph_task_exec_info();
  if (!only || only->empty()) return true;  // every leaf of the graph
  const auto info = only->find(accumulator.get());
  return info != only->end() && info->second.needed_;
}

// Autograd adds to a leaf's .grad on the stream of the leaf's accumulator, and
// backward() puts its caller's stream behind that one.  Rows added in place are
// added on the stream of the forward instead, which may be another one (where
// the accumulator was made by an earlier use of the leaf): it waits for what the
// accumulator's has done so far, and that one for the rows.
class AccumulatorOrder {
 public:
  explicit AccumulatorOrder(const Tensor& leaf) : here_(c10::cuda::getCurrentCUDAStream(leaf.device().index())) {
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(leaf);
    if (accumulator) there_ = accumulator->stream();
    if (there_ && (there_->device_type() != c10::DeviceType::CUDA || *there_ == here_)) there_.reset();
    if (!there_) return;
    TORCH_CHECK(capturing(here_) == capturing(*there_),
                "grad_in_place: this backward pass is captured, but the weight's gradient accumulator belongs to "
                "a graph that was made outside the capture; delete that graph first");
    order(*there_, here_);
  }
  void added() const {
    if (there_) order(here_, *there_);
  }

 private:
  static bool capturing(const c10::Stream& s) {
    const c10::cuda::CUDAStreamGuard guard(s);
    return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
  }
  static void order(const c10::Stream& first, const c10::Stream& then) {
    c10::Event e(c10::DeviceType::CUDA);
    e.record(first);
    e.block(then);
  }
  c10::Stream here_;
  std::optional<c10::Stream> there_;  // the accumulator's, if another
};

// The lookup and the table's gradient are each other's gradient.
Tensor table_grad(const Tensor& dy, const Tensor& tokens, at::IntArrayRef shape, at::ScalarType dtype,
                  const Call& call);

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& tokens, Call call,
                        at::ScalarType out_dtype, bool in_place) {
    TORCH_CHECK_VALUE(weight.dim() == 2, "weight must be a matrix");
    const Tensor flat = tokens.contiguous();
    ctx->saved_data["call"] = call.save();
    ctx->saved_data["table"] = std::vector<int64_t>{weight.size(0), weight.size(1),
                                                    static_cast<int64_t>(weight.scalar_type())};
    if (in_place) ctx->saved_data["leaf"] = weight;
    ctx->save_for_backward({flat, call.mask.state});
    std::vector<int64_t> sizes(tokens.sizes().begin(), tokens.sizes().end());
    sizes.push_back(weight.size(1));
    Tensor out = at::empty(sizes, weight.options().dtype(out_dtype));
    run_embedding(flat, weight, out, call.scale, call.mask);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dys) {
    const variable_list saved = ctx->get_saved_variables();
    const Call call = Call::load(ctx->saved_data["call"].toIntVector(), saved[1]);
    const std::vector<int64_t> table = ctx->saved_data["table"].toIntVector();
    Tensor dw;
    if (dys[0].defined() && ctx->needs_input_grad(0)) {
      const auto leaf = ctx->saved_data.find("leaf");
      Tensor into;
      if (leaf != ctx->saved_data.end() && accumulates(leaf->second.toTensor()))
        into = leaf->second.toTensor().grad();
      if (into.defined()) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "grad_in_place does not support create_graph");
        const Tensor dy = token_rows(dys[0], saved[0].numel(), table[1]);
        const AccumulatorOrder order(leaf->second.toTensor());
        run_grad(saved[0], dy, into, call.scale, call.padding, call.mask, true);
        order.added();
        written(into);
      } else {
        dw = table_grad(dys[0], saved[0], {table[0], table[1]}, static_cast<at::ScalarType>(table[2]), call);
      }
    }
    return {dw, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct TableGrad : torch::autograd::Function<TableGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& dy, const Tensor& tokens, std::vector<int64_t> shape,
                        at::ScalarType dtype, Call call) {
    ctx->saved_data["call"] = call.save();
    ctx->saved_data["dy"] = static_cast<int64_t>(dy.scalar_type());
    ctx->save_for_backward({tokens, call.mask.state});
    const Tensor rows = token_rows(dy, tokens.numel(), shape[1]);
    Tensor dw = at::empty(shape, dy.options().dtype(dtype).memory_format(at::MemoryFormat::Contiguous));
    run_grad(tokens, rows, dw, call.scale, call.padding, call.mask, false);
    return dw;
  }
  // The padding row gets no gradient, so none flows back from it: its rows are
  // looked up in a copy where it is zero.
  static variable_list backward(AutogradContext* ctx, variable_list ddw) {
    const variable_list saved = ctx->get_saved_variables();
    const Call call = Call::load(ctx->saved_data["call"].toIntVector(), saved[1]);
    Tensor ddy;
    if (ddw[0].defined() && ctx->needs_input_grad(0)) {
      Tensor w = ddw[0];
      if (call.padding >= 0) {
        w = w.clone();
        w.select(0, call.padding).zero_();
      }
      if (!row_matrix(w)) w = w.contiguous();
      ddy = Embedding::apply(w, saved[0], call, static_cast<at::ScalarType>(ctx->saved_data["dy"].toInt()), false);
    }
    return {ddy, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor table_grad(const Tensor& dy, const Tensor& tokens, at::IntArrayRef shape, at::ScalarType dtype,
                  const Call& call) {
  return TableGrad::apply(dy, tokens, shape.vec(), dtype, call);
}

// ---- Python arguments ----------------------------------------------------------------
const Tensor& tensor_arg(PyObject* o, const char* what) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be a tensor");
  return THPVariable_Unpack(o);
}

Tensor optional_tensor(PyObject* o, const char* what) { return o == Py_None ? Tensor() : tensor_arg(o, what); }

double double_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

int64_t int_arg(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

// Modulo 2^64.
uint64_t word_arg(PyObject* o) {
  const unsigned long long v = PyLong_AsUnsignedLongLongMask(o);
  if (v == ~0ull && PyErr_Occurred()) throw python_error();
  return v;
}

std::optional<int64_t> optional_int(PyObject* o) {
  return o == Py_None ? std::nullopt : std::optional<int64_t>(int_arg(o));
}

// p, seed, offset, state
Mask mask_arg(PyObject* const* a) {
  Mask m{double_arg(a[0]), word_arg(a[1]), word_arg(a[2]), optional_tensor(a[3], "state")};
  m.check();
  return m;
}

bool arity(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return false;
}

}  // namespace

PyObject* dfc_py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 5)) return nullptr;
  HANDLE_TH_ERRORS
  f_dropout = reinterpret_cast<decltype(f_dropout)>(word_arg(a[0]));
  f_embedding = reinterpret_cast<decltype(f_embedding)>(word_arg(a[1]));
  f_scratch = reinterpret_cast<decltype(f_scratch)>(word_arg(a[2]));
  f_grad = reinterpret_cast<decltype(f_grad)>(word_arg(a[3]));
  Py_INCREF(a[4]);
  Py_XSETREF(check_status, a[4]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// dropout(x, out, p, seed, offset, state, residual) -> out
PyObject* dfc_py_dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 7)) return nullptr;
  HANDLE_TH_ERRORS
  const Mask m = mask_arg(a + 2);
  run_dropout(tensor_arg(a[0], "x"), optional_tensor(a[6], "residual"), tensor_arg(a[1], "out"), m);
  written(THPVariable_Unpack(a[1]));
  Py_INCREF(a[1]);
  return a[1];
  END_HANDLE_TH_ERRORS
}

// embedding(tokens, table, out, scale, p, seed, offset, state) -> out
PyObject* dfc_py_embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 8)) return nullptr;
  HANDLE_TH_ERRORS
  const Mask m = mask_arg(a + 4);
  run_embedding(tensor_arg(a[0], "tokens"), tensor_arg(a[1], "table"), tensor_arg(a[2], "out"), double_arg(a[3]), m);
  written(THPVariable_Unpack(a[2]));
  Py_INCREF(a[2]);
  return a[2];
  END_HANDLE_TH_ERRORS
}

// embedding_grad(tokens, dy, grad, scale, padding_idx, p, seed, offset, state, accumulate) -> grad
PyObject* dfc_py_embedding_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 10)) return nullptr;
  HANDLE_TH_ERRORS
  const Tensor& grad = tensor_arg(a[2], "grad");
  row_pitch(grad, "grad");
  const Mask m = mask_arg(a + 5);
  const int accumulate = PyObject_IsTrue(a[9]);
  if (accumulate < 0) throw python_error();
  run_grad(tensor_arg(a[0], "tokens"), tensor_arg(a[1], "dy"), grad, double_arg(a[3]),
           padding_row(optional_int(a[4]), grad.size(0)), m, accumulate != 0);
  written(grad);
  Py_INCREF(a[2]);
  return a[2];
  END_HANDLE_TH_ERRORS
}

// check_tokens(device index)
PyObject* dfc_py_check_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 1)) return nullptr;
  HANDLE_TH_ERRORS
  check_flag(static_cast<int>(int_arg(a[0])));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// nn_dropout(x, p, seed, offset, state, residual) -> y, with its gradients
PyObject* dfc_py_nn_dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 6)) return nullptr;
  HANDLE_TH_ERRORS
  const Tensor& x = tensor_arg(a[0], "x");
  std::optional<Tensor> residual;
  if (a[5] != Py_None) {
    residual = tensor_arg(a[5], "residual");
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(),
                      "residual must have x's shape and dtype");
  }
  Call call;
  call.mask = mask_arg(a + 1);
  return THPVariable_Wrap(Dropout::apply(x, residual, call));
  END_HANDLE_TH_ERRORS
}

// nn_embedding(tokens, weight, scale, padding_idx, p, seed, offset, state, out_dtype, grad_in_place)
PyObject* dfc_py_nn_embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 10)) return nullptr;
  HANDLE_TH_ERRORS
  const Tensor& tokens = tensor_arg(a[0], "tokens");
  const Tensor& weight = tensor_arg(a[1], "weight");
  TORCH_CHECK_VALUE(weight.dim() == 2, "weight must be a matrix");
  Call call;
  call.scale = double_arg(a[2]);
  call.padding = padding_row(optional_int(a[3]), weight.size(0));
  call.mask = mask_arg(a + 4);
  at::ScalarType out = weight.scalar_type();
  if (a[8] != Py_None) {
    TORCH_CHECK_TYPE(THPDtype_Check(a[8]), "out_dtype must be a torch.dtype");
    out = reinterpret_cast<THPDtype*>(a[8])->scalar_type;
  }
  const int in_place = PyObject_IsTrue(a[9]);
  if (in_place < 0) throw python_error();
  TORCH_CHECK_VALUE(!in_place || weight.is_leaf(), "grad_in_place needs a leaf weight");
  return THPVariable_Wrap(Embedding::apply(weight, tokens, call, out, in_place != 0));
  END_HANDLE_TH_ERRORS
}
