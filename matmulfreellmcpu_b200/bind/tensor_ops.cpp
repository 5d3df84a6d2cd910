// tensor_ops.cpp -- the recurrent-block operators on torch tensors: checks a call's tensors,
// makes its outputs and calls the C ABI (include/mmfree_cuda.h) on the right device and stream.
//
// A CPython extension over the C ABI rather than ctypes: a step has up to twelve tensors, and
// reading their types, devices, shapes and strides from Python took 30 to 45 us a call, ten
// times as long as the kernel of one token. matmulfreellmcpu_b200/api.py documents the functions.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>

#include "mmfree_cuda.h"

namespace {

PyObject* g_error = nullptr;  // matmulfreellmcpu_b200.MmfreeError

struct Failure {
  int code;
  std::string message;
};

[[noreturn]] void refuse(const std::string& what) { throw Failure{MMFREE_E_INVALID, what}; }
inline void need(bool ok, const char* what) {
  if (!ok) refuse(what);
}
void check(int rc) {
  if (rc != MMFREE_OK) throw Failure{rc, mmfree_cuda_last_error()};
}

std::string shape_text(at::IntArrayRef s) {
  std::string t = "[";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + "]";
}

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MMFREE_T_F32;
    case at::kBFloat16: return MMFREE_T_BF16;
    case at::kHalf: return MMFREE_T_F16;
    case at::kChar: return MMFREE_T_S8;
    case at::kFloat8_e4m3fn: return MMFREE_T_E4M3;
    default: return -1;
  }
}

int row_type(at::ScalarType t, const char* name) {
  const int code = type_code(t);
  if (code < 0 || code > MMFREE_T_F16) refuse(std::string(name) + " must be float32, bfloat16 or float16");
  return code;
}

// One argument: a tensor, or None where `optional`.
struct Arg {
  const at::Tensor* t = nullptr;
  const char* name;

  Arg(PyObject* o, const char* n, bool optional = false) : name(n) {
    if (o == Py_None && optional) return;
    if (!THPVariable_Check(o)) refuse(std::string(n) + " must be a tensor");
    t = &THPVariable_Unpack(o);
    if (t->layout() != at::kStrided) refuse(std::string(n) + " must be a strided tensor");
    if (t->requires_grad() && at::GradMode::is_enabled())
      refuse(std::string(n) + " requires a gradient, and this operator has no backward pass");
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t->_fw_grad(0).defined())
      refuse(std::string(n) + " has a tangent, and this operator has no forward-mode gradient");
  }
  explicit operator bool() const { return t != nullptr; }
  void* data() const { return t ? t->data_ptr() : nullptr; }
  int64_t size(int64_t d) const { return t->size(d); }
  int64_t dim() const { return t->dim(); }

  void on(at::Device device) const {
    if (t->device() != device) refuse(std::string(name) + " is on " + t->device().str() + ", not on " + device.str());
  }
  void typed(at::ScalarType type) const {
    if (t->scalar_type() != type) refuse(std::string(name) + " must be " + at::toString(type) + ", not " + at::toString(t->scalar_type()));
  }
  void shaped(at::IntArrayRef want) const {
    if (t->sizes() != want) refuse(std::string(name) + " must be " + shape_text(want) + ", not " + shape_text(t->sizes()));
  }
  // row pitch of a [rows, cols] operand with contiguous rows
  size_t pitch(int64_t rows, int64_t cols, at::ScalarType type, at::Device device) const {
    on(device);
    typed(type);
    shaped({rows, cols});
    if (cols > 1 && t->stride(1) != 1) refuse(std::string(name) + "'s rows must be contiguous");
    return static_cast<size_t>(t->stride(0));
  }
  void dense(at::IntArrayRef shape, at::ScalarType type, at::Device device) const {
    on(device);
    typed(type);
    shaped(shape);
    if (!t->is_contiguous()) refuse(std::string(name) + " must be contiguous");
  }
  std::pair<const char*, const char*> span() const {
    const char* b = static_cast<const char*>(t->data_ptr());
    if (t->numel() == 0) return {b, b};
    int64_t last = 0;
    for (int64_t d = 0; d < t->dim(); ++d) last += (t->size(d) - 1) * t->stride(d);
    return {b, b + (last + 1) * static_cast<int64_t>(t->element_size())};
  }
  // A call has written the tensor: a graph that saved it must not use it any more. (Tensors made in inference mode have no
  // versions.)
  void written() const {
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  }
  // Bytes of a row (all dimensions but the first), or 0 where a row has gaps.
  int64_t row_bytes() const {
    int64_t n = 1;
    for (int64_t d = t->dim() - 1; d > 0; --d) {
      if (t->size(d) > 1 && t->stride(d) != n) return 0;
      n *= t->size(d);
    }
    return n * static_cast<int64_t>(t->element_size());
  }
  // Whether the tensors, whose starts are `offset` bytes apart, are different columns of rows with one pitch (two slices of
  // a wider buffer): their spans overlap, but they do not.
  bool beside(const Arg& o, int64_t offset) const {
    if (dim() < 2 || o.dim() < 2) return false;
    const int64_t pitch = t->stride(0) * static_cast<int64_t>(t->element_size()), mine = row_bytes(), other = o.row_bytes();
    if (pitch <= 0 || pitch != o.t->stride(0) * static_cast<int64_t>(o.t->element_size()) || mine == 0 || other == 0) return false;
    const int64_t at = (offset % pitch + pitch) % pitch;  // of the other's row behind the start of mine
    return at >= mine && at + other <= pitch;
  }
  void apart(const Arg& o) const {
    if (!o) return;
    const auto a = span(), b = o.span();
    if (a.first < b.second && b.first < a.second && !beside(o, b.first - a.first))
      refuse(std::string(name) + " overlaps " + o.name);
  }
};

// The device and stream of one call. Outputs are made, and the entry point runs, under the
// tensors' device; with a stream of the caller's the outputs belong to that stream and the
// inputs' memory is held until it has passed the call.
class On {
 public:
  On(const Arg& x, PyObject* stream) : device_(x.t->device()) {
    need(device_.is_cuda(), "the tensors must be on a CUDA device");
    guard_.emplace(device_);
    if (stream == Py_None) {
      stream_ = c10::cuda::getCurrentCUDAStream(device_.index());
      return;
    }
    const auto attr = [&](const char* n) {
      PyObject* v = PyObject_GetAttrString(stream, n);
      const int64_t i = v ? PyLong_AsLongLong(v) : -1;
      Py_XDECREF(v);
      if (PyErr_Occurred()) {
        PyErr_Clear();
        refuse("stream must be a torch.cuda.Stream");
      }
      return i;
    };
    const int64_t index = attr("device_index");
    stream_ = c10::cuda::CUDAStream::unpack3(attr("stream_id"), static_cast<c10::DeviceIndex>(index),
                                             static_cast<c10::DeviceType>(attr("device_type")));
    need(index == device_.index(), "the stream is on another device than the tensors");
    stream_guard_.emplace(*stream_);
    given_ = true;
  }
  at::Device device() const { return device_; }
  void* raw() const { return stream_->stream(); }
  at::Tensor empty(at::IntArrayRef shape, at::ScalarType type) const {
    return at::empty(shape, at::TensorOptions().device(device_).dtype(type));
  }
  void hold(std::initializer_list<const Arg*> args) const {
    if (!given_) return;
    for (const Arg* a : args)
      if (*a) a->t->record_stream(*stream_);
  }

 private:
  at::Device device_;
  std::optional<c10::cuda::CUDAGuard> guard_;
  std::optional<c10::cuda::CUDAStream> stream_;
  std::optional<c10::cuda::CUDAStreamGuard> stream_guard_;
  bool given_ = false;
};

int64_t integer(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(std::string(name) + " must be an integer");
  }
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) {
    PyErr_Clear();
    refuse("a flag must be a truth value");
  }
  return v != 0;
}

// (sequences, states) of a call over packed rows.
std::pair<int64_t, int64_t> sequences(const On& on, int64_t rows, const Arg& starts, const Arg& slots, const Arg& state, bool step) {
  int64_t seqs = 1;
  if (step) {
    seqs = rows;
  } else if (starts) {
    need(starts.dim() == 1 && starts.size(0) >= 1, "seq_starts must be [sequences + 1]");
    seqs = starts.size(0) - 1;
    starts.dense({seqs + 1}, at::kInt, on.device());
  }
  if (slots) {
    need(static_cast<bool>(state), "slots need a state");
    slots.dense({seqs}, at::kInt, on.device());
  }
  const int64_t count = state ? state.size(0) : seqs;
  need(slots || count >= seqs, "fewer states than sequences");
  return {seqs, count};
}

// (x, weight, residual, eps, code is int8, group, stream)
PyObject* add_rmsnorm_quant(PyObject* const* v) {
  const Arg x(v[0], "x"), weight(v[1], "weight"), residual(v[2], "residual", true);
  const int kind = row_type(x.t->scalar_type(), "x");
  need(x.dim() == 2, "x must be [rows, cols]");
  const at::ScalarType type = x.t->scalar_type();
  const int64_t rows = x.size(0), cols = x.size(1), group = integer(v[5], "group");
  const On on(x, v[6]);
  const size_t ldx = x.pitch(rows, cols, type, on.device());
  weight.dense({cols}, at::kFloat, on.device());
  need(group == 0 || group == 32 || group == 64 || group == 128, "group must be 0, 32, 64 or 128");
  size_t ldr = 0;
  if (residual) {
    ldr = residual.pitch(rows, cols, type, on.device());
    residual.apart(x);
    residual.apart(weight);
  }
  const double eps = PyFloat_AsDouble(v[3]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    refuse("eps must be a number");
  }
  const bool s8 = truth(v[4]);
  const at::Tensor codes = on.empty({rows, cols}, s8 ? at::kChar : at::kFloat8_e4m3fn);
  const at::Tensor scales = on.empty({rows, group ? (cols + group - 1) / group : 1}, at::kFloat);
  on.hold({&x, &weight, &residual});
  check(mmfree_cuda_add_rmsnorm_quant(codes.data_ptr(), static_cast<float*>(scales.data_ptr()), x.data(), ldx, residual.data(), ldr,
                                      static_cast<const float*>(weight.data()), rows, cols, static_cast<float>(eps), kind,
                                      s8 ? MMFREE_T_S8 : MMFREE_T_E4M3, group, on.raw()));
  residual.written();
  return Py_BuildValue("NN", THPVariable_Wrap(codes), THPVariable_Wrap(scales));
}

// (x, codes, scales, group, zeros, x_scales, out_dtype, stream)
PyObject* int4_matvec(PyObject* const* v) {
  const Arg x(v[0], "x"), codes(v[1], "codes"), scales(v[2], "scales"), zeros(v[4], "zeros", true), xs(v[5], "x_scales", true);
  const at::ScalarType type = x.t->scalar_type();
  const int kind = type_code(type);
  need(kind >= 0, "x must be float32, bfloat16, float16, int8 or float8_e4m3fn");
  need(x.dim() == 2 && codes.dim() == 2, "x and codes must have two dimensions");
  const int64_t rows = x.size(0), in_dim = x.size(1), out_dim = codes.size(0), group = integer(v[3], "group");
  const On on(x, v[7]);
  const size_t ldx = x.pitch(rows, in_dim, type, on.device());
  const size_t ldw = codes.pitch(out_dim, (in_dim + 1) / 2, at::kByte, on.device());
  need(group >= 32 && group % 32 == 0, "group must be a multiple of 32");
  const int64_t parts = (in_dim + group - 1) / group;
  const int scale_kind = row_type(scales.t->scalar_type(), "scales");
  scales.dense({out_dim, parts}, scales.t->scalar_type(), on.device());
  if (zeros) zeros.dense({out_dim, parts}, at::kByte, on.device());
  need(static_cast<bool>(xs) == (kind >= MMFREE_T_S8), "x_scales go with 8-bit rows, and only with them");
  int64_t x_group = 0;
  if (xs) {
    if (xs.dim() == 2 && parts > 1 && xs.size(1) == parts) x_group = group;
    xs.dense({rows, x_group ? parts : 1}, at::kFloat, on.device());
  }
  at::ScalarType out_type = kind <= MMFREE_T_F16 ? type : at::kFloat;
  if (v[6] != Py_None) {
    need(THPDtype_Check(v[6]), "out_dtype must be a torch.dtype");
    out_type = reinterpret_cast<THPDtype*>(v[6])->scalar_type;
  }
  const int out_kind = row_type(out_type, "out_dtype");
  const at::Tensor out = on.empty({rows, out_dim}, out_type);
  on.hold({&x, &codes, &scales, &zeros, &xs});
  check(mmfree_cuda_int4_matvec(out.data_ptr(), x.data(), ldx, static_cast<const float*>(xs.data()),
                                static_cast<const uint8_t*>(codes.data()), ldw, scales.data(),
                                static_cast<const uint8_t*>(zeros.data()), rows, in_dim, out_dim, group, x_group, kind, scale_kind,
                                out_kind, on.raw()));
  return THPVariable_Wrap(out);
}

// The caller's output, or a new one.
at::Tensor output(const On& on, const Arg& out, int64_t rows, int64_t channels, at::ScalarType type) {
  return out ? *out.t : on.empty({rows, channels}, type);
}

// (x, weight, bias, state, seq_starts, slots, silu, out, stream, step)
PyObject* causal_conv(PyObject* const* v) {
  const Arg x(v[0], "x"), weight(v[1], "weight"), bias(v[2], "bias", true), state(v[3], "state", true),
      starts(v[4], "seq_starts", true), slots(v[5], "slots", true), given(v[7], "out", true);
  const bool step = truth(v[9]);
  const at::ScalarType type = x.t->scalar_type();
  const int kind = row_type(type, "x");
  need(!step || state, "a step needs a state");
  need(x.dim() == 2 && weight.dim() == 2, "x and weight must have two dimensions");
  const int64_t rows = x.size(0), channels = x.size(1), width = weight.size(1);
  const On on(x, v[8]);
  mmfree_cuda_conv_args a{};
  a.ldx = x.pitch(rows, channels, type, on.device());
  need(width >= 2 && width <= MMFREE_CUDA_MAX_CONV_WIDTH, "weight must be [channels, 2 to 8]");
  weight.dense({channels, width}, at::kFloat, on.device());
  if (bias) bias.dense({channels}, at::kFloat, on.device());
  if (state) {
    need(state.dim() == 3, "state must be [states, width - 1, channels]");
    state.dense({state.size(0), width - 1, channels}, type, on.device());
    state.apart(x);
  }
  const auto [seqs, count] = sequences(on, rows, starts, slots, state, step);
  const at::Tensor out = output(on, given, rows, channels, type);
  a.ld_out = static_cast<size_t>(channels);
  if (given) {
    a.ld_out = given.pitch(rows, channels, type, on.device());
    for (const Arg* o : {&x, &weight, &bias, &state, &starts, &slots}) given.apart(*o);
  }
  a.out = out.data_ptr();
  a.x = x.data();
  a.weight = static_cast<const float*>(weight.data());
  a.bias = static_cast<const float*>(bias.data());
  a.state = state.data();
  a.seq_starts = static_cast<const int32_t*>(starts.data());
  a.slots = static_cast<const int32_t*>(slots.data());
  a.tokens = rows;
  a.seqs = seqs;
  a.slot_count = count;
  a.channels = channels;
  a.width = width;
  a.type = kind;
  a.silu = truth(v[6]);
  on.hold({&x, &weight, &bias, &state, &starts, &slots, &given});
  check(step ? mmfree_cuda_causal_conv_step(&a, on.raw()) : mmfree_cuda_causal_conv(&a, on.raw()));
  state.written();
  given.written();
  return THPVariable_Wrap(out);
}

// (x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, seq_starts, slots, out, stream, step)
PyObject* selective(PyObject* const* v) {
  const Arg x(v[0], "x"), dt(v[1], "dt"), A(v[2], "A"), B(v[3], "B"), Cm(v[4], "C"), D(v[5], "D", true), z(v[6], "z", true),
      dt_bias(v[7], "dt_bias", true), state(v[9], "state", true), starts(v[10], "seq_starts", true), slots(v[11], "slots", true),
      given(v[12], "out", true);
  const bool step = truth(v[14]);
  const at::ScalarType type = x.t->scalar_type();
  const int kind = row_type(type, "x");
  need(!step || state, "a step needs a state");
  need(x.dim() == 2 && A.dim() == 2, "x and A must have two dimensions");
  const int64_t rows = x.size(0), channels = x.size(1), states = A.size(1);
  const On on(x, v[13]);
  mmfree_cuda_ssm_args a{};
  a.ldx = x.pitch(rows, channels, type, on.device());
  a.ld_dt = dt.pitch(rows, channels, type, on.device());
  if (z) a.ldz = z.pitch(rows, channels, type, on.device());
  need(states >= 1 && states <= MMFREE_CUDA_MAX_STATES, "A must be [channels, 1 to 256]");
  A.dense({channels, states}, at::kFloat, on.device());
  need(B.dim() == 2 || B.dim() == 3, "B must be [rows, states] or [rows, groups, states]");
  const bool grouped = B.dim() == 3;
  const int64_t groups = grouped ? B.size(1) : 1;
  need(groups >= 1 && channels % groups == 0, "the groups must divide the channels");
  const auto mixed = [&](const Arg& m) {
    m.on(on.device());
    m.typed(type);
    if (grouped) m.shaped({rows, groups, states});
    else m.shaped({rows, states});
    if ((states > 1 && m.t->stride(-1) != 1) || (groups > 1 && m.t->stride(1) != states)) refuse(std::string(m.name) + "'s rows must be contiguous");
    return static_cast<size_t>(m.t->stride(0));
  };
  a.ldb = mixed(B);
  a.ldc = mixed(Cm);
  if (D) D.dense({channels}, at::kFloat, on.device());
  if (dt_bias) dt_bias.dense({channels}, at::kFloat, on.device());
  if (state) {
    need(state.dim() == 3, "state must be [states, channels, A's columns]");
    state.dense({state.size(0), channels, states}, at::kFloat, on.device());
    for (const Arg* o : {&x, &dt, &A, &B, &Cm, &D, &z, &dt_bias}) state.apart(*o);
  }
  const auto [seqs, count] = sequences(on, rows, starts, slots, state, step);
  const at::Tensor out = output(on, given, rows, channels, type);
  a.ld_out = static_cast<size_t>(channels);
  if (given) {
    a.ld_out = given.pitch(rows, channels, type, on.device());
    for (const Arg* o : {&x, &dt, &A, &B, &Cm, &D, &z, &dt_bias, &state, &starts, &slots}) given.apart(*o);
  }
  a.out = out.data_ptr();
  a.x = x.data();
  a.dt = dt.data();
  a.z = z.data();
  a.B = B.data();
  a.C = Cm.data();
  a.A = static_cast<const float*>(A.data());
  a.D = static_cast<const float*>(D.data());
  a.dt_bias = static_cast<const float*>(dt_bias.data());
  a.state = static_cast<float*>(state.data());
  a.seq_starts = static_cast<const int32_t*>(starts.data());
  a.slots = static_cast<const int32_t*>(slots.data());
  a.tokens = rows;
  a.seqs = seqs;
  a.slot_count = count;
  a.channels = channels;
  a.states = states;
  a.groups = groups;
  a.type = kind;
  a.dt_softplus = truth(v[8]);
  on.hold({&x, &dt, &A, &B, &Cm, &D, &z, &dt_bias, &state, &starts, &slots, &given});
  check(step ? mmfree_cuda_selective_step(&a, on.raw()) : mmfree_cuda_selective_scan(&a, on.raw()));
  state.written();
  given.written();
  return THPVariable_Wrap(out);
}

// Runs one function; its failures become MmfreeError, torch's errors what torch raises.
template <PyObject* (*kFunction)(PyObject* const*), Py_ssize_t kArgs>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", kArgs, n);
    return nullptr;
  }
  try {
    return kFunction(args);
  } catch (const Failure& f) {
    PyObject* e = g_error ? PyObject_CallFunction(g_error, "is", f.code, f.message.c_str()) : nullptr;
    if (e) {
      PyErr_SetObject(g_error, e);
      Py_DECREF(e);
    } else if (!PyErr_Occurred()) {
      PyErr_SetString(PyExc_RuntimeError, f.message.c_str());
    }
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());  // torch's own, out of memory among them
  }
  return nullptr;
}

PyObject* set_error(PyObject*, PyObject* o) {
  Py_INCREF(o);
  Py_XSETREF(g_error, o);
  Py_RETURN_NONE;
}

#define MMFREE_FASTCALL(f, n) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<f, n>)), METH_FASTCALL, nullptr

PyMethodDef kMethods[] = {
    {"set_error", set_error, METH_O, nullptr},
    {"add_rmsnorm_quant", MMFREE_FASTCALL(add_rmsnorm_quant, 7)},
    {"int4_matvec", MMFREE_FASTCALL(int4_matvec, 8)},
    {"causal_conv", MMFREE_FASTCALL(causal_conv, 10)},
    {"selective", MMFREE_FASTCALL(selective, 15)},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "mmfree_tensor_ops", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_mmfree_tensor_ops() { return PyModule_Create(&kModule); }
