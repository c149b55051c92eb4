// The token mixer's calls on torch tensors: checks of shapes, types and
// devices, outputs and scratch from torch's allocator, the call on torch's
// current stream.  Compiled because a serving step makes five such calls a
// layer, of 3 to 8 us on the GPU, and the same checks in Python cost twice
// that (one token of linear attention 11.9 us a call, from here 5.2, of rotary
// 11.6 and 5.7).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/core/GradMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdint>
#include <utility>

#include "rmoe.h"

namespace {

using at::Tensor;

// ---------------------------------------------------------------- arguments

const Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor (got ", Py_TYPE(o)->tp_name, ")");
  return THPVariable_Unpack(o);
}

// An undefined tensor for None.
Tensor tensor_or_none(PyObject* o, const char* name) {
  return o == Py_None ? Tensor() : tensor(o, name);
}

int32_t small(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v >= INT32_MIN && v <= INT32_MAX, name, " is out of range (got ", v, ")");
  return (int32_t)v;
}

int32_t integer(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return small(v, name);
}

float real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return (float)v;
}

bool flag(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

// ------------------------------------------------------------------- checks

// The index of the GPU that all of the tensors (or undefined ones) are on;
// refuses tensors that want a gradient: there is no backward pass.
template <size_t N>
int one_device(const std::array<const Tensor*, N>& all) {
  int index = -1;
  const bool grad = c10::GradMode::is_enabled();
  for (const Tensor* t : all) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->is_cuda(), "runnel_amd kernels take GPU tensors");
    const int i = t->get_device();
    TORCH_CHECK_VALUE(index < 0 || i == index, "tensors are on cuda:", index, " and cuda:", i);
    index = i;
    // (fake tensors and the like: there may be no memory behind them)
    TORCH_CHECK_VALUE(!t->key_set().has(c10::DispatchKey::Python),
                      "tensors whose operations dispatch to Python are not taken");
    TORCH_CHECK_VALUE(!grad || !t->requires_grad(),
                      "this operator has no backward pass: call it under torch.no_grad() or on "
                      "detached tensors");
  }
  return index;
}

bool is(const Tensor& t, std::initializer_list<int64_t> shape) {
  return t.sizes() == at::IntArrayRef(shape);
}

Tensor int32(const Tensor& t, const char* name, at::IntArrayRef shape) {
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must be ", shape, " (got ", t.sizes(), ")");
  if (t.scalar_type() == at::kInt && t.is_contiguous()) return t;
  TORCH_CHECK_VALUE(at::isIntegralType(t.scalar_type(), false), name, " must be int32 (got ",
                    t.scalar_type(), ")");
  return t.to(at::kInt).contiguous();
}

// bf16 [rows, heads, dim], as it lies where the kernels can read it so (a
// slice of a packed projection), else copied.
struct Heads {
  Tensor t;
  rmoe_rows rows;
  int64_t n, dim;
};

Heads heads(const Tensor& given, const char* name, int64_t rows = -1, int64_t count = -1,
            int64_t dim = -1) {
  TORCH_CHECK_VALUE(given.scalar_type() == at::kBFloat16 && given.dim() == 3, name,
                    " must be a bfloat16 [rows, heads, dim] tensor (got ", given.scalar_type(), " ",
                    given.sizes(), ")");
  const auto size = given.sizes();
  const std::array<int64_t, 3> want = {rows < 0 ? size[0] : rows, count < 0 ? size[1] : count,
                                       dim < 0 ? size[2] : dim};
  TORCH_CHECK_VALUE(size == at::IntArrayRef(want), name, " must be ", at::IntArrayRef(want),
                    " (got ", size, ")");
  Heads h{given, {}, size[0], size[2]};
  auto readable = [&] {
    const auto s = h.t.strides();
    return s[2] == 1 && s[0] % 8 == 0 && s[1] % 8 == 0 && (uintptr_t)h.t.data_ptr() % 16 == 0;
  };
  if (!readable()) {
    h.t = given.clone(at::MemoryFormat::Contiguous);
    TORCH_CHECK_VALUE(readable(), name, "'s dim must be a multiple of 8 (got ", size[2], ")");
  }
  h.rows = {static_cast<const uint16_t*>(h.t.data_ptr()), h.t.stride(0), h.t.stride(1),
            small(size[1], "the head count")};
  return h;
}

Tensor like(const Heads& h) { return at::empty(h.t.sizes(), h.t.options()); }

rmoe_paged_cache cache_of(const Tensor& k, const Tensor& v, float k_scale, float v_scale) {
  const bool eight = k.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK_VALUE(eight || k.scalar_type() == at::kBFloat16,
                    "the cache must be bfloat16 or float8_e4m3fn (got ", k.scalar_type(), ")");
  TORCH_CHECK_VALUE(k.dim() == 4, "the cache must be [pages, kv heads, page size, dim] (got ",
                    k.sizes(), ")");
  TORCH_CHECK_VALUE(v.scalar_type() == k.scalar_type() && v.sizes() == k.sizes(),
                    "k_cache and v_cache must have one type and shape");
  std::array<int64_t, 4> s;
  for (int i = 0; i < 4; ++i) {  // (a dimension of one has no stride)
    s[i] = k.size(i) == 1 ? 0 : k.stride(i);
    TORCH_CHECK_VALUE(k.size(i) == 1 || v.stride(i) == s[i],
                      "k_cache and v_cache must lie in memory alike");
  }
  TORCH_CHECK_VALUE(s[3] == 1, "the cache's last dimension must be contiguous");
  TORCH_CHECK_VALUE(eight || (k_scale == 1.0f && v_scale == 1.0f),
                    "k_scale and v_scale belong to float8_e4m3fn caches");
  return {k.data_ptr(),
          v.data_ptr(),
          s[0],
          s[1],
          s[2],
          small(k.size(0), "the page count"),
          small(k.size(2), "the page size"),
          small(k.size(1), "the head count"),
          small(k.size(3), "the cache's dim"),
          eight ? 8 : 16,
          k_scale,
          v_scale};
}

struct Rotary {
  rmoe_rotary_spec spec;
  Tensor positions;
};

Rotary rotary_of(const Tensor& inv_freq, const Tensor& positions, int64_t rows, PyObject* sections,
                 bool woven, bool adjacent) {
  TORCH_CHECK_VALUE(inv_freq.scalar_type() == at::kFloat && inv_freq.dim() == 1 &&
                        inv_freq.is_contiguous(),
                    "inv_freq must be a contiguous float32 vector");
  Rotary r{};
  r.spec.inv_freq = inv_freq.data_ptr<float>();
  r.spec.half = small(inv_freq.numel(), "inv_freq's length");
  r.spec.woven = woven;
  r.spec.adjacent = adjacent;
  if (sections == Py_None) {
    r.spec.axes = 1;
    r.spec.sections[0] = r.spec.half;
  } else {
    THPObjectPtr list(PySequence_Fast(sections, "sections must be a sequence"));
    if (!list) throw python_error();
    const int64_t axes = PySequence_Fast_GET_SIZE(list.get());
    TORCH_CHECK_VALUE(axes >= 1 && axes <= 4, "sections must name 1 to 4 axes (got ", axes, ")");
    r.spec.axes = (int32_t)axes;
    for (int i = 0; i < axes; ++i)
      r.spec.sections[i] = integer(PySequence_Fast_GET_ITEM(list.get(), i), "a section");
  }
  const std::array<int64_t, 2> shape = {r.spec.axes, rows};
  const bool flat = r.spec.axes == 1 && positions.dim() == 1;
  r.positions = int32(positions, "positions", at::IntArrayRef(shape.data() + flat, 2 - flat));
  return r;
}

rmoe_gate gate_of(const Tensor& t, const char* name, int64_t rows, int64_t count) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && is(t, {rows, count}), name,
                    " must be float32 [", rows, ", ", count, "] (got ", t.scalar_type(), " ",
                    t.sizes(), ")");
  return {t.data_ptr<float>(), t.stride(0), t.stride(1)};
}

// ----------------------------------------------------------------- the call

void raise_status(int rc) {
  THPObjectPtr lib(PyImport_ImportModule("runnel_amd._lib"));
  if (!lib) throw python_error();
  THPObjectPtr done(PyObject_CallMethod(lib.get(), "check", "i", rc));
  throw python_error();  // check() has raised
}

struct WithoutGil {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

// call(stream) on GPU `index` and torch's current stream there; other Python
// threads run meanwhile.
template <typename F>
void on_stream(int index, F call) {
  int rc;
  {
    const c10::DeviceGuard guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)index));
    void* stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex)index).stream();
    const WithoutGil without;
    rc = call(stream);
  }
  if (rc) raise_status(rc);
}

Tensor scratch(size_t bytes, const Tensor& beside) {
  return bytes ? at::empty({(int64_t)bytes}, beside.options().dtype(at::kByte)) : Tensor();
}

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

PyObject* tuple_of(std::initializer_list<Tensor> all) {
  THPObjectPtr t(PyTuple_New((Py_ssize_t)all.size()));
  if (!t) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor& x : all) PyTuple_SET_ITEM(t.get(), i++, THPVariable_Wrap(x));
  return t.release();
}

// ------------------------------------------------------------ the operators

// cached, added, block_table, free_pages, page_size, rows -> slots, positions,
// requests, cu_seqlens, lengths, counts
PyObject* paged_tables(PyObject* const* o) {
  const Tensor &cached0 = tensor(o[0], "cached"), &added0 = tensor(o[1], "added");
  const Tensor &table = tensor(o[2], "block_table"), &free0 = tensor(o[3], "free_pages");
  const int32_t page_size = integer(o[4], "page_size"), rows = integer(o[5], "rows");
  const int index = one_device<4>({&cached0, &added0, &table, &free0});
  TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2,
                    "block_table must be int32 [requests, pages]");
  const int64_t R = table.size(0), P = table.size(1);
  TORCH_CHECK_VALUE(P <= 1 || table.stride(1) == 1,
                    "block_table's rows must be contiguous (it is updated in place)");
  const Tensor cached = int32(cached0, "cached", {R}), added = int32(added0, "added", {R});
  const Tensor free_pages = int32(free0, "free_pages", {free0.numel()});
  TORCH_CHECK_VALUE(rows >= 0, "rows must not be negative (got ", rows, ")");
  const Tensor ints = at::empty({2 * (int64_t)rows + 2 * R + 4}, table.options());
  const Tensor slots = at::empty({rows}, table.options().dtype(at::kLong));
  const int64_t stride = R == 1 ? std::max(table.stride(0), P) : table.stride(0);
  int32_t* at = ints.data_ptr<int32_t>();
  on_stream(index, [&](void* stream) {
    return rmoe_paged_tables(
        cached.data_ptr<int32_t>(), added.data_ptr<int32_t>(), small(R, "the request count"),
        table.data_ptr<int32_t>(), stride, small(P, "the table's width"),
        free_pages.data_ptr<int32_t>(), small(free_pages.numel(), "the free pages' count"),
        page_size, rows, slots.data_ptr<int64_t>(), at, at + rows, at + 2 * (int64_t)rows,
        at + 2 * (int64_t)rows + R + 1, at + 2 * (int64_t)rows + 2 * R + 1, stream);
  });
  at::AutoDispatchBelowADInplaceOrView plain;  // views of whole numbers: nothing to record
  int64_t from = 0;
  auto next = [&](int64_t n) { return ints.as_strided({n}, {1}, std::exchange(from, from + n)); };
  const Tensor positions = next(rows), requests = next(rows), cu = next(R + 1), lengths = next(R);
  return tuple_of({slots, positions, requests, cu, lengths, next(3)});
}

// q, k, positions, inv_freq, sections, woven, adjacent -> q, k
PyObject* rotary(PyObject* const* o) {
  const Tensor &q0 = tensor(o[0], "q"), &k0 = tensor(o[1], "k");
  const Tensor &positions = tensor(o[2], "positions"), &inv_freq = tensor(o[3], "inv_freq");
  const int index = one_device<4>({&q0, &k0, &positions, &inv_freq});
  const Heads q = heads(q0, "q"), k = heads(k0, "k", q.n, -1, q.dim);
  const Rotary r = rotary_of(inv_freq, positions, q.n, o[4], flag(o[5]), flag(o[6]));
  const Tensor q_out = like(q), k_out = like(k);
  const int32_t n = small(q.n, "the row count"), dim = small(q.dim, "q's dim");
  on_stream(index, [&](void* stream) {
    return rmoe_rotary(&r.spec, r.positions.data_ptr<int32_t>(), n, n, dim, &q.rows,
                       static_cast<uint16_t*>(q_out.data_ptr()), &k.rows,
                       static_cast<uint16_t*>(k_out.data_ptr()), stream);
  });
  return tuple_of({q_out, k_out});
}

// q, k, v, positions, inv_freq, k_cache, v_cache, slots, sections, woven,
// adjacent, k_scale, v_scale -> q
PyObject* rotary_append(PyObject* const* o) {
  const Tensor &q0 = tensor(o[0], "q"), &k0 = tensor(o[1], "k"), &v0 = tensor(o[2], "v");
  const Tensor &positions = tensor(o[3], "positions"), &inv_freq = tensor(o[4], "inv_freq");
  const Tensor &k_cache = tensor(o[5], "k_cache"), &v_cache = tensor(o[6], "v_cache");
  const Tensor& slots0 = tensor(o[7], "slots");
  const int index = one_device<8>(
      {&q0, &k0, &v0, &positions, &inv_freq, &k_cache, &v_cache, &slots0});
  const rmoe_paged_cache cache = cache_of(k_cache, v_cache, real(o[11]), real(o[12]));
  for (const int64_t s : k_cache.strides())
    TORCH_CHECK_VALUE(s != 0, "an expanded cache cannot be written");
  TORCH_CHECK_VALUE(cache.k != cache.v, "k_cache and v_cache must be two");
  const Heads q = heads(q0, "q", -1, -1, cache.dim);
  const Heads k = heads(k0, "k", q.n, cache.kv_heads, cache.dim);
  const Heads v = heads(v0, "v", q.n, cache.kv_heads, cache.dim);
  const Rotary r = rotary_of(inv_freq, positions, q.n, o[8], flag(o[9]), flag(o[10]));
  TORCH_CHECK_VALUE(slots0.scalar_type() == at::kLong && is(slots0, {q.n}), "slots must be int64 [",
                    q.n, "] (got ", slots0.scalar_type(), " ", slots0.sizes(), ")");
  const Tensor slots = slots0.contiguous(), q_out = like(q);
  const int32_t n = small(q.n, "the row count");
  on_stream(index, [&](void* stream) {
    return rmoe_rotary_append(&r.spec, r.positions.data_ptr<int32_t>(), n, n, &q.rows,
                              static_cast<uint16_t*>(q_out.data_ptr()), &k.rows, &v.rows, &cache,
                              slots.data_ptr<int64_t>(), stream);
  });
  return THPVariable_Wrap(q_out);
}

// q, k_cache, v_cache, block_table, lengths, scale, window, k_scale, v_scale,
// return_lse -> out, or out and lse
PyObject* paged_attention(PyObject* const* o) {
  const Tensor &q0 = tensor(o[0], "q"), &k_cache = tensor(o[1], "k_cache");
  const Tensor &v_cache = tensor(o[2], "v_cache"), &table0 = tensor(o[3], "block_table");
  const Tensor& lengths0 = tensor(o[4], "lengths");
  const int index = one_device<5>({&q0, &k_cache, &v_cache, &table0, &lengths0});
  const rmoe_paged_cache cache = cache_of(k_cache, v_cache, real(o[7]), real(o[8]));
  const Heads q = heads(q0, "q", -1, -1, cache.dim);
  TORCH_CHECK_VALUE(table0.dim() == 2 && table0.size(0) == q.n, "block_table must be [", q.n,
                    ", pages] (got ", table0.sizes(), ")");
  const bool rows = table0.scalar_type() == at::kInt && table0.stride(1) == 1;
  const Tensor table = rows ? table0 : int32(table0, "block_table", table0.sizes());
  const Tensor lengths = int32(lengths0, "lengths", {q.n});
  const float scale = o[5] == Py_None ? (float)(1.0 / std::sqrt((double)q.dim)) : real(o[5]);
  const int32_t window = integer(o[6], "window"), R = small(q.n, "the request count");
  const int32_t width = small(table.size(1), "the table's width");
  const bool with_lse = flag(o[9]);
  const Tensor out = like(q);
  const Tensor lse =
      with_lse ? at::empty({q.n, q.rows.heads}, out.options().dtype(at::kFloat)) : Tensor();
  const size_t need =
      rmoe_paged_attention_workspace_bytes(&cache, q.rows.heads, R, width, window);
  const Tensor ws = scratch(need, out);
  on_stream(index, [&](void* stream) {
    return rmoe_paged_attention(&q.rows, &cache, table.data_ptr<int32_t>(), table.stride(0), width,
                                lengths.data_ptr<int32_t>(), R, window, scale,
                                static_cast<uint16_t*>(out.data_ptr()),
                                static_cast<float*>(address(lse)), address(ws), need, stream);
  });
  return with_lse ? tuple_of({out, lse}) : THPVariable_Wrap(out);
}

// q, k, v, log_decay, cu_seqlens, state, beta, state_index, scale, state_out
// -> out
PyObject* linear_attention(PyObject* const* o) {
  const Tensor &q0 = tensor(o[0], "q"), &k0 = tensor(o[1], "k"), &v0 = tensor(o[2], "v");
  const Tensor &decay0 = tensor(o[3], "log_decay"), &cu0 = tensor(o[4], "cu_seqlens");
  const Tensor& state = tensor(o[5], "state");
  const Tensor beta0 = tensor_or_none(o[6], "beta");
  const Tensor index0 = tensor_or_none(o[7], "state_index");
  const Tensor given = tensor_or_none(o[9], "state_out");
  const int index =
      one_device<9>({&q0, &k0, &v0, &decay0, &cu0, &state, &beta0, &index0, &given});
  const Tensor& state_out = given.defined() ? given : state;
  const Heads q = heads(q0, "q"), k = heads(k0, "k", q.n, q.rows.heads, q.dim);
  const Heads v = heads(v0, "v", q.n);
  TORCH_CHECK_VALUE(cu0.dim() == 1 && cu0.numel() >= 1, "cu_seqlens must be [sequences + 1]");
  const int64_t R = cu0.numel() - 1;
  const Tensor cu = int32(cu0, "cu_seqlens", {R + 1});
  const rmoe_gate decay = gate_of(decay0, "log_decay", q.n, v.rows.heads);
  rmoe_gate beta{};
  if (beta0.defined()) beta = gate_of(beta0, "beta", q.n, v.rows.heads);
  const int64_t slots = state.dim() ? state.size(0) : 0;
  for (const Tensor* t : {&state, &state_out})
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat &&
                          is(*t, {slots, v.rows.heads, q.dim, v.dim}) && t->is_contiguous(),
                      t == &state ? "state" : "state_out", " must be contiguous float32 [", slots,
                      ", ", v.rows.heads, ", ", q.dim, ", ", v.dim, "] (got ", t->scalar_type(),
                      " ", t->sizes(), ")");
  const float *from = state.data_ptr<float>(), *to = state_out.data_ptr<float>();
  TORCH_CHECK_VALUE(from == to || from + state.numel() <= to || to + state.numel() <= from,
                    "state_out must be state or lie apart from it");
  TORCH_CHECK_VALUE(index0.defined() || slots >= R, "state has ", slots, " slots for ", R,
                    " sequences");
  const Tensor at = index0.defined() ? int32(index0, "state_index", {R}) : Tensor();
  const float scale = o[8] == Py_None ? (float)(1.0 / std::sqrt((double)q.dim)) : real(o[8]);
  if (R == 0) return THPVariable_Wrap(at::zeros(v.t.sizes(), v.t.options()));
  const int32_t N = small(q.n, "the row count"), sequences = small(R, "the sequence count");
  const int32_t dk = small(q.dim, "q's dim"), dv = small(v.dim, "v's dim");
  const Tensor out = like(v);
  const size_t need = rmoe_linear_attention_workspace_bytes(N, sequences, q.rows.heads,
                                                            v.rows.heads, dk, beta0.defined());
  const Tensor ws = scratch(need, out);
  const int32_t count = small(slots, "the slot count");
  on_stream(index, [&](void* stream) {
    return rmoe_linear_attention(
        &q.rows, &k.rows, &v.rows, &decay, beta0.defined() ? &beta : nullptr,
        cu.data_ptr<int32_t>(), N, sequences, dk, dv, scale, from, const_cast<float*>(to),
        static_cast<const int32_t*>(address(at)), count, static_cast<uint16_t*>(out.data_ptr()), 1,
        address(ws), need, stream);
  });
  return THPVariable_Wrap(out);
}

// ---------------------------------------------------------------- the module

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == N, "takes ", N, " arguments (got ", n, ")");
  return F(args);
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject* const*), int N>
PyMethodDef method(const char* name) {
  return {name, (PyCFunction)(void (*)())(PyObject * (*)(PyObject*, PyObject* const*, Py_ssize_t))
                    entry<F, N>,
          METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<paged_tables, 6>("paged_tables"),
                         method<rotary, 7>("rotary"),
                         method<rotary_append, 13>("rotary_append"),
                         method<paged_attention, 10>("paged_attention"),
                         method<linear_attention, 10>("linear_attention"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mixer", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__mixer() { return PyModule_Create(&module); }
