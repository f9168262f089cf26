// Host part of the bounded-cache calls (fa_b200_page_bounds, fa_b200_page_select, fa_b200_decode_budget,
// fa_b200_token_weights, fa_b200_kv_evict) as a Python module over the C ABI.
//
// A decode step makes several of these calls with a few microseconds of GPU work each.  Argument checks, output allocation
// and the parameter struct took 12 to 14 us of Python per call: with two kernel launches a call held the host for 17 to 20 us
// while its kernels take 10 to 16.  Through this module it is 9 to 12 us (one launch: 4 to 5).  The module holds no state but
// one scratch buffer per (device, stream), which grows on demand up to 64 MB; more than that, and all scratch under stream
// capture (graph-private memory), comes from the caching allocator call by call.
#include <Python.h>

#include <cmath>
#include <cstdlib>
#include <cstring>
#include <map>
#include <utility>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/fa_b200.h"

#ifndef FA_B200_HOST_KEY
#error "build.py names the torch and Python that this is built against"
#endif

namespace {

// The library that the Python binding has loaded, in the order of `functions`.
struct Api {
  decltype(&fa_b200_page_bounds) page_bounds;
  decltype(&fa_b200_page_select) page_select;
  decltype(&fa_b200_page_select_workspace_bytes) page_select_bytes;
  decltype(&fa_b200_decode_budget) decode_budget;
  decltype(&fa_b200_decode_budget_workspace_bytes) decode_budget_bytes;
  decltype(&fa_b200_token_weights) token_weights;
  decltype(&fa_b200_token_weights_workspace_bytes) token_weights_bytes;
  decltype(&fa_b200_kv_evict) kv_evict;
  decltype(&fa_b200_status_string) status_string;
  decltype(&fa_b200_last_cuda_error) last_cuda_error;
};
constexpr const char* functions[] = {
    "fa_b200_page_bounds", "fa_b200_page_select", "fa_b200_page_select_workspace_bytes", "fa_b200_decode_budget",
    "fa_b200_decode_budget_workspace_bytes", "fa_b200_token_weights", "fa_b200_token_weights_workspace_bytes", "fa_b200_kv_evict",
    "fa_b200_status_string", "fa_b200_last_cuda_error"};
constexpr Py_ssize_t kFunctions = sizeof(functions) / sizeof(functions[0]);
static_assert(sizeof(Api) == kFunctions * sizeof(void*), "one name per function");
Api api;
void* profile_events[2] = {nullptr, nullptr};

// ---- arguments -------------------------------------------------------------------------------------
const at::Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}
at::Tensor optional_tensor(PyObject* o, const char* name) { return o == Py_None ? at::Tensor() : tensor(o, name); }
int32_t integer(PyObject* o, const char* name) {
  PyObject* i = PyNumber_Index(o);
  if (!i) throw python_error();
  const long long v = PyLong_AsLongLong(i);
  Py_DECREF(i);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  TORCH_CHECK(v >= INT32_MIN && v <= INT32_MAX, name, " is out of range");
  return static_cast<int32_t>(v);
}
float number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return static_cast<float>(v);
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
void arguments(Py_ssize_t got, Py_ssize_t want) {
  TORCH_CHECK(api.page_bounds, "bind() comes first");
  TORCH_CHECK_TYPE(got == want, "expected ", want, " arguments, got ", got);
}

bool is_fp8(at::ScalarType t) { return t == at::kFloat8_e4m3fn || t == at::kFloat8_e5m2; }
bool is_half(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
int code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return FA_B200_F16;
    case at::kBFloat16: return FA_B200_BF16;
    case at::kFloat8_e4m3fn: return FA_B200_E4M3;
    case at::kFloat8_e5m2: return FA_B200_E5M2;
    default: return -1;
  }
}
int index_of(const at::Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }
bool dense_last(const at::Tensor& t) { return t.stride(-1) == 1 || t.size(-1) <= 1; }
void forward_only(std::initializer_list<const at::Tensor*> ts) {
  if (!c10::GradMode::is_enabled()) return;
  for (const at::Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->requires_grad(),
                                "the B200 hot path is forward only: call under torch.no_grad() or detach inputs");
}

// A paged pool (num_blocks, page, h_k, d) with d contiguous (and the values beside the keys): its device.
int check_cache(const at::Tensor& k, const char* what, const at::Tensor* v = nullptr) {
  const int index = index_of(k);
  TORCH_CHECK(index >= 0 && k.dim() == 4 && k.stride(3) == 1, what,
              ": k_cache must be a CUDA tensor (num_blocks, page_size, nheads_k, d) with contiguous last dimension");
  TORCH_CHECK(code(k.scalar_type()) >= 0, what, ": the cache must be fp16, bf16, fp8 e4m3 or fp8 e5m2");
  if (v)
    TORCH_CHECK(v->sizes() == k.sizes() && v->scalar_type() == k.scalar_type() && index_of(*v) == index && v->stride(3) == 1, what,
                ": v_cache must be like k_cache, with contiguous last dimension");
  return index;
}
// An int32 block table (b, n) with the lengths (b) beside it.
void check_tables(const at::Tensor& table, const at::Tensor& lens, int index, const char* what) {
  TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kInt && index_of(table) == index && dense_last(table), what,
              ": block_table must be an int32 tensor (batch, max_num_blocks_per_seq) on the cache's device with contiguous last dimension");
  TORCH_CHECK(lens.dim() == 1 && lens.size(0) == table.size(0) && lens.scalar_type() == at::kInt && index_of(lens) == index && lens.is_contiguous(),
              what, ": cache_seqlens must be a contiguous int32 tensor (batch,) on the cache's device");
}

// fp32 token weights (b, h_k, capacity), capacity contiguous; `out` undefined: in place.  Fills the struct's fields.
template <class P>
at::Tensor set_weights(P& p, const at::Tensor& in, const at::Tensor& out_, int64_t b, int64_t h_k, int index, const char* what) {
  const at::Tensor& out = out_.defined() ? out_ : in;
  TORCH_CHECK(out.defined(), what, ": token_weights is required");
  for (const at::Tensor* w : {&in, &out})
    if (w->defined())
      TORCH_CHECK(w->scalar_type() == at::kFloat && index_of(*w) == index && w->dim() == 3 && w->size(0) == b && w->size(1) == h_k && dense_last(*w),
                  what, ": token weights must be a float32 tensor (batch, nheads_k, capacity) on the cache's device with contiguous last "
                  "dimension");
  TORCH_CHECK(!in.defined() || in.size(2) == out.size(2), what, ": token_weights_out must have the shape of token_weights");
  TORCH_CHECK(!in.defined() || !out_.defined() || at::get_overlap_status(in, out) != at::MemOverlapStatus::Partial, what,
              ": token_weights_out must be token_weights or not overlap it");
  p.weights_in = in.defined() ? static_cast<const float*>(in.const_data_ptr()) : nullptr;
  p.weights_out = static_cast<float*>(out.mutable_data_ptr());
  const at::Tensor& i = in.defined() ? in : out;
  p.weights_in_batch_stride = i.stride(0);
  p.weights_in_head_stride = i.stride(1);
  p.weights_out_batch_stride = out.stride(0);
  p.weights_out_head_stride = out.stride(1);
  TORCH_CHECK(out.size(2) <= INT32_MAX, what, ": token weights are too long");
  p.weights_capacity = static_cast<int32_t>(out.size(2));
  return out;
}

// ---- the call ----------------------------------------------------------------------------------------
void check_status(int status, const char* what) {
  if (status == FA_B200_OK) return;
  if (status == FA_B200_ERR_CUDA) TORCH_CHECK(false, what, ": ", api.status_string(status), " (", api.last_cuda_error(), ")");
  TORCH_CHECK(false, what, ": ", api.status_string(status));
}

// `call(stream)` with device `index` current; p's scratch is the (device, stream)'s buffer, grown when the library refuses it as
// too small (which it does before any launch), `size()` bytes; under capture a fresh one.  Beyond kKeptBytes it goes back to the
// caching allocator after the call (in stream order), which a call with that much to do does not notice.
constexpr int64_t kKeptBytes = 64 << 20;
template <class P, class Call, class Size>
void run_with_scratch(int index, const char* what, P& p, Call call, Size size) {
  using Key = std::pair<int, void*>;
  static auto* buffers = new std::map<Key, at::Tensor>();   // not freed at exit: the CUDA context may be gone by then
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream();
  const auto bytes = at::TensorOptions().dtype(at::kByte).device(at::kCUDA, index);
  auto offer = [&](const at::Tensor& t) {
    p.workspace = t.defined() ? t.mutable_data_ptr() : nullptr;
    p.workspace_bytes = t.defined() ? static_cast<size_t>(t.numel()) : 0;
  };
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
    const int64_t n = static_cast<int64_t>(size());
    const at::Tensor own = n > 0 ? at::empty({n}, bytes) : at::Tensor();
    offer(own);
    check_status(call(stream), what);
    return;
  }
  at::Tensor& kept = (*buffers)[Key(index, stream)];
  offer(kept);
  int status = call(stream);
  if (status == FA_B200_ERR_WORKSPACE) {
    const int64_t n = std::max<int64_t>(static_cast<int64_t>(size()), 1 << 20);
    at::Tensor grown = at::empty({n}, bytes);
    offer(grown);
    status = call(stream);
    if (n <= kKeptBytes) kept = std::move(grown);
  }
  check_status(status, what);
}
template <class Call>
void run(int index, const char* what, Call call) {
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
  check_status(call(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream()), what);
}

template <class P>
P sized() {
  P p;
  memset(&p, 0, sizeof(p));
  p.struct_size = sizeof(p);
  return p;
}
template <class P>
void set_keys(P& p, const at::Tensor& k, const at::Tensor& table, const at::Tensor& lens) {
  p.k_block_stride = k.stride(0);
  p.k_row_stride = k.stride(1);
  p.k_head_stride = k.stride(2);
  p.block_table = static_cast<const int32_t*>(table.const_data_ptr());
  p.block_table_batch_stride = table.stride(0);
  p.cache_seqlens = static_cast<const int32_t*>(lens.const_data_ptr());
  p.num_blocks = static_cast<int32_t>(k.size(0));
  p.page_size = static_cast<int32_t>(k.size(1));
  p.h_k = static_cast<int32_t>(k.size(2));
  p.d = static_cast<int32_t>(k.size(3));
  p.b = static_cast<int32_t>(table.size(0));
  p.max_blocks_per_seq = static_cast<int32_t>(table.size(-1));
}
PyObject* wrap(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!r) throw python_error();
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
    if (!o) { Py_DECREF(r); throw python_error(); }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// page_bounds(k_cache, block_table, cache_seqlens, bounds, new_tokens) -> bounds
PyObject* page_bounds(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 5);
  const at::Tensor &k = tensor(a[0], "k_cache"), &table = tensor(a[1], "block_table"), &lens = tensor(a[2], "cache_seqlens"),
                   &bounds = tensor(a[3], "page_bounds");
  forward_only({&k});
  const int index = check_cache(k, "page_bounds");
  check_tables(table, lens, index, "page_bounds");
  const at::ScalarType kt = k.scalar_type(), bt = bounds.scalar_type();
  TORCH_CHECK(bounds.dim() == 4 && bounds.size(0) == k.size(0) && bounds.size(1) == k.size(2) && bounds.size(2) == 2 && bounds.size(3) == k.size(3) &&
                  bounds.is_contiguous() && index_of(bounds) == index && is_half(bt) && (is_fp8(kt) || bt == kt),
              "page_bounds: bounds must be a contiguous tensor (num_blocks, nheads_k, 2, d) of the cache's type (fp16 or bf16 for an fp8 cache) "
              "on the cache's device");
  auto p = sized<fa_b200_page_bounds_params>();
  set_keys(p, k, table, lens);
  p.k_cache = k.const_data_ptr();
  p.page_bounds = bounds.mutable_data_ptr();
  p.new_tokens = integer(a[4], "new_tokens");
  p.dtype = code(kt);
  p.bounds_dtype = code(bt);
  run(index, "page_bounds", [&](cudaStream_t s) { return api.page_bounds(&p, s); });
  return Py_NewRef(a[3]);
  END_HANDLE_TH_ERRORS
}

// page_select(q, bounds, block_table, cache_seqlens, page_size, num_pages, sink_pages, recent_pages) -> page_table, seqlens, page_index
PyObject* page_select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 8);
  at::Tensor q = tensor(a[0], "q");
  const at::Tensor &bounds = tensor(a[1], "page_bounds"), &table = tensor(a[2], "block_table"), &lens = tensor(a[3], "cache_seqlens");
  forward_only({&q, &bounds});
  const int index = index_of(q);
  TORCH_CHECK(index >= 0 && q.dim() == 4 && is_half(q.scalar_type()), "page_select: q must be an fp16 / bf16 CUDA tensor (batch, seqlen_q, nheads, d)");
  if (q.stride(3) != 1) q = q.contiguous();
  TORCH_CHECK(bounds.dim() == 4 && bounds.size(2) == 2 && bounds.size(3) == q.size(3) && bounds.is_contiguous() &&
                  bounds.scalar_type() == q.scalar_type() && index_of(bounds) == index,
              "page_select: page_bounds must be a contiguous tensor (num_blocks, nheads_k, 2, d) of q's type on q's device");
  check_tables(table, lens, index, "page_select");
  TORCH_CHECK(table.size(0) == q.size(0), "page_select: block_table batch mismatch");
  auto p = sized<fa_b200_page_select_params>();
  p.num_pages = integer(a[5], "num_pages");
  TORCH_CHECK(p.num_pages > 0, "page_select: num_pages must be positive");
  const int64_t b = q.size(0), h_k = bounds.size(1);
  const auto ints = q.options().dtype(at::kInt);
  const at::Tensor pages = at::empty({b, h_k, p.num_pages}, ints), place = at::empty({b, h_k, p.num_pages}, ints), kept = at::empty({b, h_k}, ints);
  p.q = q.const_data_ptr();
  p.q_batch_stride = q.stride(0);
  p.q_row_stride = q.stride(1);
  p.q_head_stride = q.stride(2);
  p.page_bounds = bounds.const_data_ptr();
  p.block_table = static_cast<const int32_t*>(table.const_data_ptr());
  p.block_table_batch_stride = table.stride(0);
  p.cache_seqlens = static_cast<const int32_t*>(lens.const_data_ptr());
  p.page_table = static_cast<int32_t*>(pages.mutable_data_ptr());
  p.page_index = static_cast<int32_t*>(place.mutable_data_ptr());
  p.seqlens_out = static_cast<int32_t*>(kept.mutable_data_ptr());
  p.b = static_cast<int32_t>(b);
  p.seqlen_q = static_cast<int32_t>(q.size(1));
  p.h = static_cast<int32_t>(q.size(2));
  p.h_k = static_cast<int32_t>(h_k);
  p.d = static_cast<int32_t>(q.size(3));
  p.page_size = integer(a[4], "page_size");
  p.num_blocks = static_cast<int32_t>(bounds.size(0));
  p.max_blocks_per_seq = static_cast<int32_t>(table.size(1));
  p.sink_pages = integer(a[6], "sink_pages");
  p.recent_pages = integer(a[7], "recent_pages");
  p.dtype = code(q.scalar_type());
  run_with_scratch(index, "page_select", p, [&](cudaStream_t s) { return api.page_select(&p, s); }, [&] { return api.page_select_bytes(&p); });
  return wrap({pages, kept, place});
  END_HANDLE_TH_ERRORS
}

// fp32 descale of one element or shape (batch, h_k) -> pointer and strides.
void descale(const at::Tensor& t, const char* name, int64_t b, int64_t h_k, int index, const float*& ptr, int64_t& sb, int64_t& sh) {
  if (!t.defined()) return;
  TORCH_CHECK(t.scalar_type() == at::kFloat && index_of(t) == index, name, " must be a float32 tensor on q's device");
  ptr = static_cast<const float*>(t.const_data_ptr());
  if (t.numel() == 1) return;
  TORCH_CHECK(t.dim() == 2 && t.size(0) == b && t.size(1) == h_k, name, " must have one element or shape (batch, nheads_k)");
  sb = t.stride(0);
  sh = t.stride(1);
}

// decode_budget(q, k_cache, v_cache, block_table, seqlens, softmax_scale or None, is_causal, out, s_aux, window_left, token_weights,
//               token_weights_out, decay, q_descale, k_descale, v_descale, need_lse) -> out, softmax_lse or None, token weights or None
PyObject* decode_budget(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 17);
  at::Tensor q = tensor(a[0], "q"), table = tensor(a[3], "the block table"), sink = optional_tensor(a[8], "s_aux");
  const at::Tensor &k = tensor(a[1], "k_cache"), &v = tensor(a[2], "v_cache"), &lens = tensor(a[4], "the lengths");
  at::Tensor out = optional_tensor(a[7], "out");
  const at::Tensor w_in = optional_tensor(a[10], "token_weights"), w_out = optional_tensor(a[11], "token_weights_out");
  forward_only({&q, &k, &v});
  TORCH_CHECK_NOT_IMPLEMENTED(!(v.dim() == 4 && v.stride(3) != 1 && v.stride(1) == 1),
                              "a transposed V pool (layout 0) is outside the B200 hot path of this build");
  const int index = check_cache(k, "decode_budget", &v);
  const at::ScalarType qt = q.scalar_type(), kt = k.scalar_type();
  const bool fp8_kv = is_half(qt) && is_fp8(kt);
  TORCH_CHECK(q.dim() == 4 && index_of(q) == index, "q must be a CUDA tensor (batch, seqlen_q, nheads, d) on the caches' device");
  TORCH_CHECK(is_half(qt) || qt == at::kFloat8_e4m3fn, "FlashAttention only support fp16, bf16 and fp8 e4m3 data type");
  TORCH_CHECK(fp8_kv || kt == qt, "query and key must have the same dtype");
  if (q.stride(3) != 1) q = q.contiguous();
  const int64_t b = q.size(0), sq = q.size(1), h = q.size(2), h_k = k.size(2);
  TORCH_CHECK(k.size(3) == q.size(3), "query and key must have the same head dimension");
  TORCH_CHECK(h_k > 0 && h % h_k == 0, "Number of heads in key/value must divide number of heads in query");
  TORCH_CHECK(sq >= 1, "q must hold at least one token per sequence");
  TORCH_CHECK_NOT_IMPLEMENTED(!(fp8_kv && a[13] != Py_None), "an fp8 KV cache under 16-bit queries with q_descale is outside the B200 hot path "
                                                            "of this build");
  const bool per_head = table.dim() == 3;
  TORCH_CHECK((per_head || table.dim() == 2) && table.scalar_type() == at::kInt && index_of(table) == index && table.size(0) == b &&
                  (!per_head || table.size(1) == h_k),
              "the block table must be int32, (batch, n) or (batch, nheads_k, n), on q's device");
  if (!dense_last(table)) table = table.contiguous();
  TORCH_CHECK(lens.scalar_type() == at::kInt && index_of(lens) == index && lens.is_contiguous() && lens.dim() == (per_head ? 2 : 1) &&
                  lens.size(0) == b && (!per_head || lens.size(1) == h_k),
              "the lengths must be a contiguous int32 tensor, (batch,) or with a table for each kv head (batch, nheads_k)");
  at::ScalarType ot = qt == at::kFloat8_e4m3fn ? at::kBFloat16 : qt;
  if (out.defined()) {
    TORCH_CHECK(is_half(out.scalar_type()), "Output must be fp16 or bf16");
    TORCH_CHECK(qt == at::kFloat8_e4m3fn || out.scalar_type() == qt, "Output must have the same dtype as inputs");
    TORCH_CHECK(out.sizes() == q.sizes() && out.stride(3) == 1 && index_of(out) == index,
                "out must have the shape of q and a contiguous last dimension");
    ot = out.scalar_type();
  } else {
    out = at::empty(q.sizes(), q.options().dtype(ot));
  }
  const at::Tensor lse = truth(a[16]) ? at::empty({b, h, sq}, q.options().dtype(at::kFloat)) : at::Tensor();
  auto e = sized<fa_b200_decode_budget_params>();
  e.decay = number(a[12]);
  at::Tensor w;
  if (w_in.defined() || w_out.defined()) w = set_weights(e, w_in, w_out, b, h_k, index, "token weights");
  auto p = sized<fa_b200_decode_params>();
  set_keys(p, k, table, lens);
  if (per_head) {
    e.per_kv_head = 1;
    e.block_table_head_stride = table.stride(1);
  }
  p.q = q.const_data_ptr();
  p.k_cache = k.const_data_ptr();
  p.v_cache = v.const_data_ptr();
  p.out = out.mutable_data_ptr();
  p.softmax_lse = lse.defined() ? static_cast<float*>(lse.mutable_data_ptr()) : nullptr;
  p.q_batch_stride = q.stride(0);
  p.q_row_stride = q.stride(1);
  p.q_head_stride = q.stride(2);
  p.o_batch_stride = out.stride(0);
  p.o_row_stride = out.stride(1);
  p.o_head_stride = out.stride(2);
  p.v_block_stride = v.stride(0);
  p.v_row_stride = v.stride(1);
  p.v_head_stride = v.stride(2);
  p.h = static_cast<int32_t>(h);
  p.seqlen_q = static_cast<int32_t>(sq);
  p.softmax_scale = a[5] == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(q.size(3)))) : number(a[5]);
  p.dtype = code(qt);
  p.out_dtype = code(ot);
  descale(optional_tensor(a[13], "q_descale"), "q_descale", b, h_k, index, p.q_descale, p.q_descale_batch_stride, p.q_descale_head_stride);
  descale(optional_tensor(a[14], "k_descale"), "k_descale", b, h_k, index, p.k_descale, p.k_descale_batch_stride, p.k_descale_head_stride);
  descale(optional_tensor(a[15], "v_descale"), "v_descale", b, h_k, index, p.v_descale, p.v_descale_batch_stride, p.v_descale_head_stride);
  // looked at on every call, so that a process may change it while it runs
  if (const char* part = std::getenv("FA_B200_DECODE_PARTITION")) p.partition_tokens = std::atoi(part);
  p.profile_start_event = profile_events[0];
  p.profile_stop_event = profile_events[1];
  if (sink.defined()) {
    TORCH_CHECK(index_of(sink) == index && sink.dim() == 1 && sink.numel() == h, "s_aux must have shape (nheads,)");
    TORCH_CHECK(is_half(sink.scalar_type()) || sink.scalar_type() == at::kFloat, "s_aux must be fp16, bf16 or fp32");
    sink = sink.contiguous();
    p.s_aux = sink.const_data_ptr();
    p.s_aux_dtype = sink.scalar_type() == at::kFloat ? FA_B200_F32 : code(sink.scalar_type());
  }
  const int32_t left = integer(a[9], "window_size");
  if (left >= 0) {
    p.has_window = 1;
    p.window_left = left;
  }
  p.is_causal = truth(a[6]) ? 1 : 0;
  p.kv_e4m3 = fp8_kv ? 1 : 0;
  p.kv_e5m2 = fp8_kv && kt == at::kFloat8_e5m2 ? 1 : 0;
  run_with_scratch(index, "decode_budget", p, [&](cudaStream_t s) { return api.decode_budget(&p, &e, s); },
                   [&] { return api.decode_budget_bytes(&p, &e); });
  return wrap({out, lse, w});
  END_HANDLE_TH_ERRORS
}

// token_weights(q, k_cache, softmax_lse, cu_seqlens_q, max_seqlen_q, cache_seqlens, block_table, weights, softmax_scale or None,
//               is_causal, decay, weights_out) -> weights_out
PyObject* token_weights(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 12);
  at::Tensor q = tensor(a[0], "q");
  const at::Tensor &k = tensor(a[1], "k_cache"), &lse = tensor(a[2], "softmax_lse"), &cu = tensor(a[3], "cu_seqlens_q"),
                   &lens = tensor(a[5], "cache_seqlens"), &table = tensor(a[6], "block_table");
  forward_only({&q, &k});
  const int index = check_cache(k, "token_weights");
  check_tables(table, lens, index, "token_weights");
  TORCH_CHECK(q.dim() == 3 && index_of(q) == index, "token_weights: q must be (total_q, nheads, d) on the cache's device");
  TORCH_CHECK_NOT_IMPLEMENTED(is_half(q.scalar_type()) && k.scalar_type() == q.scalar_type(),
                              "token_weights with other than fp16 or bf16 queries and a cache of their type is outside the B200 hot path of this "
                              "build");
  if (q.stride(2) != 1) q = q.contiguous();
  const int64_t total = q.size(0), h = q.size(1), h_k = k.size(2), b = table.size(0);
  TORCH_CHECK(k.size(3) == q.size(2) && h_k > 0 && h % h_k == 0, "token_weights: q and k_cache must have the same d, and nheads_k must divide nheads");
  TORCH_CHECK(lse.scalar_type() == at::kFloat && index_of(lse) == index && lse.dim() == 2 && lse.size(0) == h && lse.size(1) == total && dense_last(lse),
              "token_weights: softmax_lse must be a float32 tensor (nheads, total_q) with contiguous last dimension");
  TORCH_CHECK(cu.scalar_type() == at::kInt && index_of(cu) == index && cu.dim() == 1 && cu.size(0) == b + 1 && cu.is_contiguous(),
              "token_weights: cu_seqlens_q must be a contiguous int32 tensor (batch + 1,)");
  auto p = sized<fa_b200_token_weights_params>();
  set_keys(p, k, table, lens);
  const at::Tensor w = set_weights(p, optional_tensor(a[7], "token_weights"), optional_tensor(a[11], "token_weights_out"), b, h_k, index, "token_weights");
  p.q = q.const_data_ptr();
  p.q_row_stride = q.stride(0);
  p.q_head_stride = q.stride(1);
  p.softmax_lse = static_cast<const float*>(lse.const_data_ptr());
  p.lse_head_stride = lse.stride(0);
  p.cu_seqlens_q = static_cast<const int32_t*>(cu.const_data_ptr());
  p.k_cache = k.const_data_ptr();
  p.decay = number(a[10]);
  p.total_q = total;
  p.max_seqlen_q = integer(a[4], "max_seqlen_q");
  p.h = static_cast<int32_t>(h);
  p.softmax_scale = a[8] == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(q.size(2)))) : number(a[8]);
  p.is_causal = truth(a[9]) ? 1 : 0;
  p.dtype = code(q.scalar_type());
  run_with_scratch(index, "token_weights", p, [&](cudaStream_t s) { return api.token_weights(&p, s); }, [&] { return api.token_weights_bytes(&p); });
  return THPVariable_Wrap(w);
  END_HANDLE_TH_ERRORS
}

// kv_evict(k_cache, v_cache, block_table, cache_seqlens, weights, budget, sink_tokens, recent_tokens, new_block_table, weights_out)
//   -> kept_index, new lengths
PyObject* kv_evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 10);
  const at::Tensor &k = tensor(a[0], "k_cache"), &v = tensor(a[1], "v_cache"), &table = tensor(a[2], "block_table"),
                   &lens = tensor(a[3], "cache_seqlens");
  const at::Tensor w = optional_tensor(a[4], "token_weights"), w_out = optional_tensor(a[9], "token_weights_out");
  TORCH_CHECK(w.defined(), "kv_evict: token_weights is required");
  const at::Tensor fresh = optional_tensor(a[8], "new_block_table");
  forward_only({&k, &v});
  const int index = check_cache(k, "kv_evict", &v);
  check_tables(table, lens, index, "kv_evict");
  const int64_t b = table.size(0), h_k = k.size(2);
  auto p = sized<fa_b200_kv_evict_params>();
  set_keys(p, k, table, lens);
  set_weights(p, w, w_out, b, h_k, index, "kv_evict");
  p.budget = integer(a[5], "budget");
  TORCH_CHECK(p.budget > 0, "kv_evict: budget must be positive");
  p.sink_tokens = integer(a[6], "sink_tokens");
  p.recent_tokens = integer(a[7], "recent_tokens");
  if (fresh.defined()) {
    TORCH_CHECK(fresh.scalar_type() == at::kInt && fresh.dim() == 2 && index_of(fresh) == index && fresh.size(0) == b && dense_last(fresh),
                "kv_evict: new_block_table must be like block_table");
    p.new_block_table = static_cast<const int32_t*>(fresh.const_data_ptr());
    p.new_block_table_batch_stride = fresh.stride(0);
    p.new_max_blocks_per_seq = static_cast<int32_t>(fresh.size(1));
  }
  p.k_cache = k.mutable_data_ptr();
  p.v_cache = v.mutable_data_ptr();
  p.v_block_stride = v.stride(0);
  p.v_row_stride = v.stride(1);
  p.v_head_stride = v.stride(2);
  p.dtype = code(k.scalar_type());
  const auto ints = k.options().dtype(at::kInt);
  const at::Tensor kept = at::empty({b, h_k, p.budget}, ints), now = at::empty({b}, ints);
  p.kept_index = static_cast<int32_t*>(kept.mutable_data_ptr());
  p.seqlens_out = static_cast<int32_t*>(now.mutable_data_ptr());
  run(index, "kv_evict", [&](cudaStream_t s) { return api.kv_evict(&p, s); });
  return wrap({kept, now});
  END_HANDLE_TH_ERRORS
}

// bind(addresses): the library's functions, in the order of FUNCTIONS.
PyObject* bind(PyObject*, PyObject* addresses) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(PyTuple_Check(addresses) && PyTuple_GET_SIZE(addresses) == kFunctions, "bind: a tuple of ", kFunctions, " addresses");
  void* p[kFunctions];
  for (Py_ssize_t i = 0; i < kFunctions; ++i) {
    p[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(addresses, i));
    if (!p[i]) throw python_error();
  }
  memcpy(&api, p, sizeof(api));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// set_profile_events(start, stop): CUDA event handles (0: none) recorded around the main kernel of decode_budget.
PyObject* set_profile_events(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 2);
  for (int i = 0; i < 2; ++i) {
    profile_events[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) throw python_error();
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, nullptr},
    {"set_profile_events", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(set_profile_events)), METH_FASTCALL, nullptr},
    {"page_bounds", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(page_bounds)), METH_FASTCALL,
     "fa_b200_page_bounds: (k_cache, block_table, cache_seqlens, bounds, new_tokens) -> bounds"},
    {"page_select", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(page_select)), METH_FASTCALL,
     "fa_b200_page_select: (q, bounds, block_table, cache_seqlens, page_size, num_pages, sink_pages, recent_pages) -> (page_table, "
     "seqlens, page_index)"},
    {"decode_budget", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(decode_budget)), METH_FASTCALL,
     "fa_b200_decode_budget: (q, k_cache, v_cache, block_table, seqlens, softmax_scale, is_causal, out, s_aux, window_left, token_weights, "
     "token_weights_out, decay, q_descale, k_descale, v_descale, need_lse) -> (out, softmax_lse, token weights)"},
    {"token_weights", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(token_weights)), METH_FASTCALL,
     "fa_b200_token_weights: (q, k_cache, softmax_lse, cu_seqlens_q, max_seqlen_q, cache_seqlens, block_table, weights, softmax_scale, "
     "is_causal, decay, weights_out) -> weights_out"},
    {"kv_evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(kv_evict)), METH_FASTCALL,
     "fa_b200_kv_evict: (k_cache, v_cache, block_table, cache_seqlens, weights, budget, sink_tokens, recent_tokens, new_block_table, "
     "weights_out) -> (kept_index, new lengths)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fa_b200_host", "Host part of the bounded-cache calls of libfa_b200.so", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fa_b200_host() {
  PyObject* m = PyModule_Create(&module);
  PyObject* names = PyTuple_New(kFunctions);
  bool ok = m && names;
  for (Py_ssize_t i = 0; ok && i < kFunctions; ++i) {
    PyObject* name = PyUnicode_FromString(functions[i]);
    ok = name != nullptr;
    if (ok) PyTuple_SET_ITEM(names, i, name);
  }
  ok = ok && PyModule_AddObjectRef(m, "FUNCTIONS", names) == 0 && PyModule_AddStringConstant(m, "BUILT_FOR", FA_B200_HOST_KEY) == 0;
  Py_XDECREF(names);
  if (!ok) Py_CLEAR(m);
  return m;
}
