// The host side of a call in native code: reads the tensors' addresses, sizes and strides, allocates the results
// and fills the C ABI's argument structs (include/splash_b200.h), which python did field by field through ctypes.
// forward() takes 12 us and backward() 25 (three launches), launches included; a whole forward pass of 256 tokens went
// from 39 to 21 us, a training step of 2 x 1024 from 176 to 114.  attention() is the autograd function in native code too, for
// calls without segment ids, sinks and a fixed maximum: a whole pass of those two 21.0 -> 16.5 and 118.8 -> 93.1 us.  The checks of
// arguments, the schedules and the autograd function of the other calls are in splash_attention_kernel.py.
#include <torch/csrc/utils/pybind.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <ATen/ATen.h>
#include <ATen/ExpandUtils.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <memory>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/splash_b200.h"

namespace {

// entry points of libsplash_b200.so, as ctypes resolved them
struct Library {
  int (*fwd)(const SplashFwdArgs*, const SplashShards*, void*) = nullptr;
  int (*bwd)(const SplashBwdArgs*, const SplashShards*, void*) = nullptr;
  size_t (*workspace_bytes)(int64_t, int64_t, int64_t) = nullptr;
  size_t (*fused_workspace_bytes)(int64_t, int64_t, int64_t) = nullptr;
} lib;

void bind_library(uintptr_t fwd, uintptr_t bwd, uintptr_t workspace_bytes, uintptr_t fused_workspace_bytes) {
  lib.fwd = reinterpret_cast<decltype(lib.fwd)>(fwd);
  lib.bwd = reinterpret_cast<decltype(lib.bwd)>(bwd);
  lib.workspace_bytes = reinterpret_cast<decltype(lib.workspace_bytes)>(workspace_bytes);
  lib.fused_workspace_bytes = reinterpret_cast<decltype(lib.fused_workspace_bytes)>(fused_workspace_bytes);
}

// `t` if the kernels can read it in place, else a contiguous copy
at::Tensor usable(const at::Tensor& t) {
  TORCH_CHECK(t.dim() == 4, "expected a tensor of rank 4, got rank ", t.dim());
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && t.stride(i) % 8 == 0;
  if (ok) return t;
  const at::Tensor copy = t.contiguous();  // (t itself where it is contiguous and begins between two boundaries of 16 bytes)
  return copy.data_ptr() == t.data_ptr() ? copy.clone(at::MemoryFormat::Contiguous) : copy;
}

// The kernels follow every address that they are given: each must be one of their own device, that of `q`.
void require_beside(const at::Tensor& t, const at::Tensor& q) {
  TORCH_CHECK(t.device() == q.device(), "expected all tensors on the device of q, ", q.device(), ", got one on ", t.device());
}

SplashTensor describe(const at::Tensor& t, const at::Tensor& q) {
  TORCH_CHECK(t.dim() == 4, "expected a tensor of rank 4, got rank ", t.dim());
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, "expected bfloat16 operands, got ", t.scalar_type());
  require_beside(t, q);
  SplashTensor d{};
  d.data = t.data_ptr();
  d.dtype = SPLASH_BF16;
  for (int i = 0; i < 4; ++i) d.size[i] = t.size(i), d.stride[i] = t.stride(i);
  return d;
}

template <typename T>
T* pointer(const at::Tensor& t, const at::Tensor& q) {
  require_beside(t, q);
  return static_cast<T*>(t.data_ptr());
}
template <typename T>
T* pointer(const std::optional<at::Tensor>& t, const at::Tensor& q) {
  return t.has_value() ? pointer<T>(*t, q) : nullptr;
}

template <typename T>
const T& at_address(uintptr_t a) {
  return *reinterpret_cast<const T*>(a);
}

using Maybe = std::optional<at::Tensor>;

// Gives the interpreter's lock up, where this thread holds it.
class WithoutGil {
  std::optional<pybind11::gil_scoped_release> release_;

 public:
  WithoutGil() {
    if (PyGILState_Check()) release_.emplace();
  }
};

// `sched`, `mask_fn`, `o_peer`: addresses of the structs (o_peer: 0 for none).  Returns the status, the operands as
// the kernel read them, and the results.
std::tuple<int, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> forward(
    const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in, const Maybe& q_seg, const Maybe& kv_seg,
    const Maybe& q_sequence, const Maybe& sinks, const Maybe& max_logit, const at::Tensor& error_record, uintptr_t sched,
    uintptr_t mask_fn, double scale, double mask_value, double soft_cap, int head_shards, int q_shards, uintptr_t o_peer) {
  const at::Tensor q = usable(q_in), k = usable(k_in), v = usable(v_in);
  const int64_t b = q.size(0), hq = q.size(1), sq = q.size(2);
  // (like q, it keeps q's dense stride order, e.g. [B,T,H,D] storage stays [B,T,H,D])
  const at::Tensor o = v.size(3) == q.size(3) ? at::empty_like(q) : at::empty({b, hq, sq, v.size(3)}, q.options());
  const auto f32 = q.options().dtype(at::kFloat);
  const at::Tensor lse = at::empty({b, hq, sq}, f32), max_logits = at::empty({b, hq, sq}, f32);
  SplashFwdArgs a{};
  a.q = describe(q, q);
  a.k = describe(k, q);
  a.v = describe(v, q);
  a.o = describe(o, q);
  a.logsumexp = pointer<float>(lse, q);
  a.max_logits = static_cast<float*>(max_logits.data_ptr());
  a.q_segment_ids = pointer<int32_t>(q_seg, q);
  a.kv_segment_ids = pointer<int32_t>(kv_seg, q);
  a.q_sequence = pointer<int32_t>(q_sequence, q);
  a.sched = at_address<SplashDeviceSchedule>(sched);
  a.mask_fn = at_address<SplashMaskFn>(mask_fn);
  a.scale = (float)scale;
  a.mask_value = (float)mask_value;
  a.error_record = pointer<uint32_t>(error_record, q);
  a.sinks = pointer<float>(sinks, q);
  a.max_logit_value = pointer<float>(max_logit, q);
  a.soft_cap = (float)soft_cap;
  if (o_peer != 0) a.o_peer = at_address<SplashPeerOutput>(o_peer);
  const SplashShards shards{head_shards, q_shards};
  int status;
  {
    const WithoutGil release;
    const c10::OptionalDeviceGuard guard(q.device());
    status = lib.fwd(&a, &shards, c10::cuda::getCurrentCUDAStream(q.device().index()).stream());
  }
  return {status, q, k, v, o, lse, max_logits};
}

// `peers`: addresses of three SplashPeerOutput, or zeros.  Returns the status, the gradients and the workspace.
std::tuple<int, at::Tensor, at::Tensor, at::Tensor, at::Tensor> backward(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& o, const at::Tensor& lse,
    const at::Tensor& d_o_in, const Maybe& q_seg, const Maybe& kv_seg, const Maybe& q_sequence, const at::Tensor& error_record,
    uintptr_t sched_dq, uintptr_t sched_dkv, uintptr_t mask_fn, double scale, double soft_cap, bool fused, int head_shards,
    int q_shards, uintptr_t dq_peer, uintptr_t dk_peer, uintptr_t dv_peer) {
  const at::Tensor d_o = usable(d_o_in);
  const at::Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
  SplashBwdArgs a{};
  a.q = describe(q, q);
  a.k = describe(k, q);
  a.v = describe(v, q);
  a.o = describe(o, q);
  a.d_o = describe(d_o, q);
  a.dq = describe(dq, q);
  a.dk = describe(dk, q);
  a.dv = describe(dv, q);
  const size_t bytes = (fused ? lib.fused_workspace_bytes : lib.workspace_bytes)(q.size(0), q.size(1), q.size(2));
  const at::Tensor workspace = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  a.flags = fused ? SPLASH_BWD_FUSED_DQ : 0;
  a.logsumexp = pointer<float>(lse, q);
  a.q_segment_ids = pointer<int32_t>(q_seg, q);
  a.kv_segment_ids = pointer<int32_t>(kv_seg, q);
  a.q_sequence = pointer<int32_t>(q_sequence, q);
  a.sched_dq = at_address<SplashDeviceSchedule>(sched_dq);
  a.sched_dkv = at_address<SplashDeviceSchedule>(sched_dkv);
  a.mask_fn = at_address<SplashMaskFn>(mask_fn);
  a.scale = (float)scale;
  a.workspace = workspace.data_ptr();
  a.workspace_bytes = bytes;
  a.error_record = pointer<uint32_t>(error_record, q);
  a.soft_cap = (float)soft_cap;
  if (dq_peer != 0) a.dq_peer = at_address<SplashPeerOutput>(dq_peer);
  if (dk_peer != 0) a.dk_peer = at_address<SplashPeerOutput>(dk_peer);
  if (dv_peer != 0) a.dv_peer = at_address<SplashPeerOutput>(dv_peer);
  const SplashShards shards{head_shards, q_shards};
  int status;
  {
    const WithoutGil release;
    const c10::OptionalDeviceGuard guard(q.device());
    status = lib.bwd(&a, &shards, c10::cuda::getCurrentCUDAStream(q.device().index()).stream());
  }
  return {status, dq, dk, dv, workspace};
}

// The schedules of one kernel object on one device, with the tensors that hold them.
struct Tables {
  SplashDeviceSchedule fwd, dq, dkv;
  std::vector<at::Tensor> held;
  at::Tensor error_record;
  Maybe q_sequence;
  int q_shards;

  Tables(uintptr_t fwd, uintptr_t dq, uintptr_t dkv, std::vector<at::Tensor> held, at::Tensor error_record, Maybe q_sequence,
         int q_shards)
      : fwd(at_address<SplashDeviceSchedule>(fwd)),
        dq(at_address<SplashDeviceSchedule>(dq)),
        dkv(at_address<SplashDeviceSchedule>(dkv)),
        held(std::move(held)),
        error_record(std::move(error_record)),
        q_sequence(std::move(q_sequence)),
        q_shards(q_shards) {}
};

// What the backward of a call needs beside its tensors.
struct Call : torch::CustomClassHolder {
  std::shared_ptr<const Tables> tables;
  SplashMaskFn mask_fn;
  double scale, mask_value, soft_cap;
  bool fused;
  int head_shards;
};

// `_native.check`, held for the life of the process: raises the package's exception for a status that is not zero
PyObject* check_status = nullptr;

// From a thread that does not hold the interpreter's lock, as python's own exception.
void raise_status(int status, const char* what) {
  pybind11::gil_scoped_acquire gil;
  Py_XDECREF(PyObject_CallFunction(check_status, "is", status, what));
  python_error error;
  error.persist();
  throw std::move(error);
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// As _SplashFunction of splash_attention_kernel.py.
struct Attention : torch::autograd::Function<Attention> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                               const c10::intrusive_ptr<Call>& call) {
    const Tables& t = *call->tables;
    auto [status, q, k, v, o, lse, max_logits] = ::forward(
        q_in, k_in, v_in, {}, {}, t.q_sequence, {}, {}, t.error_record, reinterpret_cast<uintptr_t>(&t.fwd),
        reinterpret_cast<uintptr_t>(&call->mask_fn), call->scale, call->mask_value, call->soft_cap, call->head_shards, t.q_shards, 0);
    if (status != 0) raise_status(status, "splash_fwd");
    ctx->save_for_backward({q, k, v, o, lse});
    ctx->saved_data["call"] = c10::IValue::make_capsule(call);
    ctx->mark_non_differentiable({lse, max_logits});
    ctx->set_materialize_grads(false);  // no zeros made up for the gradients of lse and max_logits
    return {o, lse, max_logits};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &lse = saved[4];
    const auto call = c10::static_intrusive_pointer_cast<Call>(ctx->saved_data["call"].toCapsule());
    const Tables& t = *call->tables;
    const at::Tensor d_o = grads[0].defined() ? grads[0] : at::zeros_like(o);  // an undefined gradient of o is zero
    auto [status, dq, dk, dv, workspace] = ::backward(
        q, k, v, o, lse, d_o, {}, {}, t.q_sequence, t.error_record, reinterpret_cast<uintptr_t>(&t.dq),
        reinterpret_cast<uintptr_t>(&t.dkv), reinterpret_cast<uintptr_t>(&call->mask_fn), call->scale, call->soft_cap,
        call->fused, call->head_shards, t.q_shards, 0, 0, 0);
    if (status != 0) raise_status(status, "splash_bwd");
    return {dq, dk, dv, at::Tensor()};
  }
};

// Output, logsumexp and max_logits, the output differentiable.
std::tuple<at::Tensor, at::Tensor, at::Tensor> attention(const std::shared_ptr<Tables>& tables, const at::Tensor& q,
                                                         const at::Tensor& k, const at::Tensor& v, uintptr_t mask_fn,
                                                         double scale, double mask_value, double soft_cap, bool fused,
                                                         int head_shards) {
  auto call = c10::make_intrusive<Call>();
  call->tables = tables;
  call->mask_fn = at_address<SplashMaskFn>(mask_fn);
  call->scale = scale;
  call->mask_value = mask_value;
  call->soft_cap = soft_cap;
  call->fused = fused;
  call->head_shards = head_shards;
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    out = Attention::apply(q, k, v, call);
  }
  return {out[0], out[1], out[2]};
}

// ------------------------------------------------------------------------------------------------------------------
// the quantised key / value cache (kv_cache.py): checks of arguments, results, launches
// ------------------------------------------------------------------------------------------------------------------
struct CacheLibrary {
  int (*append)(const SplashCacheAppendArgs*, void*) = nullptr;
  int (*read)(const SplashCacheReadArgs*, void*) = nullptr;
  int (*attend)(const SplashCacheAttendArgs*, void*) = nullptr;
  size_t (*attend_workspace_bytes)(const SplashCacheAttendArgs*) = nullptr;
} cache_lib;

void bind_cache_library(uintptr_t append, uintptr_t read, uintptr_t attend, uintptr_t attend_workspace_bytes) {
  cache_lib.append = reinterpret_cast<decltype(cache_lib.append)>(append);
  cache_lib.read = reinterpret_cast<decltype(cache_lib.read)>(read);
  cache_lib.attend = reinterpret_cast<decltype(cache_lib.attend)>(attend);
  cache_lib.attend_workspace_bytes = reinterpret_cast<decltype(cache_lib.attend_workspace_bytes)>(attend_workspace_bytes);
}

struct PageLibrary {
  int (*attend)(const SplashCacheAttendArgs*, void*) = nullptr;
  size_t (*attend_workspace_bytes)(const SplashCacheAttendArgs*) = nullptr;
  int (*bound)(const SplashCacheBoundArgs*, void*) = nullptr;
  int (*bound_values)(const SplashKvCache*, const SplashPageBounds*, float*, void*) = nullptr;
  int (*choose)(const SplashCacheChooseArgs*, void*) = nullptr;
  size_t (*choose_workspace_bytes)(const SplashCacheChooseArgs*) = nullptr;
} page_lib;

void bind_page_library(uintptr_t attend, uintptr_t attend_workspace_bytes, uintptr_t bound, uintptr_t bound_values, uintptr_t choose,
                       uintptr_t choose_workspace_bytes) {
  page_lib.attend = reinterpret_cast<decltype(page_lib.attend)>(attend);
  page_lib.attend_workspace_bytes = reinterpret_cast<decltype(page_lib.attend_workspace_bytes)>(attend_workspace_bytes);
  page_lib.bound = reinterpret_cast<decltype(page_lib.bound)>(bound);
  page_lib.bound_values = reinterpret_cast<decltype(page_lib.bound_values)>(bound_values);
  page_lib.choose = reinterpret_cast<decltype(page_lib.choose)>(choose);
  page_lib.choose_workspace_bytes = reinterpret_cast<decltype(page_lib.choose_workspace_bytes)>(choose_workspace_bytes);
}

// A cache's description, with the tensors that it lies in.
struct KvCache {
  SplashKvCache desc{};
  at::Tensor k_codes, k_scales, v_codes, v_scales;

  KvCache(at::Tensor k_codes_in, at::Tensor k_scales_in, at::Tensor v_codes_in, at::Tensor v_scales_in, int format, int group,
          int head_dim, int head_dim_v, int row_k, int row_v)
      : k_codes(std::move(k_codes_in)), k_scales(std::move(k_scales_in)), v_codes(std::move(v_codes_in)), v_scales(std::move(v_scales_in)) {
    for (const at::Tensor* t : {&k_codes, &k_scales, &v_codes, &v_scales})
      TORCH_CHECK_VALUE(t->is_contiguous() && t->device() == k_codes.device(), "the arrays of a cache are contiguous, on one device");
    desc.k_codes = k_codes.data_ptr();
    desc.k_scales = k_scales.data_ptr();
    desc.v_codes = v_codes.data_ptr();
    desc.v_scales = v_scales.data_ptr();
    desc.n_pages = k_codes.size(0);
    desc.kv_heads = (int32_t)k_codes.size(1);
    desc.page_size = (int32_t)k_codes.size(2);
    desc.format = format;
    desc.group = group;
    desc.head_dim = head_dim;
    desc.head_dim_v = head_dim_v;
    desc.row_k = row_k;
    desc.row_v = row_v;
  }
};

void require_on_gpu(const at::Tensor& t, const KvCache& cache, const char* name) {
  TORCH_CHECK(cache.k_codes.is_cuda(), "a cache on ", cache.k_codes.device(), ": the kernels need a CUDA device");
  TORCH_CHECK_VALUE(t.device() == cache.k_codes.device(), name, " is on ", t.device(), ", the cache on ", cache.k_codes.device());
}

// The result of a cache's operator cannot be differentiated: refused rather than cut off from its inputs without a word.
void require_no_grad(const at::Tensor& t, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(t.requires_grad() && at::GradMode::is_enabled()), name,
                              " requires a gradient: the cache's operators have none (call them under torch.no_grad())");
  TORCH_CHECK_NOT_IMPLEMENTED(!(t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode()), name,
                              " has a tangent of forward mode: the cache's operators have none");
}

// A recorded graph (of torch.jit.trace or make_fx) would hold results of this call, or what allocates them, and not the launch that
// writes them.
void require_not_recorded(const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), what, " cannot be recorded by torch.jit.trace");
  TORCH_CHECK_NOT_IMPLEMENTED(!c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(), what,
                              " cannot be recorded by make_fx");
}
void require_not_traced() { require_not_recorded("the cache's operators"); }

void require_row_type(at::ScalarType type, const char* name, bool f32_too) {
  TORCH_CHECK_NOT_IMPLEMENTED(type == at::kBFloat16 || type == at::kHalf || (f32_too && type == at::kFloat), name, ": ", type,
                              " is not built (bfloat16, float16", f32_too ? ", float32)" : ")");
}

SplashTensor describe_row_tensor(const at::Tensor& t, const char* name, bool f32_too) {
  SplashTensor d{};
  const auto type = t.scalar_type();
  require_row_type(type, name, f32_too);
  d.dtype = type == at::kBFloat16 ? SPLASH_BF16 : type == at::kHalf ? SPLASH_F16 : SPLASH_F32;
  d.data = t.data_ptr();
  TORCH_CHECK_VALUE(d.data != nullptr || t.numel() == 0, name, ": a tensor without memory (a fake or a functional one?)");
  for (int i = 0; i < 4; ++i) d.size[i] = t.size(i), d.stride[i] = t.stride(i);
  return d;
}

// Raises what `status` stands for; called with the interpreter's lock held.
void check_cache_call(int status, const char* what) {
  if (status == 0) return;
  TORCH_CHECK_NOT_IMPLEMENTED(status != SPLASH_ERR_UNSUPPORTED, what, ": not built for these sizes or types");
  Py_XDECREF(PyObject_CallFunction(check_status, "is", status, what));
  throw python_error();
}

// Memory for results, from torch's allocator without its dispatcher (a microsecond less for each).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, at::Device device) { return at::detail::empty_cuda(sizes, type, device, std::nullopt); }
// In the order of t's strides, dense.
at::Tensor fresh_like(const at::Tensor& t) {
  if (t.is_non_overlapping_and_dense()) return at::detail::empty_strided_cuda(t.sizes(), t.strides(), t.scalar_type(), t.device());
  return at::detail::empty_strided_cuda(t.sizes(), at::infer_dense_strides(t.sizes(), t.strides()), t.scalar_type(), t.device());
}

template <typename Fn>
int on_stream_of(const at::Tensor& t, Fn&& call) {
  const WithoutGil release;
  const c10::OptionalDeviceGuard guard(t.device());
  return call(static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()));
}

void cache_append(const KvCache& cache, const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& slots_in) {
  const SplashKvCache& c = cache.desc;
  require_not_traced();
  TORCH_CHECK_VALUE(k_in.dim() == 4 && v_in.dim() == 4 && slots_in.dim() == 2, "expected k and v of [B, H, T, D] and slots of [B, T]");
  TORCH_CHECK_VALUE(k_in.size(1) == c.kv_heads && k_in.size(3) == c.head_dim && v_in.size(3) == c.head_dim_v, "k ", k_in.sizes(), " / v ",
                    v_in.sizes(), " do not match a cache of ", c.kv_heads, " heads of ", c.head_dim, " / ", c.head_dim_v, " channels");
  TORCH_CHECK_VALUE(v_in.sizes().slice(0, 3) == k_in.sizes().slice(0, 3) && slots_in.size(0) == k_in.size(0) && slots_in.size(1) == k_in.size(2),
                    "k ", k_in.sizes(), ", v ", v_in.sizes(), " and slots ", slots_in.sizes(), " do not match");
  TORCH_CHECK_VALUE(k_in.scalar_type() == v_in.scalar_type(), "k and v have one type, got ", k_in.scalar_type(), " and ", v_in.scalar_type());
  const auto type = slots_in.scalar_type();
  TORCH_CHECK_VALUE(type == at::kInt || type == at::kLong, "slots are int32 or int64, got ", type);
  require_no_grad(k_in, "k");
  require_no_grad(v_in, "v");
  require_on_gpu(k_in, cache, "k");
  require_on_gpu(v_in, cache, "v");
  require_on_gpu(slots_in, cache, "slots");
  SplashCacheAppendArgs a{};
  a.cache = c;
  if (slots_in.numel() == 0) return;
  const at::Tensor k = usable(k_in), v = usable(v_in), slots = slots_in.stride(1) == 1 || slots_in.size(1) == 1 ? slots_in : slots_in.contiguous();
  a.k = describe_row_tensor(k, "k", true);
  a.v = describe_row_tensor(v, "v", true);
  a.slots = slots.data_ptr();
  a.slots_are_64 = type == at::kLong;
  a.slot_stride = slots.stride(0);
  check_cache_call(on_stream_of(k, [&](void* stream) { return cache_lib.append(&a, stream); }), "splash_cache_append");
}

// What can be said of page tables and lengths wherever they are; calls make all such checks before they ask for the device.
void require_pages(const at::Tensor& table, const at::Tensor& lengths, int64_t pages) {
  TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && lengths.scalar_type() == at::kInt, "the page table and the lengths are int32");
  TORCH_CHECK_VALUE(pages >= 1 && pages <= INT32_MAX, "a page table of ", pages, " pages");
}
// [B, pages] and [B]
void require_pages_of_sequences(const at::Tensor& table, const at::Tensor& lengths) {
  TORCH_CHECK_VALUE(table.dim() == 2 && lengths.dim() == 1 && table.size(0) == lengths.size(0), "page table ", table.sizes(), " and lengths ",
                    lengths.sizes(), " do not match: expected [B, pages] and [B]");
  require_pages(table, lengths, table.size(1));
  TORCH_CHECK_VALUE(lengths.size(0) <= 1 || lengths.stride(0) == 1, "lengths are contiguous");
}
void require_pages_on_gpu(const at::Tensor& table, const at::Tensor& lengths, const KvCache& cache) {
  require_on_gpu(table, cache, "the page table");
  require_on_gpu(lengths, cache, "lengths");
}

// A page table [B, pages] and the lengths [B] of the sequences (require_pages_of_sequences), as the kernels take them.
template <typename Args>
at::Tensor set_pages(Args& a, const KvCache& cache, const at::Tensor& table_in, const at::Tensor& lengths) {
  require_pages_on_gpu(table_in, lengths, cache);
  const at::Tensor table = table_in.size(1) <= 1 || table_in.stride(1) == 1 ? table_in : table_in.contiguous();
  a.cache = cache.desc;
  a.page_table = static_cast<const int32_t*>(table.data_ptr());
  a.table_stride = table.stride(0);
  a.n_table = (int32_t)table.size(1);
  a.lengths = static_cast<const int32_t*>(lengths.data_ptr());
  return table;
}

std::tuple<at::Tensor, at::Tensor> cache_read(const KvCache& cache, const at::Tensor& table_in, const at::Tensor& lengths, int64_t max_len,
                                              at::ScalarType type) {
  const SplashKvCache& c = cache.desc;
  require_not_traced();
  SplashCacheReadArgs a{};
  require_pages_of_sequences(table_in, lengths);
  TORCH_CHECK_VALUE(max_len >= 0, "max_len is not negative, got ", max_len);
  const at::Tensor table = set_pages(a, cache, table_in, lengths);
  const auto options = cache.k_codes.options().dtype(type);
  const at::Tensor k = at::empty({lengths.size(0), c.kv_heads, max_len, c.head_dim}, options);
  const at::Tensor v = at::empty({lengths.size(0), c.kv_heads, max_len, c.head_dim_v}, options);
  a.k = describe_row_tensor(k, "dtype", true);
  a.v = describe_row_tensor(v, "dtype", true);
  if (k.numel() != 0)
    check_cache_call(on_stream_of(k, [&](void* stream) { return cache_lib.read(&a, stream); }), "splash_cache_read");
  return {k, v};
}

std::tuple<at::Tensor, Maybe, Maybe> cache_attend(const KvCache& cache, const at::Tensor& q_in, const at::Tensor& table_in,
                                                  const at::Tensor& lengths_in, double scale, std::optional<int64_t> window,
                                                  std::optional<double> soft_cap, const Maybe& sinks_in, double mask_value, bool residuals) {
  const SplashKvCache& c = cache.desc;
  require_not_traced();
  require_no_grad(q_in, "q");
  if (sinks_in.has_value()) require_no_grad(*sinks_in, "sinks");
  TORCH_CHECK_VALUE(q_in.dim() == 4 && q_in.size(3) == c.head_dim && q_in.size(1) % c.kv_heads == 0, "q ", q_in.sizes(),
                    " does not match a cache of ", c.kv_heads, " heads of ", c.head_dim, " channels: expected [B, heads, T, D]");
  SplashCacheAttendArgs a{};
  const bool by_head = table_in.dim() == 4;  // a table for each kv head and query
  at::Tensor table, lengths = lengths_in;
  if (by_head) {
    TORCH_CHECK_VALUE(lengths.dim() == 3 && table_in.sizes().slice(0, 3) == lengths.sizes() && table_in.size(0) == q_in.size(0) &&
                          table_in.size(1) == c.kv_heads && table_in.size(2) == q_in.size(2),
                      "page tables ", table_in.sizes(), " and lengths ", lengths.sizes(), " do not match: expected [B, kv_heads, T, pages] and [B, kv_heads, T]");
    TORCH_CHECK_VALUE(!window.has_value(), "local_window_size goes by places in the sequence, which tables of chosen pages do not say");
    require_pages(table_in, lengths, table_in.size(3));
    require_pages_on_gpu(table_in, lengths, cache);
    table = table_in.contiguous();  // (rows one behind the other)
    lengths = lengths.contiguous();
    a.cache = cache.desc;
    a.page_table = static_cast<const int32_t*>(table.data_ptr());
    a.table_stride = table.size(3);
    a.n_table = (int32_t)table.size(3);
    a.lengths = static_cast<const int32_t*>(lengths.data_ptr());
  } else {
    require_pages_of_sequences(table_in, lengths);
    TORCH_CHECK_VALUE(q_in.size(0) == lengths.size(0), "q of ", q_in.size(0), " sequences, lengths of ", lengths.size(0));
    table = set_pages(a, cache, table_in, lengths);
  }
  TORCH_CHECK_VALUE(!window.has_value() || (*window >= 0 && *window <= INT32_MAX), "local_window_size is not negative");
  TORCH_CHECK_VALUE(!soft_cap.has_value() || (float)*soft_cap > 0, "logits_soft_cap is positive (in 32 bits), got ", *soft_cap);
  TORCH_CHECK_VALUE(!std::isnan(scale), "logits_scale is NaN");
  require_on_gpu(q_in, cache, "q");
  const int64_t b = q_in.size(0), heads = q_in.size(1), t = q_in.size(2);
  Maybe sinks;
  if (sinks_in.has_value()) {
    TORCH_CHECK_VALUE(sinks_in->dim() == 1 && sinks_in->size(0) == heads, "sinks ", sinks_in->sizes(), " for ", heads, " q heads");
    require_on_gpu(*sinks_in, cache, "sinks");
    sinks = sinks_in->to(at::kFloat).contiguous();
    a.sinks = static_cast<const float*>(sinks->data_ptr());
  }
  const at::Tensor q = usable(q_in);
  a.q = describe_row_tensor(q, "q", false);
  // (like q, it keeps q's dense stride order)
  const at::Tensor o = c.head_dim_v == c.head_dim ? fresh_like(q) : fresh({b, heads, t, c.head_dim_v}, q.scalar_type(), q.device());
  a.o = describe_row_tensor(o, "o", false);
  Maybe lse, max_logits;
  if (residuals) {
    lse = at::empty({b, heads, t}, q.options().dtype(at::kFloat));
    max_logits = at::empty({b, heads, t}, q.options().dtype(at::kFloat));
    a.logsumexp = static_cast<float*>(lse->data_ptr());
    a.max_logits = static_cast<float*>(max_logits->data_ptr());
  }
  if (o.numel() == 0) return {o, lse, max_logits};
  a.scale = (float)scale;
  a.soft_cap = (float)soft_cap.value_or(0.0);
  a.window = window.has_value() ? (int32_t)*window : -1;
  a.mask_value = (float)mask_value;
  a.workspace_bytes = (by_head ? page_lib.attend_workspace_bytes : cache_lib.attend_workspace_bytes)(&a);
  at::Tensor workspace;
  if (a.workspace_bytes != 0) {
    workspace = fresh({(int64_t)a.workspace_bytes}, at::kByte, q.device());
    a.workspace = workspace.data_ptr();
  }
  check_cache_call(on_stream_of(q, [&](void* stream) { return (by_head ? page_lib.attend : cache_lib.attend)(&a, stream); }),
                   by_head ? "splash_cache_attend_tables" : "splash_cache_attend");
  return {o, lse, max_logits};
}

// The bounds of the keys of a cache's pages, with the tensors that they lie in.
struct PageBounds {
  SplashPageBounds desc{};
  at::Tensor codes, scales;

  PageBounds(at::Tensor codes_in, at::Tensor scales_in) : codes(std::move(codes_in)), scales(std::move(scales_in)) {
    TORCH_CHECK_VALUE(codes.is_contiguous() && scales.is_contiguous() && codes.device() == scales.device(),
                      "the arrays of page bounds are contiguous, on one device");
    desc.codes = static_cast<int8_t*>(codes.data_ptr());
    desc.scales = static_cast<float*>(scales.data_ptr());
  }
};

void require_bounds_of(const PageBounds& bounds, const KvCache& cache) {
  const SplashKvCache& c = cache.desc;
  require_on_gpu(bounds.codes, cache, "the page bounds");
  TORCH_CHECK_VALUE(bounds.codes.sizes() == at::IntArrayRef({c.n_pages, c.kv_heads, 2, c.row_k}) &&
                        bounds.scales.sizes() == at::IntArrayRef({c.n_pages, c.kv_heads}),
                    "page bounds of ", bounds.codes.sizes(), " are not of a cache of ", c.n_pages, " pages, ", c.kv_heads, " heads and rows of ", c.row_k);
}

void cache_bound(const KvCache& cache, const PageBounds& bounds, const at::Tensor& table_in, const at::Tensor& lengths, int64_t newest) {
  require_not_traced();
  SplashCacheBoundArgs a{};
  require_pages_of_sequences(table_in, lengths);
  TORCH_CHECK_VALUE(newest >= 0, "newest is not negative, got ", newest);
  const at::Tensor table = set_pages(a, cache, table_in, lengths);
  require_bounds_of(bounds, cache);
  a.bounds = bounds.desc;
  a.batch = lengths.size(0);
  a.newest = newest;
  if (a.batch != 0) check_cache_call(on_stream_of(table, [&](void* stream) { return page_lib.bound(&a, stream); }), "splash_cache_bound");
}

at::Tensor cache_bound_values(const KvCache& cache, const PageBounds& bounds) {
  const SplashKvCache& c = cache.desc;
  require_not_traced();
  require_bounds_of(bounds, cache);
  const at::Tensor values = fresh({c.n_pages, c.kv_heads, 2, c.head_dim}, at::kFloat, bounds.codes.device());
  check_cache_call(on_stream_of(values, [&](void* stream) { return page_lib.bound_values(&c, &bounds.desc, static_cast<float*>(values.data_ptr()), stream); }),
                   "splash_cache_bound_values");
  return values;
}

std::tuple<at::Tensor, at::Tensor> cache_choose(const KvCache& cache, const PageBounds& bounds, const at::Tensor& q_in, const at::Tensor& table_in,
                                                const at::Tensor& lengths, int64_t count, int64_t first, int64_t last) {
  const SplashKvCache& c = cache.desc;
  require_not_traced();
  require_no_grad(q_in, "q");
  TORCH_CHECK_VALUE(q_in.dim() == 4 && q_in.size(3) == c.head_dim && q_in.size(1) % c.kv_heads == 0 && q_in.size(1) > 0, "q ", q_in.sizes(),
                    " does not match a cache of ", c.kv_heads, " heads of ", c.head_dim, " channels: expected [B, heads, T, D]");
  SplashCacheChooseArgs a{};
  require_pages_of_sequences(table_in, lengths);
  TORCH_CHECK_VALUE(q_in.size(0) == lengths.size(0), "q of ", q_in.size(0), " sequences, lengths of ", lengths.size(0));
  TORCH_CHECK_VALUE(first >= 0 && last >= 1 && first <= INT32_MAX && last <= INT32_MAX && count <= INT32_MAX && first + last <= count,
                    "expected first >= 0, last >= 1 and count >= first + last, got first ", first, ", last ", last, ", count ", count);
  const at::Tensor table = set_pages(a, cache, table_in, lengths);
  require_bounds_of(bounds, cache);
  require_on_gpu(q_in, cache, "q");
  const at::Tensor q = usable(q_in);
  a.bounds = bounds.desc;
  a.q = describe_row_tensor(q, "q", false);
  const at::Tensor tables = fresh({q.size(0), c.kv_heads, q.size(2), count}, at::kInt, q.device());
  const at::Tensor table_lengths = fresh({q.size(0), c.kv_heads, q.size(2)}, at::kInt, q.device());
  if (tables.numel() == 0) return {tables, table_lengths};
  a.tables = static_cast<int32_t*>(tables.data_ptr());
  a.table_lengths = static_cast<int32_t*>(table_lengths.data_ptr());
  a.count = (int32_t)count, a.first = (int32_t)first, a.last = (int32_t)last;
  a.workspace_bytes = page_lib.choose_workspace_bytes(&a);
  at::Tensor workspace;
  if (a.workspace_bytes != 0) {
    workspace = at::empty({(int64_t)a.workspace_bytes}, q.options().dtype(at::kByte));
    a.workspace = workspace.data_ptr();
  }
  check_cache_call(on_stream_of(q, [&](void* stream) { return page_lib.choose(&a, stream); }), "splash_cache_choose");
  return {tables, table_lengths};
}

// ------------------------------------------------------------------------------------------------------------------
// rotary positions (rotary.py)
// ------------------------------------------------------------------------------------------------------------------
int (*rotate_library)(const SplashRotateArgs*, void*) = nullptr;

void bind_rotary_library(uintptr_t rotate) { rotate_library = reinterpret_cast<decltype(rotate_library)>(rotate); }

// What the layers of a model share.
struct RotaryTable {
  at::Tensor turns;  // int64 [dim / 2], the bits of unsigned numbers
  int dim;
  bool interleaved;
  double factor;
};

// Positions [B, T] as the kernel reads them, which takes their extents from the rows: int32 or int64, tokens one behind the other.
at::Tensor usable_positions(const at::Tensor& given, const at::Tensor& x) {
  const auto type = given.scalar_type();
  TORCH_CHECK_VALUE(type == at::kInt || type == at::kLong, "positions are int32 or int64, got ", type);
  TORCH_CHECK_VALUE(x.dim() == 4 && (given.dim() == 1 || given.dim() == 2), "expected q and k of [B, heads, T, D] and positions of [B, T] or [T]");
  const at::Tensor positions = given.dim() == 1 ? given.unsqueeze(0) : given;
  TORCH_CHECK_VALUE((positions.size(0) == 1 || positions.size(0) == x.size(0)) && positions.size(1) == x.size(2), "positions ", given.sizes(),
                    " do not match q ", x.sizes());
  TORCH_CHECK_VALUE(positions.device() == x.device(), "positions are on ", positions.device(), ", q on ", x.device());
  return positions.size(1) > 1 && positions.stride(1) != 1 ? positions.contiguous() : positions;
}

// x and, where there is one, z, turned by their positions (or back).
std::tuple<at::Tensor, at::Tensor> rotated(const RotaryTable& table, const at::Tensor& positions, const at::Tensor& x, const Maybe& z, bool inverse) {
  at::Tensor out[2];
  SplashRotateArgs a{};
  at::Tensor in[2];
  bool any = false;
  for (int i = 0; i < 2; ++i) {
    if (i == 1 && !z.has_value()) continue;
    const at::Tensor& t = i == 0 ? x : *z;
    in[i] = usable(t);
    out[i] = fresh_like(in[i]);
    if (out[i].numel() == 0) continue;
    any = true;
    a.x[i] = describe_row_tensor(in[i], "rotate", true);
    a.y[i] = describe_row_tensor(out[i], "rotate", true);
  }
  if (any) {
    a.positions = positions.data_ptr();
    a.positions_are_64 = positions.scalar_type() == at::kLong;
    a.position_stride = positions.size(0) == 1 ? 0 : positions.stride(0);
    a.turns = static_cast<const uint64_t*>(table.turns.data_ptr());
    a.dim = table.dim;
    a.interleaved = table.interleaved;
    a.inverse = inverse;
    a.factor = (float)table.factor;
    const int status = on_stream_of(x, [&](void* stream) { return rotate_library(&a, stream); });
    if (status != 0) raise_status(status, "splash_rotate");
  }
  return {out[0], out[1]};
}

struct RotaryCall : torch::CustomClassHolder {
  std::shared_ptr<const RotaryTable> table;
  bool inverse;
};

// Its own gradient, the other way round: it can be differentiated any number of times.
struct Rotation : torch::autograd::Function<Rotation> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& positions, const at::Tensor& x, const Maybe& z,
                               const c10::intrusive_ptr<RotaryCall>& call) {
    auto [y, w] = rotated(*call->table, positions, x, z, call->inverse);
    ctx->save_for_backward({positions});
    ctx->saved_data["call"] = c10::IValue::make_capsule(call);
    ctx->set_materialize_grads(false);
    variable_list constant;  // (rows that no gradient is asked of stay so: a cache takes no others)
    if (!x.requires_grad()) constant.push_back(y);
    if (z.has_value() && !z->requires_grad()) constant.push_back(w);
    ctx->mark_non_differentiable(constant);
    return z.has_value() ? variable_list{y, w} : variable_list{y};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const at::Tensor saved = ctx->get_saved_variables()[0];
    const auto call = c10::static_intrusive_pointer_cast<RotaryCall>(ctx->saved_data["call"].toCapsule());
    auto back = c10::make_intrusive<RotaryCall>();
    back->table = call->table;
    back->inverse = !call->inverse;
    at::Tensor found[2];
    const at::Tensor dy = ctx->needs_input_grad(1) ? grads[0] : at::Tensor();
    const at::Tensor dw = grads.size() > 1 && ctx->needs_input_grad(2) ? grads[1] : at::Tensor();
    if (dy.defined() || dw.defined()) {
      // (hooks of saved tensors may give back anything)
      const at::Tensor positions = usable_positions(saved, dy.defined() ? dy : dw);
      const variable_list out = Rotation::apply(positions, dy.defined() ? dy : dw, dy.defined() && dw.defined() ? Maybe(dw) : Maybe(), back);
      if (dy.defined()) found[0] = out[0];
      if (dw.defined()) found[1] = out[dy.defined() ? 1 : 0];
    }
    return {at::Tensor(), found[0], found[1], at::Tensor()};
  }
};

std::tuple<at::Tensor, Maybe> rotate(const std::shared_ptr<RotaryTable>& table, const at::Tensor& positions_in, const at::Tensor& q, const Maybe& k) {
  require_not_recorded("rotate");
  const at::Tensor positions = usable_positions(positions_in, q);
  const at::Tensor* const both[2] = {&q, k.has_value() ? &*k : nullptr};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor* const t = both[i];
    if (t == nullptr) continue;
    const char* const name = i == 0 ? "q" : "k";
    TORCH_CHECK_VALUE(t->dim() == 4 && t->size(0) == q.size(0) && t->size(2) == q.size(2) && t->size(3) == q.size(3), "k ", t->sizes(),
                      " does not match q ", q.sizes());
    TORCH_CHECK_VALUE(t->scalar_type() == q.scalar_type(), "q and k have one type, got ", q.scalar_type(), " and ", t->scalar_type());
    TORCH_CHECK_NOT_IMPLEMENTED(!(t->_fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode()), name,
                                " has a tangent of forward mode: rotate has none");
    require_row_type(t->scalar_type(), name, true);
  }
  TORCH_CHECK_VALUE(q.size(3) % 8 == 0 && table->dim <= q.size(3), "rows of ", q.size(3), " channels: expected a multiple of 8, ", table->dim, " at least");
  TORCH_CHECK_NOT_IMPLEMENTED(q.size(3) <= 256, "rows of ", q.size(3), " channels are not built (256 at most)");
  for (int i = 0; i < 2; ++i) {
    if (both[i] == nullptr) continue;
    const at::Device device = both[i]->device();
    TORCH_CHECK(device.is_cuda(), i == 0 ? "q" : "k", " is on ", device, ": the kernels need a CUDA device");
    TORCH_CHECK_VALUE(device == table->turns.device(), i == 0 ? "q" : "k", " is on ", device, ", the rotary table on ", table->turns.device());
  }
  if (!(at::GradMode::is_enabled() && (q.requires_grad() || (k.has_value() && k->requires_grad())))) {
    const auto [y, w] = rotated(*table, positions, q, k, false);
    return {y, k.has_value() ? Maybe(w) : Maybe()};
  }
  auto call = c10::make_intrusive<RotaryCall>();
  call->table = table;
  call->inverse = false;
  variable_list out;
  {
    const WithoutGil release;
    out = Rotation::apply(positions, q, k, call);
  }
  return {out[0], k.has_value() ? Maybe(out[1]) : Maybe()};
}

}  // namespace

PYBIND11_MODULE(_splash_torch, m) {
  m.def("bind_library", &bind_library);
  m.def("bind_cache_library", &bind_cache_library);
  pybind11::class_<KvCache>(m, "KvCache")
      .def(pybind11::init<at::Tensor, at::Tensor, at::Tensor, at::Tensor, int, int, int, int, int, int>());
  m.def("bind_page_library", &bind_page_library);
  m.def("bind_rotary_library", &bind_rotary_library);
  pybind11::class_<PageBounds>(m, "PageBounds").def(pybind11::init<at::Tensor, at::Tensor>());
  m.def("cache_bound", torch::wrap_pybind_function(cache_bound));
  m.def("cache_bound_values", torch::wrap_pybind_function(cache_bound_values));
  m.def("cache_choose", torch::wrap_pybind_function(cache_choose));
  pybind11::class_<RotaryTable, std::shared_ptr<RotaryTable>>(m, "RotaryTable").def(pybind11::init<at::Tensor, int, bool, double>());
  m.def("rotate", torch::wrap_pybind_function(rotate));
  m.def("cache_append", torch::wrap_pybind_function(cache_append));
  m.def("cache_read", torch::wrap_pybind_function(cache_read));
  m.def("cache_attend", torch::wrap_pybind_function(cache_attend));
  m.def("forward", torch::wrap_pybind_function(forward));
  m.def("backward", torch::wrap_pybind_function(backward));
  m.def("bind_check", [](pybind11::object check) { check_status = check.release().ptr(); });
  pybind11::class_<Tables, std::shared_ptr<Tables>>(m, "Tables")
      .def(pybind11::init<uintptr_t, uintptr_t, uintptr_t, std::vector<at::Tensor>, at::Tensor, Maybe, int>());
  m.def("attention", torch::wrap_pybind_function(attention));
}
