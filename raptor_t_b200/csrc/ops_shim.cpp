// pybind11 module `raptor_ops`: the calls of ops.py whose kernels take a few microseconds, from tensors to the C ABI without a
// Python statement for each argument.  A call through ctypes costs the host 9 to 17 us (checks, addresses, output tensors), through this
// module 5 to 8; the kernels of a single token's step take 3 to 7.
//
// Every function checks its tensors, makes its outputs and calls one entry point of include/raptor_b200.h, at the address that
// ops.py passes in: the library that the rest of the process uses, whichever file that came from.
#include <torch/extension.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <array>
#include <cstdint>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/raptor_b200.h"

namespace {

namespace py = pybind11;
using torch::Tensor;
using OptTensor = std::optional<Tensor>;

struct Entries {
  decltype(&rt_last_error) last_error = nullptr;
  decltype(&rt_kv_cache_write) kv_cache_write = nullptr;
  decltype(&rt_kv_cache_read) kv_cache_read = nullptr;
  decltype(&rt_cached_attention) cached_attention = nullptr;
  decltype(&rt_token_logprobs) token_logprobs = nullptr;
  decltype(&rt_token_logprobs_backward) token_logprobs_backward = nullptr;
} entry;

void bind(uintptr_t last_error, uintptr_t write, uintptr_t read, uintptr_t attention, uintptr_t scores, uintptr_t scores_grad) {
  entry.last_error = reinterpret_cast<decltype(entry.last_error)>(last_error);
  entry.kv_cache_write = reinterpret_cast<decltype(entry.kv_cache_write)>(write);
  entry.kv_cache_read = reinterpret_cast<decltype(entry.kv_cache_read)>(read);
  entry.cached_attention = reinterpret_cast<decltype(entry.cached_attention)>(attention);
  entry.token_logprobs = reinterpret_cast<decltype(entry.token_logprobs)>(scores);
  entry.token_logprobs_backward = reinterpret_cast<decltype(entry.token_logprobs_backward)>(scores_grad);
}

// capi.RtError, as the ctypes calls raise it
void check(rt_status s) {
  if (s == RT_OK) return;
  py::object type = py::module_::import("raptor_t_b200.capi").attr("RtError");
  py::object e = type(static_cast<int>(s), std::string(entry.last_error()));
  PyErr_SetObject(type.ptr(), e.ptr());
  throw py::error_already_set();
}

std::string shape_of(c10::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

int dtype16(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return RT_BF16;
  if (t.scalar_type() == at::kHalf) return RT_F16;
  throw py::type_error(std::string("expected float16 or bfloat16, got ") + c10::toString(t.scalar_type()));
}

// Kernels run on the current device's current stream: the tensors have to be there, too.
void* stream_for(int device) {
  if (device < 0) throw std::runtime_error("raptor_t_b200 ops need CUDA tensors (there is no CPU path)");
  if (device != c10::cuda::current_device())
    throw std::runtime_error("tensors on cuda:" + std::to_string(device) + ", but the current device is cuda:" +
                             std::to_string(c10::cuda::current_device()));
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}

int fits(int64_t v, const char* name) {
  if (v < 0 || v > INT32_MAX) throw py::value_error(std::string(name) + ": " + std::to_string(v) + " is out of range");
  return static_cast<int>(v);
}

// The most rows of one sequence: all rows where the caller does not say, and 0 counts as 1.
int most_of(int64_t most, int rows, const char* name) { return most < 0 ? rows : std::max(1, fits(most, name)); }

int index_of(const Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }

// Address of a contiguous tensor of that type and shape on that device.
void* flat(const Tensor& t, const char* name, at::ScalarType type, c10::IntArrayRef shape, int device) {
  if (t.scalar_type() != type)
    throw py::type_error(std::string(name) + ": expected " + c10::toString(type) + ", got " + c10::toString(t.scalar_type()));
  if (t.sizes() != shape || !t.is_contiguous() || index_of(t) != device)
    throw py::value_error(std::string(name) + ": expected a contiguous tensor of shape " + shape_of(shape) + " on cuda:" +
                          std::to_string(device) + ", got " + shape_of(t.sizes()) + " with strides " + shape_of(t.strides()) + " on " +
                          t.device().str());
  return t.data_ptr();
}

Tensor empty(c10::IntArrayRef shape, at::ScalarType type, int device) {
  return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device)), std::nullopt);
}

// A contiguous tensor in `base`'s memory.  Outputs of a call that are used together share one allocation, one for each type (torch.save wants
// that): each of their own costs the host 0.6 us.
Tensor part(const Tensor& base, int64_t byte, c10::IntArrayRef shape, at::ScalarType type) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                      c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(byte / static_cast<int64_t>(c10::elementSize(type)));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
  return t;
}

// The tensors of a KvCache with the C ABI's view of them.
struct Cache {
  Tensor k, v, k_scale, v_scale;
  rt_kv_cache c{};
  int device = -1;
  Cache(Tensor k_, Tensor v_, Tensor ks, Tensor vs) : k(k_), v(v_), k_scale(ks), v_scale(vs) {
    const auto type = k.scalar_type();
    if (type != at::kFloat8_e4m3fn && type != at::kChar)
      throw py::type_error(std::string("expected float8_e4m3fn or int8, got ") + c10::toString(type));
    if (k.dim() != 4 || k.size(2) != 64 || k.size(3) != 64) throw py::value_error("a cache is [blocks, kv_heads, 64, 64]");
    device = index_of(k);
    if (device < 0) throw std::runtime_error("raptor_t_b200 ops need CUDA tensors (there is no CPU path)");
    const auto shape = k.sizes();
    c.k_dev = flat(k, "k", type, shape, device);
    c.v_dev = flat(v, "v", type, shape, device);
    c.k_scale_dev = static_cast<float*>(flat(k_scale, "k_scale", at::kFloat, shape.slice(0, 2), device));
    c.v_scale_dev = static_cast<float*>(flat(v_scale, "v_scale", at::kFloat, shape.slice(0, 2), device));
    c.blocks = fits(k.size(0), "blocks");
    c.kv_heads = fits(k.size(1), "kv_heads");
    c.format = type == at::kChar ? RT_KV_INT8 : RT_KV_E4M3;
  }
};

// The arguments that say which tokens a call is about.
struct Ragged {
  const int32_t *table, *lengths, *first;
  int width, n;
  Ragged(const Tensor& t, const Tensor& l, const Tensor& f, int device) {
    const int64_t count = l.dim() == 1 ? l.size(0) : -1, wide = t.dim() == 2 ? t.size(1) : 0;
    if (count < 0 || wide <= 0) throw py::value_error("a block table is [sequences, width], lengths are [sequences]");
    n = fits(count, "sequences");
    width = fits(wide, "block table");
    table = static_cast<const int32_t*>(flat(t, "block table", at::kInt, {count, wide}, device));
    lengths = static_cast<const int32_t*>(flat(l, "lengths", at::kInt, {count}, device));
    first = static_cast<const int32_t*>(flat(f, "first rows", at::kInt, {count + 1}, device));
  }
};

void kv_cache_write(const Cache& c, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& start, const Tensor& first,
                    int64_t max_tokens, bool head_major) {
  void* st = stream_for(c.device);
  const int dt = dtype16(k);
  const int64_t heads = c.c.kv_heads, tokens = k.dim() > 0 ? k.size(0) : 0;
  int64_t ts = 0, hs = 0;
  if (head_major) {
    flat(k, "k", k.scalar_type(), {tokens, heads * 64}, c.device);
    flat(v, "v", k.scalar_type(), {tokens, heads * 64}, c.device);
  } else {
    // the stride over one token or one head says nothing
    auto strides = [&](const Tensor& t) {
      return std::array<int64_t, 2>{tokens > 1 ? t.stride(0) : 64 * heads, heads > 1 ? t.stride(1) : 64};
    };
    if (k.dim() != 3 || k.size(1) != heads || k.size(2) != 64 || k.sizes() != v.sizes() || strides(k) != strides(v) ||
        k.stride(2) != 1 || v.stride(2) != 1 || v.scalar_type() != k.scalar_type() || index_of(k) != c.device || index_of(v) != c.device)
      throw py::value_error("k and v: expected [tokens, kv_heads, 64] of the same type and strides, on the cache's device");
    ts = strides(k)[0];
    hs = strides(k)[1];
    if (ts == 0) throw py::value_error("k and v: rows without a stride");
  }
  const Ragged r(table, start, first, c.device);
  const int n = fits(tokens, "tokens");
  check(entry.kv_cache_write(&c.c, k.data_ptr(), v.data_ptr(), ts, hs, r.table, r.width, r.lengths, r.first, r.n, n,
                             most_of(max_tokens, n, "max_tokens"), dt, st));
}

std::tuple<Tensor, Tensor> kv_cache_read(const Cache& c, const Tensor& table, const Tensor& start, const Tensor& first, int64_t tokens,
                                         at::ScalarType type, int64_t max_tokens, OptTensor out_k, OptTensor out_v) {
  void* st = stream_for(c.device);
  const int n = fits(tokens, "tokens");
  const int64_t shape[3] = {tokens, c.c.kv_heads, 64};
  Tensor k, v;
  if (out_k && out_v) {
    k = *out_k;
    v = *out_v;
  } else {
    const int64_t both[4] = {2, tokens, c.c.kv_heads, 64}, bytes = tokens * c.c.kv_heads * 64 * static_cast<int64_t>(c10::elementSize(type));
    const Tensor base = empty(both, type, c.device);
    k = out_k ? *out_k : part(base, 0, shape, type);
    v = out_v ? *out_v : part(base, bytes, shape, type);
  }
  const int dt = dtype16(k);
  const Ragged r(table, start, first, c.device);
  check(entry.kv_cache_read(&c.c, flat(k, "k", type, shape, c.device), flat(v, "v", type, shape, c.device), r.table, r.width, r.lengths,
                            r.first, r.n, n, most_of(max_tokens, n, "max_tokens"), dt, st));
  return {k, v};
}

Tensor cached_attention(const Tensor& q, const Cache& c, const Tensor& table, const Tensor& context, const Tensor& first, int64_t max_q,
                        int64_t max_context, double scale, bool causal, OptTensor out) {
  void* st = stream_for(c.device);
  const int dt = dtype16(q);
  if (q.dim() != 3 || q.size(2) != 64 || q.stride(2) != 1 || (q.stride(1) != 64 && q.size(1) != 1) || index_of(q) != c.device)
    throw py::value_error("q: expected [tokens, heads, 64] with adjacent heads, on the cache's device");
  Tensor o = out ? *out : empty(q.sizes(), q.scalar_type(), c.device);
  const Ragged r(table, context, first, c.device);
  const int n = fits(q.size(0), "tokens");
  check(entry.cached_attention(flat(o, "out", q.scalar_type(), q.sizes(), c.device), q.data_ptr(), n > 1 ? q.stride(0) : 64 * q.size(1), &c.c, r.table, r.width,
                               r.lengths, r.first, r.n, n, most_of(max_q, n, "max_q"), fits(max_context, "max_context"),
                               fits(q.size(1), "heads"), static_cast<float>(scale), causal, dt, st));
  return o;
}

struct Logits {
  int rows, vocab, type;
  int64_t pitch;
  Logits(const Tensor& z, const char* name) {
    switch (z.scalar_type()) {
      case at::kHalf: type = RT_F16; break;
      case at::kBFloat16: type = RT_BF16; break;
      case at::kFloat: type = RT_F32; break;
      default:
        throw py::type_error(std::string(name) + ": expected float16, bfloat16 or float32, got " + c10::toString(z.scalar_type()));
    }
    if (z.dim() != 2 || (z.stride(1) != 1 && z.size(1) != 1))
      throw py::value_error(std::string(name) + ": expected [rows, vocab] with rows of adjacent values");
    rows = fits(z.size(0), "rows");
    vocab = fits(z.size(1), "vocab");
    pitch = rows > 1 ? z.stride(0) : std::max<int64_t>(z.stride(0), vocab);
  }
};

std::tuple<OptTensor, Tensor, Tensor, OptTensor, OptTensor> token_logprobs(const Tensor& logits, OptTensor targets, int64_t top_k) {
  const Logits z(logits, "logits");
  const int device = index_of(logits);
  void* st = stream_for(device);
  const int top = fits(top_k, "top_k");
  // stats, entropy, logp if there are targets, best; ids
  const int64_t rows = z.rows, scores = targets ? 4 : 3;
  const Tensor base = empty({scores + top_k, rows}, at::kFloat, device);
  Tensor stats = part(base, 0, {rows, 2}, at::kFloat), entropy = part(base, rows * 8, {rows}, at::kFloat);
  OptTensor logp, ids, best;
  const int32_t* t = nullptr;
  if (targets) {
    t = static_cast<const int32_t*>(flat(*targets, "targets", at::kInt, {z.rows}, device));
    logp = part(base, rows * 12, {rows}, at::kFloat);
  }
  if (top > 0) {
    ids = empty({rows, top_k}, at::kInt, device);
    best = part(base, rows * scores * 4, {rows, top_k}, at::kFloat);
  }
  check(entry.token_logprobs(logits.data_ptr(), z.pitch, t, z.rows, z.vocab, top, logp ? logp->data_ptr<float>() : nullptr,
                             entropy.data_ptr<float>(), stats.data_ptr<float>(), ids ? ids->data_ptr<int32_t>() : nullptr,
                             best ? best->data_ptr<float>() : nullptr, z.type, st));
  return {logp, entropy, stats, ids, best};
}

Tensor token_logprobs_backward(const Tensor& logits, OptTensor targets, const Tensor& stats, OptTensor entropy, OptTensor grad_logp,
                               OptTensor grad_entropy, OptTensor top_ids, OptTensor grad_top, OptTensor out) {
  const Logits z(logits, "logits");
  const int device = index_of(logits);
  void* st = stream_for(device);
  Tensor d;
  if (out) {
    d = *out;
  } else {  // as few spare columns as give the rows the alignment of the logits' own
    const int64_t pitch = z.vocab + (z.pitch - z.vocab) % (16 / logits.element_size());
    d = empty({z.rows, pitch}, logits.scalar_type(), device);
    if (pitch != z.vocab) d = d.narrow(1, 0, z.vocab);
  }
  if (d.sizes() != logits.sizes() || index_of(d) != device) throw py::value_error("out: expected the logits' shape and device");
  if (d.scalar_type() != logits.scalar_type())
    throw py::type_error(std::string("out: expected ") + c10::toString(logits.scalar_type()) + ", got " + c10::toString(d.scalar_type()));
  const Logits o(d, "out");
  auto f = [&](const OptTensor& t, const char* name) {
    return t ? static_cast<const float*>(flat(*t, name, at::kFloat, {z.rows}, device)) : nullptr;
  };
  int top = 0;
  const int32_t* ids = nullptr;
  const float* g_top = nullptr;
  if (grad_top) {
    if (grad_top->dim() != 2) throw py::value_error("grad_top: expected [rows, k]");
    const int64_t k = grad_top->size(1);
    g_top = static_cast<const float*>(flat(*grad_top, "grad_top", at::kFloat, {z.rows, k}, device));
    if (k > 0 && !top_ids) throw py::value_error("grad_top needs top_ids");
    if (k > 0) ids = static_cast<const int32_t*>(flat(*top_ids, "top_ids", at::kInt, {z.rows, k}, device));
    top = fits(k, "alternatives");
  }
  if (grad_logp && !targets) throw py::value_error("grad_logp needs the targets");
  if (grad_entropy && !entropy) throw py::value_error("grad_entropy needs the entropy");
  const int32_t* t = targets ? static_cast<const int32_t*>(flat(*targets, "targets", at::kInt, {z.rows}, device)) : nullptr;
  check(entry.token_logprobs_backward(d.data_ptr(), o.pitch, logits.data_ptr(), z.pitch, t,
                                      static_cast<const float*>(flat(stats, "stats", at::kFloat, {z.rows, 2}, device)), f(entropy, "entropy"),
                                      z.rows, z.vocab, f(grad_logp, "grad_logp"), f(grad_entropy, "grad_entropy"), top, ids, g_top, z.type,
                                      st));
  return d;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "Short calls of raptor_t_b200.ops on the raptor_b200 C ABI (B200, sm_100a)";
  m.def("bind", &bind);
  py::class_<Cache>(m, "Cache").def(py::init<Tensor, Tensor, Tensor, Tensor>());
  m.def("kv_cache_write", &kv_cache_write);
  m.def("kv_cache_read", &kv_cache_read);
  m.def("cached_attention", &cached_attention);
  m.def("token_logprobs", &token_logprobs);
  m.def("token_logprobs_backward", &token_logprobs_backward);
}
