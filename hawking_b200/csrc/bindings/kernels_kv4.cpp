// torch bindings of the 4-bit paged KV cache kernels (kv4_cache.cu, kv4_decode.cu,
// kv4_prefill.cu).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>

#include "../kernels/kernels_api.h"
#include "../kernels/kv4.h"

namespace py = pybind11;
using at::Tensor;
using c10::optional;

namespace {

template <typename T> T* ptr(const Tensor& t) { return reinterpret_cast<T*>(t.data_ptr()); }
template <typename T> T* optr(const optional<Tensor>& t) { return t.has_value() ? ptr<T>(*t) : nullptr; }

// Numbers enter the messages as strings: the check macros format everything else through streams.
std::string num(int64_t v) { return std::to_string(v); }

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// A vector of int32 on the cache's (or the step's) device.
const int* ints(const Tensor& t, int64_t n, const at::Device& dev, const char* name) {
  TORCH_CHECK(t.device() == dev && t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() >= n, "kv4: ", name,
              " must be contiguous int32 of at least ", num(n), " elements on ", dev.str());
  return t.data_ptr<int>();
}
int* ints_out(const Tensor& t, int64_t n, const at::Device& dev, const char* name) {
  return const_cast<int*>(ints(t, n, dev, name));
}

struct Shape {
  int64_t blocks;
  int nkv, hd, block_size;
};

Shape cache_shape(const Tensor& c) {
  TORCH_CHECK(c.is_cuda() && c.dim() == 4 && c.scalar_type() == at::kByte && c.is_contiguous(),
              "kv4: the cache must be contiguous uint8 [blocks, kv_heads, block_size / 16, 18 * head_dim] on the GPU");
  const int64_t hd = c.size(3) / 18;
  TORCH_CHECK(c.size(3) % 18 == 0 && (hd == 64 || hd == 128 || hd == 256),
              "kv4: head_dim must be 64, 128 or 256 (units of 18 * head_dim bytes), not units of ", num(c.size(3)), " bytes");
  TORCH_CHECK(c.size(1) > 0 && c.size(2) > 0, "kv4: the cache must have kv heads and a block size of at least 16");
  TORCH_CHECK(aligned16(c.data_ptr()), "kv4: the cache must start on a 16-byte boundary");
  TORCH_CHECK(c.size(0) * c.size(2) * 16 < (int64_t(1) << 31), "kv4: KV pool too large for int32 slot ids");
  return {c.size(0), (int)c.size(1), (int)hd, (int)c.size(2) * 16};
}

// [table_rows, max_blocks] int32
const int* tables_of(const Tensor& t, const at::Device& dev, int& rows, int& cols) {
  TORCH_CHECK(t.device() == dev && t.dim() == 2 && t.scalar_type() == at::kInt && t.is_contiguous(),
              "kv4: block_tables must be contiguous int32 [rows, max_blocks] on ", dev.str());
  rows = (int)t.size(0);
  cols = (int)t.size(1);
  return t.data_ptr<int>();
}

void kv4_plan(const Tensor& seq_rows, const Tensor& cached, const Tensor& fresh, const Tensor& tables,
              int64_t block_size, const Tensor& positions, const Tensor& row_seq, const Tensor& row_ctx,
              const Tensor& slots, const optional<Tensor>& free_blocks, const optional<Tensor>& taken,
              const optional<Tensor>& status, bool pdl) {
  TORCH_CHECK(tables.is_cuda(), "kv4: block_tables must be on the GPU");
  const at::Device dev = tables.device();
  hk::Kv4PlanArgs a{};
  a.S = (int)seq_rows.numel();
  TORCH_CHECK(a.S <= 8192, "kv4 plan: at most 8192 requests, got ", num(a.S));
  a.seq_rows = ints(seq_rows, a.S, dev, "seq_rows");
  a.cached = ints(cached, a.S, dev, "cached");
  a.fresh = ints(fresh, a.S, dev, "new");
  TORCH_CHECK(cached.numel() == a.S && fresh.numel() == a.S, "kv4 plan: seq_rows, cached and new must have one length");
  a.tables = const_cast<int*>(tables_of(tables, dev, a.table_rows, a.max_blocks));
  TORCH_CHECK(block_size > 0 && block_size <= 65536, "kv4 plan: block_size must be positive");
  TORCH_CHECK((int64_t)a.max_blocks * block_size < (int64_t(1) << 31), "kv4 plan: positions must fit int32");
  a.block_size = (int)block_size;
  a.cap = (int)positions.numel();
  a.positions = ints_out(positions, a.cap, dev, "positions");
  a.row_seq = ints_out(row_seq, a.cap, dev, "row_seq");
  a.row_ctx = ints_out(row_ctx, a.cap, dev, "row_ctx");
  a.slots = ints_out(slots, a.cap, dev, "slots");
  TORCH_CHECK(row_seq.numel() == a.cap && row_ctx.numel() == a.cap && slots.numel() == a.cap,
              "kv4 plan: positions, row_seq, row_ctx and slots must have one length");
  if (free_blocks.has_value()) {
    a.n_free = (int)free_blocks->numel();
    a.free_blocks = ints(*free_blocks, a.n_free, dev, "free_blocks");
    static const int none = 0;
    if (a.n_free == 0) a.free_blocks = &none;  // an empty list is a list: nothing is read from it
  }
  if (taken.has_value()) a.taken = ints_out(*taken, 1, dev, "taken");
  if (status.has_value()) a.status = ints_out(*status, 1, dev, "status");
  const c10::cuda::CUDAGuard g(dev);
  hk::kv4_plan_launch(a, at::cuda::getCurrentCUDAStream().stream(), pdl);
}

void kv4_append(const Tensor& qkv, const Tensor& positions, const optional<Tensor>& slots, const Tensor& rope,
                int64_t rot_dim, int64_t style, const Tensor& q_out, const Tensor& cache, int64_t nh, int64_t nkv,
                int64_t hd, const optional<Tensor>& bias, const optional<Tensor>& q_norm,
                const optional<Tensor>& k_norm, double eps, const optional<Tensor>& block_tables,
                const optional<Tensor>& row_seq, bool pdl) {
  const Shape sh = cache_shape(cache);
  const at::Device dev = cache.device();
  TORCH_CHECK(nkv == sh.nkv && hd == sh.hd && nh > 0, "kv4 append: the cache holds ", num(sh.nkv), " kv heads of ",
              num(sh.hd), ", the rows ", num(nkv), " of ", num(hd));
  const int64_t width = (nh + 2 * nkv) * hd;
  TORCH_CHECK(qkv.device() == dev && qkv.dim() == 2 && qkv.scalar_type() == at::kFloat && qkv.size(1) == width &&
                  qkv.stride(1) == 1 && (qkv.size(0) < 2 || (qkv.stride(0) >= width && qkv.stride(0) % 4 == 0)) &&
                  aligned16(qkv.data_ptr()),
              "kv4 append: qkv must be 16-byte aligned fp32 rows of ", num(width), " elements");
  hk::Kv4AppendArgs a{};
  a.R = (int)qkv.size(0);
  a.nh = (int)nh;
  a.nkv = (int)nkv;
  a.hd = (int)hd;
  a.qkv = ptr<float>(qkv);
  a.qkv_stride = qkv.stride(0);
  const auto vec = [&](const optional<Tensor>& t, int64_t n, const char* name) -> const float* {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == dev && t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == n,
                "kv4 append: ", name, " must be contiguous fp32 of ", num(n), " elements");
    return t->data_ptr<float>();
  };
  a.bias = vec(bias, width, "bias");
  a.q_norm = vec(q_norm, hd, "q_norm");
  a.k_norm = vec(k_norm, hd, "k_norm");
  a.eps = (float)eps;
  a.positions = ints(positions, a.R, dev, "positions");
  if (slots.has_value()) {
    a.slots = ints(*slots, a.R, dev, "slots");
  } else {
    TORCH_CHECK(block_tables.has_value() && row_seq.has_value(), "kv4 append: slots or block tables required");
    a.block_tables = tables_of(*block_tables, dev, a.table_rows, a.max_blocks);
    a.row_seq = ints(*row_seq, a.R, dev, "row_seq");
  }
  TORCH_CHECK(rot_dim >= 0 && rot_dim % 2 == 0 && rot_dim <= hd, "kv4 append: rot_dim must be even and at most head_dim");
  TORCH_CHECK(style == 0 || style == 1, "kv4 append: style 0 (adjacent pairs) or 1 (halves)");
  TORCH_CHECK(rope.device() == dev && rope.scalar_type() == at::kFloat && rope.is_contiguous() && rope.dim() == 3 &&
                  rope.size(1) * 2 == rot_dim && rope.size(2) == 2 && reinterpret_cast<uintptr_t>(rope.data_ptr()) % 8 == 0,
              "kv4 append: rope must be 8-byte aligned contiguous fp32 [positions, rot_dim / 2, 2]");
  a.rope = rope.data_ptr<float>();
  a.rope_rows = (int)rope.size(0);
  a.rot_dim = (int)rot_dim;
  a.rope_style = (int)style;
  TORCH_CHECK(q_out.device() == dev && q_out.scalar_type() == at::kBFloat16 && q_out.dim() == 3 && q_out.size(0) == a.R &&
                  q_out.size(1) == nh && q_out.size(2) == hd && q_out.stride(2) == 1 && q_out.stride(1) == hd &&
                  (a.R < 2 || (q_out.stride(0) % 8 == 0 && q_out.stride(0) >= nh * hd)) && aligned16(q_out.data_ptr()),
              "kv4 append: q_out must be 16-byte aligned bf16 [rows, heads, head_dim], no rows over one another");
  a.q_out = ptr<uint16_t>(q_out);
  a.q_stride = q_out.stride(0);
  a.cache = ptr<uint8_t>(cache);
  a.cache_blocks = sh.blocks;
  a.block_size = sh.block_size;
  const c10::cuda::CUDAGuard g(dev);
  hk::kv4_append_launch(a, at::cuda::getCurrentCUDAStream().stream(), pdl);
}

void kv4_gather(const Tensor& cache, const Tensor& slots, const optional<Tensor>& k, const optional<Tensor>& v,
                bool pdl) {
  const Shape sh = cache_shape(cache);
  const at::Device dev = cache.device();
  hk::Kv4GatherArgs a{};
  a.cache = ptr<uint8_t>(cache);
  a.cache_blocks = sh.blocks;
  a.N = (int)slots.numel();
  a.slots = ints(slots, a.N, dev, "slots");
  a.nkv = sh.nkv;
  a.hd = sh.hd;
  a.block_size = sh.block_size;
  const auto rows = [&](const optional<Tensor>& t, const char* name) -> uint16_t* {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == dev && t->scalar_type() == at::kBFloat16 && t->is_contiguous() &&
                    t->numel() == (int64_t)a.N * sh.nkv * sh.hd && aligned16(t->data_ptr()),
                "kv4 gather: ", name, " must be 16-byte aligned contiguous bf16 [slots, kv_heads, head_dim]");
    return ptr<uint16_t>(*t);
  };
  a.k = rows(k, "k");
  a.v = rows(v, "v");
  const c10::cuda::CUDAGuard g(dev);
  hk::kv4_gather_launch(a, at::cuda::getCurrentCUDAStream().stream(), pdl);
}

void kv4_attention(bool prefill, const Tensor& q, const Tensor& cache, const Tensor& block_tables,
                   const Tensor& row_seq, const Tensor& row_ctx, double scale, const optional<Tensor>& out,
                   const optional<Tensor>& out_bf16, const optional<Tensor>& sinks, const Tensor& status, const Tensor& part, const Tensor& counters,
                   int64_t sms, bool pdl, int64_t wait_polls) {
  const Shape sh = cache_shape(cache);
  const at::Device dev = cache.device();
  TORCH_CHECK(q.device() == dev && q.dim() == 3 && q.scalar_type() == at::kBFloat16 && q.size(2) == sh.hd &&
                  q.stride(2) == 1 && q.stride(1) == sh.hd && (q.size(0) < 2 || q.stride(0) % 8 == 0) &&
                  aligned16(q.data_ptr()),
              "kv4 attention: q must be 16-byte aligned bf16 [rows, heads, ", num(sh.hd), "]");
  hk::Kv4AttnArgs a{};
  a.R = (int)q.size(0);
  a.nh = (int)q.size(1);
  a.nkv = sh.nkv;
  a.hd = sh.hd;
  a.block_size = sh.block_size;
  TORCH_CHECK(a.nh > 0 && a.nh % a.nkv == 0 && a.nh / a.nkv <= 16,
              "kv4 attention: query heads must be a multiple of the kv heads, at most 16 each (", num(a.nh),
              " and ", num(a.nkv), ")");
  TORCH_CHECK(!prefill || sh.hd <= 128, "kv4 attention prefill: head_dim 64 or 128");
  a.q = ptr<uint16_t>(q);
  a.q_stride = q.stride(0);
  a.cache = ptr<uint8_t>(cache);
  a.cache_blocks = sh.blocks;
  a.block_tables = tables_of(block_tables, dev, a.table_rows, a.max_blocks);
  TORCH_CHECK((int64_t)a.max_blocks * sh.block_size < (int64_t(1) << 31) - 65536, "kv4 attention: contexts must fit int32");
  a.row_seq = ints(row_seq, a.R, dev, "row_seq");
  a.row_ctx = ints(row_ctx, a.R, dev, "row_ctx");
  TORCH_CHECK(scale > 0 && std::isfinite(scale), "kv4 attention: scale must be positive");
  a.scale = (float)scale;
  const auto rows = [&](const optional<Tensor>& t, at::ScalarType ty, int64_t& stride, const char* name) -> void* {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == dev && t->scalar_type() == ty && t->dim() == 2 && t->size(0) == a.R &&
                    t->size(1) == (int64_t)a.nh * a.hd && t->stride(1) == 1 &&
                    (a.R < 2 || (t->stride(0) % 8 == 0 && t->stride(0) >= t->size(1))) && aligned16(t->data_ptr()),
                "kv4 attention: ", name, " must be 16-byte aligned [rows, heads * head_dim], no rows over one another");
    stride = t->stride(0);
    return t->data_ptr();
  };
  a.out_bf16 = static_cast<uint16_t*>(rows(out_bf16, at::kBFloat16, a.out_stride, "out_bf16 (bf16)"));
  a.out = static_cast<float*>(rows(out, at::kFloat, a.outf_stride, "out (fp32)"));
  TORCH_CHECK(a.out || a.out_bf16, "kv4 attention: out or out_bf16 required");
  if (sinks.has_value()) {
    TORCH_CHECK(sinks->device() == dev && sinks->scalar_type() == at::kFloat && sinks->is_contiguous() &&
                    sinks->numel() == a.nh, "kv4 attention: sinks must be fp32 [heads]");
    a.sinks = sinks->data_ptr<float>();
  }
  a.status = ints_out(status, 1, dev, "status");
  TORCH_CHECK(wait_polls >= 0 && wait_polls <= hk::kKv4WaitPolls, "kv4 attention: wait_polls must be 0 to ",
              num(hk::kKv4WaitPolls));
  a.wait_polls = (uint32_t)wait_polls;
  TORCH_CHECK(part.device() == dev && part.scalar_type() == at::kFloat && part.is_contiguous() &&
                  part.numel() >= hk::kKv4PartFloats((int)sms) && sms > 0 && 3 * sms <= hk::kKv4Counters,
              "kv4 attention: the workspace's partials are too small");
  const hk::Kv4Workspace ws{part.data_ptr<float>(), ints_out(counters, hk::kKv4Counters, dev, "counters"), (int)sms};
  const c10::cuda::CUDAGuard g(dev);
  const cudaStream_t s = at::cuda::getCurrentCUDAStream().stream();
  if (prefill) hk::kv4_attention_prefill_launch(a, ws, s, pdl);
  else hk::kv4_attention_decode_launch(a, ws, s, pdl);
}

}  // namespace

namespace hk {
void register_kv4_kernels(py::module_& m) {
  m.def("kv4_plan", &kv4_plan, py::arg("seq_rows"), py::arg("cached"), py::arg("new"), py::arg("block_tables"),
        py::arg("block_size"), py::arg("positions"), py::arg("row_seq"), py::arg("row_ctx"), py::arg("slots"),
        py::arg("free_blocks") = py::none(), py::arg("taken") = py::none(), py::arg("status") = py::none(),
        py::arg("pdl") = false);
  m.def("kv4_append", &kv4_append, py::arg("qkv"), py::arg("positions"), py::arg("slots"), py::arg("rope"),
        py::arg("rot_dim"), py::arg("style"), py::arg("q_out"), py::arg("cache"), py::arg("nh"), py::arg("nkv"),
        py::arg("hd"), py::arg("bias") = py::none(), py::arg("q_norm") = py::none(), py::arg("k_norm") = py::none(),
        py::arg("eps") = 1e-6, py::arg("block_tables") = py::none(), py::arg("row_seq") = py::none(),
        py::arg("pdl") = false);
  m.def("kv4_gather", &kv4_gather, py::arg("cache"), py::arg("slots"), py::arg("k"), py::arg("v"),
        py::arg("pdl") = false);
  m.def("kv4_attention", &kv4_attention, py::arg("prefill"), py::arg("q"), py::arg("cache"), py::arg("block_tables"),
        py::arg("row_seq"), py::arg("row_ctx"), py::arg("scale"), py::arg("out"), py::arg("out_bf16"),
        py::arg("sinks"), py::arg("status"), py::arg("part"), py::arg("counters"), py::arg("sms"),
        py::arg("pdl") = false, py::arg("wait_polls") = (int64_t)hk::kKv4WaitPolls);
  m.attr("KV4_WAIT_POLLS") = (int64_t)hk::kKv4WaitPolls;
  m.def("kv4_workspace_sizes", [](int64_t sms) { return std::make_pair(hk::kKv4PartFloats((int)sms), hk::kKv4Counters); });
}
}  // namespace hk
