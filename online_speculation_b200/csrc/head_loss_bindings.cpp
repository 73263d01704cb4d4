// PyTorch bindings of the vocabulary-head losses and the top logits (head_loss.cu, top_logits.cu).
//
// Scratch and saved tensors come from PyTorch's allocator on every call: two graphs, or two
// streams, never share them.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "head_loss.h"
#include "head_loss_bindings.h"
#include "top_logits.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

void check(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, " failed: ", cudaGetErrorString(e));
}

// A tensor on the current device, past the dispatcher: small calls are bound by the host.
Tensor device_tensor(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

// Bytes of the current stream that live as long as the call.
struct Scratch {
  c10::DataPtr data;
  explicit Scratch(size_t bytes) : data(c10::cuda::CUDACachingAllocator::get()->allocate(bytes)) {}
  char* base() const { return static_cast<char*>(data.get()); }
};

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// Rows the tile loads can address: unit inner stride, 16-byte aligned starts.  Others are copied.
Tensor tile_rows(const Tensor& t) {
  const bool ok = t.stride(1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                  (t.size(0) == 1 || (t.stride(0) >= t.size(1) && t.stride(0) % 8 == 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

long long row_stride(const Tensor& t) { return t.size(0) == 1 ? t.size(1) : t.stride(0); }

void check_matrix(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && t.scalar_type() == torch::kBFloat16, name, " must be a 2-D CUDA bf16 tensor");
}

// Per-row state of one call, carved out of one byte buffer (saved for the backward pass).
struct Carve {
  char* base;
  size_t at = 0;
  template <typename T>
  T* take(long long n) {
    T* p = reinterpret_cast<T*>(base + at);
    at += (static_cast<size_t>(n) * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

size_t bind_state(osb::HeadLossState& s, char* base) {
  Carve c{base};
  const long long listed = static_cast<long long>(s.R) * s.K;
  s.hc = c.take<__nv_bfloat16>(static_cast<long long>(s.rpad) * s.H);
  s.row_of = c.take<int>(s.rpad);
  s.compact_of = c.take<int>(s.R);
  s.count = c.take<int>(1);
  s.list_id = c.take<int>(listed);
  s.list_logit = c.take<float>(listed);
  s.list_mass = c.take<float>(s.divergence ? listed : 0);
  s.rest_mass = c.take<float>(s.divergence ? s.R : 0);
  s.all_mass = c.take<float>(s.divergence ? s.R : 0);
  s.row_stat = c.take<float4>(s.R);
  return c.at;
}

osb::HeadLossState make_state(const Tensor& w, int64_t R, int64_t H, int64_t K, const OptTensor& inv_temp,
                              bool divergence, bool rest_bucket, double smoothing, double z_loss, const Tensor& status) {
  TORCH_CHECK(R >= 1 && H >= 8 && H % 8 == 0, "hidden rows must be a multiple of 8 wide");
  TORCH_CHECK(w.size(0) >= 1 && w.size(0) < (1ll << 31) - 65536 && R < (1ll << 31) - 65536, "too many rows");
  TORCH_CHECK(K >= 1 && K <= osb::kHeadMaxListed, "listed columns per row: 1 to ", osb::kHeadMaxListed);
  TORCH_CHECK(status.is_cuda() && status.scalar_type() == torch::kInt32, "status word");
  osb::HeadLossState s{};
  s.R = static_cast<int>(R);
  s.H = static_cast<int>(H);
  s.V = static_cast<int>(w.size(0));
  s.K = static_cast<int>(K);
  s.rpad = static_cast<int>((R + osb::kHeadRowPad - 1) / osb::kHeadRowPad * osb::kHeadRowPad);
  s.w = reinterpret_cast<const __nv_bfloat16*>(w.data_ptr());
  s.ldw = row_stride(w);
  s.divergence = divergence;
  s.rest_bucket = rest_bucket;
  s.smoothing = static_cast<float>(smoothing);
  s.z_loss = static_cast<float>(z_loss);
  s.status = status.data_ptr<int>();
  if (given(inv_temp)) {
    TORCH_CHECK(inv_temp->is_cuda() && inv_temp->scalar_type() == torch::kFloat32 && inv_temp->is_contiguous() &&
                    inv_temp->numel() == R,
                "inv_temp needs one contiguous float per row");
    s.inv_temp = inv_temp->data_ptr<float>();
  }
  return s;
}

// ids [R] (cross entropy) or [R, K] with teacher logits [R, K].  Returns (loss [R], saved bytes, kept logits or
// an undefined tensor).
std::tuple<Tensor, Tensor, Tensor> head_loss_forward(Tensor h, Tensor weight, Tensor ids, OptTensor teacher,
                                             OptTensor teacher_lse, OptTensor inv_temp, int64_t ignore_index,
                                             double smoothing, double z_loss, bool keep, Tensor status) {
  check_matrix(h, "h");
  check_matrix(weight, "weight");
  TORCH_CHECK(h.size(1) == weight.size(1) && h.device() == weight.device(), "h and weight differ in width or device");
  TORCH_CHECK(ids.is_cuda() && ids.device() == h.device() && ids.is_contiguous(), "ids must be contiguous on the device of h");
  TORCH_CHECK(ids.scalar_type() == torch::kInt32 || ids.scalar_type() == torch::kInt64, "ids must be int32 or int64");
  const int64_t R = h.size(0), H = h.size(1);
  const bool divergence = given(teacher);
  TORCH_CHECK(ids.dim() == (divergence ? 2 : 1) && ids.size(0) == R, "one row of ids for every row of h");
  const int64_t K = divergence ? ids.size(1) : 1;
  c10::cuda::CUDAGuard guard(h.device());
  check(cudaSetDevice(h.get_device()), "cudaSetDevice");   // see head_loss_backward
  const Tensor rows = tile_rows(h), w = tile_rows(weight);
  osb::HeadLossState s = make_state(w, R, H, K, inv_temp, divergence, given(teacher_lse), smoothing, z_loss, status);
  Tensor saved = device_tensor({static_cast<int64_t>(bind_state(s, nullptr))}, torch::kUInt8, h);
  bind_state(s, static_cast<char*>(saved.data_ptr()));
  s.h = reinterpret_cast<const __nv_bfloat16*>(rows.data_ptr());
  s.ldh = row_stride(rows);
  Tensor loss = device_tensor({R}, torch::kFloat32, h);
  s.loss = loss.data_ptr<float>();

  osb::HeadTargets t{};
  t.ids = ids.data_ptr();
  t.ids_i64 = ids.scalar_type() == torch::kInt64;
  t.ignore_index = ignore_index;
  if (divergence) {
    TORCH_CHECK(teacher->is_cuda() && teacher->is_contiguous() && teacher->sizes() == ids.sizes(),
                "teacher logits must be contiguous and shaped like ids");
    TORCH_CHECK(teacher->scalar_type() == torch::kFloat32 || teacher->scalar_type() == torch::kBFloat16,
                "teacher logits must be fp32 or bf16");
    t.teacher = teacher->data_ptr();
    t.teacher_bf16 = teacher->scalar_type() == torch::kBFloat16;
    if (given(teacher_lse)) {
      TORCH_CHECK(teacher_lse->is_cuda() && teacher_lse->scalar_type() == torch::kFloat32 &&
                      teacher_lse->is_contiguous() && teacher_lse->numel() == R,
                  "teacher_lse needs one contiguous float per row");
      t.teacher_lse = teacher_lse->data_ptr<float>();
    }
  }
  osb::HeadStatsScratch p{};
  Tensor kept;
  const osb::HeadKept keeps = keep ? osb::head_loss_kept(s.R, s.H, s.V) : osb::HeadKept{};
  if (keeps.bytes > 0) {
    kept = device_tensor({keeps.bytes}, torch::kUInt8, h);
    p.kept = static_cast<char*>(kept.data_ptr());
  }
  p.tiles = osb::head_loss_vocab_tiles(s.R, s.V, keeps.bytes > 0);
  const long long parts = static_cast<long long>(s.rpad) * p.tiles;
  Carve size{nullptr};
  size.take<float2>(keeps.part_at > 0 ? 0 : parts);
  size.take<float>(smoothing != 0.0 ? parts : 0);
  size.take<unsigned char>(R);
  const Scratch scratch(size.at);
  Carve c{scratch.base()};
  p.part = c.take<float2>(keeps.part_at > 0 ? 0 : parts);
  if (keeps.part_at > 0) p.part = reinterpret_cast<float2*>(p.kept + keeps.part_at);
  float* part_sum = c.take<float>(smoothing != 0.0 ? parts : 0);
  p.part_sum = smoothing != 0.0 ? part_sum : nullptr;
  t.active = c.take<unsigned char>(R);
  const auto stream = at::cuda::getCurrentCUDAStream();
  check(osb::head_loss_rows_launch(s, t, stream), "head loss rows");
  check(osb::head_loss_forward_launch(s, p, stream), "head loss forward");
  return {loss, saved, kept};
}

// Gradients of sum_r g[r] loss[r]: (dh [R, H] or undefined, dW [V, H] or undefined), bf16.
std::tuple<OptTensor, OptTensor> head_loss_backward(Tensor saved, Tensor kept, Tensor weight, OptTensor inv_temp, Tensor g,
                                                    int64_t K, bool divergence, bool rest_bucket, double smoothing,
                                                    double z_loss, bool need_dh, bool need_dw, int64_t piece,
                                                    Tensor status) {
  check_matrix(weight, "weight");
  TORCH_CHECK(g.is_cuda() && g.scalar_type() == torch::kFloat32 && g.is_contiguous() && g.dim() == 1, "g: one float per row");
  const int64_t R = g.size(0), H = weight.size(1), V = weight.size(0);
  c10::cuda::CUDAGuard guard(weight.device());
  // binds the device's context to this thread: the tensor maps are made by the driver, which needs one, and
  // an autograd thread may not have called the runtime yet
  check(cudaSetDevice(weight.get_device()), "cudaSetDevice");
  const Tensor w = tile_rows(weight);
  osb::HeadLossState s = make_state(w, R, H, K, inv_temp, divergence, rest_bucket, smoothing, z_loss, status);
  TORCH_CHECK(saved.scalar_type() == torch::kUInt8 && saved.numel() == static_cast<int64_t>(bind_state(s, nullptr)),
              "saved state does not belong to these arguments");
  bind_state(s, static_cast<char*>(saved.data_ptr()));
  osb::HeadGradArgs a{};
  a.g = g.data_ptr<float>();
  if (kept.defined()) a.kept = static_cast<const char*>(kept.data_ptr());
  if (piece > 0) {
    TORCH_CHECK(piece % 256 == 0, "pieces are multiples of 256 columns");
    a.piece = static_cast<int>(std::min<int64_t>(piece, (V + 255) / 256 * 256));
  } else {
    a.piece = osb::head_loss_piece(s.R, s.V);
  }
  a.splits = need_dh ? osb::head_loss_splits(s.R, s.H, a.piece, s.V, need_dw) : 1;
  OptTensor dh, dw;
  if (need_dh) {
    dh = device_tensor({R, H}, torch::kBFloat16, weight);
    a.dh = reinterpret_cast<__nv_bfloat16*>(dh->data_ptr());
  }
  if (need_dw) {
    dw = device_tensor({V, H}, torch::kBFloat16, weight);
    a.dw = reinterpret_cast<__nv_bfloat16*>(dw->data_ptr());
  }
  const long long dl = static_cast<long long>(osb::head_loss_grad_rows(s.R)) * a.piece;
  const long long parts = need_dh ? static_cast<long long>(a.splits) * s.rpad * H : 0;
  Carve size{nullptr};
  size.take<__nv_bfloat16>(dl);
  size.take<float>(parts);
  size.take<float4>(s.rpad);
  size.take<float>(R * K);
  const Scratch scratch(size.at);
  Carve c{scratch.base()};
  a.dl = c.take<__nv_bfloat16>(dl);
  a.dh_part = c.take<float>(parts);
  a.row_coef = c.take<float4>(s.rpad);
  a.list_grad = c.take<float>(R * K);
  check(osb::head_loss_backward_launch(s, a, at::cuda::getCurrentCUDAStream()), "head loss backward");
  return {dh, dw};
}

// The loss as an autograd node: the backward pass runs on the engine's thread without the interpreter.
struct HeadLossNode : public torch::autograd::Function<HeadLossNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& h, const Tensor& weight, const Tensor& ids,
                        const OptTensor& teacher, const OptTensor& teacher_lse, const OptTensor& inv_temp,
                        int64_t ignore_index, double smoothing, double z_loss, int64_t piece, bool keep,
                        const Tensor& status) {
    auto [loss, saved, kept] = head_loss_forward(h, weight, ids, teacher, teacher_lse, inv_temp, ignore_index, smoothing,
                                           z_loss, keep, status);
    ctx->save_for_backward({saved, weight, given(inv_temp) ? *inv_temp : Tensor(), kept});
    // one word a device, shared by all kernels and reset when an error is reported: no input whose changes count
    ctx->saved_data["status"] = status;
    ctx->saved_data["k"] = given(teacher) ? ids.size(1) : 1;
    ctx->saved_data["divergence"] = given(teacher);
    ctx->saved_data["rest"] = given(teacher_lse);
    ctx->saved_data["smoothing"] = smoothing;
    ctx->saved_data["z"] = z_loss;
    ctx->saved_data["piece"] = piece;
    return loss;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "the head losses are differentiable once: create_graph is not supported");
    const auto saved = ctx->get_saved_variables();
    const Tensor g = grads[0].to(torch::kFloat32).contiguous();
    OptTensor inv_temp;
    if (saved[2].defined()) inv_temp = saved[2];
    auto& d = ctx->saved_data;
    auto [dh, dw] = head_loss_backward(saved[0], saved[3], saved[1], inv_temp, g, d["k"].toInt(), d["divergence"].toBool(),
                                       d["rest"].toBool(), d["smoothing"].toDouble(), d["z"].toDouble(),
                                       ctx->needs_input_grad(0), ctx->needs_input_grad(1), d["piece"].toInt(), d["status"].toTensor());
    torch::autograd::variable_list out(12);
    if (given(dh)) out[0] = *dh;
    if (given(dw)) out[1] = *dw;
    return out;
  }
};

Tensor head_loss(const Tensor& h, const Tensor& weight, const Tensor& ids, const OptTensor& teacher,
                 const OptTensor& teacher_lse, const OptTensor& inv_temp, int64_t ignore_index, double smoothing,
                 double z_loss, int64_t piece, const Tensor& status) {
  // a piece that the caller chose bounds the memory: nothing is kept
  const bool keep = piece <= 0 && at::GradMode::is_enabled() && (h.requires_grad() || weight.requires_grad());
  return HeadLossNode::apply(h, weight, ids, teacher, teacher_lse, inv_temp, ignore_index, smoothing, z_loss, piece, keep,
                             status);
}

std::tuple<Tensor, Tensor, Tensor> top_logits(Tensor logits, int64_t k, OptTensor inv_temp) {
  // a single column may have any inner stride, contiguous or not
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) == 1),
              "logits must be 2-D CUDA rows of unit inner stride");
  TORCH_CHECK(logits.scalar_type() == torch::kFloat32 || logits.scalar_type() == torch::kBFloat16, "logits must be fp32 or bf16");
  const int64_t R = logits.size(0), V = logits.size(1);
  TORCH_CHECK(R >= 1 && k >= 1 && k <= V && k <= osb::kTopLogitsMax && V < (1ll << 31) - 65536, "top_logits sizes");
  osb::TopLogitsArgs a{};
  if (given(inv_temp)) {
    TORCH_CHECK(inv_temp->is_cuda() && inv_temp->scalar_type() == torch::kFloat32 && inv_temp->is_contiguous() &&
                    inv_temp->numel() == R,
                "inv_temp needs one contiguous float per row");
    a.inv_temp = inv_temp->data_ptr<float>();
  }
  c10::cuda::CUDAGuard guard(logits.device());
  Tensor values = device_tensor({R, k}, torch::kFloat32, logits), ids = device_tensor({R, k}, torch::kInt32, logits);
  Tensor lse = device_tensor({R}, torch::kFloat32, logits);
  a.logits = logits.data_ptr();
  a.bf16 = logits.scalar_type() == torch::kBFloat16;
  a.ld = row_stride(logits);
  a.V = static_cast<int>(V);
  a.k = static_cast<int>(k);
  a.splits = osb::top_logits_splits(static_cast<int>(std::min<int64_t>(R, 1 << 20)), a.V, a.k);
  TORCH_CHECK(R * a.splits < (1ll << 31), "too many rows");
  a.R = static_cast<int>(R);
  a.values = values.data_ptr<float>();
  a.ids = ids.data_ptr<int>();
  a.lse = lse.data_ptr<float>();
  c10::optional<Scratch> scratch;
  if (a.splits > 1) {
    Carve size{nullptr};
    size.take<unsigned long long>(R * a.splits * k);
    size.take<float2>(R * a.splits);
    scratch.emplace(size.at);
    Carve c{scratch->base()};
    a.keys = c.take<unsigned long long>(R * a.splits * k);
    a.part = c.take<float2>(R * a.splits);
  }
  check(osb::top_logits_launch(a, at::cuda::getCurrentCUDAStream()), "top logits");
  return {values, ids, lse};
}

}  // namespace

void register_head_losses(pybind11::module_& m) {
  m.def("head_loss", &head_loss);
  m.def("top_logits", &top_logits);
}
