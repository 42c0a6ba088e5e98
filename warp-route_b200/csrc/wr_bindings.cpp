// wr_bindings.cpp — the `warp_route._C` torch extension.
//
// Keeps warp-route's binding surface (src/bindings.cpp:145-152):
//   naive_moe_forward, fused_moe_forward, batched_fused_moe_forward, each
//   (Tensor hidden, Tensor gate_w, Tensor weight_buf, int E, int H, int I,
//    int top_k) -> Tensor,
// with the same argument checks and messages (src/bindings.cpp:9-23,40-43,
// 75-83), raised as RuntimeError.  Differences: float32 or bfloat16 inputs
// (one dtype for all three tensors; the output is always float32), top_k up
// to num_experts, work on the current torch stream, and no device-wide
// synchronisation after the launch.  Everything below the tensor checks is a
// call into the C ABI (include/warp_route_b200.h); torch is only the binding.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <tuple>
#include <utility>

#include "warp_route_b200.h"

namespace {

#define CHECK_CONTIGUOUS(t) TORCH_CHECK((t).is_contiguous(), #t " must be contiguous")
#define CHECK_CUDA(t) TORCH_CHECK((t).is_cuda(), #t " must be a CUDA tensor")
#define CHECK_DTYPE(t)                                                                     \
  TORCH_CHECK((t).scalar_type() == torch::kFloat32 || (t).scalar_type() == torch::kBFloat16, \
              #t " must be float32 or bfloat16")

// warp-route's validate_1d/2d (src/bindings.cpp:13-23) stringify their own
// parameter ("t must be ..."); these name the argument instead.
void check_tensor(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16, name,
              " must be float32 or bfloat16");
}

void validate_1d(const torch::Tensor& t, const char* name, int64_t expected) {
  check_tensor(t, name);
  TORCH_CHECK(t.dim() == 1 && t.size(0) == expected, name, " must have shape [", expected,
              "], got shape ", t.sizes());
}

void validate_2d(const torch::Tensor& t, const char* name, int64_t rows, int64_t cols) {
  check_tensor(t, name);
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, name,
              " must have shape [", rows, ", ", cols, "], got shape ", t.sizes());
}

int32_t dtype_code(const torch::Tensor& t) {
  return t.scalar_type() == torch::kBFloat16 ? WR_DTYPE_BF16 : WR_DTYPE_F32;
}

void check_same(const torch::Tensor& a, const torch::Tensor& b, const char* an, const char* bn) {
  TORCH_CHECK(a.scalar_type() == b.scalar_type(), an, " and ", bn,
              " must have the same dtype, got ", a.scalar_type(), " and ", b.scalar_type());
  TORCH_CHECK(a.device() == b.device(), an, " and ", bn, " must be on the same device");
}

void check_status(wr_status_t st) {
  TORCH_CHECK(st == WR_OK, wr_last_error_string());
}

// One zero-initialised workspace per (device, stream), grown on demand.  Calls
// on one stream are ordered, so sharing is safe; distinct streams get distinct
// workspaces.  The map is never destroyed (process exit frees device memory).
struct WsCache {
  std::mutex mu;
  std::map<std::pair<int, cudaStream_t>, torch::Tensor> bufs;
};
WsCache& ws_cache() {
  static WsCache* c = new WsCache();
  return *c;
}

torch::Tensor workspace_for(const torch::Device& dev, cudaStream_t stream, size_t bytes) {
  auto& c = ws_cache();
  std::lock_guard<std::mutex> lk(c.mu);
  auto key = std::make_pair((int)dev.index(), stream);
  auto it = c.bufs.find(key);
  if (it != c.bufs.end() && (size_t)it->second.numel() >= bytes) return it->second;
  size_t grow = bytes < (1u << 20) ? (1u << 20) : bytes;
  torch::Tensor t = torch::zeros({(int64_t)grow}, torch::TensorOptions().dtype(torch::kUInt8).device(dev));
  c.bufs[key] = t;
  return t;
}

wr_moe_desc_t make_desc(const torch::Tensor& hidden, int E, int H, int I, int top_k,
                        const c10::optional<torch::Tensor>& bias, int ep_first, int ep_num) {
  wr_moe_desc_t d{};
  d.num_experts = E;
  d.hidden_dim = H;
  d.intermediate_dim = I;
  d.top_k = top_k;
  d.dtype = dtype_code(hidden);
  d.ep_first_expert = ep_first;
  d.ep_num_local = ep_num;
  d.router_bias = nullptr;
  if (bias.has_value() && bias->defined()) {
    const auto& b = *bias;
    CHECK_CUDA(b);
    CHECK_CONTIGUOUS(b);
    TORCH_CHECK(b.scalar_type() == torch::kFloat32, "router_bias must be float32");
    TORCH_CHECK(b.dim() == 1 && b.size(0) == E, "router_bias must have shape [", E, "], got shape ",
                b.sizes());
    d.router_bias = b.data_ptr<float>();
  }
  return d;
}

void check_weight_buf(const torch::Tensor& hidden, const torch::Tensor& weight_buf) {
  CHECK_CUDA(weight_buf);
  CHECK_CONTIGUOUS(weight_buf);
  CHECK_DTYPE(weight_buf);
  check_same(hidden, weight_buf, "hidden", "weight_buf");
}

// Shared body of the fused entry points.  hidden: [H] or [T,H].
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> fused_impl(
    const torch::Tensor& hidden, const torch::Tensor& gate_w, const torch::Tensor& weight_buf,
    int E, int H, int I, int top_k, const c10::optional<torch::Tensor>& bias, int ep_first,
    int ep_num, bool want_routing, wr_comm_t comm = nullptr) {
  const bool one = hidden.dim() == 1;
  const int64_t T = one ? 1 : hidden.size(0);
  validate_2d(gate_w, "gate_w", E, H);
  check_same(hidden, gate_w, "hidden", "gate_w");
  check_weight_buf(hidden, weight_buf);
  const c10::cuda::CUDAGuard guard(hidden.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(hidden.device().index()).stream();
  wr_moe_desc_t d = make_desc(hidden, E, H, I, top_k, bias, ep_first, ep_num);
  auto fopt = torch::TensorOptions().dtype(torch::kFloat32).device(hidden.device());
  torch::Tensor out = one ? torch::empty({H}, fopt) : torch::empty({T, H}, fopt);
  torch::Tensor ids, w;
  if (want_routing) {
    ids = torch::empty({T, top_k}, fopt.dtype(torch::kInt32));
    w = torch::empty({T, top_k}, fopt);
  }
  if (T == 0) return {out, ids, w};
  const size_t need = wr_fused_moe_workspace_size(&d, (int32_t)T);
  TORCH_CHECK(need > 0, wr_last_error_string());
  torch::Tensor ws = workspace_for(hidden.device(), stream, need);
  const int64_t wbytes = weight_buf.numel() * (int64_t)weight_buf.element_size();
  wr_status_t st;
  if (comm)
    st = wr_fused_moe_allreduce(&d, (int32_t)T, hidden.data_ptr(), gate_w.data_ptr(),
                                weight_buf.data_ptr(), wbytes, out.data_ptr<float>(),
                                want_routing ? ids.data_ptr<int32_t>() : nullptr,
                                want_routing ? w.data_ptr<float>() : nullptr, ws.data_ptr(),
                                (size_t)ws.numel(), comm, stream);
  else if (one)
    st = wr_fused_moe(&d, hidden.data_ptr(), gate_w.data_ptr(), weight_buf.data_ptr(), wbytes,
                      out.data_ptr<float>(), want_routing ? ids.data_ptr<int32_t>() : nullptr,
                      want_routing ? w.data_ptr<float>() : nullptr, ws.data_ptr(),
                      (size_t)ws.numel(), stream);
  else
    st = wr_batched_fused_moe(&d, (int32_t)T, hidden.data_ptr(), gate_w.data_ptr(),
                              weight_buf.data_ptr(), wbytes, out.data_ptr<float>(),
                              want_routing ? ids.data_ptr<int32_t>() : nullptr,
                              want_routing ? w.data_ptr<float>() : nullptr, ws.data_ptr(),
                              (size_t)ws.numel(), stream);
  check_status(st);
  return {out, ids, w};
}

// ---- warp-route's three entry points ---------------------------------------

torch::Tensor naive_moe_forward_torch(torch::Tensor hidden, torch::Tensor gate_w,
                                      torch::Tensor weight_buf, int num_experts, int hidden_dim,
                                      int intermediate_dim, int top_k) {
  validate_1d(hidden, "hidden", hidden_dim);
  validate_2d(gate_w, "gate_w", num_experts, hidden_dim);
  check_same(hidden, gate_w, "hidden", "gate_w");
  check_weight_buf(hidden, weight_buf);
  const c10::cuda::CUDAGuard guard(hidden.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(hidden.device().index()).stream();
  wr_moe_desc_t d = make_desc(hidden, num_experts, hidden_dim, intermediate_dim, top_k,
                              c10::nullopt, 0, 0);
  const size_t need = wr_naive_moe_workspace_size(&d);
  TORCH_CHECK(need > 0, wr_last_error_string());
  torch::Tensor ws = workspace_for(hidden.device(), stream, need);
  torch::Tensor out =
      torch::empty({hidden_dim}, torch::TensorOptions().dtype(torch::kFloat32).device(hidden.device()));
  check_status(wr_naive_moe(&d, hidden.data_ptr(), gate_w.data_ptr(), weight_buf.data_ptr(),
                            weight_buf.numel() * (int64_t)weight_buf.element_size(),
                            out.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(), stream));
  return out;
}

torch::Tensor fused_moe_forward_torch(torch::Tensor hidden, torch::Tensor gate_w,
                                      torch::Tensor weight_buf, int num_experts, int hidden_dim,
                                      int intermediate_dim, int top_k) {
  validate_1d(hidden, "hidden", hidden_dim);
  return std::get<0>(fused_impl(hidden, gate_w, weight_buf, num_experts, hidden_dim,
                                intermediate_dim, top_k, c10::nullopt, 0, 0, false));
}

torch::Tensor batched_fused_moe_forward_torch(torch::Tensor hidden_batch, torch::Tensor gate_w,
                                              torch::Tensor weight_buf, int num_experts,
                                              int hidden_dim, int intermediate_dim, int top_k) {
  CHECK_CUDA(hidden_batch);
  CHECK_CONTIGUOUS(hidden_batch);
  CHECK_DTYPE(hidden_batch);
  TORCH_CHECK(hidden_batch.dim() == 2 && hidden_batch.size(1) == hidden_dim,
              "hidden_batch must have shape [batch_size, ", hidden_dim, "], got shape ",
              hidden_batch.sizes());
  return std::get<0>(fused_impl(hidden_batch, gate_w, weight_buf, num_experts, hidden_dim,
                                intermediate_dim, top_k, c10::nullopt, 0, 0, false));
}

// ---- additions (keyword-only extras in warp_route.functional) -------------

// Layer with optional router bias / expert-parallel shard, returning the
// routing as well: (out fp32 [..,H], ids int32 [T,K], weights fp32 [T,K]).
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> fused_moe_routed(
    torch::Tensor hidden, torch::Tensor gate_w, torch::Tensor weight_buf, int num_experts,
    int hidden_dim, int intermediate_dim, int top_k, c10::optional<torch::Tensor> router_bias,
    int ep_first_expert, int ep_num_local) {
  CHECK_CUDA(hidden);
  CHECK_CONTIGUOUS(hidden);
  CHECK_DTYPE(hidden);
  TORCH_CHECK((hidden.dim() == 1 && hidden.size(0) == hidden_dim) ||
                  (hidden.dim() == 2 && hidden.size(1) == hidden_dim),
              "hidden must have shape [", hidden_dim, "] or [batch_size, ", hidden_dim,
              "], got shape ", hidden.sizes());
  return fused_impl(hidden, gate_w, weight_buf, num_experts, hidden_dim, intermediate_dim, top_k,
                    router_bias, ep_first_expert, ep_num_local, true);
}

// Router only: (logits fp32 [T,E], ids int32 [T,K], weights fp32 [T,K]).
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> router_topk(
    torch::Tensor hidden, torch::Tensor gate_w, int num_experts, int hidden_dim, int top_k,
    c10::optional<torch::Tensor> router_bias) {
  CHECK_CUDA(hidden);
  CHECK_CONTIGUOUS(hidden);
  CHECK_DTYPE(hidden);
  const int64_t T = hidden.dim() == 1 ? 1 : hidden.size(0);
  TORCH_CHECK(hidden.size(-1) == hidden_dim, "hidden last dimension must be ", hidden_dim);
  validate_2d(gate_w, "gate_w", num_experts, hidden_dim);
  check_same(hidden, gate_w, "hidden", "gate_w");
  const c10::cuda::CUDAGuard guard(hidden.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(hidden.device().index()).stream();
  wr_moe_desc_t d = make_desc(hidden, num_experts, hidden_dim, 1, top_k, router_bias, 0, 0);
  auto fopt = torch::TensorOptions().dtype(torch::kFloat32).device(hidden.device());
  torch::Tensor logits = torch::empty({T, num_experts}, fopt);
  torch::Tensor ids = torch::empty({T, top_k}, fopt.dtype(torch::kInt32));
  torch::Tensor w = torch::empty({T, top_k}, fopt);
  check_status(wr_router_topk(&d, (int32_t)T, hidden.data_ptr(), gate_w.data_ptr(),
                              logits.data_ptr<float>(), ids.data_ptr<int32_t>(),
                              w.data_ptr<float>(), stream));
  return {logits, ids, w};
}

// ---- communicator for the all-reduce fused into the layer ---------------
// The handle is the C pointer as an integer; the Python wrapper owns it.

int64_t comm_create(int rank, int world_size, int hidden_dim) {
  wr_comm_t c = nullptr;
  check_status(wr_comm_create(rank, world_size, hidden_dim, &c));
  return reinterpret_cast<int64_t>(c);
}

torch::Tensor comm_handle(int64_t comm) {
  torch::Tensor h = torch::empty({(int64_t)wr_comm_handle_bytes()}, torch::kUInt8);
  check_status(wr_comm_get_handle(reinterpret_cast<wr_comm_t>(comm), h.data_ptr()));
  return h;
}

void comm_open(int64_t comm, torch::Tensor handles) {
  TORCH_CHECK(handles.device().is_cpu() && handles.scalar_type() == torch::kUInt8 &&
                  handles.is_contiguous(),
              "handles must be a contiguous uint8 CPU tensor");
  check_status(wr_comm_open(reinterpret_cast<wr_comm_t>(comm), handles.data_ptr()));
}

void comm_destroy(int64_t comm) { check_status(wr_comm_destroy(reinterpret_cast<wr_comm_t>(comm))); }

void comm_set_peer_timeout_ns(int64_t comm, int64_t ns) {
  TORCH_CHECK(ns >= 0, "peer timeout must be >= 0 ns");
  check_status(wr_comm_set_peer_timeout_ns(reinterpret_cast<wr_comm_t>(comm), (uint64_t)ns));
}

void comm_reset(int64_t comm) {
  cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  check_status(wr_comm_reset(reinterpret_cast<wr_comm_t>(comm), stream));
}

// This rank's shard of the layer with the ranks' outputs summed in-kernel:
// (out fp32 [..,H], ids int32 [T,K], weights fp32 [T,K]).
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> fused_moe_allreduce(
    torch::Tensor hidden, torch::Tensor gate_w, torch::Tensor weight_buf, int num_experts,
    int hidden_dim, int intermediate_dim, int top_k, int64_t comm,
    c10::optional<torch::Tensor> router_bias, int ep_first_expert, int ep_num_local) {
  CHECK_CUDA(hidden);
  CHECK_CONTIGUOUS(hidden);
  CHECK_DTYPE(hidden);
  TORCH_CHECK(comm != 0, "comm must not be NULL");
  TORCH_CHECK((hidden.dim() == 1 && hidden.size(0) == hidden_dim) ||
                  (hidden.dim() == 2 && hidden.size(1) == hidden_dim),
              "hidden must have shape [", hidden_dim, "] or [batch_size, ", hidden_dim,
              "], got shape ", hidden.sizes());
  return fused_impl(hidden, gate_w, weight_buf, num_experts, hidden_dim, intermediate_dim, top_k,
                    router_bias, ep_first_expert, ep_num_local, true,
                    reinterpret_cast<wr_comm_t>(comm));
}

// One layer of a decode stack with the residual fused (wr_moe_decode_layer):
// returns out = hidden + layer(hidden) (fp32, summed over the ranks when comm
// is given) and writes next_x = out in hidden's dtype when next_x is given.
torch::Tensor moe_decode_layer(torch::Tensor hidden, torch::Tensor gate_w,
                               torch::Tensor weight_buf, int num_experts, int hidden_dim,
                               int intermediate_dim, int top_k, int64_t comm,
                               c10::optional<torch::Tensor> router_bias, int ep_first_expert,
                               int ep_num_local, c10::optional<torch::Tensor> next_x) {
  CHECK_CUDA(hidden);
  CHECK_CONTIGUOUS(hidden);
  CHECK_DTYPE(hidden);
  TORCH_CHECK((hidden.dim() == 1 && hidden.size(0) == hidden_dim) ||
                  (hidden.dim() == 2 && hidden.size(1) == hidden_dim),
              "hidden must have shape [", hidden_dim, "] or [batch_size, ", hidden_dim,
              "], got shape ", hidden.sizes());
  validate_2d(gate_w, "gate_w", num_experts, hidden_dim);
  check_same(hidden, gate_w, "hidden", "gate_w");
  check_weight_buf(hidden, weight_buf);
  void* nx = nullptr;
  if (next_x.has_value() && next_x->defined()) {
    const auto& n = *next_x;
    CHECK_CUDA(n);
    CHECK_CONTIGUOUS(n);
    check_same(hidden, n, "hidden", "next_x");
    TORCH_CHECK(n.sizes() == hidden.sizes(), "next_x must have hidden's shape ", hidden.sizes(),
                ", got ", n.sizes());
    nx = n.data_ptr();
  }
  const c10::cuda::CUDAGuard guard(hidden.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(hidden.device().index()).stream();
  wr_moe_desc_t d = make_desc(hidden, num_experts, hidden_dim, intermediate_dim, top_k,
                              router_bias, ep_first_expert, ep_num_local);
  const int64_t T = hidden.dim() == 1 ? 1 : hidden.size(0);
  auto fopt = torch::TensorOptions().dtype(torch::kFloat32).device(hidden.device());
  torch::Tensor out = torch::empty(hidden.sizes(), fopt);
  if (T == 0) return out;
  const size_t need = wr_fused_moe_workspace_size(&d, (int32_t)T);
  TORCH_CHECK(need > 0, wr_last_error_string());
  torch::Tensor ws = workspace_for(hidden.device(), stream, need);
  check_status(wr_moe_decode_layer(&d, (int32_t)T, hidden.data_ptr(), gate_w.data_ptr(),
                                   weight_buf.data_ptr(),
                                   weight_buf.numel() * (int64_t)weight_buf.element_size(),
                                   out.data_ptr<float>(), nx, nullptr, nullptr, ws.data_ptr(),
                                   (size_t)ws.numel(), reinterpret_cast<wr_comm_t>(comm), stream));
  return out;
}

// One rank's shard of per-expert weight lists packed on the device
// (wr_pack_experts): experts [ep_first, ep_first + ep_num), intermediate
// slice tp_rank of tp_size.  Entries outside the shard are not read.
torch::Tensor pack_experts(const std::vector<torch::Tensor>& gate,
                           const std::vector<torch::Tensor>& up,
                           const std::vector<torch::Tensor>& down, int num_experts,
                           int hidden_dim, int intermediate_dim, int ep_first, int ep_num,
                           int tp_rank, int tp_size) {
  TORCH_CHECK((int)gate.size() == num_experts && (int)up.size() == num_experts &&
                  (int)down.size() == num_experts,
              "gate_proj, up_proj and down_proj must each hold num_experts=", num_experts,
              " tensors");
  TORCH_CHECK(ep_num >= 1 && ep_first >= 0 && ep_first + ep_num <= num_experts,
              "expert shard [", ep_first, ", ", ep_first + ep_num, ") is outside [0, ",
              num_experts, ")");
  const torch::Tensor& ref = gate[ep_first];
  CHECK_CUDA(ref);
  CHECK_DTYPE(ref);
  std::vector<const void*> g(num_experts, nullptr), u(num_experts, nullptr),
      d(num_experts, nullptr);
  for (int e = ep_first; e < ep_first + ep_num; ++e) {
    const torch::Tensor* mats[3] = {&gate[e], &up[e], &down[e]};
    const char* names[3] = {"gate_proj", "up_proj", "down_proj"};
    for (int m = 0; m < 3; ++m) {
      const torch::Tensor& t = *mats[m];
      CHECK_CUDA(t);
      CHECK_CONTIGUOUS(t);
      check_same(ref, t, "gate_proj", names[m]);
      const int64_t rows = m == 2 ? hidden_dim : intermediate_dim;
      const int64_t cols = m == 2 ? intermediate_dim : hidden_dim;
      TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, names[m], "[", e,
                  "] must have shape [", rows, ", ", cols, "], got shape ", t.sizes());
    }
    g[e] = gate[e].data_ptr();
    u[e] = up[e].data_ptr();
    d[e] = down[e].data_ptr();
  }
  TORCH_CHECK(tp_size >= 1 && intermediate_dim % tp_size == 0,
              "tp_size must divide intermediate_dim");
  const int elt = (int)ref.element_size();
  const int64_t stride = wr_total_weight_bytes(1, hidden_dim, intermediate_dim / tp_size, elt);
  const c10::cuda::CUDAGuard guard(ref.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(ref.device().index()).stream();
  torch::Tensor buf = torch::empty({ep_num * stride / elt}, ref.options());
  check_status(wr_pack_experts(num_experts, hidden_dim, intermediate_dim,
                               ref.scalar_type() == torch::kBFloat16 ? WR_DTYPE_BF16
                                                                     : WR_DTYPE_F32,
                               ep_first, ep_num, tp_rank, tp_size, g.data(), u.data(), d.data(),
                               buf.data_ptr(), ep_num * stride, stream));
  return buf;
}

// ---- paged cache, shared-prefix attention, sampling --------------------------

void check_on(const torch::Tensor& t, const char* name, const torch::Tensor& ref, const char* ref_name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == ref.device(), name, " and ", ref_name, " must be on the same device");
}

void check_list(const torch::Tensor& t, const char* name, torch::ScalarType type, int64_t n,
                const torch::Tensor& ref, const char* ref_name) {
  check_on(t, name, ref, ref_name);
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n, name, " must have shape [", n, "], got shape ", t.sizes());
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// A length of one has no stride that counts: 0 is as good as any.
int64_t stride_of(const torch::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

int32_t narrow(int64_t v, const char* what) {
  TORCH_CHECK(v >= 0 && v <= INT32_MAX, what, " is out of range: ", v);
  return (int32_t)v;
}

wr_paged_kv_t make_cache(const torch::Tensor& k, const torch::Tensor& v) {
  TORCH_CHECK(k.is_cuda(), "k_cache must be a CUDA tensor");
  TORCH_CHECK(k.scalar_type() == torch::kFloat32 || k.scalar_type() == torch::kBFloat16,
              "k_cache must be float32 or bfloat16");
  TORCH_CHECK(k.dim() == 4, "k_cache must have shape [num_pages, num_kv_heads, page_size, head_dim], got shape ",
              k.sizes());
  check_same(k, v, "k_cache", "v_cache");
  TORCH_CHECK(v.sizes() == k.sizes() && v.strides() == k.strides(),
              "v_cache must have k_cache's shape and strides, got shape ", v.sizes(), " and ", k.sizes());
  TORCH_CHECK(k.stride(3) == 1 || k.size(3) == 1, "the caches' last dimension must be contiguous");
  wr_paged_kv_t c{};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.page_stride = stride_of(k, 0);
  c.head_stride = stride_of(k, 1);
  c.slot_stride = stride_of(k, 2);
  c.num_pages = narrow(k.size(0), "num_pages");
  c.num_kv_heads = narrow(k.size(1), "num_kv_heads");
  c.page_size = narrow(k.size(2), "page_size");
  c.head_dim = narrow(k.size(3), "head_dim");
  c.dtype = dtype_code(k);
  return c;
}

wr_rows_t make_rows(const torch::Tensor& t, const char* name, int64_t tokens, int64_t heads,
                    const torch::Tensor& cache) {
  check_on(t, name, cache, "k_cache");
  TORCH_CHECK(t.scalar_type() == cache.scalar_type(), name, " and k_cache must have the same dtype, got ",
              t.scalar_type(), " and ", cache.scalar_type());
  TORCH_CHECK(t.dim() == 3 && t.size(0) == tokens && (heads < 0 || t.size(1) == heads) &&
                  t.size(2) == cache.size(3),
              name, " must have shape [", tokens, ", ", heads < 0 ? std::string("heads") : std::to_string(heads),
              ", ", cache.size(3), "], got shape ", t.sizes());
  TORCH_CHECK(t.stride(2) == 1, name, "'s last dimension must be contiguous");
  return wr_rows_t{t.data_ptr(), stride_of(t, 0), stride_of(t, 1)};
}

// Writes k and v into the caches, in place; returns the rotated q or None.
c10::optional<torch::Tensor> append_paged_kv(torch::Tensor k, torch::Tensor v, torch::Tensor k_cache,
                                             torch::Tensor v_cache, torch::Tensor slots,
                                             c10::optional<torch::Tensor> positions,
                                             c10::optional<torch::Tensor> inv_freq,
                                             c10::optional<torch::Tensor> q, bool interleaved) {
  const wr_paged_kv_t cache = make_cache(k_cache, v_cache);
  TORCH_CHECK(k.dim() == 3, "k must have shape [tokens, heads, head_dim], got shape ", k.sizes());
  const int64_t T = k.size(0);
  const wr_rows_t kr = make_rows(k, "k", T, k_cache.size(1), k_cache);
  const wr_rows_t vr = make_rows(v, "v", T, k_cache.size(1), k_cache);
  check_list(slots, "slots", torch::kInt64, T, k_cache, "k_cache");
  TORCH_CHECK(positions.has_value() == inv_freq.has_value(), "positions and inv_freq go together");
  int32_t rot = 0;
  if (positions.has_value()) {
    check_list(*positions, "positions", torch::kInt64, T, k_cache, "k_cache");
    TORCH_CHECK(inv_freq->dim() == 1, "inv_freq must have shape [rot_dim / 2], got shape ", inv_freq->sizes());
    check_list(*inv_freq, "inv_freq", torch::kFloat32, inv_freq->size(0), k_cache, "k_cache");
    rot = narrow(2 * inv_freq->size(0), "rot_dim");
  }
  const c10::cuda::CUDAGuard guard(k_cache.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(k_cache.device().index()).stream();
  wr_rows_t qr{};
  torch::Tensor out;
  int32_t hq = 0;
  if (q.has_value()) {
    qr = make_rows(*q, "q", T, -1, k_cache);
    hq = narrow(q->size(1), "num_q_heads");
    out = torch::empty({T, hq, k_cache.size(3)}, k_cache.options());
    if (T == 0) return out;
  }
  check_status(wr_append_paged_kv(&cache, narrow(T, "num_tokens"), &kr, &vr, slots.data_ptr<int64_t>(),
                                  rot ? positions->data_ptr<int64_t>() : nullptr,
                                  rot ? inv_freq->data_ptr<float>() : nullptr, rot, interleaved ? 1 : 0, hq,
                                  q.has_value() ? &qr : nullptr, q.has_value() ? out.data_ptr() : nullptr,
                                  stream));
  if (!q.has_value()) return c10::nullopt;
  return out;
}

std::tuple<torch::Tensor, c10::optional<torch::Tensor>> shared_prefix_attention(
    torch::Tensor q, torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor block_tables,
    torch::Tensor context_lens, c10::optional<torch::Tensor> prefix_pages, int64_t prefix_len,
    c10::optional<torch::Tensor> q_start, double scale, bool want_lse) {
  const wr_paged_kv_t cache = make_cache(k_cache, v_cache);
  TORCH_CHECK(q.dim() == 3, "q must have shape [tokens, heads, head_dim], got shape ", q.sizes());
  const int64_t T = q.size(0);
  const wr_rows_t qr = make_rows(q, "q", T, -1, k_cache);
  check_on(block_tables, "block_tables", k_cache, "k_cache");
  TORCH_CHECK(block_tables.scalar_type() == torch::kInt32, "block_tables must be ", torch::kInt32, ", got ",
              block_tables.scalar_type());
  TORCH_CHECK(block_tables.dim() == 2, "block_tables must have shape [num_seqs, pages], got shape ",
              block_tables.sizes());
  TORCH_CHECK(block_tables.size(1) <= 1 || block_tables.stride(1) == 1,
              "block_tables' last dimension must be contiguous");
  const int64_t B = block_tables.size(0);
  check_list(context_lens, "context_lens", torch::kInt32, B, k_cache, "k_cache");
  if (q_start.has_value()) check_list(*q_start, "q_start", torch::kInt32, B + 1, k_cache, "k_cache");
  else TORCH_CHECK(T == B, "without q_start q must have one token a sequence, got ", T, " tokens and ", B,
                   " sequences");
  TORCH_CHECK(prefix_len >= 0, "prefix_len must be >= 0, got ", prefix_len);
  if (prefix_len > 0) {
    TORCH_CHECK(prefix_pages.has_value(), "prefix_pages must be given when prefix_len > 0");
    check_list(*prefix_pages, "prefix_pages", torch::kInt32, prefix_pages->size(0), k_cache, "k_cache");
    TORCH_CHECK(prefix_pages->size(0) * k_cache.size(2) >= prefix_len, "prefix_pages holds ",
                prefix_pages->size(0), " pages of ", k_cache.size(2), ", too few for prefix_len ", prefix_len);
  }
  wr_attn_desc_t d{};
  d.num_tokens = narrow(T, "num_tokens");
  d.num_seqs = narrow(B, "num_seqs");
  d.num_q_heads = narrow(q.size(1), "num_q_heads");
  d.table_width = narrow(block_tables.size(1), "table_width");
  d.table_stride = stride_of(block_tables, 0);
  d.prefix_len = narrow(prefix_len, "prefix_len");
  d.scale = (float)scale;
  const c10::cuda::CUDAGuard guard(k_cache.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(k_cache.device().index()).stream();
  torch::Tensor out = torch::empty({T, q.size(1), q.size(2)}, k_cache.options());
  c10::optional<torch::Tensor> lse;
  if (want_lse) lse = torch::empty({T, q.size(1)}, k_cache.options().dtype(torch::kFloat32));
  const size_t need = wr_shared_prefix_attention_workspace_size(&cache, &d, q_start.has_value() ? 1 : 0);
  TORCH_CHECK(need > 0, wr_last_error_string());
  if (T == 0) return {out, lse};
  // From torch's allocator for this call alone: in a captured graph it is the
  // graph's own memory, so two graphs never share one.
  torch::Tensor ws = torch::empty({(int64_t)need}, k_cache.options().dtype(torch::kUInt8));
  check_status(wr_shared_prefix_attention(
      &cache, &d, &qr, block_tables.data_ptr<int32_t>(), context_lens.data_ptr<int32_t>(),
      q_start.has_value() ? q_start->data_ptr<int32_t>() : nullptr,
      prefix_len > 0 ? prefix_pages->data_ptr<int32_t>() : nullptr, out.data_ptr(),
      want_lse ? lse->data_ptr<float>() : nullptr, ws.data_ptr(), need, stream));
  return {out, lse};
}

// Each setting: its number, or a tensor with one for each row.
torch::Tensor sample_tokens(torch::Tensor logits, torch::Tensor uniforms, double temperature,
                            c10::optional<torch::Tensor> temperatures, int64_t top_k,
                            c10::optional<torch::Tensor> top_ks, double top_p,
                            c10::optional<torch::Tensor> top_ps, double min_p,
                            c10::optional<torch::Tensor> min_ps) {
  CHECK_CUDA(logits);
  CHECK_DTYPE(logits);
  TORCH_CHECK(logits.dim() == 2, "logits must have shape [rows, vocab], got shape ", logits.sizes());
  TORCH_CHECK(logits.stride(1) == 1 || logits.size(1) == 1, "logits' last dimension must be contiguous");
  const int64_t R = logits.size(0);
  check_list(uniforms, "uniforms", torch::kFloat32, R, logits, "logits");
  wr_sampling_t s{};
  s.temperature = (float)temperature;
  s.top_p = (float)top_p;
  s.min_p = (float)min_p;
  s.top_k = (int32_t)std::min<int64_t>(std::max<int64_t>(top_k, 0), INT32_MAX);
  if (temperatures.has_value()) {
    check_list(*temperatures, "temperature", torch::kFloat32, R, logits, "logits");
    s.temperatures = temperatures->data_ptr<float>();
  }
  if (top_ps.has_value()) {
    check_list(*top_ps, "top_p", torch::kFloat32, R, logits, "logits");
    s.top_ps = top_ps->data_ptr<float>();
  }
  if (min_ps.has_value()) {
    check_list(*min_ps, "min_p", torch::kFloat32, R, logits, "logits");
    s.min_ps = min_ps->data_ptr<float>();
  }
  if (top_ks.has_value()) {
    check_list(*top_ks, "top_k", torch::kInt32, R, logits, "logits");
    s.top_ks = top_ks->data_ptr<int32_t>();
  }
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(logits.device().index()).stream();
  torch::Tensor ids = torch::empty({R}, logits.options().dtype(torch::kInt64));
  check_status(wr_sample_tokens(R, narrow(logits.size(1), "vocab"), dtype_code(logits), logits.data_ptr(),
                                stride_of(logits, 0), uniforms.data_ptr<float>(), &s,
                                ids.data_ptr<int64_t>(), stream));
  return ids;
}

int64_t workspace_status(torch::Tensor hidden) {
  // Reads and clears the status word of this device/stream's cached workspace.
  const c10::cuda::CUDAGuard guard(hidden.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(hidden.device().index()).stream();
  torch::Tensor ws = workspace_for(hidden.device(), stream, 256);
  return (int64_t)wr_workspace_status(ws.data_ptr(), stream);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("naive_moe_forward", &naive_moe_forward_torch,
        "Naive multi-kernel MoE forward (float32 or bfloat16 inputs, float32 output)");
  m.def("fused_moe_forward", &fused_moe_forward_torch,
        "Fused MoE forward for one decode token (float32 or bfloat16 inputs, float32 output)");
  m.def("batched_fused_moe_forward", &batched_fused_moe_forward_torch,
        "Fused MoE forward for B decode tokens (float32 or bfloat16 inputs, float32 output)");
  m.def("fused_moe_routed", &fused_moe_routed, "Fused MoE forward returning (out, ids, weights)",
        py::arg("hidden"), py::arg("gate_w"), py::arg("weight_buf"), py::arg("num_experts"),
        py::arg("hidden_dim"), py::arg("intermediate_dim"), py::arg("top_k"),
        py::arg("router_bias") = py::none(), py::arg("ep_first_expert") = 0,
        py::arg("ep_num_local") = 0);
  m.def("router_topk", &router_topk, "Router + softmax + top-K: (logits, ids, weights)",
        py::arg("hidden"), py::arg("gate_w"), py::arg("num_experts"), py::arg("hidden_dim"),
        py::arg("top_k"), py::arg("router_bias") = py::none());
  m.def("comm_create", &comm_create, "Communicator of one rank (returns an opaque handle)",
        py::arg("rank"), py::arg("world_size"), py::arg("hidden_dim"));
  m.def("comm_handle", &comm_handle, "This rank's IPC handle bytes (uint8 CPU tensor)");
  m.def("comm_open", &comm_open, "Map every rank's buffer (handles in rank order)");
  m.def("comm_destroy", &comm_destroy, "Unmap and free a communicator");
  m.def("comm_set_peer_timeout_ns", &comm_set_peer_timeout_ns,
        "Bound of each wait for a peer's partial outputs (ns; 0 = default)");
  m.def("comm_reset", &comm_reset,
        "Back to the initial state after a timed-out call (every rank, between host barriers)");
  m.def("fused_moe_allreduce", &fused_moe_allreduce,
        "This rank's shard of the layer with the ranks' outputs summed in the same kernel",
        py::arg("hidden"), py::arg("gate_w"), py::arg("weight_buf"), py::arg("num_experts"),
        py::arg("hidden_dim"), py::arg("intermediate_dim"), py::arg("top_k"), py::arg("comm"),
        py::arg("router_bias") = py::none(), py::arg("ep_first_expert") = 0,
        py::arg("ep_num_local") = 0);
  m.def("moe_decode_layer", &moe_decode_layer,
        "Layer with the residual fused: out = hidden + layer(hidden); next_x = out in the "
        "layer dtype",
        py::arg("hidden"), py::arg("gate_w"), py::arg("weight_buf"), py::arg("num_experts"),
        py::arg("hidden_dim"), py::arg("intermediate_dim"), py::arg("top_k"), py::arg("comm"),
        py::arg("router_bias") = py::none(), py::arg("ep_first_expert") = 0,
        py::arg("ep_num_local") = 0, py::arg("next_x") = py::none());
  m.def("pack_experts", &pack_experts,
        "Pack one rank's shard (experts, intermediate slice) of per-expert weights on the "
        "device");
  m.def("append_paged_kv", &append_paged_kv,
        "Keys and values into a paged cache, rotated by position; returns the rotated q",
        py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"), py::arg("slots"),
        py::arg("positions") = py::none(), py::arg("inv_freq") = py::none(),
        py::arg("q") = py::none(), py::arg("interleaved") = false);
  m.def("shared_prefix_attention", &shared_prefix_attention,
        "Attention of a batch over a paged cache with a prefix shared by all: (out, lse or None)",
        py::arg("q"), py::arg("k_cache"), py::arg("v_cache"), py::arg("block_tables"),
        py::arg("context_lens"), py::arg("prefix_pages"), py::arg("prefix_len"),
        py::arg("q_start"), py::arg("scale"), py::arg("return_lse"));
  m.def("sample_tokens", &sample_tokens,
        "A token for each row of logits by temperature, top-k, top-p and min-p",
        py::arg("logits"), py::arg("uniforms"), py::arg("temperature"), py::arg("temperatures"),
        py::arg("top_k"), py::arg("top_ks"), py::arg("top_p"), py::arg("top_ps"),
        py::arg("min_p"), py::arg("min_ps"));
  m.def("workspace_status", &workspace_status,
        "Read and clear the device status word of the current stream's workspace");
  m.def("version", []() { return std::string(wr_version()); });
}
