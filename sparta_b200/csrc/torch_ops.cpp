// The training operators as torch autograd functions: dropout, rotary positions, fused sparse attention.  They check
// and lay out tensors, call the C ABI of include/sparta_b200.h and record the backward pass, all without Python: the
// operators' kernels take microseconds at small sizes, where an autograd function written in Python costs its user
// 50 to 100 microseconds per step (rotary positions of 1777 tokens, forward and backward: 157 us from Python, 76 us from here).
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "../../include/sparta_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

void check_status(int status, const char* where) {
  TORCH_CHECK(status == SPARTA_OK, where, ": status ", status, " (", sparta_status_string(status), ")");
}
void check_cuda(const Tensor& x) {
  TORCH_CHECK(x.is_cuda(), "sparta_b200 operators run on CUDA tensors only (no CPU fallback)");
}
int dtype_code(const Tensor& x) {
  switch (x.scalar_type()) {
    case at::kFloat: return SPARTA_F32;
    case at::kHalf: return SPARTA_F16;
    case at::kBFloat16: return SPARTA_BF16;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", x.scalar_type(), ": expected float32, float16 or bfloat16");
  }
}
void* stream_of(const Tensor& x) { return at::cuda::getCurrentCUDAStream(x.get_device()).stream(); }

const int64_t* rng_pointer(const OptTensor& rng, const Tensor& x) {
  if (!rng) return nullptr;
  TORCH_CHECK_VALUE(rng->scalar_type() == at::kLong && rng->numel() == 2 && rng->is_contiguous(),
                    "rng has to be a contiguous int64 tensor of two numbers (seed, call number)");
  TORCH_CHECK_VALUE(rng->device() == x.device(), "rng is on ", rng->device(), ", the input on ", x.device());
  return rng->const_data_ptr<int64_t>();
}
OptTensor optional_of(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
Tensor tensor_of(const OptTensor& t) { return t ? *t : Tensor(); }

// ---- dropout ----------------------------------------------------------------------------------------------------
struct Blocks {  // BCSR indexes of block values; absent for dense tensors
  OptTensor idx, nnz;
  int64_t BH = 0, BW = 0, stride = 0;
};

Tensor run_dropout(const Tensor& input, double p, const OptTensor& rng, int64_t seed, int64_t call, const Blocks& blocks) {
  const Tensor x = input.contiguous();
  Tensor y = at::empty_like(x);
  const int64_t n = x.numel(), dim = x.dim();
  if (n == 0) return y;
  const int dtype = dtype_code(x);
  const int64_t* numbers = rng_pointer(rng, x);
  const c10::cuda::CUDAGuard guard(x.device());
  if (!blocks.idx) {
    const int64_t W = dim > 0 ? x.size(-1) : 1, H = dim > 1 ? x.size(-2) : 1, B = n / (H * W);
    TORCH_CHECK_VALUE(W <= INT_MAX && H <= INT_MAX && B <= INT_MAX, "dropout: a dimension beyond 31 bits");
    check_status(sparta_dropout(x.const_data_ptr(), y.mutable_data_ptr(), (int)B, (int)H, (int)W, p, numbers, (uint64_t)seed,
                                (uint64_t)call, dtype, stream_of(x)), "sparta_dropout");
  } else {
    check_status(sparta_dropout_blocks(x.const_data_ptr(), y.mutable_data_ptr(), blocks.idx->const_data_ptr<int32_t>(),
                                       blocks.nnz->const_data_ptr<int32_t>(), (int)(n / x.size(-1)), (int)blocks.BH,
                                       (int)blocks.BW, blocks.stride, p, numbers, (uint64_t)seed, (uint64_t)call, dtype,
                                       stream_of(x)), "sparta_dropout_blocks");
  }
  return y;
}

struct DropoutFn : torch::autograd::Function<DropoutFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& rng, const OptTensor& idx, const OptTensor& nnz,
                        double p, int64_t seed, int64_t call, int64_t BH, int64_t BW, int64_t stride) {
    // numbers that are rewritten before the backward pass would drop other positions: saved, so that autograd refuses
    ctx->save_for_backward({tensor_of(rng), tensor_of(idx), tensor_of(nnz)});
    ctx->saved_data["p"] = p;
    ctx->saved_data["n"] = std::vector<int64_t>{seed, call, BH, BW, stride};
    return run_dropout(x, p, rng, seed, call, {idx, nnz, BH, BW, stride});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(10);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const double p = ctx->saved_data["p"].toDouble();
    const auto n = ctx->saved_data["n"].toIntVector();
    const OptTensor rng = optional_of(saved[0]), idx = optional_of(saved[1]), nnz = optional_of(saved[2]);
    // linear: the gradient's own gradient is the same operator
    out[0] = at::GradMode::is_enabled() ? DropoutFn::apply(grads[0], rng, idx, nnz, p, n[0], n[1], n[2], n[3], n[4])
                                        : run_dropout(grads[0], p, rng, n[0], n[1], {idx, nnz, n[2], n[3], n[4]});
    return out;
  }
};

Tensor dropout(const Tensor& x, double p, const OptTensor& rng, int64_t seed, int64_t call, const OptTensor& idx,
               const OptTensor& nnz, int64_t BH, int64_t BW, int64_t stride) {
  check_cuda(x);
  dtype_code(x);
  rng_pointer(rng, x);
  return DropoutFn::apply(x, rng, idx, nnz, p, seed, call, BH, BW, stride);
}

// ---- rotary positions ---------------------------------------------------------------------------------------------
struct RotaryPlan {
  int64_t dim, rotary_dim;
  bool interleaved;
  double magnitude;
};

// (..., N, E) as [batch, heads, n, dim] with strides, next to its positions; `x` may be replaced by what the record reads
sparta_rotary_tensor rotary_record(Tensor& x, const Tensor& y, const OptTensor& positions) {
  if (x.dim() > 4) x = x.flatten(0, -3);
  if (x.stride(-1) != 1) x = x.contiguous();
  sparta_rotary_tensor t = {};
  const int64_t n = x.size(-2);
  const int64_t rows = positions && positions->dim() == 2 ? positions->size(0) : 1;
  TORCH_CHECK_VALUE(!positions || positions->size(-1) == n, positions ? positions->size(-1) : 0, " positions for ", n, " tokens");
  int64_t batch = 1, heads = 1;
  if (x.dim() == 4) {
    batch = x.size(0);
    heads = x.size(1);
    TORCH_CHECK_VALUE(rows == 1 || rows == batch, "positions of ", rows, " sequences for a batch of ", batch);
    t.stride_batch = x.stride(0);
    t.stride_head = x.stride(1);
  } else if (x.dim() == 3) {
    TORCH_CHECK_VALUE(x.size(0) % rows == 0, "positions of ", rows, " sequences for ", x.size(0), " heads");
    batch = rows;
    heads = x.size(0) / rows;
    t.stride_batch = heads * x.stride(0);
    t.stride_head = x.stride(0);
  } else {
    TORCH_CHECK_VALUE(rows == 1, "positions of ", rows, " sequences for one");
  }
  TORCH_CHECK_VALUE(batch <= INT_MAX && heads <= INT_MAX && n <= INT_MAX, "rotary: a dimension beyond 31 bits");
  t.stride_token = x.stride(-2);
  t.batch = (int32_t)batch;
  t.heads = (int32_t)heads;
  t.n = (int32_t)n;
  t.x = x.const_data_ptr();
  t.y = y.data_ptr();
  t.positions = positions ? positions->const_data_ptr() : nullptr;
  t.positions_per_batch = rows > 1;
  return t;
}

variable_list run_rotary(const variable_list& inputs, const std::array<OptTensor, 2>& positions, const Tensor& turns,
                         const RotaryPlan& plan, bool backward) {
  variable_list held, outs;
  sparta_rotary_tensor records[2];
  int count = 0;
  bool wide = false;
  for (size_t k = 0; k < inputs.size(); ++k) {
    Tensor x = inputs[k];
    outs.push_back(at::empty(x.sizes(), x.options()));
    if (x.numel() == 0) continue;
    records[count++] = rotary_record(x, outs.back(), positions[k]);
    held.push_back(x);
    if (positions[k]) wide = positions[k]->scalar_type() == at::kLong;
  }
  if (count > 0) {
    const Tensor& x = held[0];
    const c10::cuda::CUDAGuard guard(x.device());
    check_status(sparta_rotary(records, count, reinterpret_cast<const uint64_t*>(turns.const_data_ptr<int64_t>()), (int)plan.dim,
                               (int)plan.rotary_dim, plan.interleaved, (float)plan.magnitude, backward, wide, dtype_code(x),
                               stream_of(x)), "sparta_rotary");
  }
  return outs;
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& query, const OptTensor& key, const OptTensor& query_positions,
                               const OptTensor& key_positions, const Tensor& turns, int64_t dim, int64_t rotary_dim,
                               bool interleaved, double magnitude, bool backward) {
    ctx->save_for_backward({tensor_of(query_positions), tensor_of(key_positions), turns});
    ctx->saved_data["n"] = std::vector<int64_t>{dim, rotary_dim, interleaved, backward};
    ctx->saved_data["m"] = magnitude;
    ctx->set_materialize_grads(false);
    variable_list in{query};
    if (key) in.push_back(*key);
    return run_rotary(in, {query_positions, key_positions}, turns, {dim, rotary_dim, interleaved, magnitude}, backward);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(10);
    const auto saved = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    const RotaryPlan plan{n[0], n[1], n[2] != 0, ctx->saved_data["m"].toDouble()};
    variable_list in;
    std::array<OptTensor, 2> positions;
    std::array<size_t, 2> at{};
    for (size_t k = 0; k < grads.size(); ++k)
      if (grads[k].defined() && ctx->needs_input_grad(k)) {
        at[in.size()] = k;
        positions[in.size()] = optional_of(saved[k]);
        in.push_back(grads[k]);
      }
    if (in.empty()) return out;
    const bool reverse = n[3] == 0;
    // linear: the gradient's own gradient is the same operator
    const variable_list turned =
        at::GradMode::is_enabled()
            ? RotaryFn::apply(in[0], in.size() > 1 ? OptTensor(in[1]) : std::nullopt, positions[0], positions[1], saved[2], plan.dim,
                              plan.rotary_dim, plan.interleaved, plan.magnitude, reverse)
            : run_rotary(in, positions, saved[2], plan, reverse);
    for (size_t k = 0; k < in.size(); ++k) out[at[k]] = turned[k];
    return out;
  }
};

void check_rotary(const Tensor& x, const OptTensor& positions, const Tensor& first, int64_t dim) {
  check_cuda(x);
  dtype_code(x);
  TORCH_CHECK_VALUE(x.dim() >= 2 && x.size(-1) == dim, "expected (..., N, ", dim, "), got ", x.sizes());
  TORCH_CHECK_VALUE(x.scalar_type() == first.scalar_type() && x.device() == first.device(),
                    "queries and keys have to be of one type on one device");
  if (!positions) return;
  TORCH_CHECK_VALUE((positions->scalar_type() == at::kInt || positions->scalar_type() == at::kLong) &&
                        (positions->dim() == 1 || positions->dim() == 2),
                    "positions have to be int32 or int64, (N,) or (B, N)");
  TORCH_CHECK_VALUE(positions->device() == x.device(), "positions are on ", positions->device(), ", the input on ", x.device());
}

variable_list rotary(const Tensor& query, const OptTensor& key, OptTensor positions, OptTensor key_positions, const Tensor& turns,
                     int64_t dim, int64_t rotary_dim, bool interleaved, double magnitude) {
  check_rotary(query, positions, query, dim);
  if (key) {
    if (!key_positions) key_positions = positions;
    check_rotary(*key, key_positions, query, dim);
    if (positions && key_positions && positions->scalar_type() != key_positions->scalar_type()) {
      positions = positions->to(at::kLong);
      key_positions = key_positions->to(at::kLong);
    }
    if (key_positions) key_positions = key_positions->contiguous();
  }
  if (positions) positions = positions->contiguous();
  return RotaryFn::apply(query, key, positions, key ? key_positions : std::nullopt, turns, dim, rotary_dim, interleaved, magnitude,
                         false);
}

// ---- fused sparse attention ---------------------------------------------------------------------------------------
constexpr int64_t kBlock = 64;

// (..., n, E) as the contiguous, 16-byte aligned (heads, n, E) that the kernels read
Tensor attention_rows(const Tensor& x, int64_t n) {
  Tensor y = x.reshape({-1, n, x.size(-1)}).contiguous();
  return reinterpret_cast<uintptr_t>(y.const_data_ptr()) % 16 == 0 ? y : y.clone();
}

struct AttentionCall {
  double p, scale;
  int64_t seed, call, nnz, Nt, Ns;
  bool check;  // read the kernels' status words after every launch
};

sparta_attn_train_args attention_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lse,
                                      const Tensor& row_ptr, const Tensor& bcsr, const OptTensor& mask, const Tensor& status,
                                      const OptTensor& rng, const AttentionCall& c) {
  sparta_attn_train_args a = {};
  a.Q = q.const_data_ptr();
  a.K = k.const_data_ptr();
  a.V = v.const_data_ptr();
  a.O = out.data_ptr();
  a.lse = lse.defined() ? lse.data_ptr<float>() : nullptr;
  a.row_ptr = row_ptr.const_data_ptr<int32_t>();
  a.bcsr_idx = bcsr.const_data_ptr<int32_t>();
  a.mask = mask ? mask->const_data_ptr<uint8_t>() : nullptr;
  a.rng = rng_pointer(rng, q);
  a.seed = (uint64_t)c.seed;
  a.call = (uint64_t)c.call;
  a.nnz_hint = c.nnz;
  a.status = status.data_ptr<int32_t>();
  a.dropout = c.p;
  a.scale = (float)c.scale;
  a.heads = (int32_t)q.size(0);
  a.kv_heads = (int32_t)k.size(0);
  a.Nt = (int32_t)c.Nt;
  a.Ns = (int32_t)c.Ns;
  a.D = (int32_t)q.size(2);
  a.BLK = kBlock;
  a.dtype = dtype_code(q);
  return a;
}
void check_words(const Tensor& status, const AttentionCall& c) {
  if (c.check)
    TORCH_CHECK(!status.any().item<bool>(), "fused sparse attention: a bounded wait ran out on the device; the output is invalid");
}

void run_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lse, const Tensor& row_ptr,
                   const Tensor& bcsr, const OptTensor& mask, const Tensor& status, const OptTensor& rng, const AttentionCall& c) {
  if (out.numel() == 0) return;
  const c10::cuda::CUDAGuard guard(q.device());
  const sparta_attn_train_args a = attention_args(q, k, v, out, lse, row_ptr, bcsr, mask, status, rng, c);
  check_status(sparta_attn_train_fwd(&a, stream_of(q)), "sparta_attn_train_fwd");
  check_words(status, c);
}

struct AttentionFn : torch::autograd::Function<AttentionFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& row_ptr,
                        const Tensor& bcsr, const OptTensor& mask, const Tensor& status, const OptTensor& rng, double p, double scale,
                        std::vector<int64_t> n) {
    const AttentionCall c{p, scale, n[0], n[1], n[2], n[3], n[4], n[5] != 0};
    const Tensor q = attention_rows(query, c.Nt), k = attention_rows(key, c.Ns), v = attention_rows(value, c.Ns);
    Tensor out = at::empty(query.sizes(), query.options());
    Tensor lse = at::empty({q.size(0), c.Nt}, query.options().dtype(at::kFloat));
    run_attention(q, k, v, out, lse, row_ptr, bcsr, mask, status, rng, c);
    // an element mask and the random numbers are read again: autograd refuses if they were rewritten in place since
    ctx->save_for_backward({q, k, v, out, lse, row_ptr, bcsr, tensor_of(mask), status, tensor_of(rng)});
    ctx->saved_data["p"] = p;
    ctx->saved_data["s"] = scale;
    ctx->saved_data["n"] = std::move(n);
    ctx->saved_data["k"] = key.sizes().vec();
    ctx->saved_data["v"] = value.sizes().vec();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(11);
    const bool want_q = ctx->needs_input_grad(0), want_k = ctx->needs_input_grad(1), want_v = ctx->needs_input_grad(2);
    const auto s = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    const AttentionCall c{ctx->saved_data["p"].toDouble(), ctx->saved_data["s"].toDouble(), n[0], n[1], n[2], n[3], n[4], n[5] != 0};
    const Tensor &q = s[0], &k = s[1], &v = s[2], &out = s[3];
    if (!grads[0].defined() || !(want_q || want_k || want_v)) return result;
    {
      const at::NoGradGuard no_grad;
      const Tensor grad = attention_rows(grads[0], c.Nt);
      const Tensor dq = want_q ? at::empty(out.sizes(), q.options()) : Tensor();
      const Tensor dk = want_k || want_v ? at::empty(ctx->saved_data["k"].toIntVector(), k.options()) : Tensor();
      const Tensor dv = want_k || want_v ? at::empty(ctx->saved_data["v"].toIntVector(), v.options()) : Tensor();
      if (q.numel() > 0) {
        const c10::cuda::CUDAGuard guard(q.device());
        sparta_attn_train_args a = attention_args(q, k, v, out, s[4], s[5], s[6], optional_of(s[7]), s[8], optional_of(s[9]), c);
        size_t bytes = sparta_attn_train_bwd_workspace_bytes(a.heads, a.kv_heads, a.Nt, a.Ns, a.D, a.nnz_hint);
        if (c.p > 0) bytes += sparta_attn_train_bwd_dropout_bytes(a.heads, a.nnz_hint);
        const Tensor workspace = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
        a.dO = grad.const_data_ptr();
        a.dQ = want_q ? dq.data_ptr() : nullptr;
        a.dK = dk.defined() ? dk.data_ptr() : nullptr;
        a.dV = dv.defined() ? dv.data_ptr() : nullptr;
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = bytes;
        check_status(sparta_attn_train_bwd(&a, stream_of(q)), "sparta_attn_train_bwd");
        check_words(s[8], c);
      }
      result[0] = dq;
      if (want_k) result[1] = dk;
      if (want_v) result[2] = dv;
    }
    if (at::GradMode::is_enabled()) {  // a second derivative is refused where it is asked for
      auto refuse = std::make_shared<torch::autograd::DelayedError>("the fused sparse attention cannot be differentiated twice",
                                                                    (int64_t)result.size());
      variable_list in;
      for (Tensor& g : result) {
        if (g.defined()) g = g.detach().requires_grad_();
        in.push_back(g);
      }
      result = (*refuse)(std::move(in));
    }
    return result;
  }
};

void check_attention(const Tensor& x, const Tensor& query, int64_t n, int64_t dim, const char* name) {
  check_cuda(x);
  TORCH_CHECK_VALUE(x.dim() >= 2 && x.size(-2) == n && x.size(-1) == dim, "expect ", name, " shape (?, ", n, ", ", dim, "), got ",
                    x.sizes());
  TORCH_CHECK_TYPE(x.scalar_type() == query.scalar_type() && x.device() == query.device(),
                   "query, key and value have to be of one type on one device");
}

Tensor attention(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& row_ptr, const Tensor& bcsr,
                 const OptTensor& mask, const Tensor& status, const OptTensor& rng, double p, double scale, int64_t seed, int64_t call,
                 int64_t nnz, int64_t Nt, int64_t Ns, int64_t dim, bool check) {
  check_attention(query, query, Nt, dim, "query");
  check_attention(key, query, Ns, dim, "key");
  check_attention(value, query, Ns, dim, "value");
  const int64_t q_heads = query.numel() / (Nt * dim), k_heads = key.numel() / (Ns * dim), v_heads = value.numel() / (Ns * dim);
  TORCH_CHECK_VALUE(k_heads == v_heads && k_heads > 0 && q_heads % k_heads == 0, q_heads, " query heads cannot share ", k_heads,
                    " key and ", v_heads, " value heads");
  TORCH_CHECK_VALUE(q_heads <= INT_MAX && Nt <= INT_MAX && Ns <= INT_MAX, "attention: a dimension beyond 31 bits");
  TORCH_CHECK_VALUE(row_ptr.device() == query.device(), "the mask is on ", row_ptr.device(), ", the inputs on ", query.device());
  rng_pointer(rng, query);
  if (at::GradMode::is_enabled() && (query.requires_grad() || key.requires_grad() || value.requires_grad()))
    return AttentionFn::apply(query, key, value, row_ptr, bcsr, mask, status, rng, p, scale,
                              std::vector<int64_t>{seed, call, nnz, Nt, Ns, check});
  const at::NoGradGuard no_grad;  // nothing to differentiate: no row sums are kept
  const Tensor out = at::empty(query.sizes(), query.options());
  run_attention(attention_rows(query, Nt), attention_rows(key, Ns), attention_rows(value, Ns), out, Tensor(), row_ptr, bcsr, mask,
                status, rng, {p, scale, seed, call, nnz, Nt, Ns, check});
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("dropout", &dropout);
  m.def("rotary", &rotary);
  m.def("attention", &attention);
}
