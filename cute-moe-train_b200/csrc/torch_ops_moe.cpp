// torch.library registration of the MoE block's operators (router, permutation, block-scaled e4m3) in the
// `grouped_mm` namespace, over the C ABI in moe_gemm.h.  The router and the permutation carry their
// autograd here rather than in Python: their kernels take a few microseconds, which a Python autograd
// function would double or triple.  Shape inference for fake tensors is registered from Python.
// Every launch goes on the current CUDA stream of the inputs' device; nothing here synchronises.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "moe_gemm.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using torch::autograd::Variable;

void check_launch(int rc, const char* what) {
  TORCH_CHECK(rc == MGF_OK, what, ": ", mgf_status_string(rc), " (status ", rc, ") ", mgf_last_error_detail());
}

void* stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int32_t dtype_code(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return MGF_DT_BF16;
    case at::kHalf: return MGF_DT_F16;
    case at::kFloat: return MGF_DT_F32;
    default: TORCH_CHECK(false, what, ": expected bfloat16, float16 or float32, got ", t.scalar_type());
  }
  return -1;
}

int64_t round_up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// A [rows, cols] output whose row stride is padded to 16 bytes, as the grouped products take it.
Tensor padded_rows(int64_t rows, int64_t cols, const at::TensorOptions& o) {
  return at::empty_strided({rows, cols}, {round_up(cols, 16 / static_cast<int64_t>(o.dtype().itemsize())), 1}, o);
}

// Row stride of a matrix; a matrix of one row (or none) may carry any.
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.stride(0), t.size(1)); }

void check_matrix(const Tensor& t, const char* what, const char* name) {
  TORCH_CHECK(t.is_cuda(), what, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == 2, what, ": ", name, " must be 2D, got ", t.dim(), "D");
  if (t.numel() == 0) return;
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, what, ": ", name, " must have unit stride along its last dimension");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), what, ": ", name, " must be row-major");
}

// ---------------------------------------------------------------- router
int32_t check_route(const Tensor& logits, int64_t topk, int64_t score) {
  check_matrix(logits, "moe_route", "logits");
  const int64_t E = logits.size(1);
  TORCH_CHECK(E >= 1 && E <= 1024, "moe_route: the number of experts must be in [1, 1024], got ", E);
  TORCH_CHECK(topk >= 1 && topk <= std::min<int64_t>(E, 32), "moe_route: topk must be in [1, min(E, 32)], got ", topk);
  const int64_t kind = score & ~int64_t{MGF_ROUTE_BIAS_ON_SCORE};
  TORCH_CHECK(kind == MGF_ROUTE_SOFTMAX || kind == MGF_ROUTE_SIGMOID, "moe_route: unknown score");
  return dtype_code(logits, "moe_route");
}

std::tuple<Tensor, Tensor> moe_route_cuda(const Tensor& logits, int64_t topk, int64_t score, bool renormalize,
                                          double scale, const std::optional<Tensor>& bias,
                                          const std::optional<Tensor>& token_mask) {
  const int32_t dt = check_route(logits, topk, score);
  const int64_t T = logits.size(0), E = logits.size(1);
  if (bias.has_value())
    TORCH_CHECK(bias->device() == logits.device() && bias->scalar_type() == at::kFloat && bias->dim() == 1 &&
                    bias->size(0) == E && bias->is_contiguous(),
                "moe_route: bias must be a contiguous float32 [E] tensor on the logits' device");
  if (token_mask.has_value())
    TORCH_CHECK(token_mask->device() == logits.device() && token_mask->scalar_type() == at::kBool &&
                    token_mask->dim() == 1 && token_mask->size(0) == T && token_mask->is_contiguous(),
                "moe_route: token_mask must be a contiguous bool [tokens] tensor on the logits' device");
  const c10::cuda::CUDAGuard guard(logits.device());
  Tensor weights = at::empty({T, topk}, logits.options().dtype(at::kFloat));
  Tensor idx = at::empty({T, topk}, logits.options().dtype(at::kLong));
  check_launch(mgf_moe_route(logits.data_ptr(), dt, row_stride(logits), T, static_cast<int32_t>(E),
                             static_cast<int32_t>(topk), static_cast<int32_t>(score), renormalize ? 1 : 0,
                             static_cast<float>(scale), bias.has_value() ? bias->data_ptr<float>() : nullptr,
                             token_mask.has_value() ? reinterpret_cast<const uint8_t*>(token_mask->data_ptr<bool>())
                                                    : nullptr,
                             weights.data_ptr<float>(), idx.data_ptr<int64_t>(), stream()),
               "moe_route");
  return {weights, idx};
}

Tensor moe_route_bwd_cuda(const Tensor& logits, const Tensor& idx, const Tensor& grad_weights, int64_t score,
                          bool renormalize, double scale) {
  TORCH_CHECK(idx.dim() == 2 && grad_weights.dim() == 2 && idx.sizes() == grad_weights.sizes() &&
                  idx.size(0) == logits.size(0) && idx.scalar_type() == at::kLong && idx.is_contiguous() &&
                  grad_weights.scalar_type() == at::kFloat && grad_weights.is_contiguous() &&
                  idx.device() == logits.device() && grad_weights.device() == logits.device(),
              "moe_route_bwd: expert_idx int64 and grad_weights float32, contiguous [tokens, topk]");
  const int32_t dt = check_route(logits, idx.size(1), score);
  const c10::cuda::CUDAGuard guard(logits.device());
  Tensor grad = at::empty(logits.sizes(), logits.options());
  check_launch(mgf_moe_route_bwd(logits.data_ptr(), dt, row_stride(logits), logits.size(0),
                                 static_cast<int32_t>(logits.size(1)), static_cast<int32_t>(idx.size(1)),
                                 static_cast<int32_t>(score), renormalize ? 1 : 0, static_cast<float>(scale),
                                 idx.data_ptr<int64_t>(), grad_weights.data_ptr<float>(), grad.data_ptr(),
                                 grad.size(1), stream()),
               "moe_route_bwd");
  return grad;
}

// ---------------------------------------------------------------- permutation
constexpr int64_t kMaxCopies = INT32_MAX;

void check_experts(int64_t num_experts) {
  TORCH_CHECK(num_experts >= 1 && num_experts <= 1024, "moe_sort: the number of experts must be in [1, 1024], got ",
              num_experts);
}

void check_ids(const Tensor& expert_idx, int64_t num_experts) {
  TORCH_CHECK(expert_idx.is_cuda() && expert_idx.scalar_type() == at::kLong && expert_idx.dim() == 2 &&
                  expert_idx.size(1) >= 1 && expert_idx.is_contiguous(),
              "moe_sort: expert_idx must be a contiguous int64 [tokens, topk] CUDA tensor");
  check_experts(num_experts);
  TORCH_CHECK(expert_idx.numel() <= kMaxCopies, "moe_sort: too many copies, ", expert_idx.numel());
}

struct Plan {
  Tensor offs, row_of_copy, copy_of_row, workspace;
  int32_t* scratch = nullptr;
};

Plan empty_plan(const Tensor& expert_idx, int64_t num_experts) {
  const auto o = expert_idx.options().dtype(at::kInt);
  const int64_t n = expert_idx.numel(), words = mgf_moe_sort_workspace_words(n, static_cast<int32_t>(num_experts));
  Plan p{at::empty({num_experts}, o), at::empty(expert_idx.sizes(), o), at::empty({n}, o), Tensor()};
  if (words > 0) {
    p.workspace = at::empty({words}, o);
    p.scratch = p.workspace.data_ptr<int32_t>();
  }
  return p;
}

std::tuple<Tensor, Tensor, Tensor> moe_sort_cuda(const Tensor& expert_idx, int64_t num_experts) {
  check_ids(expert_idx, num_experts);
  const c10::cuda::CUDAGuard guard(expert_idx.device());
  Plan p = empty_plan(expert_idx, num_experts);
  check_launch(mgf_moe_sort(expert_idx.data_ptr<int64_t>(), expert_idx.numel(), static_cast<int32_t>(num_experts),
                            p.offs.data_ptr<int32_t>(), p.row_of_copy.data_ptr<int32_t>(),
                            p.copy_of_row.data_ptr<int32_t>(), p.scratch, stream()),
               "moe_sort");
  return {p.offs, p.row_of_copy, p.copy_of_row};
}

void check_plan(const Tensor& offs, const Tensor& row_of_copy, const Tensor& like, const char* what) {
  TORCH_CHECK(offs.device() == like.device() && row_of_copy.device() == like.device(), what,
              ": the plan must be on the tensors' device");
  TORCH_CHECK(offs.scalar_type() == at::kInt && offs.dim() == 1 && offs.numel() >= 1 && offs.is_contiguous(), what,
              ": offs must be a contiguous int32 [E] tensor");
  TORCH_CHECK(row_of_copy.scalar_type() == at::kInt && row_of_copy.dim() == 2 && row_of_copy.size(1) >= 1 &&
                  row_of_copy.is_contiguous() && row_of_copy.numel() <= kMaxCopies,
              what, ": row_of_copy must be a contiguous int32 [tokens, topk] tensor");
}

const int32_t* offs_end(const Tensor& offs) { return offs.data_ptr<int32_t>() + offs.numel() - 1; }

Tensor permute_rows_cuda(const Tensor& x, const Tensor& offs, const Tensor& row_of_copy) {
  check_matrix(x, "moe_permute", "x");
  const int32_t dt = dtype_code(x, "moe_permute");
  check_plan(offs, row_of_copy, x, "moe_permute");
  TORCH_CHECK(row_of_copy.size(0) == x.size(0), "moe_permute: the plan is for ", row_of_copy.size(0), " tokens, x has ",
              x.size(0));
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t n = row_of_copy.numel();
  Tensor rows = padded_rows(n, x.size(1), x.options());
  check_launch(mgf_moe_permute(x.data_ptr(), dt, row_stride(x), x.size(0), static_cast<int32_t>(row_of_copy.size(1)),
                               x.size(1), row_of_copy.data_ptr<int32_t>(), offs_end(offs), rows.data_ptr(),
                               rows.stride(0), n, stream()),
               "moe_permute");
  return rows;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> moe_permute_cuda(const Tensor& x, const Tensor& expert_idx,
                                                            int64_t num_experts) {
  check_matrix(x, "moe_permute", "x");
  TORCH_CHECK(expert_idx.device() == x.device(), "moe_permute: expert_idx must be on x's device");
  TORCH_CHECK(expert_idx.dim() == 2 && expert_idx.size(0) == x.size(0),
              "moe_permute: expert_idx must be [tokens, topk] for the tokens of x");
  const int32_t dt = dtype_code(x, "moe_permute");
  check_ids(expert_idx, num_experts);
  const c10::cuda::CUDAGuard guard(x.device());
  Plan p = empty_plan(expert_idx, num_experts);
  Tensor rows = padded_rows(expert_idx.numel(), x.size(1), x.options());
  check_launch(mgf_moe_sort_permute(expert_idx.data_ptr<int64_t>(), static_cast<int32_t>(num_experts), x.data_ptr(), dt,
                                    row_stride(x), x.size(0), static_cast<int32_t>(expert_idx.size(1)), x.size(1),
                                    p.offs.data_ptr<int32_t>(), p.row_of_copy.data_ptr<int32_t>(),
                                    p.copy_of_row.data_ptr<int32_t>(), rows.data_ptr(), rows.stride(0), p.scratch,
                                    stream()),
               "moe_permute");
  return {rows, p.offs, p.row_of_copy, p.copy_of_row};
}

void check_weights(const std::optional<Tensor>& weights, const Tensor& row_of_copy) {
  if (weights.has_value())
    TORCH_CHECK(weights->device() == row_of_copy.device() && weights->scalar_type() == at::kFloat &&
                    weights->sizes() == row_of_copy.sizes() && weights->is_contiguous(),
                "moe_unpermute: weights must be a contiguous float32 [tokens, topk] tensor on the rows' device");
}

Tensor moe_unpermute_cuda(const Tensor& rows, const Tensor& offs, const Tensor& row_of_copy,
                          const std::optional<Tensor>& weights) {
  check_matrix(rows, "moe_unpermute", "rows");
  const int32_t dt = dtype_code(rows, "moe_unpermute");
  check_plan(offs, row_of_copy, rows, "moe_unpermute");
  check_weights(weights, row_of_copy);
  const int64_t T = row_of_copy.size(0);
  const c10::cuda::CUDAGuard guard(rows.device());
  Tensor out = padded_rows(T, rows.size(1), rows.options());
  check_launch(mgf_moe_unpermute(rows.data_ptr(), dt, row_stride(rows), rows.size(0), T,
                                 static_cast<int32_t>(row_of_copy.size(1)), rows.size(1),
                                 row_of_copy.data_ptr<int32_t>(),
                                 weights.has_value() ? weights->data_ptr<float>() : nullptr, out.data_ptr(),
                                 out.stride(0), stream()),
               "moe_unpermute");
  return out;
}

// Gradients of moe_unpermute: (rows, weights); the one that is not wanted comes back empty.
std::tuple<Tensor, Tensor> moe_unpermute_bwd_cuda(const Tensor& grad_out, const Tensor& rows, const Tensor& offs,
                                                  const Tensor& row_of_copy, const std::optional<Tensor>& weights,
                                                  bool need_rows, bool need_weights) {
  check_matrix(grad_out, "moe_unpermute_bwd", "grad_out");
  check_matrix(rows, "moe_unpermute_bwd", "rows");
  check_plan(offs, row_of_copy, rows, "moe_unpermute_bwd");
  check_weights(weights, row_of_copy);
  TORCH_CHECK(grad_out.device() == rows.device() && grad_out.scalar_type() == rows.scalar_type() &&
                  grad_out.size(0) == row_of_copy.size(0) && grad_out.size(1) == rows.size(1),
              "moe_unpermute_bwd: grad_out must be [tokens, hidden] of the rows' type");
  const int32_t dt = dtype_code(rows, "moe_unpermute_bwd");
  const c10::cuda::CUDAGuard guard(rows.device());
  Tensor grad_rows = need_rows ? padded_rows(rows.size(0), rows.size(1), rows.options()) : at::empty({0}, rows.options());
  const auto fo = rows.options().dtype(at::kFloat);
  Tensor grad_weights = need_weights ? at::empty(row_of_copy.sizes(), fo) : at::empty({0}, fo);
  check_launch(
      mgf_moe_unpermute_bwd(grad_out.data_ptr(), row_stride(grad_out), rows.data_ptr(), row_stride(rows), dt,
                            rows.size(0), row_of_copy.size(0), static_cast<int32_t>(row_of_copy.size(1)), rows.size(1),
                            row_of_copy.data_ptr<int32_t>(), offs_end(offs),
                            weights.has_value() ? weights->data_ptr<float>() : nullptr,
                            need_rows ? grad_rows.data_ptr() : nullptr, need_rows ? grad_rows.stride(0) : 0,
                            need_weights ? grad_weights.data_ptr<float>() : nullptr, stream()),
      "moe_unpermute_bwd");
  return {grad_rows, grad_weights};
}

// ---------------------------------------------------------------- block-scaled e4m3
constexpr int64_t kBlock = 128;
int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

void check_bf16_matrix(const Tensor& x, const char* what) {
  check_matrix(x, what, "x");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, what, ": x must be BFloat16, got ", x.scalar_type());
}

std::tuple<Tensor, Tensor> block_outputs(int64_t rows, int64_t cols, const Tensor& like) {
  return {padded_rows(rows, cols, like.options().dtype(at::kFloat8_e4m3fn)),
          padded_rows(rows, blocks_of(cols), like.options().dtype(at::kFloat))};
}

std::tuple<Tensor, Tensor> quantize_rows_block_cuda(const Tensor& x) {
  check_bf16_matrix(x, "fp8_quantize_rows_block");
  const c10::cuda::CUDAGuard guard(x.device());
  auto [q, scale] = block_outputs(x.size(0), x.size(1), x);
  check_launch(mgf_fp8_block_quantize_rows(x.data_ptr(), row_stride(x), x.size(0), x.size(1), 1, nullptr, nullptr,
                                           q.data_ptr(), q.stride(0), scale.data_ptr<float>(), scale.stride(0),
                                           x.size(0), stream()),
               "fp8_quantize_rows_block");
  return {q, scale};
}

std::tuple<Tensor, Tensor> permute_rows_fp8_cuda(const Tensor& x, const Tensor& offs, const Tensor& row_of_copy) {
  check_bf16_matrix(x, "moe_permute_fp8");
  check_plan(offs, row_of_copy, x, "moe_permute_fp8");
  TORCH_CHECK(row_of_copy.size(0) == x.size(0), "moe_permute_fp8: the plan is for ", row_of_copy.size(0),
              " tokens, x has ", x.size(0));
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t n = row_of_copy.numel();
  auto [q, scale] = block_outputs(n, x.size(1), x);
  check_launch(mgf_fp8_block_quantize_rows(x.data_ptr(), row_stride(x), x.size(0), x.size(1),
                                           static_cast<int32_t>(row_of_copy.size(1)), row_of_copy.data_ptr<int32_t>(),
                                           offs_end(offs), q.data_ptr(), q.stride(0), scale.data_ptr<float>(),
                                           scale.stride(0), n, stream()),
               "moe_permute_fp8");
  return {q, scale};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> moe_permute_fp8_cuda(const Tensor& x, const Tensor& expert_idx,
                                                                        int64_t num_experts) {
  check_bf16_matrix(x, "moe_permute_fp8");
  TORCH_CHECK(expert_idx.device() == x.device(), "moe_permute_fp8: expert_idx must be on x's device");
  TORCH_CHECK(expert_idx.dim() == 2 && expert_idx.size(0) == x.size(0),
              "moe_permute_fp8: expert_idx must be [tokens, topk] for the tokens of x");
  auto [offs, row_of_copy, copy_of_row] = moe_sort_cuda(expert_idx, num_experts);
  auto [q, scale] = permute_rows_fp8_cuda(x, offs, row_of_copy);
  return {q, scale, offs, row_of_copy, copy_of_row};
}

// w [E, K, N] with unit stride along N or along K; the codes keep that layout, rows padded to 16 bytes.
std::tuple<Tensor, Tensor> quantize_weights_block_cuda(const Tensor& w) {
  TORCH_CHECK(w.is_cuda() && w.dim() == 3 && w.scalar_type() == at::kBFloat16,
              "fp8_quantize_weights_block: w must be a bf16 [E, K, N] CUDA tensor");
  const bool along_n = w.stride(2) == 1 || w.size(2) <= 1;
  TORCH_CHECK(along_n || w.stride(1) == 1 || w.size(1) <= 1,
              "fp8_quantize_weights_block: w must have unit stride along K or N");
  const c10::cuda::CUDAGuard guard(w.device());
  const Tensor src = along_n ? w : w.transpose(1, 2);
  const int64_t E = src.size(0), R = src.size(1), C = src.size(2), pitch = round_up(C, 16);
  Tensor q = at::empty_strided({E, R, C}, {R * pitch, pitch, 1}, w.options().dtype(at::kFloat8_e4m3fn));
  Tensor scale = at::empty({E, blocks_of(R), blocks_of(C)}, w.options().dtype(at::kFloat));
  check_launch(mgf_fp8_block_quantize_weights(src.data_ptr(), E, R, C, src.stride(0), src.stride(1), q.data_ptr(),
                                              q.stride(0), q.stride(1), scale.data_ptr<float>(), scale.stride(0),
                                              scale.stride(1), scale.stride(2), stream()),
               "fp8_quantize_weights_block");
  if (along_n) return {q, scale};
  return {q.transpose(1, 2), scale.transpose(1, 2)};
}

// ---------------------------------------------------------------- grouped product of block-scaled operands
// Stride of dimension i; a dimension of one element may carry any.
int64_t stride_of(const Tensor& t, int i, int64_t otherwise) { return t.size(i) > 1 ? t.stride(i) : otherwise; }

struct BlockArgs {
  mgf_block_gemm_desc g{};
  int64_t rows, n;
};

BlockArgs block_args(const Tensor& a, const Tensor& b, const Tensor& offs, const Tensor& scale_a, const Tensor& scale_b,
                     const std::optional<Tensor>& bias, const char* what) {
  TORCH_CHECK(a.is_cuda() && b.is_cuda(), what, ": inputs must be CUDA tensors");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 3, what, ": mat_a must be 2D and mat_b 3D");
  TORCH_CHECK(a.scalar_type() == at::kFloat8_e4m3fn && b.scalar_type() == at::kFloat8_e4m3fn, what,
              ": mat_a and mat_b must be float8_e4m3fn");
  const int64_t M = a.size(0), K = a.size(1), E = b.size(0), N = b.size(2);
  TORCH_CHECK(b.size(1) == K, what, ": contraction dimension of mat_a and mat_b must match");
  TORCH_CHECK(K >= 1 && N >= 1 && N % 8 == 0, what, ": N must be a positive multiple of 8 and K positive, got N=", N,
              ", K=", K);
  TORCH_CHECK(offs.scalar_type() == at::kInt && offs.dim() == 1 && offs.is_contiguous() && offs.size(0) == E, what,
              ": offs must be a contiguous int32 [E] tensor");
  TORCH_CHECK(E >= 1 && E <= 1024, what, ": group count must be in [1, 1024], got ", E);
  for (const Tensor* t : {&b, &offs, &scale_a, &scale_b})
    TORCH_CHECK(t->device() == a.device(), what, ": all tensors must be on the same device");
  TORCH_CHECK((K == 1 || a.stride(1) == 1) && (M <= 1 || a.stride(0) >= K), what, ": mat_a must be row-major");
  const bool mn = N == 1 || b.stride(2) == 1;
  TORCH_CHECK(mn || K == 1 || b.stride(1) == 1, what, ": mat_b must have unit stride along N or K");
  TORCH_CHECK(scale_a.scalar_type() == at::kFloat && scale_a.dim() == 2 && scale_a.size(0) == M &&
                  scale_a.size(1) == blocks_of(K) && (scale_a.size(1) == 1 || scale_a.stride(1) == 1),
              what, ": scale_a must be float32 [M, ceil(K / 128)] with unit stride along the blocks");
  TORCH_CHECK(scale_b.scalar_type() == at::kFloat && scale_b.dim() == 3 && scale_b.size(0) == E &&
                  scale_b.size(1) == blocks_of(K) && scale_b.size(2) == blocks_of(N),
              what, ": scale_b must be float32 [E, ceil(K / 128), ceil(N / 128)]");
  if (bias.has_value())
    TORCH_CHECK(bias->device() == a.device() && bias->scalar_type() == at::kBFloat16 && bias->dim() == 2 &&
                    bias->size(0) == E && bias->size(1) == N && bias->is_contiguous(),
                what, ": bias must be a contiguous BFloat16 [E, N] tensor");
  BlockArgs r;
  mgf_block_gemm_desc& g = r.g;
  r.rows = M;
  r.n = N;
  g.num_groups = static_cast<int32_t>(E);
  g.total_rows = M;
  g.n = N;
  g.k = K;
  g.a = a.data_ptr();
  g.lda = stride_of(a, 0, round_up(K, 16));
  g.b = b.data_ptr();
  g.b_mn_major = mn ? 1 : 0;
  g.ldb = mn ? stride_of(b, 1, round_up(N, 16)) : stride_of(b, 2, round_up(K, 16));
  g.ldb_batch = stride_of(b, 0, 16);
  g.offs = offs.data_ptr<int32_t>();
  g.scale_a = scale_a.data_ptr<float>();
  g.scale_a_stride = scale_a.stride(0);
  g.scale_b = scale_b.data_ptr<float>();
  g.scale_b_stride_e = scale_b.stride(0);
  g.scale_b_stride_k = scale_b.stride(1);
  g.scale_b_stride_n = scale_b.stride(2);
  if (bias.has_value()) {
    g.bias = bias->data_ptr();
    g.bias_stride = N;
  }
  const auto carve = at::globalContext()._SMCarveout_EXPERIMENTAL();
  g.sm_carveout = carve.has_value() ? static_cast<int32_t>(*carve) : 0;
  return r;
}

// The launch with its scratch, which the caching allocator takes back in stream order.
void launch_block(BlockArgs& r, const Tensor& a, const char* what) {
  Tensor ws;
  const int64_t bytes = mgf_block_gemm_workspace_bytes(&r.g);
  if (bytes > 0) {
    ws = at::empty({bytes}, a.options().dtype(at::kByte));
    r.g.workspace = ws.data_ptr();
  }
  check_launch(mgf_block_gemm_launch(&r.g, stream()), what);
}

Tensor mm_fp8_block_cuda(const Tensor& a, const Tensor& b, const Tensor& offs, const Tensor& scale_a,
                         const Tensor& scale_b, const std::optional<Tensor>& bias) {
  BlockArgs r = block_args(a, b, offs, scale_a, scale_b, bias, "grouped_mm_fp8_block");
  const c10::cuda::CUDAGuard guard(a.device());
  Tensor out = padded_rows(r.rows, r.n, a.options().dtype(at::kBFloat16));
  r.g.epilogue = MGF_EPI_BIAS;
  r.g.d = out.data_ptr();
  r.g.ldd = out.stride(0);
  launch_block(r, a, "grouped_mm_fp8_block");
  return out;
}

std::tuple<Tensor, Tensor> mm_swiglu_fp8_block_cuda(const Tensor& a, const Tensor& b, const Tensor& offs,
                                                    const Tensor& scale_a, const Tensor& scale_b, const Tensor& bias,
                                                    double alpha, double limit) {
  BlockArgs r = block_args(a, b, offs, scale_a, scale_b, bias, "grouped_mm_swiglu_fp8_block");
  TORCH_CHECK(r.n % 16 == 0, "grouped_mm_swiglu_fp8_block: 2*I must be a multiple of 16, got ", r.n);
  const c10::cuda::CUDAGuard guard(a.device());
  Tensor s = padded_rows(r.rows, r.n / 2, a.options().dtype(at::kBFloat16));
  Tensor aux = padded_rows(r.rows, r.n, a.options().dtype(at::kBFloat16));
  r.g.epilogue = MGF_EPI_SWIGLU;
  r.g.d = aux.data_ptr();
  r.g.ldd = aux.stride(0);
  r.g.d2 = s.data_ptr();
  r.g.ldd2 = s.stride(0);
  r.g.swiglu_alpha = static_cast<float>(alpha);
  r.g.swiglu_limit = static_cast<float>(limit);
  launch_block(r, a, "grouped_mm_swiglu_fp8_block");
  return {s, aux};
}

Tensor mm_swiglu_bwd_fp8_block_cuda(const Tensor& grad_output, const Tensor& down_w_t, const Tensor& offs,
                                    const Tensor& aux, const Tensor& scale_a, const Tensor& scale_b, double alpha,
                                    double limit) {
  BlockArgs r = block_args(grad_output, down_w_t, offs, scale_a, scale_b, std::nullopt, "grouped_mm_swiglu_bwd_fp8_block");
  TORCH_CHECK(aux.device() == grad_output.device() && aux.scalar_type() == at::kBFloat16 && aux.dim() == 2 &&
                  aux.size(0) == r.rows && aux.size(1) == 2 * r.n && aux.stride(1) == 1,
              "grouped_mm_swiglu_bwd_fp8_block: aux_biased_acc must be a row-major BFloat16 [M, 2*I] tensor");
  const c10::cuda::CUDAGuard guard(grad_output.device());
  Tensor out = padded_rows(r.rows, 2 * r.n, aux.options());
  r.g.epilogue = MGF_EPI_SWIGLU_BWD;
  r.g.d = out.data_ptr();
  r.g.ldd = out.stride(0);
  r.g.aux = aux.data_ptr();
  r.g.ld_aux = stride_of(aux, 0, round_up(2 * r.n, 8));
  r.g.swiglu_alpha = static_cast<float>(alpha);
  r.g.swiglu_limit = static_cast<float>(limit);
  launch_block(r, grad_output, "grouped_mm_swiglu_bwd_fp8_block");
  return out;
}

// ---------------------------------------------------------------- autograd of the router and the permutation
template <typename F>
auto op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

using RouteSig = std::tuple<Tensor, Tensor>(const Tensor&, int64_t, int64_t, bool, double, const std::optional<Tensor>&,
                                            const std::optional<Tensor>&);
using RouteBwdSig = Tensor(const Tensor&, const Tensor&, const Tensor&, int64_t, bool, double);
using PermuteSig = std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, int64_t);
using PermuteRowsSig = Tensor(const Tensor&, const Tensor&, const Tensor&);
using UnpermuteSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&);
using UnpermuteBwdSig = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                   const std::optional<Tensor>&, bool, bool);

std::tuple<Tensor, Tensor> call_route(const Tensor& logits, int64_t topk, int64_t score, bool renormalize, double scale,
                                      const std::optional<Tensor>& bias, const std::optional<Tensor>& mask) {
  static auto h = op<RouteSig>("grouped_mm::moe_route");
  return h.call(logits, topk, score, renormalize, scale, bias, mask);
}
Tensor call_route_bwd(const Tensor& logits, const Tensor& idx, const Tensor& g, int64_t score, bool renormalize,
                      double scale) {
  static auto h = op<RouteBwdSig>("grouped_mm::moe_route_bwd");
  return h.call(logits, idx, g, score, renormalize, scale);
}
std::tuple<Tensor, Tensor, Tensor, Tensor> call_permute(const Tensor& x, const Tensor& idx, int64_t E) {
  static auto h = op<PermuteSig>("grouped_mm::moe_permute");
  return h.call(x, idx, E);
}
Tensor call_permute_rows(const Tensor& x, const Tensor& offs, const Tensor& row_of_copy) {
  static auto h = op<PermuteRowsSig>("grouped_mm::moe_permute_rows");
  return h.call(x, offs, row_of_copy);
}
Tensor call_unpermute(const Tensor& rows, const Tensor& offs, const Tensor& row_of_copy,
                      const std::optional<Tensor>& weights) {
  static auto h = op<UnpermuteSig>("grouped_mm::moe_unpermute");
  return h.call(rows, offs, row_of_copy, weights);
}
std::tuple<Tensor, Tensor> call_unpermute_bwd(const Tensor& g, const Tensor& rows, const Tensor& offs,
                                              const Tensor& row_of_copy, const std::optional<Tensor>& weights,
                                              bool need_rows, bool need_weights) {
  static auto h = op<UnpermuteBwdSig>("grouped_mm::moe_unpermute_bwd");
  return h.call(g, rows, offs, row_of_copy, weights, need_rows, need_weights);
}

// Forward-mode derivatives are refused, not dropped: a dual tensor need not require grad, so it would go below autograd.
void no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what, ": forward-mode derivatives are not implemented");
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }

// A gradient as the kernels take it: unit stride along the last dimension, rows apart (a broadcast gradient of one
// column has rows of one element at stride 0).
Tensor row_major(const Tensor& g) {
  const bool dense = g.size(1) <= 1 || g.stride(1) == 1, apart = g.size(0) <= 1 || g.stride(0) >= g.size(1);
  return dense && apart ? g : g.contiguous();
}

// The backward passes are kernels without a derivative of their own: create_graph is refused, not ignored.
void once_only() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "grouped_mm: the MoE block operators cannot be differentiated twice");
}

struct Route : torch::autograd::Function<Route> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& logits, int64_t topk, int64_t score, bool renormalize,
                             double scale, const std::optional<Tensor>& bias, const std::optional<Tensor>& mask) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [weights, idx] = call_route(logits, topk, score, renormalize, scale, bias, mask);
    ctx->save_for_backward({logits, idx});
    ctx->saved_data["score"] = score;
    ctx->saved_data["renormalize"] = renormalize;
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);  // no zeros for the ids' missing gradient
    ctx->mark_non_differentiable({idx});
    return {weights, idx};
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list g) {
    once_only();
    const auto saved = ctx->get_saved_variables();
    Tensor gl;
    if (g[0].defined()) {
      at::AutoDispatchBelowADInplaceOrView below;
      gl = call_route_bwd(saved[0], saved[1], g[0].contiguous(), ctx->saved_data["score"].toInt(),
                          ctx->saved_data["renormalize"].toBool(), ctx->saved_data["scale"].toDouble());
    }
    return {gl, Variable(), Variable(), Variable(), Variable(), Variable(), Variable()};
  }
};

// The gradient of x: the sum of its copies' gradients.
Tensor permute_grad(AutogradContext* ctx, const Tensor& g) {
  once_only();
  if (!g.defined()) return Tensor();
  const auto saved = ctx->get_saved_variables();
  at::AutoDispatchBelowADInplaceOrView below;
  return call_unpermute(row_major(g), saved[0], saved[1], std::nullopt);
}

struct Permute : torch::autograd::Function<Permute> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& idx, int64_t E) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [rows, offs, row_of_copy, copy_of_row] = call_permute(x, idx, E);
    ctx->save_for_backward({offs, row_of_copy});
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({offs, row_of_copy, copy_of_row});
    return {rows, offs, row_of_copy, copy_of_row};
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list g) {
    return {permute_grad(ctx, g[0]), Variable(), Variable()};
  }
};

struct PermuteRows : torch::autograd::Function<PermuteRows> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& offs, const Tensor& row_of_copy) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({offs, row_of_copy});
    return {call_permute_rows(x, offs, row_of_copy)};
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list g) {
    return {permute_grad(ctx, g[0]), Variable(), Variable()};
  }
};

struct Unpermute : torch::autograd::Function<Unpermute> {
  static tensor_list forward(AutogradContext* ctx, const Tensor& rows, const Tensor& offs, const Tensor& row_of_copy,
                             const std::optional<Tensor>& weights) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({rows, offs, row_of_copy, weights.has_value() ? *weights : Tensor()});
    return {call_unpermute(rows, offs, row_of_copy, weights)};
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list g) {
    once_only();
    const auto saved = ctx->get_saved_variables();
    std::optional<Tensor> w;
    if (saved[3].defined()) w = saved[3];
    const bool need_rows = ctx->needs_input_grad(0), need_weights = w.has_value() && ctx->needs_input_grad(3);
    Tensor gr, gw;
    if (g[0].defined() && (need_rows || need_weights)) {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [a, b] = call_unpermute_bwd(row_major(g[0]), saved[0], saved[1], saved[2], w, need_rows, need_weights);
      if (need_rows) gr = a;
      if (need_weights) gw = b;
    }
    return {gr, Variable(), Variable(), gw};
  }
};

std::tuple<Tensor, Tensor> moe_route_autograd(const Tensor& logits, int64_t topk, int64_t score, bool renormalize,
                                              double scale, const std::optional<Tensor>& bias,
                                              const std::optional<Tensor>& mask) {
  no_tangent(logits, "moe_route");
  if (!wants_grad(logits)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_route(logits, topk, score, renormalize, scale, bias, mask);
  }
  auto r = Route::apply(logits, topk, score, renormalize, scale, bias, mask);
  return {r[0], r[1]};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> moe_permute_autograd(const Tensor& x, const Tensor& idx, int64_t E) {
  no_tangent(x, "moe_permute");
  if (!wants_grad(x)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_permute(x, idx, E);
  }
  auto r = Permute::apply(x, idx, E);
  return {r[0], r[1], r[2], r[3]};
}
Tensor moe_permute_rows_autograd(const Tensor& x, const Tensor& offs, const Tensor& row_of_copy) {
  no_tangent(x, "moe_permute");
  if (!wants_grad(x)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_permute_rows(x, offs, row_of_copy);
  }
  return PermuteRows::apply(x, offs, row_of_copy)[0];
}
Tensor moe_unpermute_autograd(const Tensor& rows, const Tensor& offs, const Tensor& row_of_copy,
                              const std::optional<Tensor>& weights) {
  no_tangent(rows, "moe_unpermute");
  if (weights.has_value()) no_tangent(*weights, "moe_unpermute");
  if (!wants_grad(rows) && !(weights.has_value() && wants_grad(*weights))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_unpermute(rows, offs, row_of_copy, weights);
  }
  return Unpermute::apply(rows, offs, row_of_copy, weights)[0];
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(grouped_mm, m) {
  m.def(
      "moe_route(Tensor logits, int topk, int score, bool renormalize, float scale, Tensor? bias, Tensor? token_mask)"
      " -> (Tensor, Tensor)");
  m.def(
      "moe_route_bwd(Tensor logits, Tensor expert_idx, Tensor grad_weights, int score, bool renormalize, float scale)"
      " -> Tensor");
  m.def("moe_sort(Tensor expert_idx, int num_experts) -> (Tensor, Tensor, Tensor)");
  m.def("moe_permute(Tensor x, Tensor expert_idx, int num_experts) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("moe_permute_rows(Tensor x, Tensor offs, Tensor row_of_copy) -> Tensor");
  m.def("moe_unpermute(Tensor rows, Tensor offs, Tensor row_of_copy, Tensor? weights) -> Tensor");
  m.def(
      "moe_unpermute_bwd(Tensor grad_out, Tensor rows, Tensor offs, Tensor row_of_copy, Tensor? weights,"
      " bool need_rows, bool need_weights) -> (Tensor, Tensor)");
  m.def("fp8_quantize_rows_block(Tensor x) -> (Tensor, Tensor)");
  m.def("fp8_quantize_weights_block(Tensor w) -> (Tensor, Tensor)");
  m.def("moe_permute_fp8(Tensor x, Tensor expert_idx, int num_experts) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "mm_fp8_block(Tensor mat_a, Tensor mat_b, Tensor offs, Tensor scale_a, Tensor scale_b, Tensor? bias) -> Tensor");
  m.def(
      "mm_swiglu_fp8_block(Tensor mat_a, Tensor mat_b, Tensor offs, Tensor scale_a, Tensor scale_b, Tensor bias,"
      " float swiglu_alpha, float swiglu_limit) -> (Tensor, Tensor)");
  m.def(
      "mm_swiglu_bwd_fp8_block(Tensor grad_output, Tensor down_w_t, Tensor offs, Tensor aux_biased_acc, Tensor scale_a,"
      " Tensor scale_b, float swiglu_alpha, float swiglu_limit) -> Tensor");
  m.def("moe_permute_rows_fp8(Tensor x, Tensor offs, Tensor row_of_copy) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(grouped_mm, CUDA, m) {
  m.impl("moe_route", &moe_route_cuda);
  m.impl("moe_route_bwd", &moe_route_bwd_cuda);
  m.impl("moe_sort", &moe_sort_cuda);
  m.impl("moe_permute", &moe_permute_cuda);
  m.impl("moe_permute_rows", &permute_rows_cuda);
  m.impl("moe_unpermute", &moe_unpermute_cuda);
  m.impl("moe_unpermute_bwd", &moe_unpermute_bwd_cuda);
  m.impl("fp8_quantize_rows_block", &quantize_rows_block_cuda);
  m.impl("fp8_quantize_weights_block", &quantize_weights_block_cuda);
  m.impl("moe_permute_fp8", &moe_permute_fp8_cuda);
  m.impl("mm_fp8_block", &mm_fp8_block_cuda);
  m.impl("mm_swiglu_fp8_block", &mm_swiglu_fp8_block_cuda);
  m.impl("mm_swiglu_bwd_fp8_block", &mm_swiglu_bwd_fp8_block_cuda);
  m.impl("moe_permute_rows_fp8", &permute_rows_fp8_cuda);
}

TORCH_LIBRARY_IMPL(grouped_mm, Autograd, m) {
  m.impl("moe_route", &moe_route_autograd);
  m.impl("moe_permute", &moe_permute_autograd);
  m.impl("moe_permute_rows", &moe_permute_rows_autograd);
  m.impl("moe_unpermute", &moe_unpermute_autograd);
}
