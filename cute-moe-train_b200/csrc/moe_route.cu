// Router of the MoE block: top-k experts of every token and their weights, and the logits' gradient.
//
//   key_e = l_e (+ bias_e, fp32)                     selection only; ties go to the lowest expert.  A bias that
//           balances the load by the scores (BIAS_ON_SCORE): key_e = s(l_e) + bias_e or softmax_e(l) + bias_e
//   chosen = the topk largest keys; a key of -inf is never chosen (id -1, weight 0), NaN sorts first
//   softmax:  w_j = scale * exp(l_j - m) / sum exp(l_i - m), the sum over the chosen experts
//             (renormalize) or over all experts
//   sigmoid:  w_j = scale * s(l_j), renormalised as the softmax of log s(l_j) over the chosen ones (the
//             same quotient s_j / sum s_i, but it cannot become 0 / 0 where every s underflows)
// backward, with p = w / scale and r = sum_i p_i g_i over the chosen experts:
//   softmax   renormalised dl_j = scale p_j (g_j - r);  else dl_e = scale p_e (G_e - r) for every expert
//             (G_e = g_j where e is chosen, else 0)
//   sigmoid   renormalised dl_j = scale p_j (g_j - r) (1 - s_j);  else dl_j = scale s_j (1 - s_j) g_j
//
// One warp per token, R = ceil(E / 32) logits per lane in registers.  The keys are mapped to unsigned
// integers of the same order, so that one selection is a redux.sync maximum of the key and a redux.sync
// minimum of the expert among the lanes that hold it; bf16 logits without a bias have 16-bit keys, and key
// and expert go into one word and one maximum (PACKED).  Statistics and sums are fp32.  Each pass reads
// the logits once and writes its outputs once.  24576 tokens, 128 experts, top 4, bf16: 16 us forward and 9 backward
// (8 tokens: 2.3), bound by the selections' instructions, not by the 6 MB.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "host.h"
#include "moe_gemm.h"

namespace mgf {
namespace {

constexpr int kWarpsPerBlock = 8;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }

// Unsigned key of the same order as the float: 0 for -inf (not available), all ones for NaN; -0 = +0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  if (v == -INFINITY) return 0u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(kFull, v, off);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {  // NaN is ignored: the sums that follow carry it
#pragma unroll
  for (int off = 16; off; off >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, off));
  return v;
}

// Per-lane value of the activation at a chosen logit: log s(v) (renormalised sigmoid) or v (softmax).
__device__ __forceinline__ float log_score(float v, int score) {
  return score == MGF_ROUTE_SIGMOID ? fminf(v, 0.0f) - log1pf(expf(-fabsf(v))) : v;
}

// The score itself; row_max and row_sum: of the softmax over all experts.
__device__ __forceinline__ float score_of(float v, int score, float row_max, float row_sum) {
  return score == MGF_ROUTE_SIGMOID ? 1.0f / (1.0f + expf(-v)) : expf(v - row_max) / row_sum;
}

// p_j of the chosen logits, one per lane (0 where `live` is false).
__device__ __forceinline__ float chosen_prob(float v, bool live, int score, bool renorm, float row_max, float row_sum) {
  if (renorm) {
    const float z = live ? log_score(v, score) : -INFINITY;
    const float m = warp_max(z);
    const float p = live ? expf(z - m) : 0.0f;
    const float s = warp_sum(p);
    return live ? p / s : 0.0f;
  }
  return live ? score_of(v, score, row_max, row_sum) : 0.0f;
}

template <typename T, int R, bool PACKED>
__global__ void __launch_bounds__(32 * kWarpsPerBlock)
    route_kernel(const T* __restrict__ logits, int64_t ld, int64_t tokens, int E, int topk, int score, bool renorm,
                 float scale, const float* __restrict__ bias, bool on_score, const uint8_t* __restrict__ token_mask,
                 float* __restrict__ weights, int64_t* __restrict__ idx) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (t >= tokens) return;
  int my_expert = -1;
  float my_logit = 0.0f, row_max = 0.0f, row_sum = 1.0f;
  if (token_mask == nullptr || token_mask[t] != 0) {
    const T* row = logits + t * ld;
    float v[R];
    uint32_t key[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int e = lane + 32 * i;
      v[i] = e < E ? to_f(row[e]) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int e = lane + 32 * i;
      key[i] = order_key(bias != nullptr && e < E ? v[i] + __ldg(bias + e) : v[i]);
      if (v[i] == -INFINITY) key[i] = 0u;  // an expert masked in the logits stays masked under any bias
      // the low half of a bf16 key says nothing; the earlier expert gets the larger word
      if (PACKED && key[i] != 0u) key[i] = (key[i] & 0xffff0000u) | static_cast<uint32_t>(0xffff - e);
    }
    if (score == MGF_ROUTE_SOFTMAX && (!renorm || on_score)) {
      float m = v[0], s = 0.0f;
#pragma unroll
      for (int i = 1; i < R; ++i) m = fmaxf(m, v[i]);
      row_max = warp_max(m);
#pragma unroll
      for (int i = 0; i < R; ++i) s += (lane + 32 * i < E) ? expf(v[i] - row_max) : 0.0f;
      row_sum = warp_sum(s);
    }
    if (on_score) {  // there is a bias
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int e = lane + 32 * i;
        if (e < E && v[i] != -INFINITY) key[i] = order_key(score_of(v[i], score, row_max, row_sum) + __ldg(bias + e));
      }
    }
    for (int j = 0; j < topk; ++j) {
      uint32_t best = key[0];
      int at = 0;
#pragma unroll
      for (int i = 1; i < R; ++i)
        if (key[i] > best) {
          best = key[i];
          at = i;
        }
      const uint32_t top = __reduce_max_sync(kFull, best);
      if (top == 0u) break;  // nothing left to choose
      const int e = PACKED ? 0xffff - static_cast<int>(top & 0xffffu)
                           : static_cast<int>(__reduce_min_sync(kFull, best == top ? static_cast<uint32_t>(lane + 32 * at) : ~0u));
      float ve = 0.0f;
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (i == (e >> 5)) {
          ve = v[i];
          if (lane == (e & 31)) key[i] = 0u;
        }
      ve = __shfl_sync(kFull, ve, e & 31);
      if (lane == j) {
        my_expert = e;
        my_logit = ve;
      }
    }
  }
  const bool live = my_expert >= 0;
  const float p = chosen_prob(my_logit, live, score, renorm, row_max, row_sum);
  if (lane < topk) {
    weights[t * topk + lane] = live ? scale * p : 0.0f;
    idx[t * topk + lane] = my_expert;
  }
}

template <typename T, int R>
__global__ void __launch_bounds__(32 * kWarpsPerBlock)
    route_bwd_kernel(const T* __restrict__ logits, int64_t ld, int64_t tokens, int E, int topk, int score, bool renorm,
                     float scale, const int64_t* __restrict__ idx, const float* __restrict__ grad_weights,
                     T* __restrict__ grad_logits, int64_t ldg) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (t >= tokens) return;
  const T* row = logits + t * ld;
  const bool full = score == MGF_ROUTE_SOFTMAX && !renorm;
  int id = -1;
  float g = 0.0f;
  if (lane < topk) {
    const int64_t raw = idx[t * topk + lane];
    id = raw >= 0 && raw < E ? static_cast<int>(raw) : -1;
    g = grad_weights[t * topk + lane];
  }
  const bool live = id >= 0;
  const float v = live ? to_f(row[id]) : 0.0f;
  const bool any = __any_sync(kFull, live);  // a masked token has no chosen expert: its row may hold anything
  float all[R], row_max = 0.0f, row_sum = 1.0f;
  if (full && any) {
    float m = -INFINITY, s = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int e = lane + 32 * i;
      all[i] = e < E ? to_f(row[e]) : -INFINITY;
      m = fmaxf(m, all[i]);
    }
    row_max = warp_max(m);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      all[i] = (lane + 32 * i < E) ? expf(all[i] - row_max) : 0.0f;
      s += all[i];
    }
    row_sum = warp_sum(s);
  }
  const float p = chosen_prob(v, live, score, renorm, row_max, row_sum);
  const float r = warp_sum(live ? p * g : 0.0f);
  float d = live ? g : 0.0f;  // softmax over all experts: G_e, the rest below
  if (!full) {
    d = p * (renorm ? g - r : g);
    if (score == MGF_ROUTE_SIGMOID) d *= 1.0f / (1.0f + expf(v));
    d = live ? scale * d : 0.0f;
  }
  float out[R];
#pragma unroll
  for (int i = 0; i < R; ++i) out[i] = 0.0f;
  for (int j = 0; j < topk; ++j) {
    const int e = __shfl_sync(kFull, id, j);
    const float de = __shfl_sync(kFull, d, j);
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (e == lane + 32 * i) out[i] = de;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int e = lane + 32 * i;
    if (e < E) grad_logits[t * ldg + e] = from_f<T>(full ? (any ? scale * (all[i] / row_sum) * (out[i] - r) : 0.0f) : out[i]);
  }
}

template <typename T, typename F>
int for_width(int E, F&& f) {
  if (E <= 32) return f(std::integral_constant<int, 1>{});
  if (E <= 64) return f(std::integral_constant<int, 2>{});
  if (E <= 128) return f(std::integral_constant<int, 4>{});
  if (E <= 256) return f(std::integral_constant<int, 8>{});
  if (E <= 512) return f(std::integral_constant<int, 16>{});
  return f(std::integral_constant<int, 32>{});
}

bool route_args_ok(int32_t dtype, int64_t tokens, int32_t E, int32_t topk, int32_t score) {
  return dtype >= MGF_DT_BF16 && dtype <= MGF_DT_F32 && tokens >= 0 && tokens <= INT32_MAX && E >= 1 && E <= 1024 &&
         topk >= 1 && topk <= 32 && topk <= E && (score == MGF_ROUTE_SOFTMAX || score == MGF_ROUTE_SIGMOID);
}

}  // namespace
}  // namespace mgf

extern "C" int mgf_moe_route(const void* logits, int32_t dtype, int64_t ld, int64_t tokens, int32_t num_experts,
                             int32_t topk, int32_t score, int32_t renormalize, float scale, const float* bias,
                             const uint8_t* token_mask, float* weights, int64_t* expert_idx, void* stream) {
  using namespace mgf;
  forget_cuda_error();
  const bool on_score = (score & MGF_ROUTE_BIAS_ON_SCORE) != 0 && bias != nullptr;
  score &= ~MGF_ROUTE_BIAS_ON_SCORE;
  if (!route_args_ok(dtype, tokens, num_experts, topk, score)) return MGF_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return MGF_OK;
  if (logits == nullptr || weights == nullptr || expert_idx == nullptr) return MGF_ERR_INVALID_ARGUMENT;
  const unsigned grid = static_cast<unsigned>((tokens + kWarpsPerBlock - 1) / kWarpsPerBlock);
  auto run = [&](auto tag) {
    using T = decltype(tag);
    return for_width<T>(num_experts, [&](auto r) {
      constexpr int R = decltype(r)::value;
      constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
      auto kern = kBf16 && bias == nullptr ? route_kernel<T, R, kBf16> : route_kernel<T, R, false>;
      kern<<<grid, 32 * kWarpsPerBlock, 0, static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T*>(logits), ld, tokens, num_experts, topk, score, renormalize != 0, scale, bias,
          on_score, token_mask, weights, expert_idx);
      return cudaGetLastError() == cudaSuccess ? MGF_OK : MGF_ERR_CUDA;
    });
  };
  if (dtype == MGF_DT_BF16) return run(__nv_bfloat16{});
  if (dtype == MGF_DT_F16) return run(__half{});
  return run(float{});
}

extern "C" int mgf_moe_route_bwd(const void* logits, int32_t dtype, int64_t ld, int64_t tokens, int32_t num_experts,
                                 int32_t topk, int32_t score, int32_t renormalize, float scale,
                                 const int64_t* expert_idx, const float* grad_weights, void* grad_logits, int64_t ldg,
                                 void* stream) {
  using namespace mgf;
  forget_cuda_error();
  score &= ~MGF_ROUTE_BIAS_ON_SCORE;  // the bias is not in the weights
  if (!route_args_ok(dtype, tokens, num_experts, topk, score)) return MGF_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return MGF_OK;
  if (logits == nullptr || expert_idx == nullptr || grad_weights == nullptr || grad_logits == nullptr)
    return MGF_ERR_INVALID_ARGUMENT;
  const unsigned grid = static_cast<unsigned>((tokens + kWarpsPerBlock - 1) / kWarpsPerBlock);
  auto run = [&](auto tag) {
    using T = decltype(tag);
    return for_width<T>(num_experts, [&](auto r) {
      route_bwd_kernel<T, decltype(r)::value><<<grid, 32 * kWarpsPerBlock, 0, static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T*>(logits), ld, tokens, num_experts, topk, score, renormalize != 0, scale, expert_idx,
          grad_weights, static_cast<T*>(grad_logits), ldg);
      return cudaGetLastError() == cudaSuccess ? MGF_OK : MGF_ERR_CUDA;
    });
  };
  if (dtype == MGF_DT_BF16) return run(__nv_bfloat16{});
  if (dtype == MGF_DT_F16) return run(__half{});
  return run(float{});
}
