// e4m3 quantisers with one power-of-two scale for each block of 128.
//
//   s = 2^ceil(log2(amax / 448)), the smallest power of two with amax / s <= 448 (1 for a block of zeros),
//   q = e4m3(x / s), round to nearest even.  x / s is exact, so the only rounding is the code's own.
// A power of two costs nothing in the normal range (e4m3 keeps its four significant bits at any scale); it
// loses at most one bit at the bottom of the code's exponent range.  A NaN or infinite element becomes a NaN
// code and does not enter amax, so the rest of its block stays what it was.
//
//   rows     1 x 128 blocks of a [tokens, cols] activation, optionally copied to the topk rows that a plan
//            gives each token (permute fused with the quantiser: the token's row is read once and the
//            bf16 rows in expert order are never written);
//   weights  128 x 128 blocks of [E, R, C], unit stride along C; the codes keep the layout, so one set of
//            codes is the forward's operand (unit stride along n) and, transposed, the input gradient's
//            (unit stride along its k).
// One read and one write each, bound by HBM: the block is held in registers between its maximum and its
// codes.  Weights 32 x 2880 x 5760: 248-262 us in calls back to back, 6.1-6.4 TB/s (240 in a loop of its own); 8192
// tokens x 7168 to 65536 rows: 97 us, 6.2 TB/s; 98304 x 2880 without a plan 279 us, 3.0 TB/s (short-lived warps).
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "host.h"
#include "moe_gemm.h"

namespace mgf {

unsigned int* status_word_address();

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kBlock = 128;
constexpr int kWarps = 8;

// Biased exponent of the scale of a block whose largest finite magnitude is `amax`: amax = m * 2^x with
// m <= 1.75 gives 2^(x - 8) (448 = 1.75 * 2^8), else 2^(x - 7); never subnormal, so that 1 / s is finite.
__device__ __forceinline__ int scale_exponent(float amax) {
  if (amax == 0.0f) return 127;
  const int e = static_cast<int>((__float_as_uint(amax) + (0x7FFFFFu - 0x600000u)) >> 23) - 8;
  return e < 1 ? 1 : e;
}
__device__ __forceinline__ float pow2_of(int biased) { return __uint_as_float(static_cast<uint32_t>(biased) << 23); }

// Magnitudes of bf16 pairs order like their bits without the sign, and those of NaN and infinity are the largest:
// one packed maximum per pair finds amax and whether anything is not finite.  (Unpacking, comparing and testing
// every element took 10 instructions each, as long as the memory traffic.)
constexpr uint32_t kNotFinite = 0x7F80u;
__device__ __forceinline__ uint32_t max_bits(uint32_t m, uint32_t pair) { return __vmaxu2(m, pair & 0x7FFF7FFFu); }
__device__ __forceinline__ uint32_t larger_half(uint32_t m) { return max(m & 0xFFFFu, m >> 16); }
// The same over finite elements only.
__device__ __forceinline__ uint32_t max_finite_bits(uint32_t m, uint32_t pair) {
  const uint32_t a = pair & 0x7FFFu, b = (pair >> 16) & 0x7FFFu;
  return max(m, max(a < kNotFinite ? a : 0u, b < kNotFinite ? b : 0u));
}
__device__ __forceinline__ float of_bits(uint32_t bf16) { return __uint_as_float(bf16 << 16); }

// Two codes.  Finite values never saturate (|x / s| <= 448); where the block holds others, they become NaN.
__device__ __forceinline__ uint32_t code2(float a, float b, float inv) {
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3));
}
__device__ __forceinline__ float no_infinity(float v) { return isinf(v) ? __uint_as_float(0x7FC00000u) : v; }

__device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// ---------------------------------------------------------------- rows
// A lane holds 16 consecutive elements, 8 lanes a block, a warp 512 elements of one token.
template <bool VEC>
__global__ void __launch_bounds__(32 * kWarps)
    quantize_rows_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, int64_t tokens, int64_t cols, int topk,
                         int64_t chunks, const int32_t* __restrict__ row_of_copy, const int32_t* __restrict__ offs_end,
                         int64_t n_rows, uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale, int64_t lds,
                         unsigned int* __restrict__ status) {
  const int lane = threadIdx.x & 31;
  const int64_t u = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (u < tokens * chunks) {
    const int64_t t = u / chunks;
    const int64_t col = (u - t * chunks) * 512 + lane * 16;
    const __nv_bfloat16* xr = x + t * ldx;
    uint32_t w[8];
    const bool whole = col + 16 <= cols;
    if (VEC && whole) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(xr + col));
      const uint4 b = __ldg(reinterpret_cast<const uint4*>(xr + col) + 1);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
      w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t l = col + 2 * i < cols ? __bfloat16_as_ushort(xr[col + 2 * i]) : 0u;
        const uint32_t h = col + 2 * i + 1 < cols ? __bfloat16_as_ushort(xr[col + 2 * i + 1]) : 0u;
        w[i] = l | (h << 16);
      }
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_bits(m, w[i]);
    m = larger_half(m);
#pragma unroll
    for (int off = 4; off; off >>= 1) m = max(m, __shfl_xor_sync(kFull, m, off));
    const bool all_finite = m < kNotFinite;
    if (__any_sync(kFull, !all_finite)) {
      uint32_t f = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) f = max_finite_bits(f, w[i]);
#pragma unroll
      for (int off = 4; off; off >>= 1) f = max(f, __shfl_xor_sync(kFull, f, off));
      m = f;
    }
    const int e = scale_exponent(of_bits(m));
    const float inv = pow2_of(254 - e);
    uint32_t c[4];
    if (all_finite) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        c[i] = code2(lo(w[2 * i]), hi(w[2 * i]), inv) | (code2(lo(w[2 * i + 1]), hi(w[2 * i + 1]), inv) << 16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        c[i] = code2(no_infinity(lo(w[2 * i])), no_infinity(hi(w[2 * i])), inv) |
               (code2(no_infinity(lo(w[2 * i + 1])), no_infinity(hi(w[2 * i + 1])), inv) << 16);
    }
    for (int j = 0; j < topk; ++j) {
      int64_t row = t;
      if (row_of_copy != nullptr) {
        row = __ldg(row_of_copy + t * topk + j);
        if (row < 0) continue;
        if (row >= n_rows) {  // a wrong plan: report it, touch nothing
          atomicOr(status, MGF_DEV_ROW_OUT_OF_RANGE);
          continue;
        }
      }
      uint8_t* d = q + row * ldq + col;
      if (whole) {
        *reinterpret_cast<uint4*>(d) = make_uint4(c[0], c[1], c[2], c[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (col + i < cols) d[i] = static_cast<uint8_t>(c[i >> 2] >> (8 * (i & 3)));
      }
      if ((lane & 7) == 0 && col < cols) scale[row * lds + col / kBlock] = pow2_of(e);
    }
  }
  // rows behind the last one: zero codes, zero scales
  if (offs_end != nullptr) {
    int64_t kept = __ldg(offs_end);
    if (kept < 0) kept = 0;
    const int64_t w0 = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int64_t nw = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
    const int64_t nb = (cols + kBlock - 1) / kBlock;
    for (int64_t r = kept + w0; r < n_rows; r += nw) {
      for (int64_t c = lane * 16; c < cols; c += 512) {
        if (c + 16 <= cols) *reinterpret_cast<uint4*>(q + r * ldq + c) = make_uint4(0, 0, 0, 0);
        else for (int64_t i = c; i < cols; ++i) q[r * ldq + i] = 0;
      }
      for (int64_t b = lane; b < nb; b += 32) scale[r * lds + b] = 0.0f;
    }
  }
}

// ---------------------------------------------------------------- weights
// One 256-thread block per 128 x 128 block: 16 threads to a row of 128, eight rows each, all in registers.
template <bool VEC>
__global__ void __launch_bounds__(256)
    quantize_weights_kernel(const __nv_bfloat16* __restrict__ w, int64_t R, int64_t C, int64_t se, int64_t sr,
                            uint8_t* __restrict__ q, int64_t qe, int64_t qr, float* __restrict__ scale, int64_t ss_e,
                            int64_t ss_r, int64_t ss_c) {
  __shared__ uint32_t red[8];
  const int tid = threadIdx.x;
  const int64_t e = blockIdx.z, rb = blockIdx.y, cb = blockIdx.x;
  const int64_t r0 = rb * kBlock + (tid >> 4), c0 = cb * kBlock + (tid & 15) * 8;
  const __nv_bfloat16* src = w + e * se + c0;
  uint4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + 16 * i;
    v[i] = make_uint4(0, 0, 0, 0);
    if (r < R) {
      if (VEC && c0 + 8 <= C) {
        v[i] = __ldg(reinterpret_cast<const uint4*>(src + r * sr));
      } else {
        uint32_t* p = reinterpret_cast<uint32_t*>(&v[i]);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c0 + k < C) p[k >> 1] |= static_cast<uint32_t>(__bfloat16_as_ushort(src[r * sr + k])) << (16 * (k & 1));
      }
    }
  }
  // the block's largest magnitude; every thread takes part in every reduction
  auto block_max = [&](uint32_t m) -> uint32_t {
    m = __reduce_max_sync(kFull, m);
    __syncthreads();  // the words of an earlier reduction have been read
    if ((tid & 31) == 0) red[tid >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, red[i]);
    return m;
  };
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max_bits(max_bits(max_bits(max_bits(m, v[i].x), v[i].y), v[i].z), v[i].w);
  m = block_max(larger_half(m));
  const bool all_finite = m < kNotFinite;  // the same for all threads
  if (!all_finite) {
    uint32_t f = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f = max_finite_bits(max_finite_bits(max_finite_bits(max_finite_bits(f, v[i].x), v[i].y), v[i].z), v[i].w);
    m = block_max(f);
  }
  const int ex = scale_exponent(of_bits(m));
  const float inv = pow2_of(254 - ex);
  if (tid == 0) scale[e * ss_e + rb * ss_r + cb * ss_c] = pow2_of(ex);
  auto code4 = [&](uint32_t x, uint32_t y) -> uint32_t {
    if (all_finite) return code2(lo(x), hi(x), inv) | (code2(lo(y), hi(y), inv) << 16);
    return code2(no_infinity(lo(x)), no_infinity(hi(x)), inv) | (code2(no_infinity(lo(y)), no_infinity(hi(y)), inv) << 16);
  };
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + 16 * i;
    if (r >= R) break;
    const uint32_t c[2] = {code4(v[i].x, v[i].y), code4(v[i].z, v[i].w)};
    uint8_t* d = q + e * qe + r * qr + c0;
    if (c0 + 8 <= C) {
      *reinterpret_cast<uint2*>(d) = make_uint2(c[0], c[1]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c0 + k < C) d[k] = static_cast<uint8_t>(c[k >> 2] >> (8 * (k & 3)));
    }
  }
}

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1u)) == 0; }

}  // namespace
}  // namespace mgf

extern "C" int mgf_fp8_block_quantize_rows(const void* x, int64_t ldx, int64_t tokens, int64_t cols, int32_t topk,
                                           const int32_t* row_of_copy, const int32_t* offs_end, void* q, int64_t ldq,
                                           float* scale, int64_t lds, int64_t n_rows, void* stream) {
  using namespace mgf;
  forget_cuda_error();
  if (tokens < 0 || cols < 0 || topk < 1 || n_rows < 0 || n_rows > INT32_MAX || tokens > INT32_MAX / topk)
    return MGF_ERR_INVALID_ARGUMENT;
  if (row_of_copy == nullptr && (topk != 1 || n_rows != tokens || offs_end != nullptr)) return MGF_ERR_INVALID_ARGUMENT;
  if (n_rows == 0 || cols == 0) return MGF_OK;
  if (q == nullptr || scale == nullptr || (tokens > 0 && x == nullptr) || (row_of_copy != nullptr && offs_end == nullptr))
    return MGF_ERR_INVALID_ARGUMENT;
  if (!aligned(q, 16) || ldq % 16 != 0) return MGF_ERR_ALIGNMENT;
  unsigned int* status = status_word_address();
  if (status == nullptr) return MGF_ERR_CUDA;
  const int64_t chunks = (cols + 511) / 512, blocks = (tokens * chunks + kWarps - 1) / kWarps;
  if (blocks > INT32_MAX) return MGF_ERR_INVALID_ARGUMENT;
  const unsigned grid = static_cast<unsigned>(blocks > 0 ? blocks : 1);
  auto kern = aligned(x, 16) && ldx % 8 == 0 ? quantize_rows_kernel<true> : quantize_rows_kernel<false>;
  kern<<<grid, 32 * kWarps, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(x), ldx, tokens, cols, topk, chunks, row_of_copy, offs_end, n_rows,
      static_cast<uint8_t*>(q), ldq, scale, lds, status);
  return cudaGetLastError() == cudaSuccess ? MGF_OK : MGF_ERR_CUDA;
}

extern "C" int mgf_fp8_block_quantize_weights(const void* w, int64_t E, int64_t R, int64_t C, int64_t s_e, int64_t s_r,
                                              void* q, int64_t q_e, int64_t q_r, float* scale, int64_t ss_e,
                                              int64_t ss_r, int64_t ss_c, void* stream) {
  using namespace mgf;
  forget_cuda_error();
  if (E < 0 || R < 0 || C < 0 || E > 65535 || R > 65535ll * kBlock || C > int64_t(INT32_MAX) * kBlock)
    return MGF_ERR_INVALID_ARGUMENT;
  if (E == 0 || R == 0 || C == 0) return MGF_OK;
  if (w == nullptr || q == nullptr || scale == nullptr) return MGF_ERR_INVALID_ARGUMENT;
  if (!aligned(q, 8) || q_e % 8 != 0 || q_r % 8 != 0) return MGF_ERR_ALIGNMENT;
  const dim3 grid(static_cast<unsigned>((C + kBlock - 1) / kBlock), static_cast<unsigned>((R + kBlock - 1) / kBlock),
                  static_cast<unsigned>(E));
  auto kern = aligned(w, 16) && s_e % 8 == 0 && s_r % 8 == 0 ? quantize_weights_kernel<true>
                                                             : quantize_weights_kernel<false>;
  kern<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const __nv_bfloat16*>(w), R, C, s_e, s_r,
                                                            static_cast<uint8_t*>(q), q_e, q_r, scale, ss_e, ss_r,
                                                            ss_c);
  return cudaGetLastError() == cudaSuccess ? MGF_OK : MGF_ERR_CUDA;
}
