// Epilogue helpers of the grouped GEMMs: row access in whole sectors, bf16 packing and the clamped SwiGLU.
#pragma once

#include <cuda_bf16.h>

#include <cstdint>

#include "ptx.cuh"

namespace mgf {

#ifndef MGF_AUX_NOALLOC
#define MGF_AUX_NOALLOC 1
#endif
// One chunk of aux words (32 packed (gate, up) pairs = 128 bytes of one row) as four 32-byte loads;
// words past n read as zero.  Each sector is requested once, so nothing relies on L1 reuse.
// v8 = false (aux rows only 16-byte aligned): eight 16-byte loads.
__device__ __forceinline__ void load_aux_chunk(const __nv_bfloat16* row, int col0, int n, bool valid, bool v8,
                                               uint4 (&aw)[8]) {
  const uint4* ap = reinterpret_cast<const uint4*>(row + 2 * col0);
  if (!v8) {
#pragma unroll
    for (int g = 0; g < 8; ++g) aw[g] = (valid && col0 + 4 * g < n) ? __ldg(ap + g) : make_uint4(0, 0, 0, 0);
    return;
  }
#pragma unroll
  for (int g = 0; g < 8; g += 2) {
    if (valid && col0 + 4 * g < n) {
      if (MGF_AUX_NOALLOC) ptx::ld_nc_v8_noalloc(ap + g, aw[g], aw[g + 1]);
      else ptx::ld_nc_v8(ap + g, aw[g], aw[g + 1]);
    } else {
      aw[g] = make_uint4(0, 0, 0, 0);
      aw[g + 1] = make_uint4(0, 0, 0, 0);
    }
  }
}

// Store the first `nvalid` of NU 16-byte units of one output row; pairs of units go out as one
// 32-byte store when v8 (the row and its 32-byte pairs aligned).
template <int NU>
__device__ __forceinline__ void store_units(void* dst, const uint4 (&u)[NU], int nvalid, bool v8) {
  uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll
  for (int g = 0; g < NU; g += 2) {
    if (v8 && g + 1 < nvalid) {
      ptx::st_v8(d + g, u[g], u[g + 1]);
    } else {
      if (g < nvalid) d[g] = u[g];
      if (g + 1 < nvalid) d[g + 1] = u[g + 1];
    }
  }
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// min and max that keep a NaN, as the formula's clamps do (fminf and fmaxf give the other operand).
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// sigma(z) = 0.5 * tanh(z / 2) + 0.5, the form the reference's SwiGLU visitors use
// (csrc/grouped_mm_swiglu_visitor.cuh:309-334, csrc/grouped_mm_swiglu_bwd_visitor.cuh:35-68), on the
// hardware tanh approximation (one MUFU operation; max relative error about 2^-11, below bf16's 2^-8).
__device__ __forceinline__ float tanh_approx(float x) {
  float y;
  asm("tanh.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoidf_fast(float z) { return fmaf(0.5f, tanh_approx(0.5f * z), 0.5f); }

// SwiGLU forward on one (gate, up) pair of bf16-rounded values.
__device__ __forceinline__ float swiglu_fwd(float g, float u, float alpha, float limit) {
  const float gc = min_nan(g, limit);
  const float uc = max_nan(min_nan(u, limit), -limit);
  return gc * sigmoidf_fast(alpha * gc) * (uc + 1.0f);
}

// SwiGLU backward for one packed (gate, up) word of aux; returns packed (d_gate, d_up), each 0 where its own input is
// clamped or NaN; a NaN of the other input or of gs stays one.
__device__ __forceinline__ uint32_t swiglu_bwd_word(float gs, uint32_t aux_word, float alpha, float limit) {
  const float g = bf16_lo(aux_word);
  const float u = bf16_hi(aux_word);
  const float gc = min_nan(g, limit);
  const float uc = max_nan(min_nan(u, limit), -limit);
  const float sig = sigmoidf_fast(alpha * gc);
  float d_gate = gs * (uc + 1.0f) * sig * (1.0f + alpha * gc * (1.0f - sig));
  float d_up = gs * gc * sig;
  d_gate = (g <= limit) ? d_gate : 0.0f;
  d_up = (u >= -limit && u <= limit) ? d_up : 0.0f;
  return pack_bf16x2(d_gate, d_up);
}

}  // namespace mgf
