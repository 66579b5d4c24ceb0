// Host helpers shared by the launchers (defined in moe_gemm_sm100.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace mgf {

// Rows of a product: a tile's row index, up to 256 past the last row, is a 32-bit number.
constexpr int64_t kMaxRows = INT32_MAX - 256;

struct DeviceInfo {
  int sms = 0;
  int major = 0;
};
DeviceInfo device_info(int dev);

// Encode a tiled tensor map of rank 1..4 (strides in bytes, innermost dimension dense); false with the
// error text recorded where the driver refuses it.
bool encode_bf16(CUtensorMap* m, const void* base, int rank, const uint64_t* dims, const uint64_t* strides_bytes,
                 const uint32_t* box, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B,
                 CUtensorMapDataType dtype = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);

// The text behind mgf_last_error_detail() on this host thread.
void clear_error();
void record_error(const char* what, cudaError_t e);

// Called before a launch whose status is read with cudaGetLastError: an error that an unrelated runtime call left would
// otherwise be reported as the launch's.
inline void forget_cuda_error() { cudaGetLastError(); }

bool bind_device(int dev);  // a current driver context for this host thread
bool debug_sync();          // MGF_DEBUG_SYNC=1

// Device address of the status word of the current device.
unsigned int* status_word_address();

}  // namespace mgf
