// mt_host.h -- host-side services of mt_api.cu for the library's other translation units:
// the thread's error text and path string, the launch counter, device properties, scratch
// memory and the tensor-map encoder.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mt {
namespace host {

// Records the calling thread's error text (printf form) and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int cuda_fail(cudaError_t e, const char* what);
// MT_OK after a clean launch (counted), else the recorded error.
int launched(const char* what);
void set_path(const char* path);
int sm_count();
int scratch_alloc(void** p, size_t bytes, cudaStream_t st, const char* who);
void scratch_free(void* p, size_t bytes, cudaStream_t st);
// cuTensorMapEncodeTiled for a 2-D or 3-D map of bfloat16 elements with 128-byte swizzle:
// extents d[0] (contiguous) .. d[rank-1], byte strides s[0..rank-2] of dims 1.., box b.
bool encode_bf16(CUtensorMap* m, const void* base, int rank, const uint64_t* d, const uint64_t* s, const uint32_t* b);
// The same for a 2-D map of bytes with 64-byte swizzle: d[0] (contiguous), d[1], byte stride s of
// dim 1, box b.
bool encode_u8(CUtensorMap* m, const void* base, const uint64_t* d, uint64_t s, const uint32_t* b);

// Device status word of mt_lowbit.cu (see mt_device_status); reset != 0 clears it.
int lowbit_device_status(int reset);

}  // namespace host
}  // namespace mt
