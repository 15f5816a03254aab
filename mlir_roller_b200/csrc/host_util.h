// Host-side helpers defined in capi.cu and used by the other entry points' translation units.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace rb200 {

// Records the text behind roller_b200_last_cuda_error, clears the error, returns ROLLER_ERR_CUDA.
int report_cuda_error(cudaError_t e, const char* what);

// Zeroes device memory that a plan has just got, and returns when that is done: the first launch may come at
// once, on a stream that does not wait for the default one, and a word left over from an earlier owner of the
// memory would end its waits or pass for a flag. (On a stream of its own where the default one is busy, which may
// be for long.)
cudaError_t zero_now(void* words, size_t bytes);

// Tensor map of a batch of `z` row-major 16-bit matrices. base, ld and z_stride have to be
// multiples of 16 bytes.
int encode_batch16(CUtensorMap* tm, const void* base, long long cols, long long rows, long long z,
                   long long ld, long long z_stride, int box_cols, int box_rows,
                   CUtensorMapSwizzle swz, bool bf16);

}  // namespace rb200
