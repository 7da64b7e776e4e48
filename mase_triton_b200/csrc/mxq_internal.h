// Host-side helpers shared by the translation units of libmxq.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mxq {
constexpr int MX_MAX_GROUPS = 1024;      // groups of rows of one mxq_mx_grouped_linear (its table lies in shared memory)
// Records the error of a failed launch for mxq_last_cuda_error(); returns MXQ_OK or MXQ_ELAUNCH.
int check_launch();
void set_last_cuda_error(cudaError_t e);
// One-pass quantise + pack of a left GEMM operand (mxq_elementwise.cu); MXQ_ESIZE = not covered.
int quantize_pack_left_operand(const void* x, int x_dtype, int64_t M, int64_t K, int eb, int fb, uint8_t* hw_codes,
                               uint8_t* hw_sf, int64_t sf_bytes, int* hw_format, cudaStream_t st);
// The same for per-tensor minifloat FP8 codes with unit block scales (mxq_elementwise.cu).
int minifloat_quantize_pack_left_operand(const void* x, int x_dtype, int64_t M, int64_t K, int eb, int fb, uint8_t* hw_codes,
                                         uint8_t* hw_sf, int64_t sf_bytes, int* hw_format, cudaStream_t st);
// Reference element code -> byte the tensor cores read (mxq_gemm.cu): of the same value, of half the value, and a bit per code
// that has no such byte; false for an element format that is none of the presets.
bool hw_code_tables(int eb, int fb, uint8_t (&plain)[256], uint8_t (&halved)[256], uint32_t (&bad)[8], int* hw_format);
}  // namespace mxq
