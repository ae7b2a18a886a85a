/* C entry points of the 4-bit microscaled format: quantisation, the way back, and products on the block-scaled tensor cores.
 * No counterpart in the reference; see csrc/src/mx4.cu.
 *
 * A tensor [rows, cols] (cols a multiple of 32) is
 *   data    rows x cols / 2 bytes, row-major: e2m1 values, the even column in a byte's low half
 *   scales  a byte per 32 columns of a row, a power of two 2^(byte - 127), 255: the block stands for NaNs. In the order in which the tensor
 *           cores take them: blocks of 512 bytes for 128 rows x 128 columns, [rows / 128 up][cols / 128 up][row % 32][row / 32 % 4][col / 32 % 4];
 *           what lies past the tensor's edges is 0. */
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { PURLIN_MX4_BF16 = 0, PURLIN_MX4_FP16 = 1, PURLIN_MX4_FP32 = 2 };

size_t purlin_mx4_scale_bytes(int rows, int cols);

/* x [rows, cols] of `dtype`, row-major, 16-byte aligned. */
int purlin_mx4_quantize(const void* x, int dtype, void* data, void* scales, int rows, int cols, void* stream);
/* The values that data and scales stand for in bf16 or fp32 (`dtype`): exact for scale bytes up to 252, which are all that the quantisation makes (and 255);
 * with 253 and 254 the largest of them are past both types' range and become infinities. No output overlaps an input, here and above. */
int purlin_mx4_dequantize(const void* data, const void* scales, void* out, int dtype, int rows, int cols, void* stream);

/* C[M, N] = A[M, K] * W[N, K]^T, fp32 accumulation, bf16 output; A and W as above. epilogue: PURLIN_EPI_STORE or PURLIN_EPI_SWIGLU (W's rows
 * alternate 16 of gate and 16 of up, N a multiple of 32, C is [M, N / 2]). N a multiple of 8. C overlaps no operand. status: as in
 * purlin_ffn_forward, with k-blocks of 256. */
int purlin_mx4_gemm(const void* aData, const void* aScales, const void* wData, const void* wScales, void* C, int M, int N, int K, int epilogue,
                    uint32_t* status, void* stream);
/* The same with activations x [M, K] of `dtype`, quantised by the way: a few tokens inside the product, more into the workspace first, which has
 * purlin_mx4_workspace_bytes() (none: it may be NULL). C may overlap x, but neither w nor the workspace; a few tokens then take a workspace too,
 * of M * K / 2 + purlin_mx4_scale_bytes(M, K) bytes. */
size_t purlin_mx4_workspace_bytes(int dtype, int M, int K);
int purlin_mx4_linear(const void* x, int dtype, void* workspace, const void* wData, const void* wScales, void* C, int M, int N, int K, int epilogue,
                      uint32_t* status, void* stream);

#ifdef __cplusplus
}
#endif
