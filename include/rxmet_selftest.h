/*
 * rxmet_selftest.h — self-tests of what the kernels rely on.
 *
 * No counterpart in the reference: these entry points exist so that tests can check,
 * on the GPU, the MFMA operand/result lane layouts the GRU kernels are written against, and, on the
 * host, which form of a kernel a call takes.
 */
#ifndef RXMET_SELFTEST_H_
#define RXMET_SELFTEST_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * One wavefront computes D[16x16] = A[16xK] * B[Kx16] with the fragment layouts the GRU
 * kernels use.  which = 0: int8 inputs (K = 64, v_mfma_i32_16x16x64_i8), A/B given as
 * int8, D int32.  which = 1: bf16 inputs (K = 32, v_mfma_f32_16x16x32_bf16), A/B given as
 * fp32 values exactly representable in bf16, D fp32.  which = 2: fp32 inputs (K = 4,
 * v_mfma_f32_16x16x4_f32), D fp32.  All pointers are device memory:
 * A row-major [16][K], B row-major [K][16], D row-major [16][16].
 */
int rxmet_selftest_mfma(int which, const void *A, const void *B, void *D, void *stream);

/*
 * The form that rxmet_experts_linear_int8 takes for `rows` places of `experts` experts with `weight_rows`
 * weight rows (N, gated 2 N) each.  0, 1: few rows, four waves or one for 32 weight rows; 2, 3, 4: tiles of
 * 128 weight rows x 64 places, 128 x 128 and 256 x 256.
 */
int rxmet_selftest_experts_form(int64_t rows, int64_t experts, int64_t weight_rows);

#ifdef __cplusplus
}
#endif

#endif /* RXMET_SELFTEST_H_ */
