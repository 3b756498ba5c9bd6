/*
 * unoq_mx.h -- microscaled 4-bit (MX4) operators of libunoq_cuda.so: quantisation, the product with
 * 4-bit weights, and a mixture-of-experts layer on them.
 *
 * An MX4 matrix of rows x k holds e2m1 values (+-0, 0.5, 1, 1.5, 2, 3, 4, 6) in blocks of 32 along
 * a row, each block with one scale 2^(s - 127), s = 0..254; s = 255 makes the block NaN. It has two
 * layouts:
 *   UG_MX4_STORED   codes[r * ceil(k/2) + j/2], the even j in the low nibble, and
 *                   scales[r * ceil(k/32) + j/32]: the exchange form of files.
 *   UG_MX4_OPERAND  what the products read, 128 rows to a tile, the tiles of 128 rows next to each other:
 *                   codes in tiles of 256 values, ((r / 128) * K + j / 256) * 16384 + (r % 128) * 128 +
 *                   (j % 256) / 2 with K = ceil(k/256), and scales in tiles of 128 values,
 *                   ((r / 128) * 2K + j / 128) * 512 + (r % 32) * 16 + (r / 32 % 4) * 4 + (j / 32 % 4).
 *                   Values and scale bytes past k, up to 256 K, are zero; rows past the last, in its
 *                   tile, are zero from ug_mx4_pack and left as they were by ug_mx4_quantize.
 * A last block or tile may be partial: rows and k are free (k >= 1), as far as the kernels count in 32 bits.
 * With T = 2 ceil(k/256), the scale tiles along a row:
 *   quantise, dequantise       rows * T < 2^31, k <= 2^30
 *   pack                       the same, rows being all matrices' with their padding (ug_mx4_pack_rows)
 *   products                   k <= UG_MX4_MAX_K, m <= UG_MX4_MAX_M, (n + 127) T < 2^31, and (m + 255) T < 2^31,
 *                              with 16-bit activations (4 m + 256) T < 2^31
 *   experts                    the limits below
 *
 * Every array is DEVICE memory of one device, `stream` is a cudaStream_t of that device (NULL: its
 * legacy default stream). Calls check their arguments, launch on `stream` and return without
 * waiting; they allocate nothing and may be captured into a CUDA graph. A workspace belongs to
 * one call in flight: calls that may overlap, and graphs that may run at the same time, each need
 * their own. No call needs anything from its workspace's earlier contents. Outputs must not overlap
 * inputs. Zero rows are a call that does nothing.
 *
 * Codes: 18 a size, type, stride or layout out of range, 22 a null, host, misaligned or
 * other-device pointer or a workspace too small, 2001 CUDA error, 2002 no device. ug_last_error has
 * the reason. A device-side wait that ran out of time (about 2 s) is reported by ug_mx4_check.
 */
#ifndef UNOQ_MX_H
#define UNOQ_MX_H
#include <stddef.h>
#include <stdint.h>

#include "unoq_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

enum UgMxType { UG_F32 = 0, UG_F16 = 1, UG_BF16 = 2 };
enum UgMx4Layout { UG_MX4_STORED = 0, UG_MX4_OPERAND = 1 };

#define UG_MX4_MAX_K 65536        /* longest row of a product */
#define UG_MX4_MAX_M 2097152      /* rows of a product's activations */
#define UG_MX4_MAX_TOKENS 128     /* ug_mx4_experts: rows of x */
#define UG_MX4_MAX_EXPERTS 256
#define UG_MX4_MAX_TOP_K 16
#define UG_MX4_MAX_WIDTH 16384    /* ug_mx4_experts: model and hidden width */

/* Bytes of an MX4 matrix's two arrays in `layout`; 0 for an unknown layout. */
UG_API size_t ug_mx4_codes_bytes(int layout, uint32_t rows, uint32_t k);
UG_API size_t ug_mx4_scales_bytes(int layout, uint32_t rows, uint32_t k);

/* x (rows x k of `type`, rows `stride` elements apart) -> MX4. Per block: s = 127 + floor(log2 of the
 * largest magnitude) - 2, at least 0; values x / 2^(s - 127) to the nearest e2m1, ties to the even
 * code, at most 6 in magnitude. A block that holds a NaN or an infinity gets s = 255, codes 0. */
UG_API int ug_mx4_quantize(const void *x, int type, uint32_t rows, uint32_t k, uint64_t stride, int layout,
                           uint8_t *codes, uint8_t *scales, void *stream);
/* The values back, into y (rows x k of `type`, rows `stride` elements apart), rounded to it once. */
UG_API int ug_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, int layout, uint32_t rows, uint32_t k,
                             void *y, int type, uint64_t stride, void *stream);
/* `count` stored matrices of rows x k, one after another -> operand layout, each matrix's rows padded
 * to whole tiles of its own. paired = 1: rows is even, the first half of each matrix are gate rows
 * and the second half up rows; a tile holds 64 gate rows, then the 64 up rows beside them
 * (ug_mx4_experts reads gate_up so). Array sizes: ug_mx4_pack_rows rows of the operand layout. */
UG_API int ug_mx4_pack(const uint8_t *codes, const uint8_t *scales, uint32_t count, uint32_t rows, uint32_t k,
                       int paired, uint8_t *packed_codes, uint8_t *packed_scales, void *stream);
UG_API uint32_t ug_mx4_pack_rows(uint32_t count, uint32_t rows, int paired);

/* y[i][j] = sum_t a[i][t] * w[j][t], a m x k and w n x k in operand layout, accumulated in 32 bits and
 * rounded once to `type`; rows of y `stride` elements apart. */
UG_API int ug_mx4_matmul(const uint8_t *a_codes, const uint8_t *a_scales, uint32_t m, const uint8_t *w_codes,
                         const uint8_t *w_scales, uint32_t n, uint32_t k, void *y, int type, uint64_t stride,
                         void *stream);
/* The same with 16-bit activations x (m x k, UG_F16 or UG_BF16, rows `x_stride` elements apart), which
 * are not rounded to MX4 but held as 8-bit pieces on one scale to a block of 32: a value is kept exactly
 * while it is above 2^-12 of the largest of its block, and to within 2^-21 (UG_F16: 2^-25) of that largest
 * below, so that what is far smaller than a loud neighbour loses bits, and in the end all of them. A block with a NaN or an infinity
 * makes its row of y NaN. */
UG_API int ug_mx4_matmul_x16(const void *x, int x_type, uint64_t x_stride, uint32_t m, const uint8_t *w_codes,
                             const uint8_t *w_scales, uint32_t n, uint32_t k, void *y, int type, uint64_t stride,
                             void *workspace, size_t workspace_bytes, void *stream);
/* Bytes of that call's workspace; 0 (workspace may be NULL) for few rows. */
UG_API size_t ug_mx4_matmul_x16_workspace(uint32_t m, uint32_t k, int x_type);

/* A mixture-of-experts layer for a few tokens. */
typedef struct {
    uint32_t experts, top_k, d, f;   /* experts >= top_k >= 1; model width d, hidden width f */
    int normalize;                   /* 1: softmax over the chosen experts' logits; 0: over all experts' */
    int type;                        /* x, y and router: UG_F16 or UG_BF16 */
    const void *router;              /* experts x d */
    const float *bias;               /* experts, added to the logits; or NULL */
    const uint8_t *gate_up_codes, *gate_up_scales;   /* ug_mx4_pack(experts, 2f, d, paired) */
    const uint8_t *down_codes, *down_scales;         /* ug_mx4_pack(experts, d, f, not paired) */
} UgMx4Experts;

/* y[t] = sum over the top_k experts e of token t (largest logits x[t] . router[e] + bias[e], ties to the
 * lowest index) of p_e * down_e (silu(gate_e x[t]) * (up_e x[t])). Logits, softmax and sums are held in
 * 32 bits; a hidden value is kept to within 2^-19 of itself, or 2^-29 of the largest of its block of 32,
 * or 2^-137, where that is more. Rows of x and y are x_stride and y_stride elements apart; tokens <=
 * UG_MX4_MAX_TOKENS. A logit that is not a number comes before every number: its expert is chosen, and the
 * token's weights and its row of y are NaN. `chosen` and `weights` (tokens x top_k, either may be NULL) receive the experts in
 * falling order of their logits and the p_e. */
UG_API int ug_mx4_experts(const UgMx4Experts *layer, const void *x, uint64_t x_stride, uint32_t tokens, void *y,
                          uint64_t y_stride, int32_t *chosen, float *weights, void *workspace, size_t workspace_bytes,
                          void *stream);
UG_API size_t ug_mx4_experts_workspace(const UgMx4Experts *layer, uint32_t tokens);

/* Waits for `device` and returns 0, 2001 after a CUDA error, or 2003 when a wait inside one of the
 * product kernels ran out of time since the last check (their outputs are then undefined). */
UG_API int ug_mx4_check(int device);

#ifdef __cplusplus
}
#endif
#endif
