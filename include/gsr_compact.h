/*
 * gsr_compact.h -- C ABI of the compact-scene kernels: spherical-harmonic (SH)
 * coefficients in 4-bit microscaled floating point, colours (and their gradients)
 * straight from the codes, and eviction of the lightest Gaussians to a budget.
 * Same library (libgsr.so) and conventions as gsr.h: plain C, caller-owned device
 * pointers, void* stream = hipStream_t, 0 = success / non-zero = error with the
 * message in gsr_last_error().  Every call runs on the current device, only on
 * `stream`, allocates nothing and does not wait for the device: all of them can be
 * captured into a graph.
 *
 * Codes.  A row of K floats is cut into blocks of GSR_MX_BLOCK neighbours (the last
 * one of a row may be shorter).  Block scale: one byte s = E8M0, 2^(s - 127), with
 * s = max(floor(log2(max |x|)) - 2, -127) + 127 (s = 0 for a block of zeros); values:
 * E2M1 = sign, magnitude index into {0, .5, 1, 1.5, 2, 3, 4, 6}, rounded to nearest
 * with ties to the even index, saturating at 6.  A block that holds a NaN or an
 * infinity gets s = 255 and reads back as NaN throughout.  (The OCP MX v1.0 format
 * MXFP4 with its reference conversion.)  Row i: ceil(K / 8) 32-bit words at word
 * i * ceil(K / 8), value j in bits [4 (j % 8), 4 (j % 8) + 4) of word j / 8, the
 * unused bits of the last word 0; ceil(K / 32) scale bytes at i * ceil(K / 32).
 */
#ifndef GSR_COMPACT_H_
#define GSR_COMPACT_H_
#include <stddef.h>
#include <stdint.h>
#include "gsr.h"
#ifdef __cplusplus
extern "C" {
#endif

#define GSR_MX_BLOCK 32
#define GSR_MAX_WIDTH (1 << 20) /* words of a row, K or width below */

/* A launch has fewer than 2^32 threads: calls that would need more are refused (decoding more than 17e9
 * values, for one), before they write anything. */

/* R rows of K floats, row i at x + i * row_stride -> codes, scales (codes 4-B aligned). */
GSR_API int gsr_mx4_quantize(long long R, int K, const float* x, long long row_stride, uint32_t* codes,
                             uint8_t* scales, void* stream);
/* The other way round: x [R, K] contiguous. */
GSR_API int gsr_mx4_dequantize(long long R, int K, const uint32_t* codes, const uint8_t* scales, float* x,
                               void* stream);

/* Colours of P Gaussians from V camera positions (utils/sh_utils.py:57-112 eval_sh, + 0.5 and
 * clamp as forward.cu:20-71), colors [V, P, 3]:
 *   u = xyz - campos[v], d = u / |u| (0 where u is 0);
 *   p = 0.5 + Y_0 dc + sum_{1 <= k < (degree+1)^2} Y_k(d) rest_k;  colors = max(0, p).
 * dc: row i at dc + i * dc_stride (3 floats); codes / scales: rows of 3 (M - 1) floats
 * (coefficient-major, as the arena's features block).  0 <= degree <= 3,
 * (degree + 1)^2 <= M <= 16, 1 <= V <= GSR_MAX_VIEWS; campos: device [V, 3].  mask [V, P],
 * for the backward, or NULL: bit c of a byte is set where channel c has p >= 0 (decided in
 * 64 bits where 32 cannot). */
GSR_API int gsr_sh_colors(int P, int V, int degree, int M, const float* xyz, const float* dc, long long dc_stride,
                          const uint32_t* codes, const uint8_t* scales, const float* campos, float* colors,
                          uint8_t* mask, void* stream);
/* The same from fp32 features [P, M, 3] whose coefficients above the constant one are rounded
 * in the call.  codes / scales: rows of 3 (M - 1) values as gsr_mx4_quantize writes them, of which
 * those that `degree` reads are written; with mask what gsr_sh_colors_backward of the same
 * degree reads. */
GSR_API int gsr_sh_colors_quantize(int P, int V, int degree, int M, const float* xyz, const float* features,
                                   const float* campos, uint32_t* codes, uint8_t* scales, uint8_t* mask,
                                   float* colors, void* stream);
/* Gradients for dcolors [V, P, 3], summed over the views in order; a channel takes part
 * where the forward's mask has its bit.  Each of the outputs may be NULL: dxyz [P, 3] (0 where
 * u is 0); ddc [P, 3]; dfeatures [P, M, 3], coefficient 0 = d/d(dc), the others the gradient
 * of the decoded value (straight through the rounding), 0 above the degree. */
GSR_API int gsr_sh_colors_backward(int P, int V, int degree, int M, const float* xyz, const uint32_t* codes,
                                   const uint8_t* scales, const float* campos, const uint8_t* mask,
                                   const float* dcolors, float* dxyz, float* ddc, float* dfeatures, void* stream);

/* acc[i] <- decay * acc[i] + weights[i * stride], i < P (accumulated blend weights).  The weights
 * may be acc itself; weights that lie on another element's sum are refused. */
GSR_API int gsr_accumulate_weights(int P, const float* weights, long long stride, float decay, float* acc,
                                   void* stream);

/* Eviction to a budget.  A group is a range [begin, end) of rows (one scene of a merged
 * model); it keeps keep = min(budget, end - begin) of them: its last min(recent, keep)
 * rows and, of the others, the heaviest by weight (ties: the lowest row; NaN below
 * everything, -0 = +0).  ids gets the kept rows in ascending order, group after group
 * (sum of keep entries).  Groups are ascending and do not overlap; rows in no group are
 * not kept.  ws: gsr_keep_ws_bytes(P) bytes (0 for small P: then ws may be NULL), 16-B aligned,
 * used by this call only. */
#define GSR_KEEP_MAX_GROUPS 64
typedef struct gsr_keep_group {
    int begin, end;
    int keep;   /* 0 <= keep <= end - begin */
    int recent; /* 0 <= recent <= keep */
} gsr_keep_group;
GSR_API size_t gsr_keep_ws_bytes(int P);
GSR_API int gsr_keep_heaviest(int P, const float* weights, int n_groups, const gsr_keep_group* groups, int* ids,
                              void* ws, void* stream);

/* dst[j] = src[ids[j]], j < K, for n tensors of rows of `width` 32-bit words.  An id
 * outside [0, rows) gives a row of zeros.  `pad` words behind a destination's last row
 * are cleared too (the padding of an arena block).  A destination that overlaps the ids or
 * another tensor of the call is refused. */
typedef struct gsr_rows {
    const void* src;
    void* dst;
    int width;
    int rows;
    int pad;
} gsr_rows;
GSR_API int gsr_take_rows(int K, const int* ids, int n, const gsr_rows* tensors, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* GSR_COMPACT_H_ */
