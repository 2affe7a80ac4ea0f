/*
 * agpt_act8.h — C ABI of 8-bit activation checkpoints (libagpt_attn.so,
 * gfx950): activations that a backward pass needs again, kept in a quarter of
 * fp32's bytes, and the weight gradients formed from them.
 *
 * Shares the conventions of agpt_attn.h: int status (AGPT_OK = 0) with the
 * message in agpt_last_error(), DEVICE pointers owned by the caller, work
 * ordered on the stream passed in (NULL = default stream), deterministic
 * results. Nothing is allocated and no call waits for the GPU, so all of them
 * may be captured into a graph.
 *
 * A checkpoint of x [T, W] (W a multiple of 32) cuts each row into blocks of
 * 32 columns with one scale s = 2^(e - 127), e a byte in 1..254:
 *   relu = 0  the smallest s with max |x| <= 127 s; code 128 + rint(x / s),
 *             value (code - 128) s: off by at most s / 2
 *   relu = 1  the smallest s with max x <= 255 s; code 0 exactly where
 *             x <= 0, else rint(x / s) between 1 and 255, value code * s: off
 *             by at most s / 2, by less than s where rint would give 0, so
 *             that the mask x > 0 survives
 * (s from 2^-126 to 2^120). A block that holds an infinity, a NaN or more than
 * the top code at s = 2^120 has e = 255 and all of its values read as NaN. x / s is exact, so the codes do not depend on
 * how they are computed, and every value has at most 8 significant bits:
 * unpacking to bf16 is exact too.
 *
 * Layout: eight rows together, so that one lane's eight rows of four columns
 * are 32 consecutive bytes and their scales eight:
 *   codes  [ceil(T/8)][W/4][8 rows][4 columns]   agpt_act8_code_bytes(T, W)
 *   scales [ceil(T/8)][W/32][8 rows]             agpt_act8_scale_bytes(T, W)
 * Both 16-byte aligned. Rows past T hold the value 0.
 */
#ifndef AGPT_ACT8_H
#define AGPT_ACT8_H

#include <stdint.h>

#include "agpt_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

int64_t agpt_act8_code_bytes(int64_t T, int W);
int64_t agpt_act8_scale_bytes(int64_t T, int W);

/* Packs x [T, W] of `dtype` (AGPT_DTYPE_*), row stride ld_x elements. */
int agpt_act8_pack(const void* x, int64_t ld_x, int dtype, int relu, uint8_t* codes, uint8_t* scales, int64_t T, int W,
                   void* stream);

/* The values that a checkpoint stands for, into x [T, W] of `dtype`, row
 * stride ld_x elements. */
int agpt_act8_unpack(const uint8_t* codes, const uint8_t* scales, int relu, void* x, int64_t ld_x, int dtype, int64_t T,
                     int W, void* stream);

/* Weight and bias gradient of a linear layer whose input was checkpointed:
 *   dw [out, in] = sum over t of dy[t, :] ^T value[t, :],   db [out] = sum over t of dy[t, :]
 * dy [T, out] of `dtype`, row stride ld_dy (up to 2^25) elements; the checkpoint is [T, in];
 * dw and db fp32, written whole (db NULL: not formed). An fp32 dy enters the
 * bf16 matrix products as three parts that add up to it exactly, so nothing of
 * it is rounded (a part below 2^-126 may count as zero); the sums are fp32 in a
 * fixed order. A dy that is not finite makes the results that it enters
 * infinite or NaN. workspace: at least
 * agpt_act8_wgrad_workspace_floats(T, out, in) floats, 16-byte aligned, as dw
 * and db are. */
int64_t agpt_act8_wgrad_workspace_floats(int64_t T, int out_width, int in_width);
int agpt_act8_wgrad(const void* dy, int64_t ld_dy, int dtype, const uint8_t* codes, const uint8_t* scales, int relu,
                    float* dw, float* db, float* workspace, int64_t workspace_floats, int64_t T, int out_width,
                    int in_width, void* stream);

/* The same behind a ReLU whose outputs were checkpointed (relu = 1, [T, out],
 * its codes h_codes): dh [T, out] = dh_in where the ReLU's output was above
 * zero, else 0 (also where dh_in is not finite), and dw, db of the layer in
 * front of it, from dh and that layer's checkpointed input. One pass; dh is
 * contiguous, of `dtype`, and must not overlap dh_in. out a multiple of 32;
 * dh_in 16-byte aligned with a row stride of a multiple of 16 bytes. Takes the
 * place of agpt_relu_bwd and of the weight gradient's product where the
 * activations are checkpointed. */
int agpt_act8_relu_wgrad(const void* dh_in, int64_t ld_dh_in, int dtype, const uint8_t* h_codes, void* dh,
                         const uint8_t* codes, const uint8_t* scales, int relu, float* dw, float* db, float* workspace,
                         int64_t workspace_floats, int64_t T, int out_width, int in_width, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AGPT_ACT8_H */
