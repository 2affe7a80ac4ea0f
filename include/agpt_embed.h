/*
 * agpt_embed.h — C ABI of the token embedding (libagpt_attn.so, gfx950): a
 * scaled lookup and the table's gradient by sorted tokens.
 *
 * Shares the conventions of agpt_attn.h: int status (AGPT_OK = 0) with the
 * message in agpt_last_error(), DEVICE pointers owned by the caller, work
 * ordered on the stream passed in (NULL = default stream), deterministic
 * results. Nothing is allocated and no call waits for the GPU, so all of them
 * may be captured into a graph.
 *
 * Tokens are int32 (token_bits 32) or int64 (64). A token outside [0, V) is
 * padding: its row of x is zero and its row of dx counts nowhere.
 */
#ifndef AGPT_EMBED_H
#define AGPT_EMBED_H

#include <stdint.h>

#include "agpt_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* x[t, :] = scale * table[tokens[t], :] for t < T. table [V, D] and x [T, D]
 * are contiguous, both of `dtype` (AGPT_DTYPE_*); the product is formed in
 * fp32 and rounded once. x must not overlap table. */
int agpt_embed_fwd(const void* table, const void* tokens, int token_bits, float scale, void* x, int64_t T, int64_t V,
                   int D, int dtype, void* stream);

/* A plan of the gradient: the rows sorted by token, stable. `plan` is an int32
 * buffer of agpt_embed_plan_ints(T, V) entries,
 *     order [T]        rows in ascending token, rows of one token ascending,
 *                      padding last
 *     keys [T]         their tokens (V for padding)
 *     offsets [V + 1]  where each token's rows start, and where padding does
 * filled from tokens [T]; it holds for any dx and D until the tokens change.
 * workspace: at least agpt_embed_plan_workspace_bytes(T, V) bytes, free again
 * after the call. T and V below 2^31 - 4096. */
int64_t agpt_embed_plan_ints(int64_t T, int64_t V);
int64_t agpt_embed_plan_workspace_bytes(int64_t T, int64_t V);
int agpt_embed_plan(const void* tokens, int token_bits, int64_t T, int64_t V, int32_t* plan, void* workspace,
                    int64_t workspace_bytes, void* stream);

/* d_table [V, D] fp32, every row written (zeros for tokens that do not
 * occur):  d_table[v, :] = scale * sum over rows t of token v of dx[t, :].
 * dx [T, D] of `dtype`, row stride ld_dx elements. The sums are fp32 in an
 * order fixed by the plan alone: two calls give the same bytes. workspace: at
 * least agpt_embed_bwd_workspace_floats(T, D) floats. */
int64_t agpt_embed_bwd_workspace_floats(int64_t T, int D);
int agpt_embed_bwd(const void* dx, int64_t ld_dx, const int32_t* plan, float scale, float* d_table, float* workspace,
                   int64_t workspace_floats, int64_t T, int64_t V, int D, int dtype, void* stream);

/* The same from the tokens themselves, for a batch that comes once: short
 * batches in one launch that sorts each token range on the fly, longer ones by a
 * plan made in the workspace (at least agpt_embed_bwd_tokens_workspace_bytes
 * bytes). Its sums may be in another order than a plan's; the order depends on
 * the tokens and sizes alone. */
int64_t agpt_embed_bwd_tokens_workspace_bytes(int64_t T, int64_t V, int D);
int agpt_embed_bwd_tokens(const void* dx, int64_t ld_dx, const void* tokens, int token_bits, float scale, float* d_table,
                          void* workspace, int64_t workspace_bytes, int64_t T, int64_t V, int D, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AGPT_EMBED_H */
