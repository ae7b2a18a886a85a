/* C entry points of the gated feed-forward block for training: forward that keeps what the backward needs, and backward.
 * No counterpart in the reference; see csrc/src/gated_ffn.cu. */
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { PURLIN_ACT_SILU = 0, PURLIN_ACT_GELU = 1 };   /* GELU: the form with the tanh */

/* Bytes of the saved pre-activations of `tokens` rows (gate and up, three bytes a value). */
size_t purlin_ffn_saved_bytes(int tokens, int intermediate);

/* hOut[tokens, I] = act(x Wg^T) * (x Wu^T), bf16, with wGateUp [2 I, hidden] (16 rows of gate and 16 of up in turn), and, where `saved` is
 * given, the pre-activations in it. y[tokens, hidden] = hOut wDown^T, unless y is NULL. No output overlaps an operand or another output, here and below. All row-major, 16-byte aligned; hidden a multiple of 8,
 * intermediate of 16. Below 2^29 of each. status: 4 words that the device can write, or NULL: {code, where, tile, k-block} of the first wait inside a
 * kernel that gave up, two seconds and 4 us for every k-block of 64 that a CTA walks; what was not finished by then is not written. */
int purlin_ffn_forward(const void* x, const void* wGateUp, const void* wDown, void* hOut, void* saved, void* y, int tokens, int hidden,
                       int intermediate, int activation, uint32_t* status, void* stream);

/* Gradients for dy [tokens, hidden]; h and saved from the forward. dz [tokens, 2 I]: workspace that holds the gradient of the
 * pre-activations (interleaved like wGateUp's rows). dx, dGateUp, dDown: any of them may be NULL and is then not computed; where neither dx nor
 * dGateUp is wanted, wDown, saved and dz are not touched. workspace: as many bytes as purlin_ffn_workspace_bytes() says for the same gradients
 * on the current device; with fewer, or NULL, dx may take longer. */
size_t purlin_ffn_workspace_bytes(int tokens, int hidden, int intermediate, int wantDx, int wantGateUp, int wantDown);
int purlin_ffn_backward(const void* x, const void* wGateUp, const void* wDown, const void* h, const void* saved, const void* dy, void* dz,
                        void* dx, void* dGateUp, void* dDown, void* workspace, size_t workspaceBytes, int tokens, int hidden, int intermediate,
                        int activation, uint32_t* status, void* stream);

#ifdef __cplusplus
}
#endif
