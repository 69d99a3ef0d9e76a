/*
 * tca_op.h — C ABI of the operator programs: the operators of a transformer's
 * dense sublayer, forward and backward, as programs of hand-written kernels.
 *
 * An operator program is what tca_emit makes of a DSL program: a HIP source,
 * a launch plan and the hipcc arguments that build the code object. It loads
 * with tca_program_load and launches with tca_program_launch (or _noalloc) of
 * tca_rt.h, under the same shape contract, workspaces, streams and errors. No
 * counterpart in the reference, whose DSL has no backward pass and stores
 * contractions in f32.
 *
 * `attributes` are words separated by spaces, key=value or a flag:
 *
 *   layer_norm            elem=f32|bf16|f16 [weight=f32] [nobias] [stats]
 *       x [R, C], gamma [C], (beta [C]) -> y [R, C], (mean [R], rstd [R]);  scalar eps
 *   layer_norm_backward   elem=f32|bf16|f16 [weight=f32] [nobias] [residual]
 *       dy [R, C], x [R, C], gamma [C], mean [R], rstd [R], (dres [R, C])
 *       -> dx [R, C], dgamma [C], (dbeta [C])
 *   linear                elem=bf16|f16 [act=A] [bias] [residual] [save]
 *       x [M, K], w [K, N], (b [N]), (res [M, N]) -> y [M, N], (z [M, N])
 *       y = res + act(z), z = x w + b
 *   linear_backward       elem=bf16|f16 [act=A] [bias]
 *       dy [M, N], x [M, K], w [K, N], (z [M, N])
 *       -> (dz [M, N]), dx [M, K], dw [K, N], (db [N])      z and dz with an act
 *   gated                 elem=bf16|f16 [act=A] [bias] [save]
 *       x [M, K], wg [K, N], wu [K, N], (bg [N], bu [N]) -> h [M, N], (g, u [M, N])
 *       h = act(g) u, g = x wg + bg, u = x wu + bu
 *   gated_backward        elem=bf16|f16 [act=A] [bias]
 *       dh [M, N], x [M, K], wg [K, N], wu [K, N], g [M, N], u [M, N]
 *       -> dg [M, N], du [M, N], dx [M, K], dwg [K, N], dwu [K, N], (dbg [N], dbu [N])
 *
 * with A = none, relu, silu, gelu (by the normal distribution) or gelu_tanh;
 * a gated pair takes silu where none is given. Tensors are of type elem;
 * mean and rstd are f32, and with weight=f32 so are gamma, beta and their
 * gradients. Parentheses mark the tensors that an attribute brings. Sums are
 * 32-bit, every result is rounded once, but that the products of a backward
 * pass read dz (dg, du) as stored.
 *
 * Outputs overlap neither each other nor an input, except that y may be res
 * and dx may be dres, exactly. Any extent may be 0: K = 0 leaves the bias, M =
 * 0 or R = 0 gives zero weight gradients; rows of no elements have a mean and
 * rstd of NaN.
 */
#ifndef TCA_OP_H_
#define TCA_OP_H_

#include "tca_cg.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Emits operator `name` with `attributes` (NULL: none) for `target` (NULL:
 * gfx950). The result is read and freed with tca_emit_* of tca_cg.h. Returns
 * TCA_OK, TCA_ERR_INVALID (a null argument), TCA_ERR_NOT_FOUND (no such
 * operator) or TCA_ERR_UNSUPPORTED (an attribute or a value that it does not
 * take); the message is tca_op_last_error() of the calling thread. */
int tca_op_emit(const char* name, const char* attributes, const char* target, tca_emit_result* out);
/* The program's name as the emitted symbols carry it (owned by the result). */
const char* tca_op_program_name(tca_emit_result r);
const char* tca_op_last_error(void);
/* The operators and the attributes each takes, one line each. */
const char* tca_op_list(void);

#ifdef __cplusplus
}
#endif

#endif /* TCA_OP_H_ */
