/*
 * tca_op.h — C ABI of the operator programs: the operators of a transformer's
 * dense sublayer, forward and backward, and of its attention over a paged cache,
 * as programs of hand-written kernels.
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
 *
 * The operators of an attention sublayer work on a cache of pages, k and v
 * [PAGES, HK, PAGE, D], PAGE tokens of HK key heads each. Row s of a table [S, P]
 * names the pages of sequence s in order: its token p lies in page table[s][p /
 * PAGE], row p % PAGE, its slot being page * PAGE + row. The new tokens of all
 * sequences are the rows of one batch of T, those of sequence s from starts[s]
 * to starts[s + 1] - 1. Lengths stay on the GPU: one captured launch serves every
 * batch of its extents. Their lists (page_table's tensors, pos, slot, freq, table,
 * starts, lens, lse) may start at any element, so that slices of longer lists do; all
 * else starts on 16 bytes.
 *
 *   page_table            (no attributes; tensors i32)       free dim page, at least 1
 *       held [S], fresh [S], free [F], first [1]
 *       -> table [S, P], starts [S + 1], lens [S], pos [T], slot [T], next [1]
 *       Sequence s holds held[s] tokens and gets fresh[s] more (below 0: 0). Columns
 *       of table that its new tokens are the first in are stored, from free[first]
 *       on, in the order of the sequences; the others stay, and those of held tokens
 *       are read. next: the first page not taken. starts, lens (held and new), pos
 *       and slot of each new token; rows behind the last token are -1. A token
 *       whose page lies behind the table's P columns or the list's end has slot -1
 *       (and such a column -1), and slots have to stay below 2^31. Tokens from T on
 *       have no place in pos and slot (nothing stores their keys); table, starts,
 *       lens and next are those of all new tokens whatever T is.
 *   rotary                elem=f32|bf16|f16 [interleaved] [inverse]       scalar scale
 *       x [T, H, D], pos [T] i32, freq [F] f32 -> y [T, H, D]             2 F <= D, F <= 512
 *       (T below 2^26: a launch has less than 2^32 lanes; rotary_cache the same)
 *       pair i < F of a head, (a, b) = x[i], x[F + i] (interleaved: x[2 i], x[2 i + 1]):
 *       scale (a c - b s, b c + a s), c and s of the angle pos freq[i]; features
 *       from 2 F on are copied. inverse: s -> -s, the gradient of x from that of y.
 *   rotary_cache          elem=f32|bf16|f16 [interleaved]                 scalar scale
 *       x [T, HK G + HK + HK, D] (queries, keys, values), pos [T], slot [T] i32, freq [F] f32
 *       -> q [T, HK, G, D], k, v [PAGES, HK, PAGE, D]
 *       Queries and keys as rotary turns them; keys and values of a row whose slot
 *       lies in the cache are stored there, the rest of k and v stays. Slots of a
 *       launch differ: of rows with one slot any may be stored, in parts.
 *   paged_attention       elem=bf16|f16 [stats] [window]       scalar scale; window: a free dim, at least 1
 *       q [T, HK, G, D], k, v [PAGES, HK, PAGE, D], table [S, P], starts [S + 1], lens [S] i32
 *       -> y [T, HK, G, D], (lse [T, HK, G] f32)              D a multiple of 8, 8 to 256
 *       Sequence s holds lens[s] tokens, its n rows the last n of them. A row sees
 *       the keys up to its own (window: the last `window` of these), not those
 *       whose entry of the table names no page or lies behind its P columns.
 *       y = sum_j p_j v_j, p the softmax of scale q . k_j; lse = log sum_j exp(scale q . k_j),
 *       to merge with attention over other keys. A row that sees no key has y = 0
 *       and lse = -inf. Rows that no sequence has are left as they were; of starts that
 *       go past T, the rows that are there keep their positions; starts have to
 *       ascend (rows that two sequences name are stored by either). Scores and sums
 *       are 32-bit; probabilities are rounded to elem for the product with v. Values
 *       that are not finite reach the rows that see them only. 77 MB of workspace at
 *       128 features, up to 85; the allocation-free launch has enough for T G of at
 *       most 93 rows of 128 features.
 *
 * y may be x in rotary; otherwise nothing of theirs overlaps.
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
