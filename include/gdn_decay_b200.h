/*
 * gdn_decay_b200.h — C ABI of linear attention with a decay per head, beside
 * the gated-delta-rule entry points of gdn_b200.h (same library, same status
 * codes, same k-last state layout and pools), and of the 8-bit state cache
 * that parks pool slots of either recurrence.
 *
 * For v-head h, reading q/k head h / (HV / H), with state S [V, K]:
 *
 *   S_t = exp(g_t) S_{t-1} + v_t k_t^T        o_t = scale * S_t q_t
 *
 * g = log_decay: [HV] fp32 (decay_per_token == 0: one number per v-head) or
 * one number per token and v-head (decay_per_token == 1: [T,HV] for the
 * prefill, [B,T,HV] otherwise).  g <= 0 is meant; -inf forgets the state.
 * Values below -104, where exp rounds to zero in fp32, act like -104.
 *
 * Contract as in gdn_b200.h: device pointers, sizes and a CUDA stream of the
 * current device; nothing is allocated, the host never waits, argument errors
 * are reported before anything is launched.  K == V == 128, H >= 1,
 * HV % H == 0.  scale == 0 means 1/sqrt(K).  q, k, v, out, states, pools and
 * workspaces 16-byte aligned (the prefill's states and workspace 32),
 * log_decay 4 bytes, index arrays their own size.
 * The reference project has no counterpart of these operators.
 *
 * Values that are not finite reach the outputs and states that the formula lets
 * them reach, and no others but where it is said below.  In the prefill and the
 * verification they may arrive as NaN where the formula has an infinity: operands
 * are split into terms, and infinity times a zero term is NaN.
 */
#ifndef GDN_DECAY_B200_H_
#define GDN_DECAY_B200_H_

#include <stddef.h>
#include <stdint.h>

#include "gdn_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Variable-length prefill over N sequences packed into T tokens: q, k
 * [T,H,K] bf16, v [T,HV,V] bf16, cu_seqlens [N+1] int32 or int64 (device),
 * state (NULL: zero) / new_state [N,HV,V,K] fp32, out [T,HV,V] bf16.
 *
 * cu_seqlens is read on the device only; entries are clamped to [0, T] and an
 * end before its start counts as no tokens, so a malformed array reads and
 * writes nothing out of bounds.  A sequence without tokens keeps its state
 * (zero when state is NULL).  Tokens outside [cu_seqlens[0], cu_seqlens[N]) get a zero output and
 * are not read into any state, whatever they hold.  new_state may equal state
 * (in-place update); any other overlap of inputs and outputs is not allowed
 * (and refused for the states).
 * The products run on 64-token chunks, so a value of v that is not finite
 * spoils the outputs of its whole chunk, those of earlier tokens too.
 *
 * Precision: new_state is advanced in fp32.  For the outputs the state before a
 * chunk and the decayed scores are rounded to bf16 once each, so an output is
 * off by up to 2^-8 of scale * (|S| |q| + sum |decayed score| |v|) beside its own
 * rounding; the other operators keep two bf16 terms (2^-16) or fp32 there.
 *
 * workspace: device memory, 32-byte aligned, at least
 * gdn_decay_prefill_workspace_bytes(N, T, HV) bytes (which may be 0; the
 * workspace may then be NULL); contents on entry do not matter.  Calls whose
 * work overlaps on the GPU need a workspace each.
 */
int gdn_decay_prefill_fwd(const void *q, const void *k, const void *v, const float *state,
                          const float *log_decay, int decay_per_token, const void *cu_seqlens,
                          int cu_seqlens_is_int64, int N, int T, float scale, int H, int HV, int K,
                          int V, void *out, float *new_state, void *workspace,
                          size_t workspace_bytes, void *stream);

size_t gdn_decay_prefill_workspace_bytes(int N, int T, int HV);

/*
 * One token per batch entry: entry i advances the state in slot indices[i]
 * of pool_in (indices == NULL: slot i) and writes it to slot out_indices[i]
 * (NULL: the slot read) of pool_out.  q, k [B,H,K] bf16; v, out [B,HV,V]
 * bf16; pools [pool_size,HV,V,K] fp32 or bf16 (state_bf16; widened on load,
 * advanced in fp32, rounded to nearest-even once when stored).  pool_out may
 * equal pool_in; otherwise the two must not overlap, and only the slots that
 * are written change.  pool_in == NULL: zero states.
 *
 * An index outside [0, pool_size) marks padding: its output is zero and no
 * state is read or written.  An output slot outside the pool skips the write.
 * No slot may be written by one entry and read or written by another.
 * A pool (here and below) may have no slots, and then no address: every entry
 * is padding.
 */
int gdn_decay_decode_fwd(const void *q, const void *k, const void *v, const void *pool_in,
                         void *pool_out, int state_bf16, const void *indices,
                         const void *out_indices, int indices_int64, const float *log_decay,
                         int decay_per_token, float scale, int B, int H, int HV, int K, int V,
                         int pool_size, void *out, void *stream);

/* The largest tree gdn_decay_verify_fwd and gdn_decay_commit take. */
#define GDN_DECAY_TREE_MAX 64

/*
 * Attention for trees of drafted tokens over the pooled states: entry i's
 * node t (T <= GDN_DECAY_TREE_MAX nodes) continues from its parent node
 * parents[i, t] (in [0, t)) or, for -1, from the state in slot indices[i].
 * out[i, t] = scale * S q_t with S the state after the path down to and
 * including node t.  No state is written; a slot may be read by several
 * entries.  q, k [B,T,H,K] bf16; v, out [B,T,HV,V] bf16; parents [B,T] int32.
 *
 * A node whose parent is below -1 or not before it is padding, and so is a
 * node whose path meets one: its output is zero and its q, k and v are not
 * used, whatever they hold.  An index outside [0, pool_size): all of the
 * entry's outputs are zero.  A v of a node in use that is not finite spoils
 * the outputs of all its tree.
 */
int gdn_decay_verify_fwd(const void *q, const void *k, const void *v, const void *pool,
                         int state_bf16, const void *indices, int indices_int64,
                         const int *parents, const float *log_decay, int decay_per_token,
                         float scale, int B, int T, int H, int HV, int K, int V, int pool_size,
                         void *out, void *stream);

/*
 * The update that follows: entry i's state is advanced over the path of node
 * accepted[i] ([B] int32) of its tree and written to slot out_indices[i]
 * (NULL: the slot read) of the same pool.  accepted[i] == -1 accepts nothing,
 * and so does a node that does not exist or is padding: the state is then
 * only copied to the output slot.  Padding entries, output slots outside the
 * pool and the rule on shared slots as in gdn_decay_decode_fwd.
 */
int gdn_decay_commit(const void *k, const void *v, void *pool, int state_bf16, const void *indices,
                     const void *out_indices, int indices_int64, const int *parents,
                     const int *accepted, const float *log_decay, int decay_per_token, int B, int T,
                     int H, int HV, int K, int V, int pool_size, void *stream);

/* values that share one scale of the 8-bit state cache */
#define GDN_STATE_CACHE_GROUP 32

/*
 * 8-bit state cache: pool slot slots[i] is written to cache slot
 * cache_slots[i] (store) or read back from it (load), i < B.  A slot is
 * slot_elems consecutive values (HV * V * K; a multiple of 32), fp32 or bf16
 * (state_bf16) in the pool, one code each in codes [cache_size, slot_elems]
 * (int8, or e4m3 when e4m3 == 1) and one exponent byte for 32 of them in
 * exps [cache_size, slot_elems / 32].
 *
 * With top = 127 (int8) or 448 (e4m3), e is the smallest integer >= -127 with
 * max |x| <= top * 2^e over the group, the codes are x / 2^e rounded to
 * nearest-even (exact but for that rounding: the scale is a power of two) and
 * the byte is e + 127.  A group with a value that is not finite has the byte
 * 255 and zero codes, and reads back as NaN.  Reading back gives
 * code * 2^e (rounded to bf16 for a bf16 pool).
 *
 * A pair with either index outside its array is padding: nothing is read or
 * written.  No two pairs may write the same slot.
 */
int gdn_state_cache_store(const void *pool, int state_bf16, const void *slots,
                          const void *cache_slots, int slots_int64, void *codes, int e4m3,
                          unsigned char *exps, int B, long long slot_elems, int pool_size,
                          int cache_size, void *stream);

int gdn_state_cache_load(const void *codes, int e4m3, const unsigned char *exps,
                         const void *cache_slots, const void *slots, int slots_int64, void *pool,
                         int state_bf16, int B, long long slot_elems, int pool_size, int cache_size,
                         void *stream);

#ifdef __cplusplus
}
#endif

#endif /* GDN_DECAY_B200_H_ */
