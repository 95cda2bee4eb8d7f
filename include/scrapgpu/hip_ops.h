/* The hip backend's serving ops: what lies between a transformer layer's q/k/v products and its
 * output product when many requests are served from a paged cache of keys and values. They run
 * through scrapgpu_op_execute, plans and scrapgpu_hip_op_execute_static like every other op; no
 * counterpart in the reference's GPU backends.
 *
 * The cache. k_cache and v_cache are [D, page_size, Hk, n_pages] tensors (any strides that are
 * multiples of 16 bytes, nb0 the element size). Request b's token j lies in page table[j / page_size, b]
 * at place j % page_size; a "slot" is page * page_size + place. page_size is a power of two; ATTENTION_PAGED
 * reads pages of 16 places or more, the other ops take smaller ones too.
 * Everything the device reads as an index (pages, slots, starts, lengths) is kept inside the tensors
 * by the kernels; what an index out of range does is said at each op.
 *
 * An output must not overlap an input or another output, except where an op allows it. */
#ifndef SCRAPGPU_HIP_OPS_H
#define SCRAPGPU_HIP_OPS_H

#include "scrapgpu/op.h"

#ifdef __cplusplus
extern "C" {
#endif

/* SCRAPGPU_OP_PAGED_PLAN: pages, slots and positions of one step, from the requests' lengths.
 * All tensors are I32. With B requests, a table of W entries a request and T tokens a step:
 *   inputs   past [B]     tokens that each request has in the cache
 *            fresh [B]    its new tokens; 0: none; negative: the request has ended
 *            free [1]     how many entries of the pool are free pages
 *   outputs  table [W, B] read and written: entry j of request b is its page j
 *            pool [n]     read and written: entries 0 .. free - 1 are the free pages, the last is taken first
 *                         (n: all pages that there are; one that comes back to a full pool is lost)
 *            left [2]     free pages after the step; requests that were refused
 *            q_start [B + 1], kv_len [B]   what ATTENTION_PAGED takes: request b's new tokens are
 *                         q_start[b] .. q_start[b + 1], its tokens with them kv_len[b] (0 if it has ended)
 *            pos [T], slots [T]   each new token's position and slot; past the last token 0 and -1
 * First the pages of ended requests go back to the pool, in order; then requests take pages in
 * order. One that would pass W pages is refused (it gets no token, kv_len = past); the first that
 * passes T or the free pages is refused with all new tokens after it. Nothing else of table and
 * pool is written. kv_len may be past itself and left's first element free itself (a step that is
 * replayed then carries its own state); otherwise no tensors may overlap. B is at most 2048. */
typedef struct scrapgpu_paged_plan_params {
    size_t struct_size;
    uint32_t page_size;
} scrapgpu_paged_plan_params;

/* SCRAPGPU_OP_ROPE_AXES: inputs [x (D x H x T), pos (I32, A x T)], output [y (D x H x T)]; x and y
 * F32, F16 or BF16. Of each head's D elements the first n_dims are turned in pairs: pair i is
 * (i, i + n_dims / 2), or (2i, 2i + 1) if `adjacent`, and
 *   y_first = x_first cos a - x_second sin a,  y_second = x_first sin a + x_second cos a,
 *   a = pos[axis(i), t] * scale * base^(-2i / n_dims);
 * the others are copied. axis(i): the first sections[0] pairs follow axis 0, the next sections[1]
 * axis 1 and so on; if `interleaved`, pair i follows axis r = i % A where r > 0 and
 * i < A * sections[r], else axis 0. sections sum to n_dims / 2 (interleaved: are checked against it);
 * all zero is one axis. A is 1 to 4. Angles are exact to 2^-24 of a turn for every 32-bit position
 * (|scale| at most 8, base at least 1).
 * y may be x itself (the same tensor). The frequencies run on from axis to axis, as text models with
 * three axes have them. Image encoders often start them anew for each of A equal sections, theta^(-2Aj / n_dims)
 * for its j-th pair: that is base = theta^A with the positions of axis a multiplied by theta^a.
 *
 * SCRAPGPU_OP_ROPE_AXES_STORE: inputs [q (D x Hq x T), k (D x Hk x T), v (D x Hk x T), pos, slots
 * (I32, T)], outputs [y (D x Hq x T), k_cache, v_cache]: q and k turned as above, q into y and k with
 * v into the cache at the tokens' slots. A slot outside the cache (-1) stores nothing. q, k, v
 * have one type, the caches one type. y may be q itself. Slots must differ. */
typedef struct scrapgpu_rope_axes_params {
    size_t struct_size;
    uint32_t n_dims;
    uint32_t sections[4];
    uint32_t adjacent;
    uint32_t interleaved;
    float base;
    float scale;
} scrapgpu_rope_axes_params;

/* y[:, h, t] = sum_j softmax_j(scale q[:, h, t] . k_j) v_j over the keys that token t sees, head h of
 * Hq reading key head h / (Hq / Hk). q, k, v are F16 or BF16 (one type), y that type or F32; D is a
 * multiple of 8, at most 256; nb0 is the element size, all other strides and offsets multiples of 16
 * bytes. Scores, maxima and sums are f32; for the second product the softmax weights are sums of terms of
 * the inputs' type: y F32 two of F16 (22 bits) or three of BF16 (24); 16-bit y two where requests have few
 * new tokens (see max_query), else one, rounded. `causal`: the i-th
 * of n new tokens of a request with m keys sees keys 0 .. m - n + i; otherwise it sees all m. A token
 * that sees no key, or that belongs to no request, gets zeros. What a token does not see does not
 * reach its result, whatever its value (NaN included); a value of Inf or NaN that it sees does, however
 * small the weight (a call that meets one where all its tokens see it reads the values twice).
 * Scores (scale q . k) may be up to 2^24 in magnitude, beyond which f32 tells few of them apart and F16 weights
 * overflow; BF16 values up to 2^100 for sums of weights and values to stay finite.
 *
 * SCRAPGPU_OP_ATTENTION_PROMPT: inputs [q (D x Hq x T), k (D x Hk x Tk), v (D x Hk x Tk), q_start
 * (I32, B + 1) and optionally k_start (I32, B + 1; q_start if absent, Tk = T then)], output [y
 * (D x Hq x T)]: request b's tokens are q_start[b] .. q_start[b + 1] of q and k_start[b] ..
 * k_start[b + 1] of k and v.
 *
 * SCRAPGPU_OP_ATTENTION_PAGED: inputs [q (D x Hq x T), k_cache, v_cache, table (I32, W x B), q_start
 * (I32, B + 1), kv_len (I32, B)], output [y]: the keys of request b are its kv_len[b] tokens in the
 * cache, its new ones among them. A page number outside the cache reads the nearest page. Pages
 * have 16 places or more.
 *
 * Starts are ascending from 0; what they do not cover or cover twice is undefined in value only.
 * max_query: no request has more new tokens than this (0: not known). It selects the kernel, so that
 * results of different values may differ in rounding; a wrong one costs time only. The same call gives
 * the same bits each time. */
typedef struct scrapgpu_attention_params {
    size_t struct_size;
    float scale;
    uint32_t causal;
    uint32_t max_query;
} scrapgpu_attention_params;

#ifdef __cplusplus
}
#endif

#endif
