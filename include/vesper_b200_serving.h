/*
 * vesper_b200 -- C ABI, operators of a serving batch: norms of queries and keys with the position rotation in one pass, attention over packed
 * prompts of different lengths, and a key / value cache held in 4 bits with the attention that reads it.  The conventions of vesper_b200.h hold:
 * borrowed pointers, nothing allocated, the caller's stream, no synchronisation, status codes; a workspace serves one call at a time, so that calls that may run
 * at once (on two streams, in two graphs) need one each.  The reference has none of these operators; they stand
 * beside the ones that replace its apply_rotary_emb (src/nn/functional.cpp:424-494), KVCache::update (src/nn/transformer.cpp:56-93) and
 * scaled_dot_product_attention (src/nn/functional.cpp:370-422).
 *
 * As they are used: the projection of a packed batch of prompts -> vb200_qk_norm_rope -> vb200_prefill_packed_fwd, and vb200_kv4_append of the same
 * keys and values; per generated token vb200_qk_norm_rope -> vb200_decode_kv4_fwd, which appends the token before it attends.
 */
#ifndef VESPER_B200_SERVING_H
#define VESPER_B200_SERVING_H

#include "vesper_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Where the tokens of a call go, or come from, in a cache of `seqs` sequences of `cap` rows each: token (b, t) belongs to row rows[b * T + t] of
 * sequence seq_ids[b * T + t] (seq_ids null: sequence b).  A negative row names no place: the token is left out (padding).  A row of cap or above, or a
 * sequence out of [0, seqs), is left out too and sets the status word (VB200_ERR_CACHE_OVERFLOW; its detail names the
 * sequence).  A call may name a place once only. */
typedef struct vb200_rows {
    const int32_t* rows;         /* device [B, T] contiguous */
    const int32_t* seq_ids;      /* device [B, T] contiguous, or null */
    int32_t seqs, cap;
} vb200_rows;

/* ---- norms of queries and keys with the rotation -------------------------------------------------
 * For every head of q and k, y = x / sqrt(mean(x^2) + eps) * weight over its D elements (norm == 0: y = x), then the pairs (y[2i], y[2i+1]) are turned
 * by the angle position * inv_freq[i] (rope.enabled == 0: not turned); all in fp32, rounded once.  The product position * inv_freq[i] is not rounded
 * to fp32 as apply_rotary_emb does it (a thousandth of a radian at position 16384): rotate the queries and the keys of one cache with one of the two.
 * Outputs stand like the inputs (and may be the same memory: q_out == q with the same strides; overlapping otherwise is not allowed, and neither are negative
 * strides, and strides of 0 in an output where there is more than one), or, with dst.rows, k_out and v_out are [dst.seqs, Hkv, dst.cap, D] caches and token (b, t) is written where `dst` says.
 * Any of q, k, v may be left out (ptr null together with its output's); v is copied, which needs an output of its own. */
typedef struct vb200_qk_norm_rope_args {
    size_t struct_size;
    int32_t device;
    void* stream;
    int32_t dtype;               /* of every tensor: VB200_F32, VB200_BF16 or VB200_F16 */
    int32_t B, Hq, Hkv, T, D;    /* D a multiple of 8, at most 128 */
    vb200_tensor4 q;             /* [B,Hq,T,D] */
    vb200_tensor4 k, v;          /* [B,Hkv,T,D] */
    vb200_tensor4 q_out, k_out, v_out;
    int32_t norm;                /* 1: normalise */
    float eps;
    const float* q_weight;       /* device fp32 [D], null: ones */
    const float* k_weight;
    vb200_rope rope;
    int32_t start_pos;           /* position of token t is start_pos + t ... */
    const int32_t* positions;    /* ... or this: device [B,T] contiguous */
    vb200_rows dst;              /* rows null: k_out and v_out stand like k and v */
} vb200_qk_norm_rope_args;
int vb200_qk_norm_rope(const vb200_qk_norm_rope_args* a);

/* ---- attention over packed prompts -----------------------------------------------------------------
 * `batch` sequences stand one behind the other: the queries of sequence i are the tokens [cu_seqlens_q[i], cu_seqlens_q[i+1]) of q and o, its keys and
 * values the tokens [cu_seqlens_k[i], cu_seqlens_k[i+1]) of k and v (null: the same as cu_seqlens_q).  The lengths stay on the device.  Causal aligns
 * the last query with the last key: query i of n_q sees key j of n_k iff j <= n_k - n_q + i.  A query that sees no key gets zeros and an lse of
 * -infinity; one whose scores are all -infinity gets NaN and an lse of -infinity (0 / 0 and ln 0).  Tokens behind the last sequence are neither read
 * (k, v) nor written (o, lse).  The running sums are fp32; the weights are rounded to `dtype` for their product with v.  NaN in a key makes the results of the
 * queries that see it NaN, the lse too.  A non-finite element of v reaches every query of its sequence that sees a key of its block of at most 112 keys (a
 * weight of zero times infinity is NaN), as in vb200_prefill_fwd.  Neither ever reaches another sequence.
 * The offsets have to ascend and to stay within the tokens given.  A sequence whose own two do not is left out; nothing outside the tensors is read or
 * written whatever they are. */
typedef struct vb200_prefill_packed_args {
    size_t struct_size;
    int32_t device;
    void* stream;
    int32_t dtype;               /* VB200_BF16 or VB200_F16 */
    int32_t batch, Hq, Hkv, D;   /* D 64 or 128; Hq a multiple of Hkv */
    int32_t total_q, total_k;    /* tokens of q / o and of k / v */
    int32_t causal;
    float scale;
    vb200_tensor4 q, o;          /* [total_q, Hq, D]: stride_s between tokens, stride_h between heads, both positive (stride_b is not looked at) */
    vb200_tensor4 k, v;          /* [total_k, Hkv, D] */
    float* lse;                  /* [Hq, total_q] contiguous fp32, nullable */
    const int32_t* cu_seqlens_q; /* device [batch + 1] */
    const int32_t* cu_seqlens_k; /* device [batch + 1] or null */
    void* workspace;             /* vb200_prefill_packed_workspace_bytes, 256-aligned */
    size_t workspace_bytes;
} vb200_prefill_packed_args;
size_t vb200_prefill_packed_workspace_bytes(const vb200_prefill_packed_args* a);
int vb200_prefill_packed_fwd(const vb200_prefill_packed_args* a);

/* ---- a cache of keys and values in 4 bits ------------------------------------------------------------
 * A row of D elements is held as D / 2 bytes of codes and, in an array of its own, D / 32 bytes of scales.  Of each 32 elements x:
 *     s = e4m3(max |x| / 7 * 2^-exponent)                       nearest, ties to even, at most 448
 *     c = sign(x) * min(7, floor(|x| * 2^-exponent / s + 1/2))  (0 where s is 0)
 * and what is read back is c * s * 2^exponent.  Byte j of a row holds c + 8 of element 2j in its low half and of element 2j + 1 in its high half.
 * A group with an infinite or NaN element gets the scale NaN: what reads it is NaN.  The exponents (for k and for v) bring tensors whose values are far
 * from one into the scales' range; s keeps its 4 significant bits for group maxima of 0.11 to 3136 times 2^exponent. */
typedef struct vb200_kv4_cache {
    void *k_codes, *v_codes;     /* [seqs, Hkv, cap, D / 2] bytes: rows of a head contiguous */
    void *k_scales, *v_scales;   /* [seqs, Hkv, cap, D / 32] e4m3 */
    int64_t stride_b, stride_h;  /* in rows, the same for all four; multiples of 8 */
    int32_t seqs, cap;           /* cap a multiple of 8; every pointer 16-byte aligned */
    int32_t k_exponent, v_exponent;   /* within [-64, 64] */
} vb200_kv4_cache;

/* Rounds k, v [B,Hkv,T,D] (VB200_BF16 or VB200_F16) into rows of the cache.  dst.rows null: token (b, t) goes to row start_row + t of sequence b
 * (dst.seqs and dst.cap are the cache's, and are not looked at). */
typedef struct vb200_kv4_rows_args {
    size_t struct_size;
    int32_t device;
    void* stream;
    int32_t dtype;
    int32_t B, Hkv, T, D;        /* D 64 or 128 */
    vb200_tensor4 k, v;
    vb200_kv4_cache cache;
    int32_t start_row;
    vb200_rows at;
} vb200_kv4_rows_args;
int vb200_kv4_append(const vb200_kv4_rows_args* a);
/* The other way: k, v are written with the values that rows of the cache stand for (exact in both types, but for values beyond fp16's range).  Tokens
 * that name no row are left as they are.  Either of k and v may be left out. */
int vb200_kv4_read(const vb200_kv4_rows_args* a);

/* One decode step over the 4-bit cache, the contract of vb200_decode_fwd without rotation and sharding: with k_new / v_new given, the new token is
 * first rounded into row seq_lens[b] of sequence b, then the query attends to rows [0, seq_lens[b] + appended) as the cache holds them, the group's query
 * heads sharing each row, split over `num_splits` CTAs and merged by a log-sum-exp combine.  A sequence without rows gets zeros and an lse of -infinity.
 * Lengths, advance_lens, max_len, num_splits and a token that does not fit: as in vb200_decode_fwd. */
typedef struct vb200_decode_kv4_args {
    size_t struct_size;
    int32_t device;
    void* stream;
    int32_t dtype;               /* VB200_BF16 or VB200_F16: q, k_new, v_new, o */
    int32_t B, Hq, Hkv, D;       /* D 64 or 128 */
    float scale;
    vb200_tensor4 q;             /* [B,Hq,1,D] */
    vb200_tensor4 k_new, v_new;  /* [B,Hkv,1,D]; ptr null: nothing to append */
    vb200_tensor4 o;             /* [B,Hq,1,D] */
    float* lse;                  /* [B,Hq] fp32, nullable */
    vb200_kv4_cache cache;       /* seqs >= B */
    int32_t* seq_lens;           /* device int32[B] or null */
    int32_t uniform_len;
    int32_t advance_lens;
    int32_t max_len;             /* upper bound of any length after the step; 0: cache.cap */
    int32_t num_splits;          /* 0: choose */
    void* workspace;             /* vb200_decode_kv4_workspace_bytes, 256-aligned */
    size_t workspace_bytes;
} vb200_decode_kv4_args;
size_t vb200_decode_kv4_workspace_bytes(const vb200_decode_kv4_args* a);
/* The most that any step over this cache needs (max_len = 1 .. cap): for a buffer that serves a whole generation. */
size_t vb200_decode_kv4_workspace_bytes_max(const vb200_decode_kv4_args* a);
int vb200_decode_kv4_fwd(const vb200_decode_kv4_args* a);

#ifdef __cplusplus
}
#endif
#endif /* VESPER_B200_SERVING_H */
