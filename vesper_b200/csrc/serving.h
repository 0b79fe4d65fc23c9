// Internal launch interfaces of the serving operators (include/vesper_b200_serving.h) between api_serving.cu and their kernels.
#pragma once

#include "../../include/vesper_b200_serving.h"
#include "kernels.h"

namespace vb200 {

constexpr int kKv4Group = 32;              // elements that share a scale

// Places of the tokens of a call in a cache; rows null: none given.
struct RowMap {
    const int* rows;
    const int* seq_ids;
    int seqs, cap;
};
struct Place {
    int seq, row;                          // row < 0: left out
};
// Beside code 2 of the status word (a sequence that is full): a place that the cache does not have; the sequence in 23 bits with its sign (beyond them, the ends).
constexpr int kNoPlace = 0x800000;
#ifdef __CUDACC__
// token (b, t) of T per sequence; out-of-range places set the status word and are left out
__device__ __forceinline__ Place find_place(const RowMap& m, int b, int t, int T, int* status) {
    const long long i = static_cast<long long>(b) * T + t;
    Place p;
    p.row = m.rows[i];
    p.seq = m.seq_ids ? m.seq_ids[i] : b;
    if (p.row >= 0 && (p.row >= m.cap || p.seq < 0 || p.seq >= m.seqs)) {
        atomicCAS(status, 0, (2 << 24) | kNoPlace | (max(-0x400000, min(p.seq, 0x3FFFFF)) & 0x7FFFFF));
        p.row = -1;
    }
    return p;
}
#endif

// ---- qk_norm_rope.cu ----
struct QkNormRopeParams {
    int dtype, B, Hq, Hkv, T, D;
    View4 q, k, v, q_out, k_out, v_out;    // ptr null: left out
    int norm;
    float eps;
    const float *q_weight, *k_weight;
    int rope, start_pos;
    const int* positions;
    RowMap dst;
    unsigned long long turns[kMaxHalfDim]; // inv_freq / (2 pi) as a fraction of 2^64, whole turns dropped
    int* status;
};
int launch_qk_norm_rope(cudaStream_t s, const QkNormRopeParams& p);

// ---- kv4_cache.cu ----
struct Kv4View {
    uint8_t *k_codes, *v_codes, *k_scales, *v_scales;
    long long stride_b, stride_h;          // rows
    int seqs, cap;
    float k_unit, v_unit;                  // 2^exponent
};
struct Kv4RowsParams {
    int dtype, B, H, T, D;
    View4 k, v;                            // ptr null: left out (reading)
    Kv4View cache;
    int start_row;
    RowMap at;                             // rows null: start_row + t of sequence b
    int* status;
};
int launch_kv4_append(cudaStream_t s, const Kv4RowsParams& p);
int launch_kv4_read(cudaStream_t s, const Kv4RowsParams& p);

// ---- decode_kv4.cu ----
constexpr int kKv4Tile = 256;              // rows that a CTA takes at a time: chunks are multiples of it
struct DecodeKv4Params {
    int dtype, B, Hq, Hkv, D;
    float scale;
    View4 q, k_new, v_new, o;
    float* lse;
    Kv4View cache;
    int* seq_lens;
    int uniform_len, advance_lens, append;
    int limit;                             // rows that a sequence may have after the step
    int per_unit, ctas, share;             // a CTA per unit, or the row of tiles in pieces of `share` (0: an equal part for each CTA)
    int* lens_used;                        // [B]: total rows | appended << 30
    int* tiles_before;                     // [B + 1]: tiles of the sequences before this one; last: the share
    float* records;                        // [ctas + units, 8, D + 2]: O / l, m, l of a CTA's part of a unit
    int* status;
};
int launch_decode_kv4(cudaStream_t s, const DecodeKv4Params& p);

// ---- prefill_packed_sm100.cu ----
struct PackedParams {
    int dtype, batch, Hq, Hkv, D, total_q, total_k, causal;
    float scale;
    View4 q, k, v, o;                      // sb unused
    float* lse;
    const int *cu_q, *cu_k;                // cu_k may equal cu_q
    void* workspace;
    int* status;
};
size_t prefill_packed_workspace(int batch, int Hq, int Hkv, int total_q);
int launch_prefill_packed(cudaStream_t s, const PackedParams& p);

}  // namespace vb200
