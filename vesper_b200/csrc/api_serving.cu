// extern "C" entry points of vesper_b200_serving.h: argument validation, plans and workspaces.
#include <algorithm>
#include <cmath>

#include "hybrid.cuh"
#include "serving.h"

namespace vb200 {

namespace {

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// base and strides of a view on 16-byte boundaries, none negative; `batch`: stride_b counts too
bool view_aligned(const vb200_tensor4& t, int size, bool batch = true) {
    auto ok = [&](int64_t s) { return s >= 0 && (s * size) % 16 == 0; };
    return aligned16(t.ptr) && ok(t.stride_h) && ok(t.stride_s) && (!batch || ok(t.stride_b));
}
// the strides of dimensions of extent 1 are never used: any value may stand there
View4 used_view(const vb200_tensor4& t, int64_t B, int64_t H, int64_t S) {
    return View4{t.ptr, B > 1 ? t.stride_b : 0, H > 1 ? t.stride_h : 0, S > 1 ? t.stride_s : 0};
}
vb200_tensor4 used(vb200_tensor4 t, int64_t B, int64_t H, int64_t S) {
    const View4 v = used_view(t, B, H, S);
    t.stride_b = v.sb; t.stride_h = v.sh; t.stride_s = v.ss;
    return t;
}

// an output: no element stands for several (a dimension of extent 1 may have any stride)
bool written_once(const vb200_tensor4& t, int64_t B, int64_t H, int64_t S) { return (B <= 1 || t.stride_b != 0) && (H <= 1 || t.stride_h != 0) && (S <= 1 || t.stride_s != 0); }
int broadcast_output() { return set_detail(VB200_ERR_UNSUPPORTED, "outputs may not be broadcast: a stride of 0 where there is more than one"); }

// f / (2 pi) as a fraction of 2^64, whole turns dropped: f = m * 2^e with a whole m of 24 bits, times 2^100 / (2 pi) as a whole number
unsigned long long turn_fraction(float f) {
    int e = 0;
    const long long m = static_cast<long long>(std::frexp(std::fabs(f), &e) * 16777216.0f);
    e -= 24;
    constexpr unsigned __int128 kInverse = (static_cast<unsigned __int128>(0x28be60db9ULL) << 64) | 0x391054a7f09d5f47ULL;
    const unsigned __int128 x = kInverse * static_cast<unsigned __int128>(m);
    const int right = 36 - e;              // x * 2^(e - 100 + 64)
    const unsigned long long t = right >= 128 || right <= -64 ? 0 : right >= 0 ? static_cast<unsigned long long>(x >> right) : static_cast<unsigned long long>(x) << -right;
    return f < 0.f ? 0 - t : t;
}

int check_rows(const vb200_rows& r) {
    if (!r.rows) return r.seq_ids ? set_detail(VB200_ERR_INVALID_ARG, "seq_ids without rows") : VB200_OK;
    if (r.seqs <= 0 || r.cap <= 0) return set_detail(VB200_ERR_INVALID_ARG, "rows: seqs and cap of the cache must be positive");
    return VB200_OK;
}
RowMap row_map(const vb200_rows& r) { return RowMap{r.rows, r.seq_ids, r.seqs, r.cap}; }

int check_cache(const vb200_kv4_cache& c, int Hkv, bool need_k = true, bool need_v = true) {
    if ((need_k && (!c.k_codes || !c.k_scales)) || (need_v && (!c.v_codes || !c.v_scales))) return set_detail(VB200_ERR_INVALID_ARG, "4-bit cache: codes and scales must be non-null");
    if (c.seqs <= 0 || c.cap <= 0) return set_detail(VB200_ERR_INVALID_ARG, "4-bit cache: seqs and cap must be positive");
    if (c.k_exponent < -64 || c.k_exponent > 64 || c.v_exponent < -64 || c.v_exponent > 64) return set_detail(VB200_ERR_INVALID_ARG, "4-bit cache: exponents must be within [-64, 64]");
    if ((Hkv > 1 && c.stride_h < c.cap) || (c.seqs > 1 && c.stride_b < c.cap)) return set_detail(VB200_ERR_INVALID_ARG, "4-bit cache: strides must be at least cap rows");
    if (!aligned16(c.k_codes) || !aligned16(c.v_codes) || !aligned16(c.k_scales) || !aligned16(c.v_scales) || c.cap % 8 != 0 || (Hkv > 1 && c.stride_h % 8 != 0) ||
        (c.seqs > 1 && c.stride_b % 8 != 0))
        return set_detail(VB200_ERR_ALIGNMENT, "4-bit cache: pointers must be 16-byte aligned, cap and strides multiples of 8 rows");
    return VB200_OK;
}
Kv4View cache_view(const vb200_kv4_cache& c, int Hkv) {
    return Kv4View{static_cast<uint8_t*>(c.k_codes), static_cast<uint8_t*>(c.v_codes), static_cast<uint8_t*>(c.k_scales), static_cast<uint8_t*>(c.v_scales),
                   c.seqs > 1 ? c.stride_b : 0, Hkv > 1 ? c.stride_h : 0, c.seqs, c.cap, std::ldexp(1.0f, c.k_exponent), std::ldexp(1.0f, c.v_exponent)};
}

int status_or_fail(int*& status) {
    status = kernel_status_word();
    return status ? VB200_OK : set_detail(VB200_ERR_CUDA, "cannot allocate the status word");
}

// most tokens and elements of one call: indexes of (token, head) stay within 31 bits
bool countable(int64_t B, int64_t T, int64_t heads) { return B * T <= INT32_MAX && B * T * heads <= INT32_MAX; }

int check_kv4_rows(const vb200_kv4_rows_args* a, bool writing) {
    if (!a || a->struct_size != sizeof(vb200_kv4_rows_args)) return set_detail(VB200_ERR_INVALID_ARG, "vb200_kv4_rows_args: null or struct_size mismatch");
    if (a->dtype != VB200_BF16 && a->dtype != VB200_F16) return set_detail(VB200_ERR_UNSUPPORTED, "4-bit cache: rows must be bf16 or fp16");
    if (a->D != 64 && a->D != 128) return set_detail(VB200_ERR_UNSUPPORTED, "4-bit cache: head_dim 64 and 128");
    if (a->B <= 0 || a->Hkv <= 0 || a->T <= 0) return set_detail(VB200_ERR_INVALID_ARG, "B, Hkv, T must be positive");
    if (!countable(a->B, a->T, a->Hkv)) return set_detail(VB200_ERR_INVALID_ARG, "4-bit cache: too many rows in one call");
    if (writing ? (!a->k.ptr || !a->v.ptr) : (!a->k.ptr && !a->v.ptr)) return set_detail(VB200_ERR_INVALID_ARG, "4-bit cache: k and v must be non-null");
    if (int rc = check_cache(a->cache, a->Hkv, a->k.ptr != nullptr, a->v.ptr != nullptr)) return rc;
    if (!a->at.rows) {
        if (a->at.seq_ids) return set_detail(VB200_ERR_INVALID_ARG, "seq_ids without rows");
        if (a->start_row < 0 || static_cast<int64_t>(a->start_row) + a->T > a->cache.cap) return set_detail(VB200_ERR_INVALID_ARG, "start_row + T exceeds the cache capacity");
        if (a->B > a->cache.seqs) return set_detail(VB200_ERR_INVALID_ARG, "B exceeds the cache's sequences");
    }
    if (!writing && ((a->k.ptr && !written_once(a->k, a->B, a->Hkv, a->T)) || (a->v.ptr && !written_once(a->v, a->B, a->Hkv, a->T)))) return broadcast_output();
    if ((a->k.ptr && !view_aligned(used(a->k, a->B, a->Hkv, a->T), 2)) || (a->v.ptr && !view_aligned(used(a->v, a->B, a->Hkv, a->T), 2)))
        return set_detail(VB200_ERR_ALIGNMENT, "k / v base and strides must be 16-byte aligned");
    return VB200_OK;
}

int kv4_rows(const vb200_kv4_rows_args* a, bool writing) {
    if (int rc = check_kv4_rows(a, writing)) return rc;
    DeviceGuard g;
    if (int rc = g.init(a->device)) return rc;
    Kv4RowsParams p{};
    p.dtype = a->dtype; p.B = a->B; p.H = a->Hkv; p.T = a->T; p.D = a->D;
    p.k = used_view(a->k, a->B, a->Hkv, a->T);
    p.v = used_view(a->v, a->B, a->Hkv, a->T);
    p.cache = cache_view(a->cache, a->Hkv);
    p.start_row = a->start_row;
    p.at = RowMap{a->at.rows, a->at.seq_ids, a->cache.seqs, a->cache.cap};
    if (int rc = status_or_fail(p.status)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(a->stream);
    return writing ? launch_kv4_append(s, p) : launch_kv4_read(s, p);
}

struct Kv4Plan {
    int limit, per_unit, ctas, share;
    int64_t units, tiles;                  // of the batch, and of its longest sequence
    size_t lens_bytes, total;
};

// A CTA per unit (a key head of a sequence with up to eight query heads) while no sequence has more than two tiles: nothing is left to merge.  Else two CTAs
// per SM share the row of all tiles.  num_splits: pieces of that part of the longest sequence, and as many CTAs as these may need.
Kv4Plan plan_kv4(const vb200_decode_kv4_args* a) {
    Kv4Plan pl{};
    pl.limit = a->max_len > 0 ? std::min(a->max_len, a->cache.cap) : a->cache.cap;
    pl.units = static_cast<int64_t>(a->B) * a->Hkv * ((a->Hq / a->Hkv + 7) / 8);
    pl.tiles = (static_cast<int64_t>(pl.limit) + kKv4Tile - 1) / kKv4Tile;
    int64_t ctas;
    if (a->num_splits > 0) {
        pl.per_unit = a->num_splits == 1;
        const int64_t share = (pl.tiles + a->num_splits - 1) / a->num_splits;
        ctas = pl.per_unit ? pl.units : pl.units * ((pl.tiles + share - 1) / share);
        pl.share = static_cast<int>(share);
    } else {
        pl.per_unit = pl.tiles <= 2;
        ctas = pl.per_unit ? pl.units : std::min<int64_t>(2 * device_sm_count(), pl.units * pl.tiles);
    }
    pl.ctas = static_cast<int>(std::min<int64_t>(ctas, INT32_MAX));
    pl.lens_bytes = up256(sizeof(int) * (2 * static_cast<size_t>(a->B) + 1));
    pl.total = pl.lens_bytes + (pl.per_unit ? 0 : up256(sizeof(float) * (pl.units + ctas) * 8 * (a->D + 2)));
    return pl;
}

bool plannable(const vb200_decode_kv4_args* a) {
    return a && a->struct_size == sizeof(vb200_decode_kv4_args) && a->B > 0 && a->Hq > 0 && a->Hkv > 0 && a->Hq % a->Hkv == 0 && a->D > 0 && a->cache.cap > 0 && a->max_len >= 0 && a->num_splits >= 0;
}

int check_packed(const vb200_prefill_packed_args* a) {
    if (!a || a->struct_size != sizeof(vb200_prefill_packed_args)) return set_detail(VB200_ERR_INVALID_ARG, "vb200_prefill_packed_args: null or struct_size mismatch");
    if (a->dtype != VB200_BF16 && a->dtype != VB200_F16) return set_detail(VB200_ERR_UNSUPPORTED, "packed attention supports bf16 and fp16");
    if (a->D != 64 && a->D != 128) return set_detail(VB200_ERR_UNSUPPORTED, "packed attention supports head_dim 64 and 128");
    if (a->batch <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->total_q <= 0 || a->total_k < 0) return set_detail(VB200_ERR_INVALID_ARG, "batch, Hq, Hkv, total_q must be positive, total_k not negative");
    if (a->Hq % a->Hkv != 0) return set_detail(VB200_ERR_INVALID_ARG, "Hq must be divisible by Hkv");
    if (!a->q.ptr || !a->o.ptr || (a->total_k > 0 && (!a->k.ptr || !a->v.ptr))) return set_detail(VB200_ERR_INVALID_ARG, "q, k, v, o must be non-null");
    if (!a->cu_seqlens_q) return set_detail(VB200_ERR_INVALID_ARG, "cu_seqlens_q must be non-null");
    if (!countable(1, static_cast<int64_t>(a->total_q) + a->batch, a->Hq) || a->batch > 65536) return set_detail(VB200_ERR_INVALID_ARG, "packed attention: at most 2^31 - 1 (token, head) pairs and 65536 sequences");
    auto dense = [](const vb200_tensor4& t, int H, int tokens) { return (H == 1 || t.stride_h > 0) && (tokens <= 1 || t.stride_s > 0); };
    if (!dense(a->q, a->Hq, a->total_q) || !dense(a->o, a->Hq, a->total_q) || !dense(a->k, a->Hkv, a->total_k) || !dense(a->v, a->Hkv, a->total_k))
        return set_detail(VB200_ERR_UNSUPPORTED, "packed attention: strides must be positive (no broadcast heads or tokens)");
    const bool k_ok = a->total_k == 0 || (view_aligned(used(a->k, 1, a->Hkv, a->total_k), 2) && view_aligned(used(a->v, 1, a->Hkv, a->total_k), 2));
    if (!view_aligned(used(a->q, 1, a->Hq, a->total_q), 2) || !view_aligned(used(a->o, 1, a->Hq, a->total_q), 2) || !k_ok)
        return set_detail(VB200_ERR_ALIGNMENT, "q / k / v / o base and strides must be 16-byte aligned");
    return VB200_OK;
}

}  // namespace
}  // namespace vb200

using namespace vb200;

extern "C" {

int vb200_qk_norm_rope(const vb200_qk_norm_rope_args* a) {
    if (!a || a->struct_size != sizeof(vb200_qk_norm_rope_args)) return set_detail(VB200_ERR_INVALID_ARG, "vb200_qk_norm_rope_args: null or struct_size mismatch");
    if (a->dtype != VB200_F32 && a->dtype != VB200_BF16 && a->dtype != VB200_F16) return set_detail(VB200_ERR_UNSUPPORTED, "unknown dtype");
    if (a->B <= 0 || a->T <= 0 || a->D <= 0 || (a->q.ptr && a->Hq <= 0) || ((a->k.ptr || a->v.ptr) && a->Hkv <= 0)) return set_detail(VB200_ERR_INVALID_ARG, "B, Hq, Hkv, T, D must be positive");
    if (a->D % 8 != 0 || a->D > 2 * kMaxHalfDim) return set_detail(VB200_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 and <= 128");
    const vb200_tensor4* in[3] = {&a->q, &a->k, &a->v};
    const vb200_tensor4* out[3] = {&a->q_out, &a->k_out, &a->v_out};
    const int heads[3] = {a->Hq, a->Hkv, a->Hkv};
    if (!a->q.ptr && !a->k.ptr && !a->v.ptr) return set_detail(VB200_ERR_INVALID_ARG, "one of q, k, v must be given");
    for (int i = 0; i < 3; ++i)
        if ((in[i]->ptr == nullptr) != (out[i]->ptr == nullptr)) return set_detail(VB200_ERR_INVALID_ARG, "each of q, k, v needs an output, and no other output may be given");
    if (!countable(a->B, a->T, static_cast<int64_t>(a->q.ptr ? a->Hq : 0) + (a->k.ptr ? a->Hkv : 0) + (a->v.ptr ? a->Hkv : 0))) return set_detail(VB200_ERR_INVALID_ARG, "too many rows in one call");
    if (a->start_pos < 0 || static_cast<int64_t>(a->start_pos) + a->T > INT32_MAX) return set_detail(VB200_ERR_INVALID_ARG, "start_pos out of range");
    if (a->norm && !(a->eps >= 0.f)) return set_detail(VB200_ERR_INVALID_ARG, "eps must be >= 0");
    if (a->rope.enabled && !a->rope.inv_freq_host) return set_detail(VB200_ERR_INVALID_ARG, "rope enabled without inv_freq_host");
    if (a->rope.enabled)
        for (int i = 0; i < a->D / 2; ++i)
            if (!std::isfinite(a->rope.inv_freq_host[i])) return set_detail(VB200_ERR_INVALID_ARG, "inv_freq must be finite");
    if (int rc = check_rows(a->dst)) return rc;
    const int size = a->dtype == VB200_F32 ? 4 : 2;
    const bool scatter = a->dst.rows != nullptr;
    for (int i = 0; i < 3; ++i) {
        if (!in[i]->ptr) continue;
        const bool to_cache = scatter && i > 0;
        if (to_cache ? !written_once(*out[i], a->dst.seqs, heads[i], a->dst.cap) : !written_once(*out[i], a->B, heads[i], a->T)) return broadcast_output();
        if (!view_aligned(used(*in[i], a->B, heads[i], a->T), size) ||
            !view_aligned(to_cache ? used(*out[i], a->dst.seqs, heads[i], a->dst.cap) : used(*out[i], a->B, heads[i], a->T), size))
            return set_detail(VB200_ERR_ALIGNMENT, "q / k / v and outputs: base and strides must be 16-byte aligned");
    }
    if ((a->norm && a->q_weight && !aligned16(a->q_weight)) || (a->norm && a->k_weight && !aligned16(a->k_weight))) return set_detail(VB200_ERR_ALIGNMENT, "norm weights must be 16-byte aligned");
    DeviceGuard g;
    if (int rc = g.init(a->device)) return rc;
    QkNormRopeParams p{};
    p.dtype = a->dtype; p.B = a->B; p.Hq = a->Hq; p.Hkv = a->Hkv; p.T = a->T; p.D = a->D;
    View4* views[6] = {&p.q, &p.k, &p.v, &p.q_out, &p.k_out, &p.v_out};
    for (int i = 0; i < 3; ++i) {
        *views[i] = used_view(*in[i], a->B, heads[i], a->T);
        *views[3 + i] = scatter && i > 0 ? used_view(*out[i], a->dst.seqs, heads[i], a->dst.cap) : used_view(*out[i], a->B, heads[i], a->T);
    }
    p.norm = a->norm; p.eps = a->eps;
    p.q_weight = a->norm ? a->q_weight : nullptr;
    p.k_weight = a->norm ? a->k_weight : nullptr;
    p.rope = a->rope.enabled; p.start_pos = a->start_pos; p.positions = a->positions;
    if (p.rope)
        for (int i = 0; i < a->D / 2; ++i) p.turns[i] = turn_fraction(a->rope.inv_freq_host[i]);
    p.dst = row_map(a->dst);
    if (int rc = status_or_fail(p.status)) return rc;
    return launch_qk_norm_rope(static_cast<cudaStream_t>(a->stream), p);
}

size_t vb200_prefill_packed_workspace_bytes(const vb200_prefill_packed_args* a) {
    if (!a || a->struct_size != sizeof(vb200_prefill_packed_args) || a->batch <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv != 0 || a->total_q <= 0) return 0;
    return prefill_packed_workspace(a->batch, a->Hq, a->Hkv, a->total_q);
}

int vb200_prefill_packed_fwd(const vb200_prefill_packed_args* a) {
    if (int rc = check_packed(a)) return rc;
    if (!a->workspace || a->workspace_bytes < vb200_prefill_packed_workspace_bytes(a)) return set_detail(VB200_ERR_WORKSPACE, "packed attention workspace too small (see vb200_prefill_packed_workspace_bytes)");
    if (reinterpret_cast<uintptr_t>(a->workspace) % 256 != 0) return set_detail(VB200_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
    DeviceGuard g;
    if (int rc = g.init(a->device)) return rc;
    PackedParams p{};
    p.dtype = a->dtype; p.batch = a->batch; p.Hq = a->Hq; p.Hkv = a->Hkv; p.D = a->D;
    p.total_q = a->total_q; p.total_k = a->total_k; p.causal = a->causal; p.scale = a->scale;
    p.q = used_view(a->q, 1, a->Hq, a->total_q);
    p.o = used_view(a->o, 1, a->Hq, a->total_q);
    p.k = used_view(a->k, 1, a->Hkv, a->total_k);
    p.v = used_view(a->v, 1, a->Hkv, a->total_k);
    p.lse = a->lse;
    p.cu_q = a->cu_seqlens_q;
    p.cu_k = a->cu_seqlens_k ? a->cu_seqlens_k : a->cu_seqlens_q;
    p.workspace = a->workspace;
    if (int rc = status_or_fail(p.status)) return rc;
    return launch_prefill_packed(static_cast<cudaStream_t>(a->stream), p);
}

int vb200_kv4_append(const vb200_kv4_rows_args* a) { return kv4_rows(a, true); }
int vb200_kv4_read(const vb200_kv4_rows_args* a) { return kv4_rows(a, false); }

size_t vb200_decode_kv4_workspace_bytes(const vb200_decode_kv4_args* a) { return plannable(a) ? plan_kv4(a).total : 0; }

size_t vb200_decode_kv4_workspace_bytes_max(const vb200_decode_kv4_args* a) {
    if (!plannable(a)) return 0;
    vb200_decode_kv4_args t = *a;
    size_t most = 0;
    for (int64_t n = 1; n < a->cache.cap + kKv4Tile; n += kKv4Tile) {        // the plan goes by whole tiles
        t.max_len = static_cast<int>(std::min<int64_t>(n, a->cache.cap));
        most = std::max(most, plan_kv4(&t).total);
    }
    return most;
}

int vb200_decode_kv4_fwd(const vb200_decode_kv4_args* a) {
    if (!a || a->struct_size != sizeof(vb200_decode_kv4_args)) return set_detail(VB200_ERR_INVALID_ARG, "vb200_decode_kv4_args: null or struct_size mismatch");
    if (a->dtype != VB200_BF16 && a->dtype != VB200_F16) return set_detail(VB200_ERR_UNSUPPORTED, "4-bit decode: q and o must be bf16 or fp16");
    if (a->D != 64 && a->D != 128) return set_detail(VB200_ERR_UNSUPPORTED, "4-bit decode: head_dim 64 and 128");
    if (a->B <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->max_len < 0 || a->num_splits < 0) return set_detail(VB200_ERR_INVALID_ARG, "B, Hq, Hkv must be positive, max_len and num_splits not negative");
    if (a->Hq % a->Hkv != 0) return set_detail(VB200_ERR_INVALID_ARG, "Hq must be divisible by Hkv");
    if (a->B > 65535 || a->Hq > 65535) return set_detail(VB200_ERR_INVALID_ARG, "4-bit decode: at most 65535 sequences and heads");
    if (!a->q.ptr || !a->o.ptr) return set_detail(VB200_ERR_INVALID_ARG, "q, o must be non-null");
    if ((a->k_new.ptr == nullptr) != (a->v_new.ptr == nullptr)) return set_detail(VB200_ERR_INVALID_ARG, "k_new and v_new must both be given or both be null");
    if (int rc = check_cache(a->cache, a->Hkv)) return rc;
    if (a->B > a->cache.seqs) return set_detail(VB200_ERR_INVALID_ARG, "B exceeds the cache's sequences");
    const bool append = a->k_new.ptr != nullptr;
    const int64_t most = a->max_len > 0 ? std::min(a->max_len, a->cache.cap) : a->cache.cap;
    if (!a->seq_lens && (a->uniform_len < 0 || static_cast<int64_t>(a->uniform_len) + append > most)) return set_detail(VB200_ERR_INVALID_ARG, "uniform_len out of range for the cache or max_len");
    if (a->advance_lens && !a->seq_lens) return set_detail(VB200_ERR_INVALID_ARG, "advance_lens needs seq_lens");
    if (!written_once(a->o, a->B, a->Hq, 1)) return broadcast_output();
    if (!view_aligned(used(a->q, a->B, a->Hq, 1), 2) || !view_aligned(used(a->o, a->B, a->Hq, 1), 2) ||
        (append && (!view_aligned(used(a->k_new, a->B, a->Hkv, 1), 2) || !view_aligned(used(a->v_new, a->B, a->Hkv, 1), 2))))
        return set_detail(VB200_ERR_ALIGNMENT, "q / k_new / v_new / o base and strides must be 16-byte aligned");
    const Kv4Plan pl = plan_kv4(a);
    // (the tiles of a step, and what rounding them up to equal shares adds, are counted in 32 bits)
    if (pl.units * pl.tiles + (a->num_splits > 0 ? 0 : pl.ctas) > INT32_MAX || a->cache.cap >= 1 << 30) return set_detail(VB200_ERR_INVALID_ARG, "4-bit decode: too many rows in one call");
    if (!a->workspace || a->workspace_bytes < pl.total) return set_detail(VB200_ERR_WORKSPACE, "decode workspace too small (see vb200_decode_kv4_workspace_bytes)");
    if (reinterpret_cast<uintptr_t>(a->workspace) % 256 != 0) return set_detail(VB200_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
    DeviceGuard g;
    if (int rc = g.init(a->device)) return rc;
    DecodeKv4Params p{};
    p.dtype = a->dtype; p.B = a->B; p.Hq = a->Hq; p.Hkv = a->Hkv; p.D = a->D; p.scale = a->scale;
    p.q = used_view(a->q, a->B, a->Hq, 1);
    p.o = used_view(a->o, a->B, a->Hq, 1);
    p.k_new = used_view(a->k_new, a->B, a->Hkv, 1);
    p.v_new = used_view(a->v_new, a->B, a->Hkv, 1);
    p.lse = a->lse;
    p.cache = cache_view(a->cache, a->Hkv);
    p.seq_lens = a->seq_lens; p.uniform_len = a->uniform_len; p.advance_lens = a->advance_lens && append; p.append = append;
    p.limit = pl.limit; p.per_unit = pl.per_unit; p.ctas = pl.ctas; p.share = pl.share;
    p.lens_used = static_cast<int*>(a->workspace);
    p.tiles_before = p.lens_used + a->B;
    p.records = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + pl.lens_bytes);
    if (int rc = status_or_fail(p.status)) return rc;
    return launch_decode_kv4(static_cast<cudaStream_t>(a->stream), p);
}

}  // extern "C"
