// Norms of queries and keys for each head, the position rotation and the append to a cache, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w          over the D elements of a head
//   (z[2i], z[2i+1]) = rotation of (y[2i], y[2i+1]) by position * inv_freq[i]
// q and k come out turned, v is copied; k and v go to plain tensors or to rows of a cache.
//
// What bounds it: HBM, each element is read once and written once.  A row of D elements is held by D / 16 neighbouring threads, 16 elements each, which
// sum the squares with shuffles.  A CTA takes a few tokens and a share of their heads: the angles of a token are computed once
// per CTA, while its first rows are on their way, and read from shared memory by all of its heads; the rows of a packed projection lie next to each other.
// 8191 tokens of 32 + 8 heads of 128, bf16: 34 us, 4.9 TB/s, issue slots 60 % busy with shuffles and reads of the angles; 65536 tokens 228 us, 5.9 TB/s.
// fp32, a call alone on a cold L2 (bf16 so: 40 us): 8191 tokens 64.5 us, 5.2 TB/s; 32768 tokens 226 us, 5.9 TB/s.
#include "hybrid.cuh"
#include "serving.h"

#include <algorithm>

namespace vb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;             // per CTA

template <typename T> struct Row8 {        // 8 elements of a row
    uint4 raw;
    __device__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
    __device__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = raw; }
    __device__ void get(float (&f)[8]) const {
        const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = Elem<T>::unpack2(u[i]);
            f[2 * i] = t.x; f[2 * i + 1] = t.y;
        }
    }
    __device__ void set(const float (&f)[8]) {
        raw = make_uint4(Elem<T>::pack2(f[0], f[1]), Elem<T>::pack2(f[2], f[3]), Elem<T>::pack2(f[4], f[5]), Elem<T>::pack2(f[6], f[7]));
    }
};
template <> struct Row8<float> {
    float4 a, b;
    __device__ void load(const float* p) { a = *reinterpret_cast<const float4*>(p); b = *reinterpret_cast<const float4*>(p + 4); }
    __device__ void store(float* p) const { *reinterpret_cast<float4*>(p) = a; *reinterpret_cast<float4*>(p + 4) = b; }
    __device__ void get(float (&f)[8]) const { f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w; }
    __device__ void set(const float (&f)[8]) { a = make_float4(f[0], f[1], f[2], f[3]); b = make_float4(f[4], f[5], f[6], f[7]); }
};

// (cos, sin) of position * inv_freq, given inv_freq as a fraction of a turn in 64 bits: the product's whole turns fall off the top, and what is left is good to
// 2^-33 of a turn at any position; its upper half as a float is rounded by up to 2^-26 of a turn more (at half a turn, less nearer to zero).  (In double
// precision, brought into [-pi, pi], the angles took as long as everything else: 8191 tokens of 32 + 8 heads of 128 41 us, with 4 tokens per CTA 57.)
__device__ __forceinline__ float2 turn_of(int position, unsigned long long fraction) {
    const long long t = static_cast<long long>(static_cast<unsigned long long>(static_cast<long long>(position)) * fraction);
    float sn, cs;
    sincospif(__int2float_rn(static_cast<int>(t >> 32)) * 4.656612873077393e-10f, &sn, &cs);      // 2^-31: half turns
    return make_float2(cs, sn);
}

// What a CTA has of its tokens: where their rows stand in the inputs and outputs (elements, without the head), and their angles.
struct Tokens {
    long long in[3][kMaxTokens], out[3][kMaxTokens];     // q, k, v; out -1: the token is left out
    float4 turn[kMaxTokens][kMaxHalfDim / 2];            // (cos, sin) of two pairs
};

constexpr int kAhead = 1;                                // rows that a thread works on, while as many are on their way

// The rows of one kind (0: q, 1: k, 2: v): heads [h0, h0 + n_heads) of n_tok tokens.  LANES: threads per row, the power of two at or above D / 16; a thread has
// the elements [8 lane, 8 lane + 8) and those 8 LANES further on.
template <typename T, int LANES, int KIND, typename F>
__device__ __forceinline__ void rows_of(const QkNormRopeParams& p, const Tokens& tk, int n_tok, int h0, int n_heads, F before_first) {
    constexpr int kRows = kThreads / LANES;
    const View4& in = KIND == 0 ? p.q : KIND == 1 ? p.k : p.v;
    const View4& out = KIND == 0 ? p.q_out : KIND == 1 ? p.k_out : p.v_out;
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    const bool live[2] = {lane * 8 < p.D, (lane + LANES) * 8 < p.D};
    const T* src = static_cast<const T*>(in.ptr) + h0 * in.sh + lane * 8;
    T* dst = static_cast<T*>(out.ptr) + h0 * out.sh + lane * 8;
    float w[2][8];
    if (KIND < 2) {
        const float* from = KIND == 0 ? p.q_weight : p.k_weight;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[c][e] = 1.f;
            if (from && live[c]) {
                const float4* f4 = reinterpret_cast<const float4*>(from) + 2 * (lane + c * LANES);
                const float4 x = f4[0], y = f4[1];
                w[c][0] = x.x; w[c][1] = x.y; w[c][2] = x.z; w[c][3] = x.w; w[c][4] = y.x; w[c][5] = y.y; w[c][6] = y.z; w[c][7] = y.w;
            }
        }
    }
    const int rows = n_tok * n_heads;
    int r = slot / n_heads, h = slot - r * n_heads;      // token and head of the next row; then kRows on
    const int step_r = kRows / n_heads, step_h = kRows - step_r * n_heads;
    const float mean = 1.0f / p.D;
    struct Row {
        Row8<T> c[2];
        int r, h;
    };
    Row x[kAhead], next[kAhead];
    auto fetch = [&](int j0, Row (&y)[kAhead]) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            y[u].r = r; y[u].h = h;
            if (j0 + u * kRows < rows) {
                const T* from = src + (tk.in[KIND][r] + h * in.sh);
                if (live[0]) y[u].c[0].load(from);
                if (live[1]) y[u].c[1].load(from + LANES * 8);
            }
            r += step_r; h += step_h;
            if (h >= n_heads) { h -= n_heads; ++r; }
        }
    };
    fetch(slot, x);
    before_first();
    for (int j0 = slot; j0 < rows; j0 += kAhead * kRows) {
        fetch(j0 + kAhead * kRows, next);                // the next rows are on their way while these are worked on
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (j0 + u * kRows >= rows) break;
            if (KIND < 2) {
                float f[2][8];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[c][e] = 0.f;
                    if (live[c]) x[u].c[c].get(f[c]);
                }
                if (p.norm) {
                    float2 sum2 = make_float2(0.f, 0.f);
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const float2 y = make_float2(f[c][e], f[c][e + 1]);
                            sum2 = __ffma2_rn(y, y, sum2);
                        }
                    float sum = sum2.x + sum2.y;
                    // the threads of this row only: another row of the warp may be past the end
                    const unsigned mask = ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES);
#pragma unroll
                    for (int o = LANES / 2; o >= 1; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
                    const float inv = rsqrtf(fmaf(sum, mean, p.eps));
                    const float2 inv2 = make_float2(inv, inv);
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const float2 y = __fmul2_rn(make_float2(f[c][e], f[c][e + 1]), __fmul2_rn(inv2, make_float2(w[c][e], w[c][e + 1])));
                            f[c][e] = y.x; f[c][e + 1] = y.y;
                        }
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (!live[c]) continue;
                    if (p.rope) {
                        const float4* at = tk.turn[x[u].r] + 2 * (lane + c * LANES);
                        const float4 c0 = at[0], c1 = at[1];
                        const float2 cs[4] = {{c0.x, c0.y}, {c0.z, c0.w}, {c1.x, c1.y}, {c1.z, c1.w}};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            // (a cos - b sin, b cos + a sin)
                            const float a = f[c][2 * e], b = f[c][2 * e + 1];
                            const float2 y = __ffma2_rn(make_float2(a, b), make_float2(cs[e].x, cs[e].x), __fmul2_rn(make_float2(-b, a), make_float2(cs[e].y, cs[e].y)));
                            f[c][2 * e] = y.x; f[c][2 * e + 1] = y.y;
                        }
                    }
                    x[u].c[c].set(f[c]);
                }
            }
            const long long to = tk.out[KIND][x[u].r];
            if (to >= 0) {
                T* into = dst + (to + x[u].h * out.sh);
                if (live[0]) x[u].c[0].store(into);
                if (live[1]) x[u].c[1].store(into + LANES * 8);
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) x[u] = next[u];
    }
}

// blockIdx.x: tokens, blockIdx.y: a share of the heads of q, k and v together
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 4 : 2) qk_norm_rope_kernel(QkNormRopeParams p, int tokens_per_cta, int heads_per_cta, int heads) {
    __shared__ Tokens tk;
    const int half = p.D / 2;
    pdl_begin();
    const int total = p.B * p.T;
    const int i0 = blockIdx.x * tokens_per_cta, n_tok = min(tokens_per_cta, total - i0);
    const int h0 = blockIdx.y * heads_per_cta, h1 = min(h0 + heads_per_cta, heads);
    if (threadIdx.x < n_tok) {
        const int i = i0 + threadIdx.x, b = i / p.T, t = i - b * p.T;
        tk.in[0][threadIdx.x] = b * p.q.sb + t * p.q.ss;
        tk.in[1][threadIdx.x] = b * p.k.sb + t * p.k.ss;
        tk.in[2][threadIdx.x] = b * p.v.sb + t * p.v.ss;
        tk.out[0][threadIdx.x] = b * p.q_out.sb + t * p.q_out.ss;
        Place c{b, t};
        if (p.dst.rows) c = find_place(p.dst, b, t, p.T, p.status);
        tk.out[1][threadIdx.x] = c.row < 0 ? -1 : c.seq * p.k_out.sb + c.row * p.k_out.ss;
        tk.out[2][threadIdx.x] = c.row < 0 ? -1 : c.seq * p.v_out.sb + c.row * p.v_out.ss;
    }
    __syncthreads();
    bool angles = !p.rope;
    auto find_angles = [&]() {                           // while the first rows are on their way; the whole block comes here
        if (angles) return;
        angles = true;
        for (int i = threadIdx.x; i < n_tok * half; i += kThreads) {
            const int r = i / half, e = i - r * half;
            const int pos = p.positions ? p.positions[i0 + r] : p.start_pos + (i0 + r) % p.T;
            reinterpret_cast<float2*>(tk.turn[r])[e] = turn_of(pos, p.turns[e]);
        }
        __syncthreads();
    };
    const int n_q = p.q.ptr ? p.Hq : 0, n_k = p.k.ptr ? p.Hkv : 0;
    if (h0 < n_q) rows_of<T, LANES, 0>(p, tk, n_tok, h0, min(h1, n_q) - h0, find_angles);
    const int k0 = max(h0, n_q) - n_q, k1 = min(h1 - n_q, n_k);
    if (k0 < k1) rows_of<T, LANES, 1>(p, tk, n_tok, k0, k1 - k0, find_angles);
    const int v0 = max(h0, n_q + n_k) - n_q - n_k, v1 = h1 - n_q - n_k;
    if (v0 < v1) rows_of<T, LANES, 2>(p, tk, n_tok, v0, v1 - v0, [] {});
}

template <typename T, int LANES>
int launch_t(cudaStream_t s, const QkNormRopeParams& p) {
    const int heads = (p.q.ptr ? p.Hq : 0) + (p.k.ptr ? p.Hkv : 0) + (p.v.ptr ? p.Hkv : 0);
    const long long total = static_cast<long long>(p.B) * p.T;
    // Four CTAs per SM as long as a CTA's share is at most 16 tokens, and then more: one round of those that fit for 16-bit types.  fp32 rows leave room for two per
    // SM, and take two rounds: 8191 tokens of 32 + 8 heads of 128 64.5 us (68.6 in one round of two per SM; 1200 tokens 21.5 and 19.5).
    const long long fit = 4LL * device_sm_count();
    const int tokens = static_cast<int>(std::min<long long>(kMaxTokens, (total + fit - 1) / fit));
    const long long blocks = (total + tokens - 1) / tokens;
    long long shares = (2LL * device_sm_count() + blocks - 1) / blocks;     // of the heads, where the tokens make fewer CTAs than two per SM
    if (shares > heads) shares = heads;
    const int per = static_cast<int>((heads + shares - 1) / shares);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((heads + per - 1) / per));
    return launch_pdl(qk_norm_rope_kernel<T, LANES>, grid, dim3(kThreads), 0, s, p, tokens, per, heads);
}

template <typename T>
int launch_d(cudaStream_t s, const QkNormRopeParams& p) {
    const int n = (p.D + 15) / 16;
    return n <= 1 ? launch_t<T, 1>(s, p) : n <= 2 ? launch_t<T, 2>(s, p) : n <= 4 ? launch_t<T, 4>(s, p) : launch_t<T, 8>(s, p);
}

}  // namespace

int launch_qk_norm_rope(cudaStream_t s, const QkNormRopeParams& p) {
    return p.dtype == VB200_F32 ? launch_d<float>(s, p) : p.dtype == VB200_BF16 ? launch_d<__nv_bfloat16>(s, p) : launch_d<__half>(s, p);
}

}  // namespace vb200
