// Norms of queries and keys for each head, the position rotation and the append to a cache, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w          over the D elements of a head
//   (z[2i], z[2i+1]) = rotation of (y[2i], y[2i+1]) by position * inv_freq[i]
// q and k come out turned, v is copied; k and v go to plain tensors or to rows of a cache.
//
// What bounds it: HBM, each element is read once and written once.  A row of D elements is held by D / 8 neighbouring threads, 8 elements each (16 bytes
// of the 16-bit types), which sum the squares with shuffles.  A CTA takes a few tokens and a share of their heads: the angles of a token are computed once
// per CTA and read from shared memory by all of its heads, and the rows of a packed projection lie next to each other.
#include "serving.h"

namespace vb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;              // per CTA

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

// (cos, sin) of position * f: the product in 64 bits, brought into [-pi, pi] there, so that the fp32 functions see a small argument at any position
__device__ __forceinline__ float2 turn_of(int position, float f) {
    const double a = static_cast<double>(position) * static_cast<double>(f);
    const double r = fma(-rint(a * 0.15915494309189535), 6.283185307179586, a);
    float sn, cs;
    sincosf(static_cast<float>(r), &sn, &cs);
    return make_float2(cs, sn);
}

// LANES: threads per row, the power of two at or above D / 8.  blockIdx.x: tokens, blockIdx.y: a share of the heads.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(QkNormRopeParams p, int tokens_per_cta, int heads_per_cta, int heads) {
    constexpr int kRows = kThreads / LANES;
    __shared__ float2 turn[kMaxTokens][kMaxHalfDim];
    __shared__ Place place[kMaxTokens];
    const int half = p.D / 2;
    const int total = p.B * p.T;
    const int i0 = blockIdx.x * tokens_per_cta, n_tok = min(tokens_per_cta, total - i0);
    const int h0 = blockIdx.y * heads_per_cta, n_heads = min(heads_per_cta, heads - h0);
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    const bool live = lane * 8 < p.D;

    if (p.rope)
        for (int j = threadIdx.x; j < n_tok * half; j += kThreads) {
            const int r = j / half, e = j - r * half;
            const int pos = p.positions ? p.positions[i0 + r] : p.start_pos + (i0 + r) % p.T;
            turn[r][e] = turn_of(pos, p.inv_freq.v[e]);
        }
    if (p.dst.rows && threadIdx.x < n_tok) place[threadIdx.x] = find_place(p.dst, (i0 + threadIdx.x) / p.T, (i0 + threadIdx.x) % p.T, p.T, p.status);
    __syncthreads();

    for (int j = slot; j < n_tok * n_heads; j += kRows) {
        const int r = j / n_heads;
        int h = h0 + j - r * n_heads;
        const int b = (i0 + r) / p.T, t = (i0 + r) % p.T;
        const int n_q = p.q.ptr ? p.Hq : 0, n_k = p.k.ptr ? p.Hkv : 0;
        const int kind = h < n_q ? 0 : h < n_q + n_k ? 1 : 2;              // q, k, v
        h -= kind == 0 ? 0 : kind == 1 ? n_q : n_q + n_k;
        const View4& in = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
        const View4& out = kind == 0 ? p.q_out : kind == 1 ? p.k_out : p.v_out;
        long long to = b * out.sb + h * out.sh + t * out.ss;
        bool keep = live;
        if (kind != 0 && p.dst.rows) {
            to = place[r].seq * out.sb + h * out.sh + place[r].row * out.ss;
            keep = live && place[r].row >= 0;
        }
        Row8<T> x;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (live) {
            x.load(static_cast<const T*>(in.ptr) + b * in.sb + h * in.sh + t * in.ss + lane * 8);
            x.get(f);
        }
        if (kind != 2) {
            if (p.norm) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf(f[e], f[e], sum);
                // the rows of a warp that is past the end are not here: name the threads of this row only
                const unsigned mask = LANES == 32 ? 0xFFFFFFFFu : ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES);
#pragma unroll
                for (int o = LANES / 2; o >= 1; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
                const float inv = rsqrtf(sum / p.D + p.eps);
                const float* w = kind == 0 ? p.q_weight : p.k_weight;
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= inv;
                if (w && live)
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= w[lane * 8 + e];
            }
            if (p.rope && live)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 cs = turn[r][lane * 4 + e];
                    const float a = f[2 * e], c = f[2 * e + 1];
                    f[2 * e] = a * cs.x - c * cs.y;
                    f[2 * e + 1] = a * cs.y + c * cs.x;
                }
            x.set(f);
        }
        if (keep) x.store(static_cast<T*>(out.ptr) + to + lane * 8);
    }
}

template <typename T, int LANES>
int launch_t(cudaStream_t s, const QkNormRopeParams& p) {
    const int heads = (p.q.ptr ? p.Hq : 0) + (p.k.ptr ? p.Hkv : 0) + (p.v.ptr ? p.Hkv : 0);
    const long long total = static_cast<long long>(p.B) * p.T;
    int tokens = kMaxTokens;
    while (tokens > 1 && (total + tokens - 1) / tokens < 296) tokens >>= 1;
    const long long blocks = (total + tokens - 1) / tokens;
    long long shares = (296 + blocks - 1) / blocks;
    if (shares > heads) shares = heads;
    const int per = static_cast<int>((heads + shares - 1) / shares);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((heads + per - 1) / per));
    qk_norm_rope_kernel<T, LANES><<<grid, kThreads, 0, s>>>(p, tokens, per, heads);
    note_launch();
    VB200_CUDA_TRY(cudaPeekAtLastError());
    return VB200_OK;
}

template <typename T>
int launch_d(cudaStream_t s, const QkNormRopeParams& p) {
    const int n = p.D / 8;
    return n <= 1 ? launch_t<T, 1>(s, p) : n <= 2 ? launch_t<T, 2>(s, p) : n <= 4 ? launch_t<T, 4>(s, p) : n <= 8 ? launch_t<T, 8>(s, p) : launch_t<T, 16>(s, p);
}

}  // namespace

int launch_qk_norm_rope(cudaStream_t s, const QkNormRopeParams& p) {
    return p.dtype == VB200_F32 ? launch_d<float>(s, p) : p.dtype == VB200_BF16 ? launch_d<__nv_bfloat16>(s, p) : launch_d<__half>(s, p);
}

}  // namespace vb200
