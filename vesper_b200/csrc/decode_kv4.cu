// One decode step over a 4-bit key / value cache.
//
//   s_j = scale q . k_j,  o = sum_j softmax(s)_j v_j,  lse = ln sum_j exp(s_j)     over the rows j < len + appended of the sequence
// with k_j, v_j as the cache holds them.  A new token is rounded into its row first and attended to as the row says.
#include "kv4.cuh"

namespace vb200 {

namespace {

constexpr int kWarps = 4;
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

// One CTA per (query head, sequence), a warp per row in turn; a lane holds D / 32 elements.
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) decode_kv4_kernel(DecodeKv4Params p) {
    constexpr int kE = D / 32;
    const int hq = blockIdx.x, b = blockIdx.y, rep = p.Hq / p.Hkv, h = hq / rep;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    __shared__ uint32_t new_codes[2][D / 8];
    __shared__ uint8_t new_scales[2][D / 32];
    __shared__ float part[kWarps][D + 2];

    const int raw = p.seq_lens ? p.seq_lens[b] : p.uniform_len;
    const long long planned = static_cast<long long>(p.num_splits) * p.chunk;
    const int limit = static_cast<int>(planned < p.cache.cap ? planned : p.cache.cap);
    const bool overflow = raw < 0 || static_cast<long long>(raw) + p.append > limit;
    const int len = raw < 0 ? 0 : min(raw, limit);
    const bool append = p.append && !overflow;
    if (overflow && hq == 0 && threadIdx.x == 0) atomicCAS(p.status, 0, (2 << 24) | (b & 0xFFFFFF));
    if (hq == 0 && threadIdx.x == 0) p.lens_used[b] = (len + append) | (append ? 1 << 30 : 0);
    const long long row0 = b * p.cache.stride_b + h * p.cache.stride_h;

    if (append && threadIdx.x < 2 * (D / 8)) {
        const int which = threadIdx.x / (D / 8), w = threadIdx.x % (D / 8);
        const View4& in = which ? p.v_new : p.k_new;
        const T* x = static_cast<const T*>(in.ptr) + b * in.sb + h * in.sh + w * 8;
        float f[8];
        for (int e = 0; e < 8; ++e) f[e] = Elem<T>::to_f(x[e]);
        uint8_t s;
        const uint32_t word = encode8(f, 1.0f / (which ? p.cache.v_unit : p.cache.k_unit), 0xFu << (threadIdx.x & 28), s);
        new_codes[which][w] = word;
        if (w % 4 == 0) new_scales[which][w / 4] = s;
        if (hq % rep == 0) {
            reinterpret_cast<uint32_t*>(which ? p.cache.v_codes : p.cache.k_codes)[(row0 + len) * (D / 8) + w] = word;
            if (w % 4 == 0) (which ? p.cache.v_scales : p.cache.k_scales)[(row0 + len) * (D / 32) + w / 4] = s;
        }
    }
    __syncthreads();

    float q[kE], acc[kE], m = -INFINITY, l = 0.f;
    const T* qp = static_cast<const T*>(p.q.ptr) + b * p.q.sb + hq * p.q.sh + lane * kE;
#pragma unroll
    for (int e = 0; e < kE; ++e) { q[e] = Elem<T>::to_f(qp[e]); acc[e] = 0.f; }
    auto value = [&](const uint8_t* codes, const uint8_t* scales, float unit, float (&x)[kE]) {
        const float s = scale_value(scales[lane * kE / 32]) * unit;
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            const int d = lane * kE + e;
            x[e] = static_cast<float>(((codes[d / 2] >> (4 * (d & 1))) & 15) - 8) * s;
        }
    };
    for (int j = warp; j < len + append; j += kWarps) {
        const bool fresh = append && j == len;
        float k[kE], v[kE];
        value(fresh ? reinterpret_cast<const uint8_t*>(new_codes[0]) : p.cache.k_codes + (row0 + j) * (D / 2), fresh ? new_scales[0] : p.cache.k_scales + (row0 + j) * (D / 32), p.cache.k_unit, k);
        value(fresh ? reinterpret_cast<const uint8_t*>(new_codes[1]) : p.cache.v_codes + (row0 + j) * (D / 2), fresh ? new_scales[1] : p.cache.v_scales + (row0 + j) * (D / 32), p.cache.v_unit, v);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < kE; ++e) s = fmaf(q[e], k[e], s);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        s *= p.scale * kLog2e;
        const float top = fmaxf(m, s), keep = m == -INFINITY ? 0.f : exp2f(m - top), w = exp2f(s - top);
        l = l * keep + w;
        m = top;
#pragma unroll
        for (int e = 0; e < kE; ++e) acc[e] = fmaf(w, v[e], acc[e] * keep);
    }
#pragma unroll
    for (int e = 0; e < kE; ++e) part[warp][lane * kE + e] = acc[e];
    if (lane == 0) { part[warp][D] = m; part[warp][D + 1] = l; }
    __syncthreads();
    if (threadIdx.x < D) {
        float top = -INFINITY, sum = 0.f, o = 0.f;
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part[w][D]);
        for (int w = 0; w < kWarps; ++w) {
            const float f = part[w][D] == -INFINITY ? 0.f : exp2f(part[w][D] - top);
            sum += part[w][D + 1] * f;
            o += part[w][threadIdx.x] * f;
        }
        static_cast<T*>(p.o.ptr)[b * p.o.sb + hq * p.o.sh + threadIdx.x] = Elem<T>::from_f(sum == 0.f ? 0.f : o / sum);
        if (p.lse && threadIdx.x == 0) p.lse[b * p.Hq + hq] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
}

__global__ void advance_kernel(DecodeKv4Params p) {
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b < p.B && StepLen::header_appended(p.lens_used[b])) p.seq_lens[b] = StepLen::header_total(p.lens_used[b]);
}

template <typename T, int D>
int launch_t(cudaStream_t s, const DecodeKv4Params& p) {
    decode_kv4_kernel<T, D><<<dim3(p.Hq, p.B), kWarps * 32, 0, s>>>(p);
    note_launch();
    if (p.advance_lens && p.seq_lens && p.append) {
        advance_kernel<<<(p.B + 127) / 128, 128, 0, s>>>(p);
        note_launch();
    }
    VB200_CUDA_TRY(cudaPeekAtLastError());
    return VB200_OK;
}

}  // namespace

int launch_decode_kv4(cudaStream_t s, const DecodeKv4Params& p) {
    if (p.dtype == VB200_BF16) return p.D == 128 ? launch_t<__nv_bfloat16, 128>(s, p) : launch_t<__nv_bfloat16, 64>(s, p);
    return p.D == 128 ? launch_t<__half, 128>(s, p) : launch_t<__half, 64>(s, p);
}

}  // namespace vb200
