// Attention over packed prompts.
//
//   s_ij = scale q_i . k_j,  key j of n_k visible to query i of n_q iff j <= n_k - n_q + i (causal) or always
//   O_i = sum_j softmax_j(s_ij) v_j,  LSE_i = ln sum_j exp(s_ij);  zeros and -infinity where no key is visible
#include "serving.h"

namespace vb200 {

namespace {

constexpr int kWarps = 4;
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

struct Sequence {
    int q0, nq, k0, nk;
};
__device__ __forceinline__ Sequence sequence_of(const PackedParams& p, int i) {
    const int a = p.cu_q[i], b = p.cu_q[i + 1], x = p.cu_k[i], y = p.cu_k[i + 1];
    const bool ok = a >= 0 && a <= b && b <= p.total_q && x >= 0 && x <= y && y <= p.total_k;
    return ok ? Sequence{a, b - a, x, y - x} : Sequence{0, 0, 0, 0};
}

// a warp per (token, query head): the keys one after the other, D / 32 elements per lane
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) prefill_packed_kernel(PackedParams p) {
    constexpr int kE = D / 32;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int token = blockIdx.x * kWarps + warp, hq = blockIdx.y, h = hq / (p.Hq / p.Hkv);
    if (token >= p.total_q) return;
    Sequence s{0, 0, 0, 0};
    for (int i = 0; i < p.batch; ++i) {
        const Sequence c = sequence_of(p, i);
        if (token >= c.q0 && token < c.q0 + c.nq) { s = c; break; }
    }
    if (s.nq == 0) return;
    const int n = p.causal ? min(s.nk, s.nk - s.nq + (token - s.q0) + 1) : s.nk;
    float q[kE], acc[kE], m = -INFINITY, l = 0.f;
    const T* qp = static_cast<const T*>(p.q.ptr) + hq * p.q.sh + token * p.q.ss + lane * kE;
#pragma unroll
    for (int e = 0; e < kE; ++e) { q[e] = Elem<T>::to_f(qp[e]); acc[e] = 0.f; }
    for (int j = 0; j < n; ++j) {
        const T* kp = static_cast<const T*>(p.k.ptr) + h * p.k.sh + (s.k0 + j) * p.k.ss + lane * kE;
        const T* vp = static_cast<const T*>(p.v.ptr) + h * p.v.sh + (s.k0 + j) * p.v.ss + lane * kE;
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < kE; ++e) x = fmaf(q[e], Elem<T>::to_f(kp[e]), x);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
        x *= p.scale * kLog2e;
        const float top = fmaxf(m, x), keep = m == -INFINITY ? 0.f : exp2f(m - top), w = exp2f(x - top);
        l = l * keep + w;
        m = top;
#pragma unroll
        for (int e = 0; e < kE; ++e) acc[e] = fmaf(w, Elem<T>::to_f(vp[e]), acc[e] * keep);
    }
    T* op = static_cast<T*>(p.o.ptr) + hq * p.o.sh + token * p.o.ss + lane * kE;
#pragma unroll
    for (int e = 0; e < kE; ++e) op[e] = Elem<T>::from_f(l == 0.f ? 0.f : acc[e] / l);
    if (p.lse && lane == 0) p.lse[static_cast<long long>(hq) * p.total_q + token] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, int D>
int launch_t(cudaStream_t s, const PackedParams& p) {
    prefill_packed_kernel<T, D><<<dim3((p.total_q + kWarps - 1) / kWarps, p.Hq), kWarps * 32, 0, s>>>(p);
    note_launch();
    VB200_CUDA_TRY(cudaPeekAtLastError());
    return VB200_OK;
}

}  // namespace

size_t prefill_packed_workspace(int, int, int, int) { return 256; }

int launch_prefill_packed(cudaStream_t s, const PackedParams& p) {
    if (p.dtype == VB200_BF16) return p.D == 128 ? launch_t<__nv_bfloat16, 128>(s, p) : launch_t<__nv_bfloat16, 64>(s, p);
    return p.D == 128 ? launch_t<__half, 128>(s, p) : launch_t<__half, 64>(s, p);
}

}  // namespace vb200
