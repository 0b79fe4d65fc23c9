// Rows of a 4-bit key / value cache: rounding 16-bit rows into it, and reading back what it stands for.
//
// What bounds it: HBM.  A thread takes 8 elements of a row (16 bytes, and one 32-bit word of codes), 4 threads share a scale.  A CTA has the places of a few tokens at hand, and each thread several rows on their way.
#include "hybrid.cuh"
#include "kv4.cuh"

#include <algorithm>

namespace vb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;             // per CTA
constexpr int kAhead = 4;                  // rows of a thread at once

// blockIdx.x: tokens; blockIdx.y: k or v.  WRITE: 16-bit rows into the cache; else the other way.
template <typename T, int D, bool WRITE>
__global__ void __launch_bounds__(kThreads) kv4_rows_kernel(Kv4RowsParams p, int tokens_per_cta) {
    constexpr int kLanes = D / 8, kRows = kThreads / kLanes;
    __shared__ long long at[kMaxTokens], row_of[kMaxTokens];                 // of a token, without the head: elements of k or v, and row of the cache (-1: left out)
    const bool value = blockIdx.y != 0;
    const View4& view = value ? p.v : p.k;
    if (!view.ptr) return;
    const int i0 = blockIdx.x * tokens_per_cta, n_tok = min(tokens_per_cta, p.B * p.T - i0);
    if (threadIdx.x < n_tok) {
        const int i = i0 + threadIdx.x, b = i / p.T, t = i - b * p.T;
        at[threadIdx.x] = b * view.sb + t * view.ss;
        const Place c = p.at.rows ? find_place(p.at, b, t, p.T, p.status) : Place{b, p.start_row + t};
        row_of[threadIdx.x] = c.row < 0 ? -1 : c.seq * p.cache.stride_b + c.row;
    }
    __syncthreads();
    T* rows16 = static_cast<T*>(view.ptr);
    uint32_t* codes = reinterpret_cast<uint32_t*>(value ? p.cache.v_codes : p.cache.k_codes);
    uint8_t* scales = value ? p.cache.v_scales : p.cache.k_scales;
    const float unit = value ? p.cache.v_unit : p.cache.k_unit;
    const int w = threadIdx.x % kLanes, slot = threadIdx.x / kLanes;
    const unsigned group = 0xFu << ((threadIdx.x & 31) & ~3);                // the threads that share this one's scale
    // token and head of the next row, tokens first (a head's rows of the cache lie next to each other); then kRows on
    int h = slot / n_tok, r = slot - h * n_tok;
    const int step_h = kRows / n_tok, step_r = kRows - step_h * n_tok, n = n_tok * p.H;
    for (int j0 = slot; j0 < n; j0 += kAhead * kRows) {
        uint4 raw[kAhead];
        uint32_t word[kAhead];
        uint8_t scale[kAhead];
        long long from[kAhead], row[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            row[u] = -1;
            if (j0 + u * kRows < n) {
                from[u] = at[r] + h * view.sh + w * 8;
                row[u] = row_of[r];
                if (row[u] >= 0) {                                           // the same for the threads of a row
                    row[u] += h * p.cache.stride_h;
                    if (WRITE) {
                        raw[u] = *reinterpret_cast<const uint4*>(rows16 + from[u]);
                    } else {
                        word[u] = codes[row[u] * kLanes + w];
                        scale[u] = scales[row[u] * (D / kKv4Group) + w / 4];
                    }
                }
            }
            r += step_r; h += step_h;
            if (r >= n_tok) { r -= n_tok; ++h; }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (row[u] < 0) continue;
            if (WRITE) {
                const uint32_t x2[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
                float x[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = Elem<T>::unpack2(x2[e]);
                    x[2 * e] = f.x; x[2 * e + 1] = f.y;
                }
                codes[row[u] * kLanes + w] = encode8(x, 1.0f / unit, group, scale[u]);
                if ((w & 3) == 0) scales[row[u] * (D / kKv4Group) + w / 4] = scale[u];
            } else {
                const float s = scale_value(scale[u]) * unit;
                uint32_t x2[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // 2^23 + n is the float of the bits 0x4B000000 | n
                    const float lo = __uint_as_float(0x4B000000u | ((word[u] >> (8 * e)) & 15)) - 8388616.0f, hi = __uint_as_float(0x4B000000u | ((word[u] >> (8 * e + 4)) & 15)) - 8388616.0f;
                    x2[e] = Elem<T>::pack2(lo * s, hi * s);
                }
                *reinterpret_cast<uint4*>(rows16 + from[u]) = make_uint4(x2[0], x2[1], x2[2], x2[3]);
            }
        }
    }
}

template <typename T, int D, bool WRITE>
int launch_t(cudaStream_t s, const Kv4RowsParams& p) {
    const long long total = static_cast<long long>(p.B) * p.T, fit = 4LL * device_sm_count();
    const int tokens = static_cast<int>(std::min<long long>(kMaxTokens, (total + fit - 1) / fit));
    kv4_rows_kernel<T, D, WRITE><<<dim3(static_cast<unsigned>((total + tokens - 1) / tokens), 2), kThreads, 0, s>>>(p, tokens);
    note_launch();
    VB200_CUDA_TRY(cudaPeekAtLastError());
    return VB200_OK;
}
template <bool WRITE>
int launch(cudaStream_t s, const Kv4RowsParams& p) {
    if (p.dtype == VB200_BF16) return p.D == 128 ? launch_t<__nv_bfloat16, 128, WRITE>(s, p) : launch_t<__nv_bfloat16, 64, WRITE>(s, p);
    return p.D == 128 ? launch_t<__half, 128, WRITE>(s, p) : launch_t<__half, 64, WRITE>(s, p);
}

}  // namespace

int launch_kv4_append(cudaStream_t s, const Kv4RowsParams& p) { return launch<true>(s, p); }
int launch_kv4_read(cudaStream_t s, const Kv4RowsParams& p) { return launch<false>(s, p); }

}  // namespace vb200
