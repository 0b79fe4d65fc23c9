// Rows of a 4-bit key / value cache: rounding 16-bit rows into it, and reading back what it stands for.
//
// What bounds it: HBM.  A thread takes 16 elements of a row, two threads share a scale.  A CTA has the places of a few tokens at hand, and each thread several
// rows on their way.  16 x 4096 tokens of 8 heads of 128 in and back: 136 us, 4.8 TB/s; 8583 tokens: 24 us, of which one round of CTAs each way is the most.
#include "hybrid.cuh"
#include "kv4.cuh"

#include <algorithm>

namespace vb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 32;             // per CTA
constexpr int kMinCtas = 4;                // per SM, of both kinds
constexpr int kAhead = 2;                  // rows of a thread at once

// blockIdx.x: tokens; blockIdx.y: k or v.  WRITE: 16-bit rows into the cache; else the other way.
template <typename T, int D, bool WRITE>
__global__ void __launch_bounds__(kThreads, kMinCtas) kv4_rows_kernel(Kv4RowsParams p, int tokens_per_cta) {
    constexpr int kLanes = D / 16, kRows = kThreads / kLanes;
    __shared__ long long at[kMaxTokens], row_of[kMaxTokens];                 // of a token, without the head: elements of k or v, and row of the cache (-1: left out)
    const bool value = blockIdx.y != 0;
    const View4& view = value ? p.v : p.k;
    pdl_begin();
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
    uint2* codes = reinterpret_cast<uint2*>(value ? p.cache.v_codes : p.cache.k_codes);
    uint8_t* scales = value ? p.cache.v_scales : p.cache.k_scales;
    const float unit = value ? p.cache.v_unit : p.cache.k_unit, back = 1.0f / unit;
    const int w = threadIdx.x % kLanes, slot = threadIdx.x / kLanes;
    const unsigned group = 3u << ((threadIdx.x & 31) & ~1);                 // the threads that share this one's scale
    // token and head of the next row, tokens first (a head's rows of the cache lie next to each other); then kRows on
    int h = slot / n_tok, r = slot - h * n_tok;
    const int step_h = kRows / n_tok, step_r = kRows - step_h * n_tok, n = n_tok * p.H;
    for (int j0 = slot; j0 < n; j0 += kAhead * kRows) {
        uint4 raw[kAhead][2];
        uint2 word[kAhead];
        uint8_t scale[kAhead];
        long long from[kAhead], row[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            row[u] = -1;
            if (j0 + u * kRows < n) {
                from[u] = at[r] + h * view.sh + w * 16;
                row[u] = row_of[r];
                if (row[u] >= 0) {                                           // the same for the threads of a row
                    row[u] += h * p.cache.stride_h;
                    if (WRITE) {
                        const uint4* x = reinterpret_cast<const uint4*>(rows16 + from[u]);
                        raw[u][0] = x[0]; raw[u][1] = x[1];
                    } else {
                        word[u] = codes[row[u] * kLanes + w];
                        scale[u] = scales[row[u] * (D / kKv4Group) + w / 2];
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
                float x[16];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t x2[4] = {raw[u][c].x, raw[u][c].y, raw[u][c].z, raw[u][c].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = Elem<T>::unpack2(x2[e]);
                        x[8 * c + 2 * e] = f.x; x[8 * c + 2 * e + 1] = f.y;
                    }
                }
                uint32_t got[2];
                encode<16>(x, back, group, got, scale[u]);
                codes[row[u] * kLanes + w] = make_uint2(got[0], got[1]);
                if ((w & 1) == 0) scales[row[u] * (D / kKv4Group) + w / 2] = scale[u];
            } else {
                const float s = scale_value(scale[u]) * unit;
                uint4* to = reinterpret_cast<uint4*>(rows16 + from[u]);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t code = c ? word[u].y : word[u].x;
                    uint32_t x2[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // 2^23 + n is the float of the bits 0x4B000000 | n
                        const float lo = __uint_as_float(0x4B000000u | ((code >> (8 * e)) & 15)) - 8388616.0f, hi = __uint_as_float(0x4B000000u | ((code >> (8 * e + 4)) & 15)) - 8388616.0f;
                        x2[e] = Elem<T>::pack2(lo * s, hi * s);
                    }
                    to[c] = make_uint4(x2[0], x2[1], x2[2], x2[3]);
                }
            }
        }
    }
}

template <typename T, int D, bool WRITE>
int launch_t(cudaStream_t s, const Kv4RowsParams& p) {
    const long long total = static_cast<long long>(p.B) * p.T, fit = kMinCtas / 2 * static_cast<long long>(device_sm_count());
    const int tokens = static_cast<int>(std::min<long long>(kMaxTokens, (total + fit - 1) / fit));
    return launch_pdl(kv4_rows_kernel<T, D, WRITE>, dim3(static_cast<unsigned>((total + tokens - 1) / tokens), 2), dim3(kThreads), 0, s, p, tokens);
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
