// Rows of a 4-bit key / value cache: rounding 16-bit rows into it, and reading back what it stands for.
//
// What bounds it: HBM.  A thread takes 8 elements of a row (16 bytes in, one 32-bit word of codes out), 4 threads share a scale.
#include "kv4.cuh"

namespace vb200 {

namespace {

constexpr int kThreads = 256;

// index of a thread -> (b, t, head, word); rows of the heads of a token lie next to each other
struct At {
    int b, t, h, w;
};
__device__ __forceinline__ At at_of(long long i, const Kv4RowsParams& p) {
    At a;
    const int words = p.D / 8;
    a.w = static_cast<int>(i % words); i /= words;
    a.h = static_cast<int>(i % p.H); i /= p.H;
    a.t = static_cast<int>(i % p.T);
    a.b = static_cast<int>(i / p.T);
    return a;
}
__device__ __forceinline__ Place place_of(const Kv4RowsParams& p, const At& a) {
    if (p.at.rows) return find_place(p.at, a.b, a.t, p.T, p.status);
    return Place{a.b, p.start_row + a.t};
}

template <typename T>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(Kv4RowsParams p, long long total) {
    const long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= total) return;                  // total is a multiple of 4 threads
    const At a = at_of(i, p);
    const Place to = place_of(p, a);
    if (to.row < 0) return;                  // the same for the threads of a group
    const unsigned lanes = 0xFu << ((threadIdx.x & 31) & ~3);
    const long long row = to.seq * p.cache.stride_b + a.h * p.cache.stride_h + to.row;
    const bool value = blockIdx.y != 0;
    const View4& in = value ? p.v : p.k;
    const float back = 1.0f / (value ? p.cache.v_unit : p.cache.k_unit);
    const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const T*>(in.ptr) + a.b * in.sb + a.h * in.sh + a.t * in.ss + a.w * 8);
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 f = Elem<T>::unpack2(u[e]);
        x[2 * e] = f.x; x[2 * e + 1] = f.y;
    }
    uint8_t scale;
    const uint32_t word = encode8(x, back, lanes, scale);
    reinterpret_cast<uint32_t*>(value ? p.cache.v_codes : p.cache.k_codes)[row * (p.D / 8) + a.w] = word;
    if ((threadIdx.x & 3) == 0) (value ? p.cache.v_scales : p.cache.k_scales)[row * (p.D / kKv4Group) + a.w / 4] = scale;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(Kv4RowsParams p, long long total) {
    const long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= total) return;
    const bool value = blockIdx.y != 0;
    const View4& out = value ? p.v : p.k;
    if (!out.ptr) return;
    const At a = at_of(i, p);
    const Place from = place_of(p, a);
    if (from.row < 0) return;
    const long long row = from.seq * p.cache.stride_b + a.h * p.cache.stride_h + from.row;
    const uint32_t word = reinterpret_cast<const uint32_t*>(value ? p.cache.v_codes : p.cache.k_codes)[row * (p.D / 8) + a.w];
    const float s = scale_value((value ? p.cache.v_scales : p.cache.k_scales)[row * (p.D / kKv4Group) + a.w / 4]) * (value ? p.cache.v_unit : p.cache.k_unit);
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        u[e] = Elem<T>::pack2(static_cast<float>(static_cast<int>((word >> (8 * e)) & 15) - 8) * s, static_cast<float>(static_cast<int>((word >> (8 * e + 4)) & 15) - 8) * s);
    *reinterpret_cast<uint4*>(static_cast<T*>(out.ptr) + a.b * out.sb + a.h * out.sh + a.t * out.ss + a.w * 8) = make_uint4(u[0], u[1], u[2], u[3]);
}

template <typename F>
int launch_rows(cudaStream_t s, const Kv4RowsParams& p, F kernel) {
    const long long total = static_cast<long long>(p.B) * p.T * p.H * (p.D / 8);
    const dim3 grid(static_cast<unsigned>((total + kThreads - 1) / kThreads), 2);
    kernel<<<grid, kThreads, 0, s>>>(p, total);
    note_launch();
    VB200_CUDA_TRY(cudaPeekAtLastError());
    return VB200_OK;
}

}  // namespace

int launch_kv4_append(cudaStream_t s, const Kv4RowsParams& p) {
    return p.dtype == VB200_BF16 ? launch_rows(s, p, kv4_append_kernel<__nv_bfloat16>) : launch_rows(s, p, kv4_append_kernel<__half>);
}
int launch_kv4_read(cudaStream_t s, const Kv4RowsParams& p) {
    return p.dtype == VB200_BF16 ? launch_rows(s, p, kv4_read_kernel<__nv_bfloat16>) : launch_rows(s, p, kv4_read_kernel<__half>);
}

}  // namespace vb200
