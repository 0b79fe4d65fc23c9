// One decode step over a 4-bit key / value cache, split over the keys.
//
//   s_j = scale q . k_j,  o = sum_j softmax(s)_j v_j,  lse = ln sum_j exp(s_j)     over the rows j < len + appended of the sequence
// with k_j, v_j as the cache holds them.  A new token is rounded into its row first and attended to as the row says.
//
// The tiles of all (sequence, key head) units stand in one row, and every CTA takes an equal piece of it, however the lengths differ: two CTAs per SM from the
// first tile to the last.  A unit that lies in one piece is finished there, the others leave records that a second kernel merges.  Tiles of 256 rows come by
// bulk copies into a ring of shared memory (the rows of a head are contiguous: a tile is four copies, codes and scales of keys and of values), four warps take
// 64 rows of a tile each.  Both products run as warp-level
// m16n8k16 products, because up to eight query heads share every row:
//   S [heads, keys] = Q K^T      A = the queries, high halves in rows 0-7 and the rest in rows 8-15, so that a score is as exact as in fp32; B = the keys
//   O^T [dims, heads] = V^T P^T  A = the values, B = the weights, which stand in the registers of S as this product wants them
// The order of the summed index is free, so every thread reads its part of a row as it lies: 32 neighbouring elements of a key (one scale), 16 neighbouring
// elements of four values.  Codes c + 8 become numbers by one and / or and one multiply-add for two of them: the bits 0x6400 | n are the fp16 number 1024 + n,
// and (1024 + n) s - 1032 s = (n - 8) s is exact in fp16 for every e4m3 scale (s is carried as s / 8, so that 1032 s stays in range).
//
// What bounds it: the instructions that expand 4.25 bits per element (logic pipe 47 %, FMA 36 %, tensor 35 % of the cycles, at two warps per scheduler: the
// registers allow no third), before HBM.  One sequence, 64 heads on 8 of 128: 265 us for 1048576 keys, 4.3 TB/s; 47 us for 131072, of which 14 are the start
// and the merge.  32 sequences of 1024-7930 keys, 32 heads on 8: 54 us.
#include "kv4.cuh"

namespace vb200 {

namespace {

constexpr int kWarps = 4;                  // 64 rows of a tile each
constexpr int kTiles8 = 8, kRows = 8 * kTiles8;
constexpr int kTile = kKv4Tile;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;
constexpr int kMinCtas = 2;
constexpr int kAtOnce = 4;                 // 8-key tiles whose products alternate
constexpr int kEarly = 2;                  // 16-row groups of values that are expanded while the largest score is looked for
constexpr int kHeads = 8;                  // query heads of a CTA, at most
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.0f;           // weights stay within 2^8 of the running reference,
constexpr float kLift = 7.0f;              // which weighs 2^7: a weight is then an fp16 number of full precision down to 2^-21 of it, and 2^-32 of it at worst
static_assert(kTile == kWarps * kRows, "the warps share a tile");

template <int D> struct Layout {
    static constexpr int kRow = D / 2, kScales = D / 32;                    // bytes of a row
    static constexpr int kKeyWords = D / 32, kValueWords = D / 64;          // 8-element words of a row that one thread takes
    static constexpr int kOutTiles = D / 16;
    static constexpr int kStageBytes = 2 * kTile * (kRow + kScales);
    static constexpr int kVCodes = kTile * kRow, kKScales = 2 * kTile * kRow, kVScales = kKScales + kTile * kScales;
    static constexpr int kSmem = kStages * kStageBytes + 2 * kStages * 8 + 16;
    static_assert(kWarps * kHeads * (D + 2) * 4 <= kStageBytes, "the warps merge in a slot of the ring");
};

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t h2(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }
__device__ __forceinline__ __half2 h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) { return h2(__hfma2(h2(a), h2(b), h2(c))); }

// the factors of two scales s (one for each half): s / 8, -1032 s / 8, and the same for codes that stand 4 bits higher
struct Scale2 {
    uint32_t s, c, s16, c16;
    Scale2() = default;
    __device__ explicit Scale2(uint32_t bytes) {                            // two e4m3 in the low 16 bits
        const __half2_raw raw = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(bytes), __NV_E4M3);
        const __half2 t = __half2(raw);
        s = h2(__hmul2(t, __float2half2_rn(0.125f)));
        c = h2(__hmul2(t, __float2half2_rn(-129.0f)));
        s16 = h2(__hmul2(t, __float2half2_rn(0.0078125f)));
        c16 = h2(__hmul2(t, __float2half2_rn(-9.0f)));
    }
};
// (w & mask) | magic in one instruction: `magic` comes from a register that the compiler does not know the value of, since two constants do not fit one
template <uint32_t kMask> __device__ __forceinline__ uint32_t pick(uint32_t w, uint32_t magic) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(kMask), "r"(magic));
    return r;
}
// nibbles (j, j + 4) of a word -> x[j] = the numbers (n - 8) s / 8, low and high half
__device__ __forceinline__ void expand(uint32_t w, const Scale2& f, uint32_t magic, uint32_t (&x)[4]) {
    x[0] = hfma2(pick<0x000F000Fu>(w, magic), f.s, f.c);
    x[1] = hfma2(pick<0x00F000F0u>(w, magic), f.s16, f.c16);
    const uint32_t u = w >> 8;
    x[2] = hfma2(pick<0x000F000Fu>(u, magic), f.s, f.c);
    x[3] = hfma2(pick<0x00F000F0u>(u, magic), f.s16, f.c16);
}

template <int N> struct Words { uint32_t w[N]; };
template <int N> __device__ __forceinline__ Words<N> load_words(const unsigned char* p) {
    Words<N> r;
    if constexpr (N == 4) { const uint4 v = *reinterpret_cast<const uint4*>(p); r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w; }
    else if constexpr (N == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); r.w[0] = v.x; r.w[1] = v.y; }
    else r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    return r;
}

// Column n of an 8-key tile of S stands for row tile_row(n): with this order the rows that the threads of a warp read at once, keys by columns and values by
// pairs of columns, lie in different banks (values: two to a bank, instead of four).
__device__ __forceinline__ int tile_row(int n) { return (n & 4) | ((n & 1) << 1) | (((n >> 1) ^ n) & 1); }

struct Step {
    int len, total;                        // rows before the step, and with the new one
    bool append, overflow;
    __device__ int tiles() const { return (total + kTile - 1) / kTile; }
    __device__ int packed() const { return total | (append ? 1 << 30 : 0); }
};
__device__ __forceinline__ Step step_of(const DecodeKv4Params& p, int b) {
    const int raw = p.seq_lens ? p.seq_lens[b] : p.uniform_len;
    Step s;
    s.overflow = raw < 0 || static_cast<long long>(raw) + p.append > p.limit;
    s.len = raw < 0 ? 0 : min(raw, p.limit);
    s.append = p.append && !s.overflow;
    s.total = s.len + s.append;
    return s;
}

// A unit is a key head of a sequence with at most eight of its query heads; its tiles, and the units, stand one behind the other.
struct Cursor {
    int b, unit, tile;                     // sequence, unit within it, tile within that
    Step st;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kMinCtas) decode_kv4_kernel(DecodeKv4Params p, int head_shares) {
    using L = Layout<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * L::kStageBytes);
    uint64_t* empty = full + kStages;
    int* abort_flag = reinterpret_cast<int*>(empty + kStages);

    const int rep = p.Hq / p.Hkv, units = p.Hkv * head_shares;               // units of a sequence
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], kWarps); }
        *abort_flag = 0;
        mbar_fence_init();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- this CTA's part of all tiles: a unit of its own, or an equal share of the whole row of them ----
    auto note = [&](int b, const Step& st) {
        p.lens_used[b] = st.packed();
        if (st.overflow) atomicCAS(p.status, 0, (2 << 24) | (b & 0xFFFFFF));
    };
    Cursor at;
    int n_tiles;
    if (p.per_unit) {
        at.b = blockIdx.x / units; at.unit = blockIdx.x % units; at.tile = 0;
        at.st = step_of(p, at.b);
        if (at.unit == 0 && tid == 0) note(at.b, at.st);
        n_tiles = at.st.tiles();
    } else {
        // every warp goes through the lengths by itself, 32 at a time: once for the sum, once (from the cache) for the place
        int all = 0;
        for (int b0 = 0; b0 < p.B; b0 += 32) {
            int n = b0 + lane < p.B ? step_of(p, b0 + lane).tiles() * units : 0;
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
            all += n;
        }
        const int share = p.share > 0 ? p.share : max(1, (all + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
        const int start = static_cast<int>(min(static_cast<long long>(blockIdx.x) * share, static_cast<long long>(all)));
        n_tiles = min(share, all - start);
        const bool notes = blockIdx.x == 0 && warp == 0;
        int before = 0;
        at.b = -1;
        for (int b0 = 0; b0 < p.B && (notes || (at.b < 0 && n_tiles > 0)); b0 += 32) {
            Step st;
            st.total = 0;
            if (b0 + lane < p.B) st = step_of(p, b0 + lane);
            const int n = st.tiles() * units;
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                if (lane >= o) upto += x;
            }
            if (notes && b0 + lane < p.B) {
                note(b0 + lane, st);
                p.tiles_before[b0 + lane] = before + upto - n;
            }
            const unsigned here = __ballot_sync(0xFFFFFFFFu, before + upto > start);
            if (at.b < 0 && n_tiles > 0 && here) {
                const int who = __ffs(here) - 1, rest = start - before - __shfl_sync(0xFFFFFFFFu, upto - n, who);
                at.b = b0 + who;
                at.st = step_of(p, at.b);
                at.unit = rest / at.st.tiles();
                at.tile = rest - at.unit * at.st.tiles();
            }
            before += __shfl_sync(0xFFFFFFFFu, upto, 31);
        }
        if (notes && lane == 0) p.tiles_before[p.B] = share;
    }
    __syncthreads();                                                         // the barriers are set up
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (n_tiles <= 0 && !p.per_unit) return;
    auto next_unit = [&](Cursor& x) {
        x.tile = 0;
        if (++x.unit < units) return;
        x.unit = 0;
        do x.st = step_of(p, ++x.b); while (x.st.total == 0);                // (asked for only while tiles are left: there is such a sequence)
    };
    const WaitCtx ctx{abort_flag, p.status};

    // ---- thread 0 brings the tiles: up to the last row that the cache held before this step, in whole 16-byte pieces of scales ----
    Cursor ahead = at;
    int brought = 0, tiles_left = 0, rows_left = 0;
    long long row = 0;                               // of the next tile, in the cache; a multiple of 8
    auto aim = [&]() {
        row = ahead.b * p.cache.stride_b + ahead.unit / head_shares * p.cache.stride_h + ahead.tile * kTile;
        rows_left = ahead.st.len - ahead.tile * kTile;
        tiles_left = ahead.st.tiles() - ahead.tile;
    };
    auto bring = [&]() {
        const int s = brought % kStages, rows = min(kTile, (rows_left + 7) & ~7);      // within the capacity: it is a multiple of 8
        unsigned char* to = smem + s * L::kStageBytes;
        if (rows <= 0) {
            mbar_arrive(&full[s]);                                                     // the new token alone
        } else {
            mbar_arrive_expect_tx(&full[s], 2 * rows * (L::kRow + L::kScales));
            bulk_load(to, p.cache.k_codes + row * L::kRow, rows * L::kRow, &full[s]);
            bulk_load(to + L::kKScales, p.cache.k_scales + row * L::kScales, rows * L::kScales, &full[s]);
            bulk_load(to + L::kVCodes, p.cache.v_codes + row * L::kRow, rows * L::kRow, &full[s]);
            bulk_load(to + L::kVScales, p.cache.v_scales + row * L::kScales, rows * L::kScales, &full[s]);
        }
        row += kTile;
        rows_left -= kTile;
        if (++brought < n_tiles && --tiles_left == 0) {
            next_unit(ahead);
            aim();
        }
    };
    if (tid == 0 && n_tiles > 0) {
        aim();
        for (int t = 0; t < min(kStages, n_tiles); ++t) bring();
    }

    const int key_row = tile_row(g);
    uint32_t magic;
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
    bool ok = true;                                  // false: a wait has expired, and only the barriers are gone through from there on
    int t = 0;                                       // tiles of this CTA that are done
    do {
        const int b = at.b, h = at.unit / head_shares, share = at.unit % head_shares;
        const int head0 = h * rep + share * kHeads, n_heads = min(kHeads, rep - share * kHeads);
        const Step st = at.st;
        const int unit_tiles = st.tiles(), n_here = min(unit_tiles - at.tile, n_tiles - t);     // of this unit
        const int begin = at.tile * kTile, end = min(st.total, begin + n_here * kTile);

        // ---- the queries of head g: 32 (or 16) neighbouring elements per thread, brought near one by a power of two, as fp16 and the rest in fp16 ----
        uint32_t hi[4 * L::kKeyWords], lo[4 * L::kKeyWords];                 // [word][pair j]: elements j and j + 4
        float q_factor;
        {
            float f[8 * L::kKeyWords], top = 0.f;
            const bool live = g < n_heads;
            const T* qp = static_cast<const T*>(p.q.ptr) + b * p.q.sb + (head0 + (live ? g : 0)) * p.q.sh + c * (8 * L::kKeyWords);
#pragma unroll
            for (int w = 0; w < L::kKeyWords; ++w) {
                const uint4 v = *reinterpret_cast<const uint4*>(qp + 8 * w);
                const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 x = Elem<T>::unpack2(u[i]);
                    f[8 * w + 2 * i] = live ? x.x : 0.f;
                    f[8 * w + 2 * i + 1] = live ? x.y : 0.f;
                    top = fmaxf(top, fmaxf(fabsf(f[8 * w + 2 * i]), fabsf(f[8 * w + 2 * i + 1])));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 1), 253);
            const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23), up = __uint_as_float(static_cast<uint32_t>(e) << 23);
            // the scale's sign goes into the queries, so that the largest product is the largest score
            const float sign = p.scale > 0.f ? 1.f : p.scale < 0.f ? -1.f : p.scale;
            // (never 0, which would make NaN of the -infinity of a masked score; below the least normal number, scores are nothing beside 1 whatever it is)
            q_factor = sign == 0.f ? 1.f : fmaxf(fabsf(p.scale) * kLog2e * 8.0f * p.cache.k_unit * up, 1.17549435e-38f);
#pragma unroll
            for (int w = 0; w < L::kKeyWords; ++w)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = f[8 * w + j] * (down * sign), y = f[8 * w + j + 4] * (down * sign);
                    const __half2 a = __floats2half2_rn(x, y);
                    const float2 back = __half22float2(a);
                    hi[4 * w + j] = h2(a);
                    lo[4 * w + j] = h2(__floats2half2_rn(x - back.x, y - back.y));
                }
        }

        // ---- the new token: rounded by the warp in whose rows it falls; threads [0, D / 8) hold the words of its key, the next D / 8 of its value ----
        const int new_row = st.append && st.len >= begin && st.len < end ? st.len - begin : -1;
        const bool holds_new = new_row >= 0 && new_row % kTile / kRows == warp;
        uint32_t new_word = 0;
        uint8_t new_scale = 0;
        if (holds_new && lane < 2 * (D / 8)) {
            const bool value = lane >= D / 8;
            const int w = lane % (D / 8);
            const View4& in = value ? p.v_new : p.k_new;
            const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const T*>(in.ptr) + b * in.sb + h * in.sh + w * 8);
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = Elem<T>::unpack2(u[i]);
                x[2 * i] = f.x; x[2 * i + 1] = f.y;
            }
            uint32_t got[1];
            encode<8>(x, 1.0f / (value ? p.cache.v_unit : p.cache.k_unit), 0xFu << (lane & 28), got, new_scale);
            new_word = got[0];
            if (share == 0) {
                const long long row = b * p.cache.stride_b + h * p.cache.stride_h + st.len;
                reinterpret_cast<uint32_t*>(value ? p.cache.v_codes : p.cache.k_codes)[row * (D / 8) + w] = new_word;
                if (w % 4 == 0) (value ? p.cache.v_scales : p.cache.k_scales)[row * L::kScales + w / 4] = new_scale;
            }
        }

        float o[L::kOutTiles][4];                    // [tile][element t or its partner of heads 2c, 2c + 1]
#pragma unroll
        for (int i = 0; i < L::kOutTiles; ++i) { o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f; }
        float m = -INFINITY, l = 0.f;                // of head g: reference of the weights (log2 units), this thread's share of their sum
        for (int j = 0; j < n_here; ++j, ++t) {
            const int s = t % kStages;
            ok = ok && mbar_wait_warp(&full[s], (t / kStages) & 1, ctx, 0x42);
            unsigned char* tile = smem + s * L::kStageBytes;
            const int live = end - (begin + j * kTile) - warp * kRows;       // rows of this warp's that exist
            if (ok && live > 0) {
                if (holds_new && new_row / kTile == j) {
                    if (lane < 2 * (D / 8)) {
                        const bool value = lane >= D / 8;
                        const int w = lane % (D / 8), r = new_row % kTile;
                        *reinterpret_cast<uint32_t*>(tile + (value ? L::kVCodes : 0) + r * L::kRow + w * 4) = new_word;
                        if (w % 4 == 0) tile[(value ? L::kVScales : L::kKScales) + r * L::kScales + w / 4] = new_scale;
                    }
                    __syncwarp();
                }
                if (live < kRows) {                                           // rows behind the last one: anything may stand there, NaN scales too
                    for (int r = lane; r < kRows; r += 32)
                        if (r >= live)
#pragma unroll
                            for (int i = 0; i < L::kScales; ++i) tile[L::kVScales + (warp * kRows + r) * L::kScales + i] = 0;
                    __syncwarp();
                }
                const unsigned char* k_codes = tile + warp * kRows * L::kRow + c * (4 * L::kKeyWords);
                const unsigned char* k_scales = tile + L::kKScales + warp * kRows * L::kScales + (D == 128 ? c : c >> 1);
                float sc[kTiles8][4];
#pragma unroll
                for (int n = 0; n < kTiles8; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
                for (int n0 = 0; n0 < kTiles8; n0 += kAtOnce) {               // independent chains of products
                    Words<L::kKeyWords> k[kAtOnce];
                    uint32_t scale[kAtOnce];
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        const int row = (n0 + i) * 8 + key_row;
                        k[i] = load_words<L::kKeyWords>(k_codes + row * L::kRow);
                        scale[i] = k_scales[row * L::kScales];
                    }
                    Scale2 f[kAtOnce];
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) f[i] = Scale2(scale[i] * 0x0101u);
#pragma unroll
                    for (int w = 0; w < L::kKeyWords; ++w)
#pragma unroll
                        for (int i = 0; i < kAtOnce; ++i) {
                            uint32_t x[4];
                            expand(k[i].w[w], f[i], magic, x);
                            mma(sc[n0 + i], hi[4 * w], lo[4 * w], hi[4 * w + 1], lo[4 * w + 1], x[0], x[1]);
                            mma(sc[n0 + i], hi[4 * w + 2], lo[4 * w + 2], hi[4 * w + 3], lo[4 * w + 3], x[2], x[3]);
                        }
                }
                const unsigned char* v_codes = tile + L::kVCodes + warp * kRows * L::kRow + g * (4 * L::kValueWords);
                const unsigned char* v_scales = tile + L::kVScales + warp * kRows * L::kScales + (D == 128 ? g >> 1 : g >> 2);
                auto values = [&](int u, uint32_t (&x)[2][2 * L::kValueWords][4]) {
                    // rows of columns 2c, 2c + 1 of both 8-key tiles: [0][.] of the first, [1][.] of the second
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int ra = u * 16 + half * 8 + tile_row(2 * c), rb = u * 16 + half * 8 + tile_row(2 * c + 1);
                        const Words<L::kValueWords> a = load_words<L::kValueWords>(v_codes + ra * L::kRow), bw = load_words<L::kValueWords>(v_codes + rb * L::kRow);
                        const Scale2 f(v_scales[ra * L::kScales] | (static_cast<uint32_t>(v_scales[rb * L::kScales]) << 8));
#pragma unroll
                        for (int w = 0; w < L::kValueWords; ++w) {
                            expand(__byte_perm(a.w[w], bw.w[w], 0x5410), f, magic, x[half][2 * w]);
                            expand(__byte_perm(a.w[w], bw.w[w], 0x7632), f, magic, x[half][2 * w + 1]);
                        }
                    }
                };
                uint32_t x[kEarly][2][2 * L::kValueWords][4];
#pragma unroll
                for (int u = 0; u < kEarly; ++u) values(u, x[u]);
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < kTiles8; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        sc[n][e] += sc[n][e + 2];
                        top = fmaxf(top, sc[n][e]);
                    }
                if (live < kRows) {                                           // the last rows of the sequence
                    top = -INFINITY;
#pragma unroll
                    for (int n = 0; n < kTiles8; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if (n * 8 + tile_row(2 * c + e) >= live) sc[n][e] = -INFINITY;
                            top = fmaxf(top, sc[n][e]);
                        }
                }
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                top *= q_factor;
                const bool grow = top > m + kRescale;
                if (__any_sync(0xFFFFFFFFu, grow)) {
                    const float next = grow ? top : m;
                    const float keep = m == -INFINITY ? 0.f : fast_exp2(m - next);
                    l *= keep;
                    m = next;
                    const float k0 = __shfl_sync(0xFFFFFFFFu, keep, 8 * c), k1 = __shfl_sync(0xFFFFFFFFu, keep, 8 * c + 4);
#pragma unroll
                    for (int i = 0; i < L::kOutTiles; ++i) { o[i][0] *= k0; o[i][1] *= k1; o[i][2] *= k0; o[i][3] *= k1; }
                }
                const float zero = m == -INFINITY ? 0.f : m - kLift;          // every score so far -infinity: weights of zero
                uint32_t weight[kTiles8];
#pragma unroll
                for (int n = 0; n < kTiles8; ++n) {
                    const float x = fast_exp2(fmaf(sc[n][0], q_factor, -zero)), y = fast_exp2(fmaf(sc[n][1], q_factor, -zero));
                    l += x + y;
                    weight[n] = h2(__floats2half2_rn(x, y));
                }
#pragma unroll
                for (int u = 0; u < kTiles8 / 2; ++u) {
                    if (u >= kEarly) values(u, x[u % kEarly]);
#pragma unroll
                    for (int i = 0; i < L::kOutTiles; ++i) {
                        // D = 128: rows of the tile are elements i and 8 + i of this thread's 16; D = 64: i and 4 + i of its 8
                        const int w0 = D == 128 ? i / 4 : 0, w1 = D == 128 ? 2 + i / 4 : 1, e = i % 4;
                        uint32_t (&y)[2][2 * L::kValueWords][4] = x[u % kEarly];
                        mma(o[i], y[0][w0][e], y[0][w1][e], y[1][w0][e], y[1][w1][e], weight[2 * u], weight[2 * u + 1]);
                    }
                }
            }
            if (j + 1 < n_here) {                                             // (the slot of a unit's last tile is needed below)
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);
            }
            // the slot of the tile before this one: the other warps are done with it by now, or nearly
            if (tid == 0 && ok && t >= 1 && t - 1 + kStages < n_tiles && mbar_wait(&empty[(t - 1) % kStages], ((t - 1) / kStages) & 1, ctx, 0x41)) bring();
        }

        // ---- merge the warps in the slot of the unit's last tile ----
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
        __syncthreads();
        const int slot = (t + kStages - 1) % kStages;                        // (of tile t - 1; a sequence without rows: any)
        float* part = reinterpret_cast<float*>(smem + slot * L::kStageBytes);                            // [warp][head][D + 2]
#pragma unroll
        for (int i = 0; i < L::kOutTiles; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = D == 128 ? 16 * g + i + 8 * (e >> 1) : 8 * g + i + 4 * (e >> 1);
                part[(warp * kHeads + 2 * c + (e & 1)) * (D + 2) + d] = o[i][e];
            }
        if (c == 0) { part[(warp * kHeads + g) * (D + 2) + D] = m - kLift; part[(warp * kHeads + g) * (D + 2) + D + 1] = l; }
        __syncthreads();
        const bool whole = n_here == unit_tiles;
        float* records = p.records + (static_cast<long long>(blockIdx.x) + b * units + at.unit) * (kHeads * (D + 2));
        if (ok && !*ctx.abort_flag)
            for (int i = tid; i < n_heads * D; i += kThreads) {
                const int r = i / D, d = i % D;
                float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part[(w * kHeads + r) * (D + 2) + D]);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float* rec = part + (w * kHeads + r) * (D + 2);
                    const float f = rec[D] == -INFINITY ? (rec[D + 1] == 0.f ? 0.f : rec[D + 1]) : fast_exp2(rec[D] - top);      // (no reference, a sum that is NaN: NaN)
                    sum += rec[D + 1] * f;
                    acc += rec[d] * f;
                }
                const float value = sum == 0.f ? 0.f : acc / sum * (8.0f * p.cache.v_unit);
                const int hq = head0 + r;
                if (whole) {
                    static_cast<T*>(p.o.ptr)[b * p.o.sb + hq * p.o.sh + d] = Elem<T>::from_f(value);
                    if (p.lse && d == 0) p.lse[b * p.Hq + hq] = sum == 0.f ? -INFINITY : (top + fast_log2(sum)) * kLn2;
                } else {
                    records[r * (D + 2) + d] = value;
                    if (d == 0) { records[r * (D + 2) + D] = top; records[r * (D + 2) + D + 1] = sum; }
                }
            }
        if (t < n_tiles) {
            fence_proxy_async_smem();                // what was written into the slot here comes before the copy that fills it next
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[slot]);
            next_unit(at);
        }
    } while (t < n_tiles);
    if (*ctx.abort_flag) {                           // copies of an abandoned tile may still be landing: far longer than one takes
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {}
    }
}

// Merges the parts of a query head whose unit several CTAs had: o = sum_i o_i l_i 2^(m_i - m) / sum_i l_i 2^(m_i - m); writes the zeros of sequences without rows
// and stores the advanced length.  Every CTA and unit that meet have a record of their own at CTA + unit: along the row of tiles both only grow, so no
// two meetings share one, and a unit's parts lie one behind the other.  THREADS / D groups of parts.
template <typename T, int D, int THREADS>
__global__ void __launch_bounds__(THREADS) decode_kv4_combine_kernel(DecodeKv4Params p, int head_shares) {
    constexpr int kGroups = THREADS / D;
    __shared__ float sum_of[kGroups][D], l_of[kGroups];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int hq = blockIdx.x, b = blockIdx.y, d = threadIdx.x % D, group = threadIdx.x / D;
    constexpr int kRecord = kHeads * (D + 2);
    const int used = p.lens_used[b], total = StepLen::header_total(used);
    if (p.advance_lens && hq == 0 && threadIdx.x == 0 && StepLen::header_appended(used)) p.seq_lens[b] = total;
    if (p.per_unit) return;
    const int rep = p.Hq / p.Hkv, units = p.Hkv * head_shares, unit = hq / rep * head_shares + hq % rep / kHeads;
    const int share = p.tiles_before[p.B], tiles = (total + kTile - 1) / kTile, start = p.tiles_before[b] + unit * tiles;
    const int first = start / share, n = tiles == 0 ? 0 : (start + tiles - 1) / share - first + 1;
    if (n == 1) return;                                                      // written by the CTA that had it
    const float* rec = p.records + (static_cast<long long>(first) + b * units + unit) * kRecord + hq % rep % kHeads * (D + 2);
    constexpr int kAhead = 8;
    float ahead[kAhead];                                                     // one round trip for the references and the first values of each group
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ahead[i] = group + i * kGroups < n ? rec[static_cast<long long>(group + i * kGroups) * kRecord + d] : 0.f;
    float m_first = -INFINITY, l_first = 0.f;                                // of part `lane`
    if ((threadIdx.x & 31) < n) { m_first = rec[(threadIdx.x & 31) * kRecord + D]; l_first = rec[(threadIdx.x & 31) * kRecord + D + 1]; }
    float top = (threadIdx.x & 31) < n ? m_first : -INFINITY;
    for (int i = 32 + (threadIdx.x & 31); i < n; i += 32) top = fmaxf(top, rec[static_cast<long long>(i) * kRecord + D]);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    float acc = 0.f, sum = 0.f;
    // (no reference and no sum: a part of scores of -infinity; no reference and a sum: NaN)
    auto weight = [&](float m, float l) { return m == -INFINITY && l == 0.f ? 0.f : l * fast_exp2(m == -INFINITY ? 0.f : m - top); };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int at = group + i * kGroups;
        const bool known = i * kGroups + kGroups <= 32;                      // the first 32 parts: from the warp's registers
        float m = __shfl_sync(0xFFFFFFFFu, m_first, at & 31), l = __shfl_sync(0xFFFFFFFFu, l_first, at & 31);
        if (at >= n) continue;
        if (!known) { m = rec[at * kRecord + D]; l = rec[at * kRecord + D + 1]; }
        const float f = weight(m, l);
        acc = fmaf(f, ahead[i], acc);
        sum += f;
    }
    for (int i = group + kAhead * kGroups; i < n; i += kGroups) {
        const float f = weight(rec[static_cast<long long>(i) * kRecord + D], rec[static_cast<long long>(i) * kRecord + D + 1]);
        acc = fmaf(f, rec[static_cast<long long>(i) * kRecord + d], acc);
        sum += f;
    }
    sum_of[group][d] = acc;
    if (d == 0) l_of[group] = sum;
    __syncthreads();
    if (group == 0) {
        acc = 0.f; sum = 0.f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) { acc += sum_of[i][d]; sum += l_of[i]; }
        static_cast<T*>(p.o.ptr)[b * p.o.sb + hq * p.o.sh + d] = Elem<T>::from_f(sum == 0.f ? 0.f : acc / sum);
        if (p.lse && d == 0) p.lse[b * p.Hq + hq] = sum == 0.f ? -INFINITY : (top + fast_log2(sum)) * kLn2;
    }
}

template <typename F, typename... Args>
cudaError_t launch_dependent(F kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, int D>
int launch_t(cudaStream_t s, const DecodeKv4Params& p) {
    static thread_local bool configured[64] = {};      // per device ordinal: the attribute belongs to the device's context
    int dev = 0;
    VB200_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return set_detail(VB200_ERR_NO_DEVICE, "device ordinal out of range");
    if (!configured[dev]) {
        VB200_CUDA_TRY(cudaFuncSetAttribute(decode_kv4_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kSmem));
        configured[dev] = true;
    }
    const int shares = (p.Hq / p.Hkv + kHeads - 1) / kHeads;
    profile_mark_begin(s);
    VB200_CUDA_TRY(launch_dependent(decode_kv4_kernel<T, D>, dim3(p.ctas), kThreads, Layout<D>::kSmem, s, p, shares));
    profile_mark_end(s);
    note_launch();
    if (!p.per_unit || p.advance_lens) {
        // Many parts to a unit: 512 threads a head (131072 keys of one sequence, 37 parts: 47.0 us, with 128 threads 49.9); few parts, but many heads: 128
        // (32 sequences of 1024-8192 keys: 54.0 us, with 512 threads 57.6).
        const dim3 grid(p.Hq, p.B);
        if (p.ctas >= 8LL * p.B * p.Hkv * shares) VB200_CUDA_TRY(launch_dependent(decode_kv4_combine_kernel<T, D, 512>, grid, 512, 0, s, p, shares));
        else VB200_CUDA_TRY(launch_dependent(decode_kv4_combine_kernel<T, D, 128>, grid, 128, 0, s, p, shares));
        note_launch();
    }
    return VB200_OK;
}

}  // namespace

int launch_decode_kv4(cudaStream_t s, const DecodeKv4Params& p) {
    if (p.dtype == VB200_BF16) return p.D == 128 ? launch_t<__nv_bfloat16, 128>(s, p) : launch_t<__nv_bfloat16, 64>(s, p);
    return p.D == 128 ? launch_t<__half, 128>(s, p) : launch_t<__half, 64>(s, p);
}

}  // namespace vb200
