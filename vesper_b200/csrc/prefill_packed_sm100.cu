// Attention over packed prompts on the tensor cores.
//
//   s_ij = scale q_i . k_j,  key j of n_k visible to query i of n_q iff j <= n_k - n_q + i (causal) or always
//   O_i = sum_j softmax_j(s_ij) v_j,  LSE_i = ln sum_j exp(s_ij);  zeros and -infinity where no key is visible
//
// A tile is 128 rows: 128 / F tokens of one sequence by F heads of one key head's group (F: the power of two of the group, at most 16), row = token * F +
// head, as one TMA box of q brings them.  Short sequences fill a tile with heads instead of padding, and the rows of a tile see nearly the same keys.  A work
// item is two tiles of neighbouring tokens that read the same blocks of keys; where the sequences are short, two blocks of heads of the same tokens
// (two_head_blocks).  The lengths are on the device: a first kernel lists the items with the longest first, then persistent CTAs, one per SM, take the next one
// of the list as they get done.  (Dealt out beforehand, up and down the CTAs: 492 us instead of 473 for 24 prompts of 16-4057 tokens, 32 heads on 8 of 128; 62
// instead of 55 for 17 of 100-1500, 16 heads on 2.)
//   warps 0-3    softmax and epilogue of tile 0, a row per thread (TMEM lane)
//   warps 4-7    the same for tile 1
//   warp  8      the items, which it tells the others of; TMA: q tiles (3 buffers, so that the next item's come while this one computes) and the ring of key and value blocks
//   warps 9, 10  tcgen05.mma issuers of tile 0 and of tile 1; warp 9 owns the TMEM
// TMEM (512 columns): per tile the scores S of a block, its weights (16 bits, two to a column) beside them, and O.  The weights do not overwrite the scores, so
// that the next block's Q K^T is made while this block's weights are computed: with head_dim 128 a block is 80 keys (2 x (80 + 40 + 128) columns), with 64 it is
// 112 (2 x (112 + 56 + 64); 128 would fit, and its scores spill registers).  (Blocks of 128 keys whose weights overwrote their scores, head_dim 128: 518 us for 24
// prompts of 16-4057 tokens, tensor pipe busy 49 %, the softmax and the products of a tile waiting for each other.)
// The last block of a tile takes only the columns and rows of V, by 16, that a row of it can see.  The rows of V behind the sequence in its last
// 16 are another sequence's, or nobody's: they are cleared in shared memory, since a weight of zero does not silence a NaN.
// What bounds it: the softmax and the products of a tile in turn (long portions: tensor pipe 67 %, special function unit 67 %).  Causal, 32 heads on 8 of 128: 24
// prompts of 16-4057 tokens 477 us, 1085 TFLOP/s (557 us where calls before it keep the card at its power limit); not causal: 8192 tokens 828 us, 1327 TFLOP/s, with
// 32 key heads of 64 742 us, 741 TFLOP/s (one after the other, at the power limit, 800-925 us).
// All weights come from the special function unit.  (One pair in eight from a polynomial on the FMA pipe gains nothing as long as it keeps NaN: 812 us for the
// 8192 tokens at a clock where this takes 802.)
// Every wait is bounded (mbar_wait); on expiry the CTA drains and returns with the status word set.
#include "hybrid.cuh"
#include "serving.h"

#include <algorithm>
#include <cstdio>
#include <type_traits>

namespace vb200 {

namespace {

constexpr int kBlockM = 128;
constexpr int kQBufs = 3;
constexpr int kProducerWarp = 8, kMmaWarp = 9;
constexpr int kThreads = 384;              // three warpgroups: registers are moved by warpgroups
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.0f;           // weights stay within 2^8 of the running reference
constexpr float kLift = 7.0f;              // which weighs 2^7, so that fp16 weights keep their precision down to 2^-21 of it
constexpr int kRegSoftmax = 216, kRegOther = 72;
static_assert(kRegSoftmax * 256 + kRegOther * 128 <= 168 * 384, "register budget");

// Two tiles of a sequence, without the head block: tokens [q0, q0 + tokens), keys [k0, k0 + keys), of which the last that token i
// sees is `last` + i (causal).
struct alignas(16) Item {
    int q0, tokens, k0, keys;
    int last, end[2];                      // keys that some row of each tile sees; -1: the tile has no tokens
    int head;                              // first head of the block (set as the item is taken from the list)
};

struct Plan {                              // workspace: the header, the items, the first item of each sequence
    int items;
    int next;                              // item that the next CTA in want of one takes
};

struct Shape {
    int fold, tokens;                      // heads and tokens of a tile
    int dual, item_tokens;                 // whether an item's tiles are two head blocks of the same tokens; tokens of an item
    int head_blocks;                       // items of the same tokens
    int max_items, room;                   // without head blocks; what a workspace holds (it does not shrink as tokens are added)
};
Shape shape_of(int batch, int Hq, int Hkv, int total_q, bool dual = false) {
    Shape s;
    const int rep = Hq / Hkv;
    s.fold = 1;
    while (s.fold < 16 && rep % (2 * s.fold) == 0) s.fold *= 2;
    s.tokens = kBlockM / s.fold;
    s.dual = dual;
    s.item_tokens = dual ? s.tokens : 2 * s.tokens;
    s.head_blocks = Hq / s.fold / (dual ? 2 : 1);
    s.max_items = total_q / s.item_tokens + batch;
    s.room = total_q / s.tokens + batch;
    return s;
}
// Sequences of about a tile leave the second tile of an item empty, or nearly: there its tiles are two blocks of heads, which costs keys and values of their own
// for both.  Lengths are known by their mean alone.  Measured over lengths spread 2- to 16-fold: with head_dim 64 it gains 5 to 27 % at a mean of 0.9 tiles and loses
// 3 to 11 % at 1.4, with 128 it gains up to 20 % at 0.7 and loses up to 14 % at 0.9 (blocks of keys are twice as large); and always where items of
// neighbouring tokens already fit the SMs at once, up to 40 %.  (40 sequences of 20-494 tokens, 16 heads of 64: 33.2 us, with tiles of neighbouring tokens 36.3.)
bool two_head_blocks(const PackedParams& p, const Shape& s) {
    return s.head_blocks % 2 == 0 && 4ll * p.total_q <= static_cast<int64_t>(p.batch) * s.tokens * (p.D == 64 ? 5 : 3) &&
           static_cast<int64_t>(p.batch) * s.head_blocks > device_sm_count();
}

// ---- the list of items, by descending number of keys ----
constexpr int kPlanThreads = 1024, kBins = 1024;

__device__ __forceinline__ int bin_of(int keys) {        // longest first
    const int blocks = (max(keys, 0) + 63) / 64;
    return kBins - 1 - (blocks < 512 ? blocks : 512 + min(511, (blocks - 512) >> 4));
}

struct Sequence {
    int q0, nq, k0, nk;
};
// a sequence whose offsets are not in order or not within the tokens is left out
__device__ __forceinline__ Sequence sequence_of(const PackedParams& p, int i) {
    const int a = p.cu_q[i], b = p.cu_q[i + 1], x = p.cu_k[i], y = p.cu_k[i + 1];
    const bool ok = a >= 0 && a <= b && b <= p.total_q && x >= 0 && x <= y && y <= p.total_k;
    return ok ? Sequence{a, b - a, x, y - x} : Sequence{0, 0, 0, 0};
}

__device__ __forceinline__ Item make_item(const PackedParams& p, const Shape& shape, const Sequence& s, int r0) {
    Item w;
    w.q0 = s.q0 + r0;
    w.tokens = min(shape.item_tokens, s.nq - r0);
    w.k0 = s.k0;
    w.keys = s.nk;
    w.last = p.causal ? s.nk - s.nq + r0 : s.nk - 1;
    w.head = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int first = shape.dual ? 0 : t * shape.tokens;                 // of the tile's tokens
        const int end = p.causal ? max(0, min(s.nk, w.last + min(w.tokens, first + shape.tokens))) : s.nk;
        w.end[t] = w.tokens > first ? end : -1;
    }
    return w;
}

constexpr int kAtHand = 1024;              // sequences that the planning block keeps in shared memory

__global__ void __launch_bounds__(kPlanThreads, 1) packed_plan_kernel(PackedParams p, Shape shape, int ctas, Plan* plan, Item* items, int* first_in_memory) {
    __shared__ int hist[kBins];
    __shared__ long long warp_sum[32];
    __shared__ int first_at_hand[kAtHand + 1];
    __shared__ Sequence at_hand[kAtHand];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, pair = shape.item_tokens, max_items = shape.max_items;
    const bool small = p.batch <= kAtHand;
    int* first_item = small ? first_at_hand : first_in_memory;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the attention kernel sets itself up meanwhile, and waits for this one
    hist[tid] = 0;
    // first item of each sequence: every thread a piece of the sequences, then a sum over the threads before it
    const int per = (p.batch + kPlanThreads - 1) / kPlanThreads, i0 = min(tid * per, p.batch), i1 = min(i0 + per, p.batch);
    long long mine = 0;                                  // (offsets that do not ascend may name more tokens than there are)
    for (int i = i0; i < i1; ++i) {
        const Sequence s = sequence_of(p, i);
        if (small) at_hand[i] = s;
        mine += (s.nq + pair - 1) / pair;
    }
    auto sequence = [&](int i) { return small ? at_hand[i] : sequence_of(p, i); };
    auto scan = [&](long long x) {                       // inclusive, over the block
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xFFFFFFFFu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) warp_sum[warp] = x;
        __syncthreads();
        if (warp == 0) {
            long long y = warp_sum[lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long z = __shfl_up_sync(0xFFFFFFFFu, y, o);
                if (lane >= o) y += z;
            }
            warp_sum[lane] = y;
        }
        __syncthreads();
        const long long before = warp > 0 ? warp_sum[warp - 1] : 0;
        __syncthreads();
        return x + before;
    };
    long long next = scan(mine) - mine;
    for (int i = i0; i < i1; ++i) {
        first_item[i] = static_cast<int>(min(next, static_cast<long long>(max_items)));
        next += (sequence(i).nq + pair - 1) / pair;
    }
    if (i1 == p.batch && i0 < i1) {
        const int n = static_cast<int>(min(next, static_cast<long long>(max_items)));      // (offsets in order leave no more than max_items)
        first_item[p.batch] = n;
        plan->items = n;
        plan->next = 2 * ctas;                           // (CTA c starts with the items c and 2 ctas - 1 - c)
    }
    __syncthreads();
    const int n = first_item[p.batch];
    auto item_at = [&](int idx) {
        int lo = 0, hi = p.batch;                        // the last sequence whose first item is at or before idx
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first_item[mid] <= idx) lo = mid; else hi = mid;
        }
        return make_item(p, shape, sequence(lo), (idx - first_item[lo]) * pair);
    };
    for (int idx = tid; idx < n; idx += kPlanThreads) {
        const Item w = item_at(idx);
        atomicAdd(&hist[bin_of(max(w.end[0], w.end[1]))], 1);
    }
    __syncthreads();
    const int count = hist[tid];
    hist[tid] = static_cast<int>(scan(count)) - count;
    __syncthreads();
    for (int idx = tid; idx < n; idx += kPlanThreads) {  // (the order within a bin is free: results do not depend on it)
        const Item w = item_at(idx);
        items[atomicAdd(&hist[bin_of(max(w.end[0], w.end[1]))], 1)] = w;
    }
}

// ---- the attention kernel ----
constexpr int kBoxes = 4;
struct __align__(16) Barriers {
    uint64_t q_full[kQBufs], q_free[kQBufs];
    uint64_t kv_full[8], kv_empty[8];
    uint64_t s_full[2], s_free[2], p_ready[2], o_done[2];
    uint64_t mma_done;
    uint64_t box_full[kBoxes], box_empty[kBoxes];
    Item box[kBoxes];                      // the producer's word to the other warps; no tokens: no more items
    uint32_t tmem_base;
    int abort_flag;
};

struct TmaMaps {
    CUtensorMap q, k, v;
};

template <int D>
struct Cfg {
    static constexpr int kN = D == 128 ? 80 : 112;               // keys of a block
    static constexpr int kStages = D == 128 ? 6 : 8;             // key / value slots
    static constexpr int kHalves = D / 64;                       // 64-column (128-byte) boxes per row
    static constexpr int kQHalf = kBlockM * 128, kQTile = kHalves * kQHalf;
    static constexpr int kKvHalf = kN * 128, kKvTile = kHalves * kKvHalf;
    static constexpr int kTile = kN + kN / 2;                    // TMEM columns of a tile's scores and weights
    static constexpr int kS(int t) { return t * (D == 128 ? 128 : kTile); }
    static constexpr int kP(int t) { return kS(t) + kN; }
    static constexpr int kO(int t) { return 512 - (2 - t) * D; }
    static constexpr int kSmemBytes = kQBufs * kQTile + kStages * kKvTile + 1024 /*alignment slack*/ + sizeof(Barriers);
    static_assert(kP(1) + kN / 2 <= kO(0) && kStages <= 8 && kSmemBytes <= 227 * 1024, "layout");
};
__device__ __forceinline__ int blocks_of(int end, int n) { return end > 0 ? (end + n - 1) / n : 0; }

template <int N> __device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// whether the phase is over, without waiting
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}

// The item of this CTA where no list is made: found by one warp, 32 sequences at a time.  Returns whether there is one.
__device__ __forceinline__ bool find_item(const PackedParams& p, const Shape& shape, Item* own) {
    const int lane = threadIdx.x & 31, pair = shape.item_tokens, want = blockIdx.x / shape.head_blocks;
    int before = 0;
    for (int i0 = 0; i0 < p.batch; i0 += 32) {
        Sequence s{0, 0, 0, 0};
        if (i0 + lane < p.batch) s = sequence_of(p, i0 + lane);
        const int n = (s.nq + pair - 1) / pair;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned here = __ballot_sync(0xFFFFFFFFu, before + upto > want);
        if (here) {
            if (lane == __ffs(here) - 1) *own = make_item(p, shape, s, (want - before - (upto - n)) * pair);
            return true;
        }
        before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    return false;
}

// kList: the items come from the list; else every CTA has at most one, which it finds itself.  kDual: Shape::dual.  (Template parameters: with a branch on the
// first head_dim 64 lost 11 %.)
template <typename T, int D, bool kList, bool kDual>
__global__ void __launch_bounds__(kThreads, 1) prefill_packed_kernel(const __grid_constant__ TmaMaps maps, PackedParams p, Shape shape, Plan* plan, const Item* items) {
    using C = Cfg<D>;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));      // 128B-swizzled tiles
    unsigned char* q_smem = smem;                                   // kQBufs tiles
    unsigned char* kv_smem = smem + kQBufs * C::kQTile;             // C::kStages tiles
    Barriers* bar = reinterpret_cast<Barriers*>(kv_smem + C::kStages * C::kKvTile);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- setup ----
    if (warp == kMmaWarp) {
        if (lane == 0) {
            for (int b = 0; b < kQBufs; ++b) { mbar_init(&bar->q_full[b], 1); mbar_init(&bar->q_free[b], 1); }
            for (int t = 0; t < 2; ++t) { mbar_init(&bar->s_full[t], 1); mbar_init(&bar->s_free[t], 4); mbar_init(&bar->p_ready[t], 4); mbar_init(&bar->o_done[t], 1); }
            for (int s = 0; s < C::kStages; ++s) { mbar_init(&bar->kv_full[s], 1); mbar_init(&bar->kv_empty[s], 2); }
            mbar_init(&bar->mma_done, 2);
            for (int s = 0; s < kBoxes; ++s) { mbar_init(&bar->box_full[s], 1); mbar_init(&bar->box_empty[s], 10); }      // two issuers, eight warps
            bar->abort_flag = 0;
            mbar_fence_init();
        }
        __syncwarp();
        tmem_alloc(&bar->tmem_base, 512);
        tmem_relinquish();
        tc_fence_before();
    } else if (warp == kProducerWarp && lane == 0) {
        tma_prefetch_desc(&maps.q); tma_prefetch_desc(&maps.k); tma_prefetch_desc(&maps.v);
    }
    __syncthreads();
    tc_fence_after();
    asm volatile("griddepcontrol.wait;" ::: "memory");              // the list of items
    __shared__ Item own;
    const int head_step = kDual ? 2 * shape.fold : shape.fold;
    if constexpr (!kList) {
        if (warp == 0) {
            const bool found = find_item(p, shape, &own);
            __syncwarp();
            if (lane == 0) {
                if (!found) own = Item{};
                own.head = blockIdx.x % shape.head_blocks * head_step;
            }
        }
        __syncthreads();
    }
    const uint32_t tmem_base = bar->tmem_base;
    const WaitCtx abort_flag{&bar->abort_flag, p.status};
    const int rep = p.Hq / p.Hkv;
    // the items of this CTA, one after the other, as the producer tells of them; null: no more (or a wait has expired)
    int taken_items = 0;
    auto take = [&](auto wait) -> const Item* {
        const int n = taken_items++;
        const Item* w = &own;
        if constexpr (kList) {
            const int s = n % kBoxes;
            if (!wait(&bar->box_full[s], (n / kBoxes) & 1)) return nullptr;
            w = &bar->box[s];
        } else if (n > 0) {
            return nullptr;
        }
        return w->tokens > 0 ? w : nullptr;
    };
    auto give_back = [&]() { if (kList) mbar_arrive(&bar->box_empty[(taken_items - 1) % kBoxes]); };

    if (warp >= 8) {
        reg_dec<kRegOther>();
        if (warp == kProducerWarp) {
            // =========================== TMA producer ===========================
            if (lane == 0) {
                int kv_item = 0;                 // running index into the ring over all items
                int q_seq = 0;                   // running index of q tiles -> buffer q_seq % kQBufs
                bool ok = true;
                auto load_q = [&](const Item& w, int t) {
                    if (w.end[t] <= 0 || !ok) return;
                    const int b = q_seq % kQBufs, use = q_seq / kQBufs;
                    if (use > 0) ok = mbar_wait(&bar->q_free[b], (use - 1) & 1, abort_flag, 0x110 + b);      // its last product has been made
                    if (!ok) return;
                    ++q_seq;
                    mbar_arrive_expect_tx(&bar->q_full[b], C::kQTile);
#pragma unroll
                    for (int h = 0; h < C::kHalves; ++h)
                        tma_load_4d(q_smem + b * C::kQTile + h * C::kQHalf, &maps.q, &bar->q_full[b], h * 64, kDual ? w.head + t * shape.fold : w.head, kDual ? w.q0 : w.q0 + t * shape.tokens, 0);
                };
                int told = 0;
                auto tell = [&](const Item& w) {
                    if constexpr (kList) {
                        const int s = told % kBoxes;
                        if (told >= kBoxes) ok = ok && mbar_wait(&bar->box_empty[s], (told / kBoxes - 1) & 1, abort_flag, 0x120);
                        if (!ok) return;
                        bar->box[s] = w;
                        mbar_arrive(&bar->box_full[s]);
                        ++told;
                    }
                };
                auto item_of = [&](int idx) {
                    Item w;
                    const int4* src = reinterpret_cast<const int4*>(items + idx / shape.head_blocks);
                    int4* dst = reinterpret_cast<int4*>(&w);
                    dst[0] = src[0]; dst[1] = src[1];
                    w.head = idx % shape.head_blocks * head_step;
                    return w;
                };
                const int n_items = kList ? plan->items * shape.head_blocks : 0;
                int next = 2 * gridDim.x - 1 - blockIdx.x;
                Item w{};
                if constexpr (!kList) w = own;
                else if (static_cast<int>(blockIdx.x) < n_items) w = item_of(blockIdx.x);
                load_q(w, 0);
                tell(w);
                load_q(w, 1);
                while (w.tokens > 0 && ok) {
                    // one item ahead: its first q tile comes during this item
                    Item wn{};
                    if (kList && next < n_items) {
                        wn = item_of(next);
                        next = atomicAdd(&plan->next, 1);                    // (looked at an item later)
                    }
                    bool announced = false;
                    auto announce = [&]() {
                        if (announced) return;
                        announced = true;
                        tell(wn);
                        load_q(wn, 0);
                    };
                    const int nmax = blocks_of(max(w.end[0], w.end[1]), C::kN);
                    // in the order in which the products take them: K0, then K(j+1), V(j)
                    for (int x = 0; x < 2 * nmax && ok; ++x) {
                        const bool value = x == 2 * nmax - 1 || (x > 0 && (x & 1) == 0);
                        const int block = x == 0 ? 0 : value ? (x - 1) / 2 : (x + 1) / 2;
                        const CUtensorMap* m = value ? &maps.v : &maps.k;
                        for (int t = 0; t < (kDual ? 2 : 1); ++t, ++kv_item) {          // (dual: tile 0's block, then tile 1's)
                            const int slot = kv_item % C::kStages;
                            if (kv_item >= C::kStages) ok = mbar_wait(&bar->kv_empty[slot], ((kv_item / C::kStages) - 1) & 1, abort_flag, 0x100);
                            if (!ok) break;
                            mbar_arrive_expect_tx(&bar->kv_full[slot], C::kKvTile);
#pragma unroll
                            for (int h = 0; h < C::kHalves; ++h)
                                tma_load_4d(kv_smem + slot * C::kKvTile + h * C::kKvHalf, m, &bar->kv_full[slot], h * 64, (w.head + t * shape.fold) / rep, w.k0 + block * C::kN, 0);
                        }
                        if (x == 0) announce();                              // (the item has had this long to come)
                    }
                    announce();
                    load_q(wn, 1);
                    w = wn;
                }
            }
        } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
            // =========================== MMA issuers, one for each tile ===========================
            // One elected thread walks the items, waits and issues: in code that the whole warp runs, a wait costs 100 to 200 cycles and a product 50.  What
            // such a thread has to do for two tiles takes longer than their softmax, so each tile has one.  (8192 keys and queries, 32 heads, a whole
            // warp for both tiles: 915 TFLOP/s, a thread for both: 1132.)
            const int t = warp - kMmaWarp;
            if (elect_one()) {
                // (bit 13 negates A: the scale's sign, so that the largest product is the largest score)
                const uint32_t idesc_qk = make_idesc_f16(Elem<T>::kFormat, 0, 0, kBlockM, C::kN) | (p.scale < 0.f ? 1u << 13 : 0u);
                constexpr uint32_t idesc_pv = make_idesc_f16(Elem<T>::kFormat, 0, 1, kBlockM, D);
                // V is MN-major for its product: 16 keys = 2048 bytes per step, second 64-column box one half-tile further (leading offset)
                const uint64_t q_desc = make_smem_desc_sw128(smem_u32(q_smem), 16, 1024), k_desc = make_smem_desc_sw128(smem_u32(kv_smem), 16, 1024);
                const uint64_t v_desc = make_smem_desc_sw128(smem_u32(kv_smem), C::kKvHalf, 1024);
                // all 512 columns are this CTA's, so they start at 0
                const uint32_t s_tmem = t ? C::kS(1) : C::kS(0), p_tmem = t ? C::kP(1) : C::kP(0), o_tmem = t ? C::kO(1) : C::kO(0);
                auto issue_pv = [&](int slot, int steps, bool accumulate) {
                    const uint64_t bd = v_desc + slot * (C::kKvTile >> 4);
                    if (steps == C::kN / 16) {
#pragma unroll
                        for (int kk = 0; kk < C::kN / 16; ++kk)
                            umma_ts(o_tmem, p_tmem + kk * 8, bd + kk * (2048 >> 4), idesc_pv, (accumulate || kk > 0) ? 1u : 0u);
                    } else {
                        for (int kk = 0; kk < steps; ++kk)
                            umma_ts(o_tmem, p_tmem + kk * 8, bd + kk * (2048 >> 4), idesc_pv, (accumulate || kk > 0) ? 1u : 0u);
                    }
                };
                int slot = 0, kv_phase = 0, qb = 0, q_phase = 0;
                auto next_slot = [&]() { if (++slot == C::kStages) { slot = 0; kv_phase ^= 1; } };
                // a block of the other tile's: handed back when it has come, so that the slot's turns stay in step
                auto skip = [&]() {
                    if (!mbar_wait(&bar->kv_full[slot], kv_phase, abort_flag, 0x201)) return false;
                    mbar_arrive(&bar->kv_empty[slot]);
                    next_slot();
                    return true;
                };
                uint32_t s_phase = 1, p_phase = 0;               // (the first wait for free scores passes: none have been made)
                bool ok = true;
                auto wait_item = [&](uint64_t* b, uint32_t parity) { return mbar_wait(b, parity, abort_flag, 0x230 + t); };
                for (const Item* at; ok && (at = take(wait_item)) != nullptr;) {
                    const Item w = *at;
                    give_back();
                    const int end = t ? w.end[1] : w.end[0], n = blocks_of(end, C::kN), nmax = blocks_of(max(w.end[0], w.end[1]), C::kN);
                    // the q tiles of an item: tile 0's buffer, if it has one, then tile 1's
                    const bool q0 = w.end[0] > 0, q1 = w.end[1] > 0;
                    auto next_q = [&]() { if (++qb == kQBufs) { qb = 0; q_phase ^= 1; } };
                    if (t == 1 && q0) next_q();
                    const int qbuf = qb;
                    const uint64_t qd = q_desc + qbuf * (C::kQTile >> 4);
                    if (n > 0) ok = mbar_wait(&bar->q_full[qbuf], q_phase, abort_flag, 0x210 + t);
                    if (t == 0 ? q0 : q1) next_q();
                    if (t == 0 && q1) next_q();
                    // j = -1: the first scores; then the scores of block j + 1 and the weighted values of block j
                    for (int j = -1; j < nmax && ok; ++j) {
                        if (j + 1 < nmax) {
                            if (kDual && t == 1) ok = skip();
                            ok = ok && mbar_wait(&bar->kv_full[slot], kv_phase, abort_flag, 0x200);
                            if (!ok) break;
                            if (j + 1 < n) {
                                // the scores before these, of this item or the one before it, have been read
                                ok = mbar_wait(&bar->s_free[t], s_phase, abort_flag, 0x220 + t);
                                if (!ok) break;
                                s_phase ^= 1;
                                tc_fence_after();
                                const uint64_t bd = k_desc + slot * (C::kKvTile >> 4);
#pragma unroll
                                for (int kk = 0; kk < D / 16; ++kk)
                                    umma_ss(s_tmem, qd + (((kk >> 2) * C::kQHalf + (kk & 3) * 32) >> 4), bd + (((kk >> 2) * C::kKvHalf + (kk & 3) * 32) >> 4), idesc_qk, kk > 0 ? 1u : 0u);
                                umma_commit(&bar->s_full[t]);
                                umma_commit(&bar->kv_empty[slot]);
                                if (j + 2 == n) umma_commit(&bar->q_free[qbuf]);      // the last product of this q tile
                            } else {
                                mbar_arrive(&bar->kv_empty[slot]);                    // a block for the other tile
                            }
                            next_slot();
                            if (kDual && t == 0) ok = skip();
                        }
                        if (j < 0) continue;
                        if (kDual && t == 1) ok = ok && skip();
                        ok = ok && mbar_wait(&bar->kv_full[slot], kv_phase, abort_flag, 0x300);
                        if (!ok) break;
                        if (j < n) {
                            const int rows = w.keys - j * C::kN;        // of the sequence in this block of V
                            if (rows < C::kN && (rows & 15) != 0) {
                                // the rest of the last 16 rows that a product may take: cleared (by both issuers, each before its own product)
                                const int m = 16 - (rows & 15);
#pragma unroll
                                for (int half = 0; half < C::kHalves; ++half)
                                    for (int i = 0; i < m * 8; ++i)
                                        *reinterpret_cast<uint4*>(kv_smem + slot * C::kKvTile + half * C::kKvHalf + rows * 128 + i * 16) = make_uint4(0, 0, 0, 0);
                                fence_proxy_async_smem();
                            }
                            ok = mbar_wait(&bar->p_ready[t], p_phase, abort_flag, 0x400 + t);
                            if (!ok) break;
                            p_phase ^= 1;
                            tc_fence_after();
                            issue_pv(slot, min(C::kN, end - j * C::kN + 15) >> 4, j > 0);
                            umma_commit(&bar->o_done[t]);
                            umma_commit(&bar->kv_empty[slot]);
                        } else {
                            mbar_arrive(&bar->kv_empty[slot]);
                        }
                        next_slot();
                        if (kDual && t == 0) ok = skip();
                    }
                }
                // everything issued so far has to retire before TMEM is released
                umma_commit(&bar->mma_done);
                mbar_wait(&bar->mma_done, 0, abort_flag, 0x600);
            }
            __syncwarp();
        }
    } else {
        // =========================== softmax / correction / epilogue ===========================
        reg_inc<kRegSoftmax>();
        const int t = warp >> 2;                     // tile of this warpgroup
        const int r = tid & 127;                     // row inside the tile = TMEM lane
        const int first = kDual ? 0 : t * shape.tokens;      // of the tile's tokens
        const int token = first + r / shape.fold, head_in = r % shape.fold + (kDual ? t * shape.fold : 0);
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem_base + lane_base + (t ? C::kS(1) : C::kS(0));
        const uint32_t p_addr = tmem_base + lane_base + (t ? C::kP(1) : C::kP(0));
        const uint32_t o_addr = tmem_base + lane_base + (t ? C::kO(1) : C::kO(0));
        // (a scale of zero: the least normal number, which keeps what is masked at -infinity)
        const float scale_log2 = p.scale == 0.f ? 1.17549435e-38f : fabsf(p.scale) * kLog2e;
        int g = 0;                                   // running count of score tiles of this query tile
        bool ok = true;

        auto wait_item = [&](uint64_t* b, uint32_t parity) { return mbar_wait_warp(b, parity, abort_flag, 0x810 + t); };
        auto done = [&]() {                          // with the item: it stays in its box meanwhile, which leaves its registers to the scores
            __syncwarp();
            if (lane == 0) give_back();
        };
        for (const Item* w; ok && (w = take(wait_item)) != nullptr; done()) {
            const int tile_end = t ? w->end[1] : w->end[0];                 // keys that some row of the tile sees
            if (tile_end < 0) continue;                                     // no tokens in this tile
            const int n = blocks_of(tile_end, C::kN);
            const int limit = p.causal ? min(w->keys - 1, w->last + token) : w->keys - 1;      // last visible key of this row
            const int all_see = p.causal ? min(w->keys, w->last + first + 1) : w->keys;      // keys that every row of the tile sees

            float m_ref = -INFINITY;
            float2 rs[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};      // partial sums of the weights
            for (int j = 0; j < n; ++j, ++g) {
                ok = mbar_wait_warp(&bar->s_full[t], g & 1, abort_flag, 0x800 + t);
                if (!ok) break;
                tc_fence_after();
                const int k0 = j * C::kN, rest = tile_end - k0;             // first key, and columns that some row sees
                uint32_t s[C::kN];
#pragma unroll
                for (int c = 0; c < C::kN / 32; ++c) tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
                if constexpr (C::kN % 32 != 0) tmem_ld16(s_addr + C::kN / 32 * 32, *reinterpret_cast<uint32_t(*)[16]>(&s[C::kN / 32 * 32]));
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar->s_free[t]);                // the next block's scores may come
                const bool masked = k0 + C::kN > all_see;
                if (masked) {
#pragma unroll
                    for (int i = 0; i < C::kN; ++i)
                        if (k0 + i > limit) s[i] = 0xFF800000u;             // -inf
                }
                // row max: 8 independent chains of 3-input max (one thread owns the whole row)
                float mx8[8];
#pragma unroll
                for (int a = 0; a < 8; ++a) mx8[a] = -INFINITY;
#pragma unroll
                for (int i = 0; i < C::kN; i += 2) mx8[(i >> 1) & 7] = fmax3(mx8[(i >> 1) & 7], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                const float mx = fmaxf(fmax3(mx8[0], mx8[1], mx8[2]), fmaxf(fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
                const float m_cand = mx * scale_log2;
                const bool grow = m_cand > m_ref + kRescale;
                // The weights before these have been multiplied, and O is whole.  Looked at here, where the answer has time: it is yes nearly always.
                bool taken = j == 0 || mbar_test(&bar->o_done[t], (g - 1) & 1);
                auto wait_taken = [&]() {
                    if (!__all_sync(0xFFFFFFFFu, taken)) ok = mbar_wait_warp(&bar->o_done[t], (g - 1) & 1, abort_flag, 0x900 + t);
                    taken = true;
                    tc_fence_after();
                };
                if (__any_sync(0xFFFFFFFFu, grow)) {
                    const float m_new = grow ? m_cand : m_ref;
                    const float alpha = (m_ref == -INFINITY) ? 0.f : fast_exp2(m_ref - m_new);
                    if (j > 0) {
                        wait_taken();
                        if (!ok) break;
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            tmem_ld32(o_addr + c * 32, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st32(o_addr + c * 32, o);
                        }
                        tmem_st_wait();
                    }
#pragma unroll
                    for (int a = 0; a < 4; ++a) { rs[a].x *= alpha; rs[a].y *= alpha; }
                    m_ref = m_new;
                }
                const float zero = m_ref == -INFINITY ? 0.f : m_ref - kLift;       // no key seen yet: weights of zero
                const float2 sc2 = make_float2(scale_log2, scale_log2), nm2 = make_float2(-zero, -zero);
                wait_taken();
                if (!ok) break;
                auto weigh = [&](int c) {                                   // columns [16 c, 16 c + 16)
                    uint32_t pk[8];
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float2 e = __ffma2_rn(make_float2(__uint_as_float(s[16 * c + i]), __uint_as_float(s[16 * c + i + 1])), sc2, nm2);
                        const float2 pp = make_float2(fast_exp2(e.x), fast_exp2(e.y));
                        rs[(i >> 1) & 3] = __fadd2_rn(rs[(i >> 1) & 3], pp);
                        pk[i >> 1] = Elem<T>::pack2(pp.x, pp.y);
                    }
                    tmem_st8(p_addr + c * 8, pk);
                };
                if (!masked) {
#pragma unroll
                    for (int c = 0; c < C::kN / 16; ++c) weigh(c);
                } else {
#pragma unroll
                    for (int c = 0; c < C::kN / 16; ++c) {
                        if (c * 16 >= rest) break;
                        weigh(c);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar->p_ready[t]);               // (one arrival per warp: those of 32 lanes take turns)
            }
            if (!ok) break;

            // ---- epilogue of this item: O / l -> global, LSE ----
            if (n > 0) {
                ok = mbar_wait_warp(&bar->o_done[t], (g - 1) & 1, abort_flag, 0xA00 + t);
                if (!ok) break;
                tc_fence_after();
            }
            const float l_sum = ((rs[0].x + rs[0].y) + (rs[1].x + rs[1].y)) + ((rs[2].x + rs[2].y) + (rs[3].x + rs[3].y));
            const bool row_live = token < w->tokens;
            const bool blind = limit < 0;                                   // sees no key: zeros; one whose scores are all -infinity: 0 / 0
            const float inv_l = 1.0f / l_sum;
            const int hq = w->head + head_in;
            T* orow = static_cast<T*>(p.o.ptr) + hq * p.o.sh + static_cast<long long>(w->q0 + token) * p.o.ss;
            const bool o32 = (reinterpret_cast<uintptr_t>(orow) & 31) == 0;     // every segment offset below is a multiple of 32 bytes
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];                          // (a tile without keys reads what stands there, and writes zeros)
                tmem_ld32(o_addr + c * 32, o);
                tmem_ld_wait();
                if (row_live) {
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        uint32_t w8[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            w8[e] = blind ? 0u : Elem<T>::pack2(__uint_as_float(o[16 * v + 2 * e]) * inv_l, __uint_as_float(o[16 * v + 2 * e + 1]) * inv_l);
                        if (o32) {
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                                         ::"l"(orow + c * 32 + v * 16), "r"(w8[0]), "r"(w8[1]), "r"(w8[2]), "r"(w8[3]), "r"(w8[4]), "r"(w8[5]),
                                           "r"(w8[6]), "r"(w8[7]) : "memory");
                        } else {                     // the interface promises 16-byte alignment only
                            uint4* o4 = reinterpret_cast<uint4*>(orow + c * 32 + v * 16);
                            o4[0] = make_uint4(w8[0], w8[1], w8[2], w8[3]);
                            o4[1] = make_uint4(w8[4], w8[5], w8[6], w8[7]);
                        }
                    }
                }
            }
            // O has been read out: the next item's first PV (issued only after this thread's next p_ready arrival) may overwrite it
            tc_fence_before();
            if (p.lse != nullptr && row_live)
                p.lse[static_cast<long long>(hq) * p.total_q + w->q0 + token] = (m_ref - kLift + fast_log2(l_sum)) * kLn2;         // (blind: -infinity)
        }
    }

    // ---- teardown ----
    tc_fence_before();
    __syncthreads();
    abort_linger(&bar->abort_flag);
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// ---- host side ----
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = []() -> EncodeTiledFn {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) != cudaSuccess || qres != cudaDriverEntryPointSuccess) return nullptr;
        return reinterpret_cast<EncodeTiledFn>(ptr);
    }();
    return fn;
}

// [tokens, H, D] view -> 4-D map (D, H, tokens, 1), box [64 columns][heads][tokens], 128-byte swizzle
int make_map(CUtensorMap* m, int dtype, const View4& v, int tokens, int H, int D, int box_heads, int box_tokens) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return set_detail(VB200_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(tokens), 1};
    cuuint64_t strides[3] = {static_cast<cuuint64_t>(v.sh) * 2, static_cast<cuuint64_t>(v.ss) * 2, 16};
    for (int i = 0; i < 2; ++i) if (strides[i] == 0) strides[i] = 16;          // (of extent 1: any legal stride)
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens), 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = enc(m, dtype == VB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, v.ptr, dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        static thread_local char buf[96];
        snprintf(buf, sizeof(buf), "cuTensorMapEncodeTiled (packed attention) failed with CUresult %d", static_cast<int>(r));
        return set_detail(VB200_ERR_CUDA, buf);
    }
    return VB200_OK;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
struct Carve {
    size_t items, first, total;            // offsets
};
Carve carve(int batch, const Shape& s) {
    Carve c;
    c.items = 256;
    c.first = c.items + up256(sizeof(Item) * static_cast<size_t>(s.room));
    c.total = c.first + up256(sizeof(int) * (static_cast<size_t>(batch) + 1));
    return c;
}

template <typename T, int D, bool kList, bool kDual>
int launch_t(cudaStream_t s, const PackedParams& p, const Shape& shape, int64_t most) {
    static thread_local bool configured[64] = {};      // per device ordinal: the attribute belongs to the device's context
    int dev = 0;
    VB200_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return set_detail(VB200_ERR_NO_DEVICE, "device ordinal out of range");
    if (!configured[dev]) {
        VB200_CUDA_TRY(cudaFuncSetAttribute(prefill_packed_kernel<T, D, kList, kDual>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmemBytes));
        configured[dev] = true;
    }
    const Carve c = carve(p.batch, shape);
    char* ws = static_cast<char*>(p.workspace);
    Plan* plan = reinterpret_cast<Plan*>(ws);
    Item* items = reinterpret_cast<Item*>(ws + c.items);
    TmaMaps maps;
    if (int rc = make_map(&maps.q, p.dtype, p.q, p.total_q, p.Hq, D, shape.fold, shape.tokens)) return rc;
    // no keys at all: no block is loaded, any map will do
    const View4 k = p.total_k > 0 ? p.k : p.q, v = p.total_k > 0 ? p.v : p.q;
    const int n_k = p.total_k > 0 ? p.total_k : p.total_q, h_k = p.total_k > 0 ? p.Hkv : p.Hq;
    if (int rc = make_map(&maps.k, p.dtype, k, n_k, h_k, D, 1, Cfg<D>::kN)) return rc;
    if (int rc = make_map(&maps.v, p.dtype, v, n_k, h_k, D, 1, Cfg<D>::kN)) return rc;
    if (kList) {
        packed_plan_kernel<<<1, kPlanThreads, 0, s>>>(p, shape, device_sm_count(), plan, items, reinterpret_cast<int*>(ws + c.first));
        note_launch();
        VB200_CUDA_TRY(cudaPeekAtLastError());
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(most, device_sm_count())));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg<D>::kSmemBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kList ? 1 : 0;
    profile_mark_begin(s);
    VB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, prefill_packed_kernel<T, D, kList, kDual>, maps, p, shape, plan, static_cast<const Item*>(items)));
    profile_mark_end(s);
    note_launch();
    return VB200_OK;
}

}  // namespace

size_t prefill_packed_workspace(int batch, int Hq, int Hkv, int total_q) { return carve(batch, shape_of(batch, Hq, Hkv, total_q)).total; }

int launch_prefill_packed(cudaStream_t s, const PackedParams& p) {
    Shape shape = shape_of(p.batch, p.Hq, p.Hkv, p.total_q);
    if (two_head_blocks(p, shape)) shape = shape_of(p.batch, p.Hq, p.Hkv, p.total_q, true);
    const int64_t most = static_cast<int64_t>(shape.max_items) * shape.head_blocks;
    // With an item per SM at most, a CTA finds its own: no list, and one launch less (eight requests of 5-96 tokens, 16 heads on 4: 9.8 us, with the list 11.6).
    const bool list = most > device_sm_count();
    auto go = [&](auto t, auto d) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        if (shape.dual) return list ? launch_t<T, D, true, true>(s, p, shape, most) : launch_t<T, D, false, true>(s, p, shape, most);
        return list ? launch_t<T, D, true, false>(s, p, shape, most) : launch_t<T, D, false, false>(s, p, shape, most);
    };
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (p.dtype == VB200_BF16) return p.D == 128 ? go(__nv_bfloat16(), D128()) : go(__nv_bfloat16(), D64());
    return p.D == 128 ? go(__half(), D128()) : go(__half(), D64());
}

}  // namespace vb200
