// Causal attention of packed prompts on the 5th-generation tensor cores (tcgen05, accumulators in
// tensor memory): 16-bit types, head_dim = v_head_dim = 64 or 128.
//
//   out_t = sum_{s <= t} p_ts v_s / l_t,  p_ts = 2^(c q_t . k_s - m_t),  c = scale log2 e,
//   l_t = sum_s p_ts [+ 2^(sink log2 e - m_t)],  lse_t = (m_t + log2 l_t) ln 2.
//
// A work item is 256 consecutive queries of one (prompt, head), as two tiles of 128 that share every
// key tile of 128.  Per key tile and query tile: S = Q K^T (M = N = 128) into tensor memory, softmax,
// P over S in the inputs' type, O += P V.  The two query tiles take turns: while one tile's scores
// are in its softmax, the tensor pipe runs the other's products, so neither waits for the other as
// long as both take about the same time (2 * 128^3 products at 4096 a cycle, 128^2 exponentials at
// 16 a cycle: 1024 cycles each).  Roles:
//  * warps 0-3 and 4-7, one warpgroup per query tile, one thread per query row: scores from tensor
//    memory, causal mask on the last key tile, online softmax with lazy rescaling (O is rescaled
//    only where the running maximum grows by more than 2^8, so p stays below 2^8), P back into tensor
//    memory; at the end O / l to the output.
//  * warps 8 and 9, one per query tile: one thread of each issues the tile's products (one thread for
//    both spent a third of its time on waits and commits with the tensor pipe idle), in turns, so that
//    the two tiles' softmaxes do not fall together.  S of key tile
//    j + 1 overwrites P of tile j, so it is issued behind P V of tile j (products of one thread execute
//    in issue order), and a warpgroup that sees S of tile j + 1 knows that O holds P V of tile j:
//    rescaling needs no further barrier.
//  * warp 10: loads Q, and K and V tiles in turn through a ring of 4 slots (TMA, 128-byte
//    swizzle, no multicast).
//  * warp 11: finds the next item while the block works on this one.  The grid holds every item, those
//    with the most keys first; a running block takes over blocks that have not started
//    (clusterlaunchcontrol), so the next item's loads and first scores overlap this one's end.
// Values that no row may see (keys behind a prompt's end, and not-finite values of keys that some rows
// of the last key tile do not see) are taken out of the V tile before its product; the rows that do see
// a not-finite value get it back in the epilogue.
// Every wait is bounded: on expiry the block raises kErrWaitTimeout, lets its copies and products
// finish, frees its tensor memory and ends.
//
// Measured (28 q and 4 kv heads of 128, bf16), with the SM clock sampled meanwhile: 16384 tokens 1.38 ms = 1394
// TFLOP/s at 1965 MHz, 83 % of the measured product rate, and 1.60 ms = 1200 TFLOP/s at the 1550 MHz that the
// power limit leaves after some 0.3 s back to back; tensor pipe and exponentials are each busy for 71 % of the time.  24
// prompts of 1 to 6000 tokens: 0.527 ms = 1107 TFLOP/s at 1965 MHz, 0.616 ms = 948 at the power limit's
// 1597, and some 0.63 ms for a first call whose inputs are in no cache; first and last key tiles.  16 q and 4 kv
// heads of 64 in fp16, 9 prompts of up to 4000 tokens: 0.136 ms = 594 TFLOP/s at 1965 MHz, 0.17 ms with cold caches; with
// half the products for the same exponentials those are the bound (0.068 ms), and short items leave the
// chain of scores, softmax and P V bare.
#include <cuda.h>

#include <atomic>

#include "gkv_device.cuh"
#include "kernels.h"
#include "prompt_tiles.cuh"
#include "../../include/glacier_kv.h"

namespace gkv {

namespace {

constexpr int kBM = 128, kBN = 128;               // query rows of a tile, keys of a tile
constexpr int kRows = 2 * kBM;                    // query rows of an item
constexpr int kEarly = 64;                        // keys whose P V starts before the others' p are there (96: 3 % slower)
constexpr int kMmaWarp = 8, kLoadWarp = 10, kPlanWarp = 11;  // kMmaWarp + t issues query tile t's products
constexpr int kThreads = 384;
constexpr int kRing = 4;
constexpr int kItems = 1;                         // item slots: the next item, while the block works on one
constexpr uint32_t kTmemCols = 512;               // S0 S1 O0 O1, 128 columns each
constexpr uint32_t kColS = 0, kColO = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleLog2 = 8.f;
// The running maximum starts at the type's lowest value: against minus infinity a row whose scores so far are all
// minus infinity would have weights of 2^(-inf + inf), NaN for good; against this they are 0, as they should be.
constexpr float kLowest = -3.402823466e+38f;
constexpr uint32_t kPolls = 1u << 24;
constexpr uint32_t kPlanNs = 100, kLoadNs = 40, kMmaNs = 0, kSoftNs = 0;

template <int D>
struct Shape {
    static constexpr uint32_t kHalf = kBN * 128;            // 128 rows x 64 dims
    static constexpr int kHalves = D / 64;
    static constexpr uint32_t kTile = kHalves * kHalf;      // a Q, K or V tile
    static constexpr uint32_t kData = 2 * kTile + kRing * kTile;
    static constexpr uint32_t kBytes = kData + 27648 + 1024;  // + bookkeeping + alignment
};

struct Item {
    int64_t row0;   // first row of the prompt
    int q0, len;    // first query in the prompt, the prompt's length
    int head;
    int n[2];       // key tiles of each query tile (0: no rows); n[0] = 0: no further item
    int number;     // of this block's items
};

struct Book {
    uint64_t q_full[2], q_empty[2];
    uint64_t ring_full[kRing], ring_empty[kRing];
    uint64_t s_full[2], p_full[2][2], o_full[2];  // p_full: of the first kEarly keys, and of the others
    uint64_t item_full[kItems], item_empty[kItems];
    uint64_t steal, drained[2], turn[2];
    alignas(16) uint32_t response[4];
    Item item[kItems];
    uint32_t tmem;
    int abort;
    // Not-finite values taken out of a query tile's last key tile: for each dim the first position with
    // NaN, +infinity, -infinity, under the complement of the item's number, so that a later item's
    // entries replace an earlier one's.  Two sets, for even and odd items: the first warpgroup may be
    // one item ahead of the second, which reads both tiles' entries, and not more.
    int poisoned[2][2];  // one more than the number of the item that the entries are of
    unsigned long long poison[2][2][3][128];
    PromptList list;  // where batch <= kListed
};
static_assert(sizeof(Book) <= 27648, "bookkeeping");

constexpr uint32_t idesc_16(int m, int n, bool b_mn_major, bool f16) {
    const uint32_t fmt = f16 ? 0u : 1u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn_major ? 1u : 0u) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ bool poll(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// Bounded wait that also ends (false) when the block has given up.  Between polls the thread sleeps
// for about `ns` nanoseconds: polls take issue slots that the other warps need.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Book* bk, uint32_t ns) {
    const uint32_t addr = smem_u32(bar);
    if (poll(addr, parity)) return true;
#pragma unroll 1
    for (uint32_t it = 0; it < kPolls; ++it) {
        if (ns) __nanosleep(ns);
        if (poll(addr, parity)) return true;
        if ((it & 15) == 15 && *reinterpret_cast<volatile int*>(&bk->abort)) return false;
    }
    return false;
}

// Asks for a block of the grid that has not started; the answer lands in `response`.
__device__ __forceinline__ void steal_block(uint32_t* response, uint64_t* bar) {
    mbar_arrive_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(response)),
                 "r"(smem_u32(bar))
                 : "memory");
}
// Its number, or -1 when there was none left.
__device__ __forceinline__ int stolen_block(const uint32_t* response) {
    uint32_t ok, x;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
        "ld.shared.b128 r, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
        : "=r"(ok), "=r"(x)
        : "r"(smem_u32(response))
        : "memory");
    return ok ? static_cast<int>(x) : -1;
}

// 32 bytes; `whole`: p is on a 32-byte boundary, which the one wide store needs (16 bytes do for the two).
__device__ __forceinline__ void store_sector(void* p, const uint32_t (&w)[8], bool whole) {
    if (whole) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                     "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
    } else {
        asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};\n\tst.global.v4.b32 [%0 + 16], {%5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
                     "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
    }
}

template <bool F16>
__device__ __forceinline__ uint32_t times_zero(uint32_t acc, uint32_t x) {  // acc + 0 * x: NaN where x is not finite
    if constexpr (F16) {
        const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(0.f), *reinterpret_cast<const __half2*>(&acc));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), __float2bfloat162_rn(0.f),
                                         *reinterpret_cast<const __nv_bfloat162*>(&acc));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}

// The last key tile of query tile t, in shared memory: thread `key` of the warpgroup takes one key row.
// Rows behind the prompt become zero; not-finite elements become zero and are noted.
template <int D, bool F16>
__device__ __forceinline__ void clean_values(uint8_t* tile, int key, int key_pos, int len, Book* bk, int number, int t) {
    constexpr uint32_t kInf = F16 ? 0x7c00u : 0x7f80u;
    if (key_pos >= len) {
#pragma unroll
        for (int h = 0; h < Shape<D>::kHalves; ++h)
#pragma unroll
            for (int c = 0; c < 8; ++c)
                *reinterpret_cast<uint4*>(tile + h * Shape<D>::kHalf + key * 128 + ((c ^ (key & 7)) << 4)) = make_uint4(0, 0, 0, 0);
        return;
    }
    uint32_t acc = 0;
#pragma unroll
    for (int h = 0; h < Shape<D>::kHalves; ++h)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const uint4 w = *reinterpret_cast<const uint4*>(tile + h * Shape<D>::kHalf + key * 128 + ((c ^ (key & 7)) << 4));
            acc = times_zero<F16>(acc, w.x);
            acc = times_zero<F16>(acc, w.y);
            acc = times_zero<F16>(acc, w.z);
            acc = times_zero<F16>(acc, w.w);
        }
    if ((acc & 0x7fff7fffu) == 0) return;
    // rare: element by element (chunk c of a row sits at c ^ (row % 8))
    for (int e = 0; e < D; ++e) {
        uint8_t* p = tile + (e >> 6) * Shape<D>::kHalf + key * 128 + ((((e & 63) >> 3) ^ (key & 7)) << 4) + (e & 7) * 2;
        const uint32_t x = *reinterpret_cast<uint16_t*>(p);
        if ((x & kInf) != kInf) continue;
        const int kind = (x & 0x7fffu) != kInf ? 0 : (x & 0x8000u) ? 2 : 1;
        atomicMin(&bk->poison[number & 1][t][kind][e],
                  (static_cast<unsigned long long>(~static_cast<uint32_t>(number)) << 32) | static_cast<uint32_t>(key_pos));
        bk->poisoned[number & 1][t] = number + 1;
        *reinterpret_cast<uint16_t*>(p) = 0;
    }
}

// 2^x, kept in program order.
__device__ __forceinline__ float exp2_in_order(float x) {
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Not-finite values that were taken out of the last key tiles (of the own one and, for the second query
// tile, of the first's), back into the row at position `pos`, whose thread has just stored it.
template <int D, bool F16>
__device__ __noinline__ void put_back(const Book* bk, int number, int t, int pos, uint8_t* out) {
    for (int e = 0; e < D; ++e) {
        bool sees[3];
        for (int k = 0; k < 3; ++k) {
            sees[k] = false;
            for (int u = 0; u <= t; ++u) {
                const unsigned long long w = *reinterpret_cast<const volatile unsigned long long*>(&bk->poison[number & 1][u][k][e]);
                sees[k] |= static_cast<uint32_t>(w >> 32) == ~static_cast<uint32_t>(number) && static_cast<uint32_t>(pos) >= static_cast<uint32_t>(w);
            }
        }
        if (!sees[0] && !sees[1] && !sees[2]) continue;
        uint16_t* p = reinterpret_cast<uint16_t*>(out) + e;
        const uint32_t was = *p;
        float x = F16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(was))) : __uint_as_float(was << 16);
        if (sees[0]) x = __uint_as_float(0x7fffffffu);
        if (sees[1]) x += INFINITY;
        if (sees[2]) x += -INFINITY;
        *p = static_cast<uint16_t>(pack_16x2<F16>(x, 0.f));
    }
}

// Weights of 32 keys: p = 2^(sl s - m) of s[0 .. 31], in pairs of the inputs' type; `sum` grows by them.
// In groups of 8 pairs, the exponentials of a group one after the other and their sums behind them: left
// to itself the compiler put each sum next to its exponential, and a warp has only one other on its
// scheduler to fill that wait.
template <bool F16>
__device__ __forceinline__ void weights(const uint32_t (&s)[32], float sl, float m, float2 (&sum)[2], uint32_t (&pk)[16]) {
    const float2 sl2 = make_float2(sl, sl), nm2 = make_float2(-m, -m);
#pragma unroll
    for (int g = 0; g < 16; g += 8) {
        float2 y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            y[e] = __ffma2_rn(make_float2(__uint_as_float(s[2 * (g + e)]), __uint_as_float(s[2 * (g + e) + 1])), sl2, nm2);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = make_float2(exp2_in_order(y[e].x), exp2_in_order(y[e].y));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sum[e & 1] = __fadd2_rn(sum[e & 1], y[e]);
            pk[g + e] = pack_16x2<F16>(y[e].x, y[e].y);
        }
    }
}
__device__ __forceinline__ float largest(const uint32_t (&s)[4][32]) {
    float mq[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) mq[k] = __uint_as_float(s[k >> 1][(k & 1) * 16]);
#pragma unroll
    for (int e = 1; e < 15; e += 2)
#pragma unroll
        for (int k = 0; k < 8; ++k)
            mq[k] = fmax3(mq[k], __uint_as_float(s[k >> 1][(k & 1) * 16 + e]), __uint_as_float(s[k >> 1][(k & 1) * 16 + e + 1]));
#pragma unroll
    for (int k = 0; k < 8; ++k) mq[k] = fmaxf(mq[k], __uint_as_float(s[k >> 1][(k & 1) * 16 + 15]));
    return fmax3(fmax3(mq[0], mq[1], mq[2]), fmax3(mq[3], mq[4], mq[5]), fmaxf(mq[6], mq[7]));
}
__device__ __forceinline__ void p_ready(uint64_t* bar) {
    tmem_wait_st();
    tc_fence_before();
    mbar_arrive(bar);
}

// The softmax of one key tile, one row per thread: p of 32 keys at a time over the first 64 columns of S.
// Here with the running maximum m as it was, next to the search for the tile's own; false, with nothing
// stored, where that is larger by more than 2^8 for some row of the warp.  Straight code: with the mask,
// the first tile or the rescaling in its blocks the compiler's order cost a long prompt 10 %.
template <bool F16>
__device__ __forceinline__ bool middle_tile(uint32_t tS, float sl, float m, float& l, uint64_t* p_full) {
    uint32_t s[4][32], pk[4][16];
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, s[c]);
    tmem_wait_ld();
#pragma unroll
    for (int c = 0; c < kEarly / 32; ++c) weights<F16>(s[c], sl, m, sum, pk[c]);
    if (__any_sync(~0u, largest(s) * sl > m + kRescaleLog2)) return false;
#pragma unroll
    for (int c = 0; c < kEarly / 32; ++c) tmem_st16(tS + c * 16, pk[c]);
    p_ready(p_full);
#pragma unroll
    for (int c = kEarly / 32; c < 4; ++c) {
        weights<F16>(s[c], sl, m, sum, pk[c]);
        tmem_st16(tS + c * 16, pk[c]);
    }
    p_ready(p_full + 1);
    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    return true;
}

// The same for any tile: keys behind `limit` masked, the tile's maximum first, O (which holds P V up to
// the tile before: its products were issued before S of this one) rescaled where it moves the running one.
template <int D, bool F16>
__device__ __forceinline__ void any_tile(uint32_t tS, uint32_t tO, float sl, int limit, bool has_o, float& m, float& l, uint64_t* p_full) {
    uint32_t s[4][32];
#pragma unroll
    for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, s[c]);
    tmem_wait_ld();
#pragma unroll
    for (int c = 0; c < 128; ++c)
        if (c > limit) s[c >> 5][c & 31] = 0xff800000u;
    const float mt = largest(s) * sl;
    const bool need = mt > m + kRescaleLog2;
    float alpha = 1.f;
    if (need) {
        alpha = fast_exp2(m - mt);  // 0 on the first tile
        m = mt;
        l *= alpha;
    }
    if (has_o && __any_sync(~0u, need)) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(tO + c * 32, o);
        }
    }
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
        weights<F16>(s[c], sl, m, sum, pk);
        tmem_st16(tS + c * 16, pk);
        if (c == kEarly / 32 - 1) p_ready(p_full);
    }
    p_ready(p_full + 1);
    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
}

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                     const __grid_constant__ CUtensorMap tmv, const __grid_constant__ PromptArgs a) {
    using Sh = Shape<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
    uint8_t* sQ = smem;
    uint8_t* sRing = sQ + 2 * Sh::kTile;
    Book* bk = reinterpret_cast<Book*>(smem + Sh::kData);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kRing; ++i) {
            mbar_init(&bk->ring_full[i], 1);
            mbar_init(&bk->ring_empty[i], 2);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&bk->q_full[t], 1);
            mbar_init(&bk->q_empty[t], 1);
            mbar_init(&bk->s_full[t], 1);
            mbar_init(&bk->p_full[t][0], 128);
            mbar_init(&bk->p_full[t][1], 128);
            mbar_init(&bk->drained[t], 1);
            mbar_init(&bk->turn[t], 1);
            mbar_init(&bk->o_full[t], 1);
            bk->poisoned[t][0] = bk->poisoned[t][1] = 0;
        }
        for (int i = 0; i < kItems; ++i) {
            mbar_init(&bk->item_full[i], 1);
            mbar_init(&bk->item_empty[i], 11);  // both warpgroups' warps, the issuers, the loader
        }
        mbar_init(&bk->steal, 1);
        bk->abort = 0;
        fence_mbar_init();
    }
    for (int i = threadIdx.x; i < 2 * 2 * 3 * 128; i += kThreads) (&bk->poison[0][0][0][0])[i] = ~0ull;
    if (warp == kMmaWarp) tmem_alloc(&bk->tmem, kTmemCols);
    const bool listed = a.batch <= kListed;
    if (listed) count_prompt_tiles<kRows>(a, bk->list, threadIdx.x, kThreads);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (listed) {
        sort_prompts(a, bk->list, threadIdx.x, kThreads);
        __syncthreads();
    }
    const uint32_t tmem = bk->tmem;
    bool ok = true;

    // registers: 384 x 168 at launch = 128 x (224 + 224 + 56)
    if (warp >= 8) {
    fewer_registers<56>();
    if (warp == kPlanWarp) {
        // ---------------- items ----------------
        // The blocks of the grid stand for the tiles, those with the most keys first (with a batch too large
        // to be listed, for each prompt), all heads of a tile in a row; some stand for none: the host knows
        // only total and batch.
        if (lane == 0) steal_block(bk->response, &bk->steal);  // the first answer is on its way meanwhile
        const int numbers = static_cast<int>(gridDim.x / a.n_heads);
        const int tiles = listed ? sum_prompt_levels(a, bk->list) : 0;
        int block = blockIdx.x, published = 0;
        uint32_t answers = 0;
        bool asking = true;
        while (true) {
            if (block == 0) check_prompts(a, lane, 32);  // by whichever block has number 0, which may have been taken over too
            PromptTile pt;
            const int x = block / a.n_heads;
            bool found = false;
            if (block >= 0 && listed) {
                found = x < tiles;
                if (found) listed_prompt_tile(a, bk->list, x, pt);
            } else if (block >= 0) {
                found = find_prompt_tile<kRows>(a, numbers - 1 - x, pt);
            }
            if (found || block < 0) {
                const int is = published % kItems;
                if (published >= kItems && !(ok = __all_sync(~0u, wait(&bk->item_empty[is], (published / kItems - 1) & 1, bk, kPlanNs)))) break;
                if (lane == 0) {
                    Item it{};
                    if (found) {
                        it.row0 = pt.row0;
                        it.q0 = pt.tile * kRows;
                        it.len = pt.len;
                        it.head = block - x * a.n_heads;
                        it.n[0] = it.q0 / kBN + 1;
                        it.n[1] = it.len - it.q0 > kBM ? it.n[0] + 1 : 0;
                        it.number = published;
                    }
                    bk->item[is] = it;
                    mbar_arrive(&bk->item_full[is]);
                }
                __syncwarp();
                if (block < 0) break;
                ++published;
            }
            if (!(ok = __all_sync(~0u, mbar_wait(&bk->steal, answers & 1)))) break;
            ++answers;
            block = stolen_block(bk->response);
            asking = block >= 0;
            __syncwarp();
            if (asking) {
                fence_proxy_async_smem();  // the answer has been read before the next one is written
                if (lane == 0) steal_block(bk->response, &bk->steal);
            }
            __syncwarp();
        }
        // an answer still on its way must land before the block's shared memory goes away
        if (!ok && asking && lane == 0) mbar_wait(&bk->steal, answers & 1);
        if (!ok && lane == 0) {
            bk->abort = 1;
            atomicOr(a.err, kErrWaitTimeout);
        }
    } else if (warp == kLoadWarp) {
        // ---------------- TMA ----------------
        // Each copy by lanes of its own, one per box of 128 rows x 64 dims: a copy holds its thread for some
        // hundred cycles.
        uint32_t slot = 0, q_loads[2] = {0, 0};
        auto empty = [&](uint64_t* bar, uint32_t parity) { return __all_sync(~0u, wait(bar, parity, bk, kLoadNs)) != 0; };
        auto load = [&](uint8_t* dst, const CUtensorMap* tm, int head, int row, uint64_t* bar) {
            if (lane == 0) mbar_arrive_expect_tx(bar, Sh::kTile);
            __syncwarp();  // the expected bytes before the first of them
            if (lane < Sh::kHalves) tma_load_3d(dst + lane * Sh::kHalf, tm, lane * 64, head, row, bar);
        };
        for (uint32_t i = 0;; ++i) {
            const int is = i % kItems;
            if (!(ok = empty(&bk->item_full[is], (i / kItems) & 1))) break;
            const Item it = bk->item[is];
            __syncwarp();
            if (lane == 0) mbar_arrive(&bk->item_empty[is]);
            if (it.n[0] == 0) break;
            const int kv = it.head / (a.n_heads / a.heads_kv), row = static_cast<int>(it.row0);
            const int nj = it.n[1] ? it.n[1] : it.n[0];
            auto load_q = [&](int t) {
                if (it.n[t] == 0) return true;
                if (q_loads[t] > 0 && !empty(&bk->q_empty[t], (q_loads[t] - 1) & 1)) return false;
                load(sQ + t * Sh::kTile, &tmq, it.head, row + it.q0 + t * kBM, &bk->q_full[t]);
                ++q_loads[t];
                return true;
            };
            if (!(ok = load_q(0))) break;
            for (int j = 0; j < 2 * nj; ++j) {  // K of tile j / 2, then V
                const int s = slot % kRing;
                if (slot >= kRing && !(ok = empty(&bk->ring_empty[s], (slot / kRing - 1) & 1))) break;
                load(sRing + s * Sh::kTile, (j & 1) ? &tmv : &tmk, kv, row + (j >> 1) * kBN, &bk->ring_full[s]);
                ++slot;
                if (j == 0 && !(ok = load_q(1))) break;
            }
            if (!ok) break;
        }
        if (!ok && lane == 0) {
            bk->abort = 1;
            atomicOr(a.err, kErrWaitTimeout);
            // every copy must land before the block's shared memory goes away
            for (int t = 0; t < 2; ++t)
                if (q_loads[t]) mbar_wait(&bk->q_full[t], (q_loads[t] - 1) & 1);
            for (uint32_t s = slot > kRing ? slot - kRing : 0; s < slot; ++s) mbar_wait(&bk->ring_full[s % kRing], (s / kRing) & 1);
        }
        __syncwarp();
    } else {
        // ---------------- products of query tile t ----------------
        // The whole warp keeps the loop, so that ring positions and descriptors are the same for all its
        // lanes (in uniform registers, where the products take them); one lane issues.
        constexpr uint32_t kIdS = idesc_16(kBM, kBN, false, F16);
        constexpr uint32_t kIdO = idesc_16(kBM, D, true, F16);
        const int t = __shfl_sync(~0u, warp, 0) - kMmaWarp;
        const uint32_t tm = __shfl_sync(~0u, tmem, 0);
        const uint32_t tS = tm + kColS + t * 128, tO = tm + kColO + t * 128;
        const bool issuer = elect_lane();
        // descriptors' low words advance by bytes / 16
        const uint64_t q_desc = umma_desc_sw128(smem_u32(sQ) + t * Sh::kTile, 16, 1024);
        const uint64_t k_desc = umma_desc_sw128(smem_u32(sRing), 16, 1024);
        const uint64_t v_desc = umma_desc_sw128(smem_u32(sRing), Sh::kHalf, 1024);
        uint32_t slot = 0;          // ring position of the next tile
        uint32_t p_count = 0, q_count = 0, turns = 0;
        auto ready = [&](uint64_t* bar, uint32_t parity) { return __all_sync(~0u, wait(bar, parity, bk, kMmaNs)) != 0; };
        auto full = [&](uint32_t at) { return ready(&bk->ring_full[at % kRing], (at / kRing) & 1); };
        auto scores = [&](uint32_t at) {  // S = Q K^T
            const uint64_t k = k_desc + (at % kRing) * (Sh::kTile / 16);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                const uint32_t off = ((kk >> 2) * Sh::kHalf + (kk & 3) * 32) / 16;
                umma_f16(tS, q_desc + off, k + off, kIdS, kk > 0 ? 1u : 0u);
            }
            umma_commit(&bk->s_full[t]);
        };
        for (uint32_t i = 0;; ++i) {
            const int is = i % kItems;
            if (!(ok = ready(&bk->item_full[is], (i / kItems) & 1))) break;
            const int n0 = __shfl_sync(~0u, bk->item[is].n[0], 0), n1 = __shfl_sync(~0u, bk->item[is].n[1], 0);
            __syncwarp();
            if (issuer) mbar_arrive(&bk->item_empty[is]);
            if (n0 == 0) break;
            const int n = t ? n1 : n0, nj = n1 ? n1 : n0;
            // a slot is free when both tiles are done with it: behind this tile's products so far, or,
            // where it has none, as soon as the slot is filled
            if (!(ok = (n == 0 || ready(&bk->q_full[t], q_count & 1)) && full(slot))) break;
            if (n > 0) ++q_count;
            tc_fence_after();
            if (issuer) {
                if (n > 0) {
                    scores(slot);
                    umma_commit(&bk->ring_empty[slot % kRing]);
                    if (n == 1) umma_commit(&bk->q_empty[t]);
                } else {
                    mbar_arrive(&bk->ring_empty[slot % kRing]);
                }
            }
            __syncwarp();
            for (int j = 0; j < nj; ++j) {
                const uint32_t vs = slot + 2 * j + 1, ks = vs + 1;  // V of tile j, K of tile j + 1
                const bool more = j + 1 < nj;
                if (!(ok = full(vs) && (!more || full(ks)))) break;
                // the tiles' products go in turns, the first tile's of every key tile first
                const uint32_t mine = (turns + (t ^ 1)) & 1;
                ++turns;
                if (!(ok = ready(&bk->turn[t], mine))) break;
                if (j >= n) {
                    if (issuer) {
                        mbar_arrive(&bk->ring_empty[vs % kRing]);
                        if (more) mbar_arrive(&bk->ring_empty[ks % kRing]);
                        mbar_arrive(&bk->turn[t ^ 1]);
                    }
                    __syncwarp();
                    continue;
                }
                const uint64_t v = v_desc + (vs % kRing) * (Sh::kTile / 16);
                if (!(ok = ready(&bk->p_full[t][0], p_count & 1))) break;
                // V tile [key][dim]: MN-major, 8-key groups 1 KB apart, dims 64-127 in the second half
                auto values = [&](int kk) { umma_f16_ts(tO, tS + kk * 8, v + kk * (2048 / 16), kIdO, (j > 0 || kk > 0) ? 1u : 0u); };
                tc_fence_after();
                if (issuer) {
#pragma unroll
                    for (int kk = 0; kk < kEarly / 16; ++kk) values(kk);
                }
                __syncwarp();
                if (!(ok = ready(&bk->p_full[t][1], p_count & 1))) break;
                tc_fence_after();
                ++p_count;
                if (issuer) {
#pragma unroll
                    for (int kk = kEarly / 16; kk < kBN / 16; ++kk) values(kk);
                    if (j + 1 < n) scores(ks);
                    else umma_commit(&bk->o_full[t]);
                    mbar_arrive(&bk->turn[t ^ 1]);
                    umma_commit(&bk->ring_empty[vs % kRing]);
                    if (more) umma_commit(&bk->ring_empty[ks % kRing]);
                    if (j + 2 == n) umma_commit(&bk->q_empty[t]);
                }
                __syncwarp();
            }
            if (!ok) break;
            slot += 2 * nj;
        }
        if (issuer) {
            if (!ok) {
                bk->abort = 1;
                atomicOr(a.err, kErrWaitTimeout);
            }
            umma_commit(&bk->drained[t]);  // every product is complete before the tensor memory is freed
            if (!mbar_wait(&bk->drained[t], 0)) atomicOr(a.err, kErrWaitTimeout);
        }
    }
    } else {
        // ---------------- softmax and epilogue ----------------
        more_registers<224>();
        const int t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t tS = tmem + kColS + t * 128 + lanes, tO = tmem + kColO + t * 128 + lanes;
        const float sl = a.scale * kLog2e;
        uint32_t s_count = 0, o_count = 0;
        uint32_t slot0 = 0;  // ring position of the item's first tile
        for (uint32_t i = 0; ok; ++i) {
            const int is = i % kItems;
            if (!(ok = __all_sync(~0u, wait(&bk->item_full[is], (i / kItems) & 1, bk, kSoftNs)))) break;
            const Item it = bk->item[is];
            __syncwarp();
            if (lane == 0) mbar_arrive(&bk->item_empty[is]);
            if (it.n[0] == 0) break;
            const int n = t ? it.n[1] : it.n[0];
            const int nj = it.n[1] ? it.n[1] : it.n[0];
            const int pos = it.q0 + t * kBM + r;
            float m_run = kLowest, l_run = 0.f;
            for (int j = 0; j < n; ++j) {
                if (j == n - 1) {  // while the scores are on their way
                    const uint32_t vs = slot0 + 2 * j + 1;
                    if (!(ok = __all_sync(~0u, wait(&bk->ring_full[vs % kRing], (vs / kRing) & 1, bk, kSoftNs)))) break;
                    clean_values<D, F16>(sRing + (vs % kRing) * Sh::kTile, r, j * kBN + r, it.len, bk, it.number, t);
                    fence_proxy_async_smem();
                }
                if (!(ok = __all_sync(~0u, wait(&bk->s_full[t], s_count & 1, bk, kSoftNs)))) break;
                ++s_count;
                tc_fence_after();
                if (j > 0 && j < n - 1 && middle_tile<F16>(tS, sl, m_run, l_run, bk->p_full[t])) continue;
                any_tile<D, F16>(tS, tO, sl, j == n - 1 ? pos - j * kBN : kBN, j > 0, m_run, l_run, bk->p_full[t]);
            }
            slot0 += 2 * nj;
            if (!ok || n == 0) continue;
            if (!(ok = __all_sync(~0u, wait(&bk->o_full[t], o_count & 1, bk, kSoftNs)))) break;
            ++o_count;
            tc_fence_after();
            // the sink joins the sum against the larger of the two maxima
            float inv, top = m_run, total = l_run;
            if (a.sinks) {
                const float sink = __ldg(a.sinks + it.head) * kLog2e;
                top = fmaxf(m_run, sink);
                const float alpha = fast_exp2(m_run - top);
                total = l_run * alpha + (sink == top ? 1.f : fast_exp2(sink - top));  // also where both are infinite
                inv = alpha / total;
            } else {
                inv = 1.f / l_run;
            }
            const int rows = min(kBM, it.len - it.q0 - t * kBM);
            const int64_t row = it.row0 + it.q0 + t * kBM;
            if (a.lse && r < rows) a.lse[(row + r) * a.n_heads + it.head] = (top + log2f(total)) * 0.6931471805599453f;
            // each row from its thread, in whole 32-byte sectors (rows are 128 or 256 bytes and dense, so the base decides)
            const bool whole = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
            uint8_t* out = static_cast<uint8_t*>(a.out) + ((row + r) * a.n_heads + it.head) * (D * 2);
#pragma unroll 1
            for (int h = 0; h < D / 64; ++h) {
                uint32_t o[2][32];
                tmem_ld32(tO + h * 64, o[0]);
                tmem_ld32(tO + h * 64 + 32, o[1]);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 64; c += 16) {
                    uint32_t w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        w[e] = pack_16x2<F16>(__uint_as_float(o[c >> 5][(c & 31) + 2 * e]) * inv, __uint_as_float(o[c >> 5][(c & 31) + 2 * e + 1]) * inv);
                    if (r < rows) store_sector(out + h * 128 + c * 2, w, whole);
                }
            }
            const volatile int* tags = bk->poisoned[it.number & 1];
            if ((tags[0] == it.number + 1 || (t && tags[1] == it.number + 1)) && r < rows) put_back<D, F16>(bk, it.number, t, pos, out);
            tc_fence_before();
        }
        if (!ok) {
            bk->abort = 1;
            atomicOr(a.err, kErrWaitTimeout);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <int D, bool F16>
cudaError_t launch(const PromptArgs& a, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
    static std::atomic<uint64_t> done_mask{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done_mask.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(prompt_tc_kernel<D, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kBytes);
        if (e != cudaSuccess) return e;
        done_mask.fetch_or(bit, std::memory_order_acq_rel);
    }
    const int64_t grid = prompt_tile_bound(a, kRows) * a.n_heads;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    prompt_tc_kernel<D, F16><<<static_cast<unsigned>(grid), kThreads, Shape<D>::kBytes, st>>>(mq, mk, mv, a);
    return cudaGetLastError();
}

// [rows][heads][d] with strides, in boxes of 128 rows x 64 dims of one head.
bool encode(CUtensorMap* m, const void* p, int d, int heads, int64_t rows, int64_t hs, int64_t ts) {
    const uint64_t dims[3] = {static_cast<uint64_t>(d), static_cast<uint64_t>(heads), static_cast<uint64_t>(rows)};
    // a stride that is never taken may be anything in the caller's tensor, but not in the map
    const uint64_t strides[2] = {static_cast<uint64_t>(heads > 1 ? hs : d) * 2, static_cast<uint64_t>(rows > 1 ? ts : d) * 2};
    const uint32_t box[3] = {64, 1, static_cast<uint32_t>(kBM)};
    return encode_bf16_map3(m, p, dims, strides, box);
}

}  // namespace

cudaError_t launch_prompt_tc(const PromptArgs& a, bool* ran, cudaStream_t st) {
    *ran = false;
    if (a.dtype == GKV_DTYPE_F32 || a.d != a.dv || (a.d != 64 && a.d != 128) || !(a.scale > 0.f) || !tmap_encoder_available())
        return cudaSuccess;
    alignas(64) CUtensorMap mq, mk, mv;
    if (!encode(&mq, a.q, a.d, a.n_heads, a.total, a.q_hs, a.q_ts) || !encode(&mk, a.k, a.d, a.heads_kv, a.total, a.k_hs, a.k_ts) ||
        !encode(&mv, a.v, a.d, a.heads_kv, a.total, a.v_hs, a.v_ts))
        return cudaSuccess;  // strides that a tensor map cannot hold
    *ran = true;
    if (a.dtype == GKV_DTYPE_BF16) return a.d == 128 ? launch<128, false>(a, mq, mk, mv, st) : launch<64, false>(a, mq, mk, mv, st);
    return a.d == 128 ? launch<128, true>(a, mq, mk, mv, st) : launch<64, true>(a, mq, mk, mv, st);
}

}  // namespace gkv
