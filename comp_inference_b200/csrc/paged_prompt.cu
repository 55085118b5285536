// Attention of many new tokens over a paged cache, on the tensor cores (tcgen05): the prompts, and parts of prompts, of a
// batch.  The same result as k_paged_attention (paged_attn.cu), which has the sequences with few.
//
// A block has two tiles of 128 query rows (one where head_dim = 256) of one key/value head: `tt` tokens by the heads that
// share it, side by side, so that grouped heads read their keys once.  It walks over tiles of 128 positions:
//   S = Q . K^T        Q and K in shared memory (128-byte swizzle), S fp32 in tensor memory
//   P = exp2(S scale - m), written back in bf16 over S by the row's own thread: no exchange between threads at all
//   O += P . V         P from tensor memory, V as it lies (its rows are the k index: an MN-major operand), O in tensor memory
// While one tile's threads are at their exponentials the tensor cores work for the other; the weights are handed over in two
// halves.  The maximum that a row's weights refer to moves only when it is exceeded by 2^8 (kLazy), so O is rarely rescaled; the
// row's own thread does that too, between two products, when nothing else touches it.  Tiles that no row sees are not
// visited; a page that does not exist is fetched from outside the tensor, which gives zeros.
//
// Blocks stay, one on each multiprocessor, and take piece after piece of the plan that k_paged_join has made (PromptPlan): one warp
// fetches the next piece and says what it sees, one issues the TMA copies, one per query tile the products, and each goes on to the
// next piece when its own part is done, so that queries, first keys and first scores of the next are there when the rows of
// this one are written (4096 tokens, 32 heads of 128 over 8: a block for each piece 134 us, 122 so; six prompts of 1024, 64 heads of
// 64 over 16, under a window of 256: 155 and 106; 16 of 256: 49 and 40).  mbarriers connect the roles.  All waits are bounded: on
// expiry a role sets the status word and the abort flag, and everyone leaves when its copies and products under way are there.
//
// A cache of 4 bits is turned into fp16 on its way into shared memory by four or eight warps, so that what codes stand for, and the
// weights, are off by 2^-11 of themselves at most and not 2^-8 (mean error of a prompt's outputs against 64 bits 0.0017; bf16's own
// rounding of the result is 0.0016).  fp16 has no range for that by itself: every key tile is scaled by the power of two that
// its largest value asks for, the values by one that changes when a tile leaves its range, O following it, and a query row by its own.
// A value tile's largest lies between 2^8 and 2^15 of its scale, so steps and lowest values down to 2^-25 of that are held exactly.  The
// scale stays above 2^-92 of the largest value of the piece so far: O of the rows that have seen that one must not overflow.
//
// What bounds it: in bf16 the chain from a tile's scores over its exponentials to its product, with two tiles in turn (4096 tokens
// 122 us, 1126 TFLOP/s, tensor pipe 61 % active, issue slots 47 %; 16001 tokens under a window of 4096: 860 to 900 us under the power
// cap, 1040 to 1090 TFLOP/s, 0.75 to 0.78 of the measured sustained rate); in 4 bits the arithmetic of turning codes, which every block
// does for itself (4096 tokens 194 us, integer pipe 42 %, issue slots 55 %), scores read twice from tensor memory, and the
// producers' meeting in every tile.
#include <cuda_fp16.h>

#include <type_traits>

#include "paged.cuh"
#include "umma.cuh"

namespace ci {

constexpr float kLazy = 8.f;
__device__ uint32_t g_prompt_status;         // code of a wait that ran out

struct PromptArgs {
    PagedBatch p;
    const uint8_t *k, *v;                    // 4 bits only
    const uint32_t *ks, *vs;
    uint32_t group, tt, negate;
    int32_t window, sinks;
    float scale_log2;                        // not negative
    uint16_t *out;
    int64_t ldo;
    const int4 *plan, *cuts;                 // see PromptPlan
    int32_t *next;                           // the first piece that no block has yet
    uint32_t count;                          // pieces and places for them, each for every head
    uint32_t polls, at_once;                 // of a wait before it gives up; the code whose waits give up at once
    float *ml, *partial;                     // of pieces: [slots][NT 128][2], [slots][NT 128][D]
};

constexpr uint32_t kItemWords = 20;          // of a piece in shared memory: PieceWords

template <int D, int BITS>
struct PromptShape {
    static constexpr uint32_t NT = D == 256 ? 1 : 2;
    static constexpr uint32_t kTile = kKt * D * 2, kBlock = kKt * 128;       // bytes: a tile of 128 rows, its 64-channel block
    static constexpr uint32_t NS = D == 64 ? 6 : D == 128 ? 4 : 2;           // ring of K and V tiles
    static constexpr uint32_t SPLIT = BITS == 4 && D > 64 ? 2 : 1;           // threads that share a position's codes
    static constexpr uint32_t PW = BITS == 16 ? 1 : 4 * SPLIT;               // producer warps
    static constexpr uint32_t kProd = 4 * NT, kMma = kProd + PW, kSched = kMma + NT;
    // Whole warpgroups (but where nothing is gained), so that registers can go where the scores are held: setmaxnreg takes them
    // up or down from what the block is launched with, within its sum.
    static constexpr bool kMove = NT == 2 || BITS == 4;
    static constexpr uint32_t kWarps = kMove ? (kSched + 4) / 4 * 4 : kSched + 1, kThreads = kWarps * 32;
    static constexpr uint32_t kLaunchRegs = 65536 / kThreads / 8 * 8;
    static constexpr uint32_t kSoftRegs = BITS == 16 ? 200 : D == 64 ? 160 : D == 128 ? 136 : 176;
    static constexpr uint32_t kProdRegs = BITS == 16 ? 104 : D == 64 ? 120 : D == 128 ? 72 : 104;
    static constexpr uint32_t kMmaRegs = BITS == 16 ? kProdRegs : D == 64 ? 72 : D == 128 ? 64 : 112;
    static_assert(!kMove || (kSoftRegs >= kLaunchRegs && kProdRegs <= kLaunchRegs && kMmaRegs <= kLaunchRegs &&
                             NT * 128 * kSoftRegs + (BITS == 16 ? 128 * kProdRegs : PW * 32 * kProdRegs + 128 * kMmaRegs) <= kThreads * kLaunchRegs), "registers");
    static constexpr uint32_t oQ = 0, oRing = NT * kTile, oBar = oRing + NS * kTile, kMisc = 640, kSmem = oBar + kMisc + 1024;
    // barriers
    static constexpr uint32_t bQ = 0, bFull = 1, bEmpty = bFull + NS, bS = bEmpty + NS, bP = bS + NT, bO = bP + 2 * NT, bRead = bO + NT, bTurn = bRead + NT,
                              bQh = bTurn + 2, bQfree = bQh + 1, bItem = bQfree + 1, bTaken = bItem + 2, bEnd = bTaken + 2;
    static constexpr uint32_t oTmem = (bEnd + 1) * 8, oAbort = oTmem + 4, oItem = oTmem + 8;
    static constexpr uint32_t oScale = oItem + 2 * kItemWords * 4, oLargest = oScale + 64;   // 4 bits: exponents of eight tiles' K and V; of warps;
    static constexpr uint32_t oTop = oLargest + 64;                          // and no tile's values of the piece had a larger one
    static_assert(oTop + 4 <= kMisc, "barrier region");
    static constexpr int kHeld = BITS == 16 ? 4 : 2;                         // groups of 32 scores that a row's thread holds
    static constexpr uint32_t cO = NT * kKt;                                 // first column of O
};

// A query tile: positions of its first and last token (p1 < p0: it has none), and which of the block's key tiles they see: the
// first tokens' and [from, to).
struct QueryTile {
    int32_t p0, p1, from, to;
};
// The key tiles that a block visits: tile i of n starts at first(i).  The first n_sink lie in front of the windows; n_first, these and
// what one query tile still has in its window, hold first tokens.
struct KeyTiles {
    int32_t lo, hi, t_lo, n_sink, n, n_first;
    __device__ __forceinline__ int32_t first(int32_t i) const { return (i < n_sink ? i : t_lo + i - n_sink) * (int32_t)kKt; }
    __device__ __forceinline__ bool seen_by(const QueryTile &q, int32_t i) const { return i < q.to && (i >= q.from || i < n_first); }
    // Of these tiles only those of one piece of several.  The first tokens of a window go with the first one.
    __device__ __forceinline__ void take(uint32_t piece, uint32_t pieces) {
        auto begin = [&](uint32_t k) {
            const int32_t x = (int32_t)((uint64_t)n * k / pieces);
            return x == 0 ? 0 : max(x, n_sink);
        };
        const int32_t i0 = begin(piece), i1 = begin(piece + 1);
        if (i0) {
            t_lo += i0 - n_sink;
            n_sink = 0;
        }
        n = i1 - i0;
    }
};

// A piece as the scheduling warp hands it to the others; sequence < 0: there is no more.
enum PieceWords : uint32_t { kSequence, kHead, kFirstRow, kPieces, kSlot, kTilesAt, kQueriesAt = kTilesAt + 6 };
static_assert(kQueriesAt + 8 <= kItemWords, "room for two query tiles");

// The same in every lane: said to the compiler, which then forms what depends on it in uniform registers.
__device__ __forceinline__ int32_t uniform(int32_t v) { return __shfl_sync(kFull, v, 0); }

// Bits 0 .. n - 1, for any n.
__device__ __forceinline__ uint32_t low_bits(int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }

__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void split(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The largest of three values, NaN where one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// 2^x of two values, x <= 2^6, in the fused multiply-add units: the integer next to x goes into the exponent field, 2^f for the rest
// in [-1/2, 1/2] is a polynomial of degree 3 fitted for the smallest largest relative error, 7.5e-5, a fiftieth of what rounding to
// bf16 loses.  The special-function unit makes four results per cycle and scheduler; a quarter of the weights comes from here
// (4096 tokens, 32 heads of 128 over 8: 121.7 us, none of them 124.0, half 140.0).  For x of
// -126 and less it gives 2^-126, not 0, and for a NaN too: not for tiles with hidden scores, nor where a row's largest is not finite.
constexpr float kExp0 = 0.99992812f, kExp1 = 0.69326097f, kExp2 = 0.24261075f, kExp3 = 0.05517141f;
__device__ __forceinline__ void ex2_poly(uint64_t x, float &r0, float &r1) {
    float x0, x1;
    split(x, x0, x1);
    x = pair(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
    const uint64_t magic = pair(12582912.f, 12582912.f), t = add2(x, magic);
    const uint64_t f = add2(x, fma2(add2(t, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), 0));
    uint64_t y = fma2(f, pair(kExp3, kExp3), pair(kExp2, kExp2));
    y = fma2(f, y, pair(kExp1, kExp1));
    y = fma2(f, y, pair(kExp0, kExp0));
    float y0, y1, t0, t1;
    split(y, y0, y1);
    split(t, t0, t1);
    r0 = __uint_as_float(__float_as_uint(y0) + (__float_as_uint(t0) << 23));
    r1 = __uint_as_float(__float_as_uint(y1) + (__float_as_uint(t1) << 23));
}

// Words that are asked for here and not where they are used: the compiler moves ordinary loads down to there.
template <int N>
__device__ __forceinline__ void ask_words(uint32_t (&w)[N], const uint32_t *p) {
    if constexpr (N == 1) {
        asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
    } else if constexpr (N == 2) {
        asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                         : "l"(p + i));
    }
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Whether p holds in all of THREADS threads, which meet here (barrier 1).
template <uint32_t THREADS>
__device__ __forceinline__ bool all_of(bool p) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred P, Q;\n\tsetp.ne.u32 P, %1, 0;\n\tbar.red.and.pred Q, 1, %2, P;\n\tselp.u32 %0, 1, 0, Q;\n\t}" : "=r"(r) : "r"((uint32_t)p), "n"(THREADS) : "memory");
    return r != 0;
}
// The smallest e with x < 2^e, for x >= 0 that is finite; others do not ask for a scale.
__device__ __forceinline__ int32_t exponent_of(float x) {
    const uint32_t e = __float_as_uint(x) >> 23 & 0xFFu;
    return e == 255 ? -126 : (int32_t)e - 126;
}
__device__ __forceinline__ float power_of_2(int32_t n) { return __uint_as_float((uint32_t)(min(max(n, -126), 127) + 127) << 23); }

// SHORT: with the limits of ci_paged_set_wait_limit; reading them at each wait costs 1 to 2 % (4 x 2000 tokens, heads of 64 in 4 bits:
// 109.0 us instead of 107.1), so the kernel that serves calls has a constant.
template <int D, int BITS, bool SHORT>
__global__ void __launch_bounds__(PromptShape<D, BITS>::kThreads, 1)
k_paged_prompt(const __grid_constant__ PromptArgs a, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
               const __grid_constant__ CUtensorMap v_map) {
    using Sh = PromptShape<D, BITS>;
    constexpr uint32_t NT = Sh::NT, NS = Sh::NS, NB = D / 64;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_s = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem = smem_raw + (smem_s - smem_u32(smem_raw));
    const uint32_t warp = uniform(threadIdx.x >> 5), lane = lane_id();
    const PagedBatch &p = a.p;
    auto bar = [&](uint32_t i) { return smem_s + Sh::oBar + i * 8; };
    volatile uint32_t *s_tmem = reinterpret_cast<volatile uint32_t *>(smem + Sh::oBar + Sh::oTmem);
    volatile uint32_t *s_abort = reinterpret_cast<volatile uint32_t *>(smem + Sh::oBar + Sh::oAbort);
    volatile int32_t *s_items = reinterpret_cast<volatile int32_t *>(smem + Sh::oBar + Sh::oItem);

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (threadIdx.x == 0) {
        mbar_init(bar(Sh::bQ), 1);
        for (uint32_t i = 0; i < NS; ++i) {
            mbar_init(bar(Sh::bFull + i), BITS == 16 ? 1 : Sh::PW);
            mbar_init(bar(Sh::bEmpty + i), NT);
        }
        for (uint32_t t = 0; t < NT; ++t) {
            mbar_init(bar(Sh::bS + t), 1);
            mbar_init(bar(Sh::bP + 2 * t), 4);
            mbar_init(bar(Sh::bP + 2 * t + 1), 4);
        }
        for (uint32_t t = 0; t < NT; ++t) {
            mbar_init(bar(Sh::bO + t), 1);
            mbar_init(bar(Sh::bRead + t), 4);
        }
        mbar_init(bar(Sh::bTurn), 1);
        mbar_init(bar(Sh::bTurn + 1), 1);
        mbar_init(bar(Sh::bQh), 4 * NT);
        mbar_init(bar(Sh::bQfree), NT);
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(bar(Sh::bItem + i), 1);
            mbar_init(bar(Sh::bTaken + i), Sh::kSched);         // all other warps
        }
        mbar_init(bar(Sh::bEnd), NT);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == Sh::kMma) tmem_alloc(smem_s + Sh::oBar + Sh::oTmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(*s_tmem);
    auto give_up = [&](uint32_t code) {
        if (lane == 0) { atomicCAS(&g_prompt_status, 0u, code); *s_abort = 1; }     // the first one's stays
    };
    // Waits of the roles on each other.  Those for what this block has in flight itself (14, and behind the last piece) go by the
    // usual limit whatever these have.
    auto polls = [&](uint32_t code) { return !SHORT ? kWaitPolls : code == a.at_once ? 0u : a.polls; };

    // ---- pieces, one after the other: the roles run ahead of each other across their borders ------------------------
    QueryTile qt[NT];
    KeyTiles kt;
    uint32_t b = 0;
    uint32_t ring0 = 0, q_count = 0;                            // tiles of K and V, and of Q, before this piece
    auto get_item = [&](uint32_t k) {                           // false: there is none (or the wait ran out)
        if (!__all_sync(kFull, mbar_wait(bar(Sh::bItem + k % 2), k / 2 & 1, polls(20)))) {
            give_up(20);
            return false;
        }
        volatile const int32_t *x = s_items + k % 2 * kItemWords;
        if (__any_sync(kFull, x[kSequence] < 0 || *s_abort)) return false;
        b = (uint32_t)uniform(x[kSequence]);
        kt = {uniform(x[kTilesAt]), uniform(x[kTilesAt + 1]), uniform(x[kTilesAt + 2]), uniform(x[kTilesAt + 3]), uniform(x[kTilesAt + 4]), uniform(x[kTilesAt + 5])};
#pragma unroll
        for (uint32_t t = 0; t < NT; ++t)
            qt[t] = {uniform(x[kQueriesAt + 4 * t]), uniform(x[kQueriesAt + 4 * t + 1]), uniform(x[kQueriesAt + 4 * t + 2]), uniform(x[kQueriesAt + 4 * t + 3])};
        return true;
    };
    auto head_of = [&](uint32_t k) { return (uint32_t)uniform(s_items[k % 2 * kItemWords + kHead]); };
    auto first_row_of = [&](uint32_t k) { return uniform(s_items[k % 2 * kItemWords + kFirstRow]); };       // first token of the piece
    auto leave_item = [&](uint32_t k) {                         // this warp has read what it wants of it
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(Sh::bTaken + k % 2));
    };
    auto end_item = [&]() {
        ring0 += 2 * (uint32_t)kt.n;
        q_count += kt.n > 0;
    };

    if (Sh::kMove) {                                            // by warpgroups: 4 bits have some of producers, one for the products
        if (warp < 4 * NT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Sh::kSoftRegs));
        else if (BITS == 4 && warp >= Sh::kMma) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Sh::kMmaRegs));
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Sh::kProdRegs));
    }
    if (warp < 4 * NT) {
        // =========================== softmax: one thread per query row ===============================================
        const uint32_t t = warp >> 2, w = warp & 3, row = w * 32 + lane;
        const uint32_t tok = row / a.group, head = row % a.group;
        uint32_t turn = 0;                                      // products of all pieces so far
        bool ok = true;
        for (uint32_t k = 0; ok && get_item(k); ++k) {
            QueryTile q = qt[0];
            if (NT == 2 && t == 1) q = qt[NT - 1];
            // (the tile's rows behind the sequence's go along with its last one; no sum of a length and more passes 2^31 so)
            const int32_t behind = q.p1 - q.p0, pos = q.p0 + max(min((int32_t)tok, behind), 0), last = min(pos, p.cap - 1);
            const bool live = tok < a.tt && (int32_t)tok <= behind;
            const uint32_t s_addr = tmem + ((w * 32u) << 16) + t * kKt, o_addr = tmem + ((w * 32u) << 16) + Sh::cO + t * D;
            float m = kNone;
            constexpr int kSums = BITS == 16 ? 4 : 2;
            uint64_t l2[kSums] = {};                                // sums of weights, two in each
            bool done = false;                                      // a product of this piece has been
            const uint32_t ids = kKt >> p.page_shift;               // pages of a tile
            auto page_id = [&](int32_t i) {                         // of tile i, one per lane; 0 where there is none to ask for
                const int32_t at = kt.first(i) + (int32_t)(lane << p.page_shift);
                return i < kt.n && lane < ids && at < kt.hi ? __ldg(p.table + (size_t)b * p.table_stride + ((uint32_t)at >> p.page_shift)) : 0;
            };
            int32_t id = page_id(0);
            float scale = a.scale_log2;
            volatile const int32_t *s_scale = reinterpret_cast<volatile const int32_t *>(smem + Sh::oBar + Sh::oScale);
            int32_t v_exp = 0;                                      // O stands for O 2^v_exp
            if (BITS == 4 && kt.n > 0) {                            // this row of Q to fp16, its largest value below 2^15
                ok = __all_sync(kFull, mbar_wait(bar(Sh::bQ), q_count & 1, polls(18)));
                if (!ok) give_up(18);
                const uint32_t q_s = smem_s + Sh::oQ + t * Sh::kTile + row * 128;
                auto chunk = [&](uint32_t c) { return q_s + (c / 8) * Sh::kBlock + ((c % 8 ^ (row & 7)) << 4); };
                float big = 0.f;
#pragma unroll 4
                for (uint32_t c = 0; c < D / 8; ++c) {
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const uint32_t x = lds_u32(chunk(c) + 4 * e);
                        big = fmaxf(big, fmaxf(fabsf(lo_bf16(x)), fabsf(hi_bf16(x))));
                    }
                }
                const int32_t e = exponent_of(big) - 15;
                const float up = power_of_2(-e / 2), up2 = power_of_2(-e - -e / 2);
#pragma unroll 4
                for (uint32_t c = 0; c < D / 8; ++c) {
                    uint32_t y[4];
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint32_t x = lds_u32(chunk(c) + 4 * j);
                        y[j] = pack_f16(lo_bf16(x) * up * up2, hi_bf16(x) * up * up2);
                    }
                    sts_v4(chunk(c), y[0], y[1], y[2], y[3]);
                }
                scale *= power_of_2(e / 2) * power_of_2(e - e / 2);
                fence_async_proxy();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(Sh::bQh));
            }
            const float row_scale = scale;
            for (int32_t i = 0; i < kt.n && ok; ++i) {
                const uint32_t gone = __ballot_sync(kFull, (uint32_t)id >= p.num_pages);    // one bit per page that does not exist
                id = page_id(i + 1);
                if (!kt.seen_by(q, i)) continue;
                const int32_t f = kt.first(i);
                const bool edge = gone || f + (int32_t)kKt - 1 > min(q.p0, p.cap - 1) ||
                                  (a.window && f <= q.p1 - a.window && f + (int32_t)kKt > a.sinks);
                if (!__all_sync(kFull, mbar_wait(bar(Sh::bS + t), turn & 1, polls(11)))) {
                    give_up(11);
                    ok = false;
                    break;
                }
                tc_fence_after();
                int32_t v_move = 0;                                 // O is to be multiplied by 2^v_move for the scale of this tile's V
                if (BITS == 4) {
                    // The tile of V cannot be replaced before this row's weights are out, so its barrier can be waited on here; the
                    // exponents of the tile were written before it.
                    const uint32_t c = ring0 + 2 * (uint32_t)i + 1, at = c / 2 % 8;
                    if (!__all_sync(kFull, mbar_wait(bar(Sh::bFull + c % NS), (c / NS) & 1, polls(19)))) {
                        give_up(19);
                        ok = false;
                        break;
                    }
                    const int32_t ke = s_scale[at], ve = s_scale[8 + at];
                    scale = fmaxf(row_scale * power_of_2(ke / 2) * power_of_2(ke - ke / 2), 1.2e-38f);
                    v_move = done ? v_exp - ve : 0;
                    v_exp = ve;
                }
                const uint64_t scale2 = pair(scale, scale);
                uint32_t x[Sh::kHeld][32];
                uint32_t any = edge ? 0u : 1u;                      // not 0: the row sees some of the tile
                auto hide = [&](uint32_t (&v)[32], int32_t c) {     // scores of positions that the row does not see
                    const int32_t f32 = f + c * 32;
                    uint32_t seen = low_bits(last + 1 - f32);
                    if (a.window) seen &= ~low_bits(pos - a.window + 1 - f32) | low_bits(a.sinks - f32);
                    if (gone)
#pragma unroll
                        for (int j = 0; j < 32; j += 16)
                            if (gone >> ((uint32_t)(c * 32 + j) >> p.page_shift) & 1) seen &= ~(0xFFFFu << j);
                    any |= seen;
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (!(seen & (1u << j))) v[j] = 0xFF800000u;
                };
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                auto largest = [&](const uint32_t (&v)[32]) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            mx4[e] = max3_nan(mx4[e], __uint_as_float(v[j + e]), __uint_as_float(v[j + 4 + e]));
                };
                auto load = [&](int first) {                        // kHeld groups of 32 scores
#pragma unroll
                    for (int c = 0; c < Sh::kHeld; ++c) tmem_ld32_start(s_addr + (first + c) * 32, x[c]);
#pragma unroll
                    for (int c = 0; c < Sh::kHeld; ++c) tmem_ld_wait(x[c]);
                    if (edge)
#pragma unroll
                        for (int c = 0; c < Sh::kHeld; ++c) hide(x[c], first + c);
                };
#pragma unroll
                for (int first = 4 - Sh::kHeld; first >= 0; first -= Sh::kHeld) {
                    load(first);
#pragma unroll
                    for (int c = 0; c < Sh::kHeld; ++c) largest(x[c]);
                }
                const float mx = max3_nan(max3_nan(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3]) * scale;
                if (any) m = fmaxf(m, kLeast);
                const bool grow = mx > m + kLazy;               // (not for a NaN: its weight is one whatever it refers to)
                // A score that is not finite (rows behind the sequence hold anything): its weight is 0 or NaN, which ex2_poly has not.
                const bool odd = BITS == 16 && !edge && live && !(fabsf(mx) < INFINITY);
                bool exact = edge;
                if (__any_sync(kFull, grow || odd || v_move != 0)) {
                    exact |= BITS == 16 && __any_sync(kFull, odd);
                    float c = grow ? ex2(m - mx) : 1.f;
                    if (grow) m = mx;
#pragma unroll
                    for (int e = 0; e < kSums; ++e) l2[e] = fma2(l2[e], pair(c, c), 0);
                    if (BITS == 4) c *= power_of_2(v_move / 2) * power_of_2(v_move - v_move / 2);
                    if (done) {
#pragma unroll 1
                        for (uint32_t j = 0; j < D / 32; ++j) {
                            uint32_t o[32];
                            tmem_ld32(o_addr + j * 32, o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * c);
                            tmem_st32(o_addr + j * 32, o);
                        }
                    }
                }
                // Rows of V that no query of the block sees become zeros: 0 times what lies there need not be 0.  A thread has the row of
                // its number; both query tiles write them, as neither waits for the other.
                if (BITS == 16 && (f + (int32_t)kKt > kt.hi || (a.window && f < kt.lo && f + (int32_t)kKt > a.sinks))) {
                    const uint32_t c = ring0 + 2 * (uint32_t)i + 1;
                    if (!__all_sync(kFull, mbar_wait(bar(Sh::bFull + c % NS), (c / NS) & 1, polls(16)))) {
                        give_up(16);
                        ok = false;
                        break;
                    }
                    const int32_t at = f + (int32_t)row;
                    if (at >= kt.hi || (a.window && at < kt.lo && at >= a.sinks)) {
                        const uint32_t v_s = smem_s + Sh::oRing + (c % NS) * Sh::kTile + row * 128;
#pragma unroll
                        for (uint32_t j = 0; j < NB * 8; ++j) sts_v4(v_s + (j / 8) * Sh::kBlock + ((j + row) % 8) * 16, 0, 0, 0, 0);
                    }
                    fence_async_proxy();
                }
                const float ref = m == kNone ? 0.f : -m;
                const uint64_t ref2 = pair(ref, ref);
                auto weights = [&](auto whole) {                    // whole: no score of the tile is hidden, none infinite or NaN
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (c && c % Sh::kHeld == 0) load(c);
                        const uint32_t(&v)[32] = x[c % Sh::kHeld];
                        uint32_t pk[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const uint64_t y = fma2(pair(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), scale2, ref2);
                            float e0, e1;
                            if (decltype(whole)::value && BITS == 16 && j % 4 == 3) {
                                ex2_poly(y, e0, e1);
                            } else {
                                split(y, e0, e1);
                                e0 = ex2(e0);
                                e1 = ex2(e1);
                            }
                            // (in the values' type, as the tensor instructions want: half a step of bf16 is 2^-8 of a weight, of fp16
                            // 2^-11; sums in fp32.  Outputs in bf16 0.0020 from 64 bits in the mean, 0.0016 of it their own rounding.)
                            l2[j % kSums] = add2(l2[j % kSums], pair(e0, e1));
                            pk[j] = BITS == 16 ? pack_bf16(e0, e1) : pack_f16(e0, e1);
                        }
                        tmem_st16(s_addr + c * 16, pk);
                        if (c % 2) {                                    // half of the weights are there
                            tmem_st_wait();
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(bar(Sh::bP + 2 * t + c / 2));
                        }
                    }
                };
                if (exact) weights(std::false_type());
                else weights(std::true_type());
                done = true;
                ++turn;
            }
            float l = 0.f;
#pragma unroll
            for (int e = 0; e < kSums; ++e) {
                float l0, l1;
                split(l2[e], l0, l1);
                l += l0 + l1;
            }
            // ---- the row's result ----------------------------------------------------------------------------------
            if (ok && !mbar_wait(bar(Sh::bO + t), k & 1, polls(12))) { give_up(12); ok = false; }
            ok = __all_sync(kFull, ok && !*s_abort);
            if (__all_sync(kFull, ok)) {
                tc_fence_after();
                const bool none = m == kNone;                         // nothing seen: zeros, whatever values have left in O
                const float inv = none ? 0.f : 1.f / l;
                const float up = BITS == 4 ? power_of_2(v_exp / 2) : 1.f, up2 = BITS == 4 ? power_of_2(v_exp - v_exp / 2) : 1.f;
                volatile const int32_t *item = s_items + k % 2 * kItemWords;
                const uint32_t pieces = (uint32_t)item[kPieces], kvh = head_of(k);
                const int32_t q_row = first_row_of(k);
                const size_t part = ((size_t)(uint32_t)item[kSlot] * p.n_kv + kvh) * (NT * 128) + t * 128 + row;
                if (pieces > 1 && live) *reinterpret_cast<float2 *>(a.ml + part * 2) = make_float2(m, l);
                uint16_t *dst = a.out + (int64_t)(q_row + (int32_t)(t * a.tt + tok)) * a.ldo + (size_t)(kvh * a.group + head) * D;
#pragma unroll 1
                for (uint32_t j = 0; j < D / 32; ++j) {
                    uint32_t o[32];
                    if (done) {                             // (zeros in both branches: one behind them takes registers from the loop over tiles)
                        tmem_ld32(o_addr + j * 32, o);
                        if (none)
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = 0;
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0;
                    }
                    if (live && pieces > 1) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            *reinterpret_cast<float4 *>(a.partial + part * D + j * 32 + e * 4) =
                                make_float4(__uint_as_float(o[4 * e]) * up * up2, __uint_as_float(o[4 * e + 1]) * up * up2,
                                            __uint_as_float(o[4 * e + 2]) * up * up2, __uint_as_float(o[4 * e + 3]) * up * up2);
                    } else if (live) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            uint32_t y[4];
#pragma unroll
                            for (int h = 0; h < 4; ++h)
                                y[h] = pack_bf16(__uint_as_float(o[8 * e + 2 * h]) * inv * up * up2, __uint_as_float(o[8 * e + 2 * h + 1]) * inv * up * up2);
                            *reinterpret_cast<uint4 *>(dst + j * 32 + e * 8) = make_uint4(y[0], y[1], y[2], y[3]);
                        }
                    }
                }
            }
            if (!ok) tmem_st_wait();                                // (nothing under way into tensor memory that is given back)
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(Sh::bRead + t));         // O may be written again
            leave_item(k);
            end_item();
        }
    } else if (warp >= Sh::kMma && warp < Sh::kMma + NT) {
        // =========================== products ======================================================================
        constexpr uint32_t kTypes = BITS == 16 ? (1u << 7) | (1u << 10) : 0u;       // both bf16, or both fp16
        constexpr uint32_t kIdescS = (1u << 4) | kTypes | ((kKt >> 3) << 17) | ((128u >> 4) << 24);
        constexpr uint32_t kIdescO = (1u << 4) | kTypes | (1u << 16) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
        // One warp per query tile, in turns: while one tile's products run, the other's rows are at their exponentials.  Without
        // turns both come to do the same at the same time (4250 cycles for a pair of query tiles and a key tile instead of 2800).
        const uint32_t t = warp - Sh::kMma, idesc_s = kIdescS | (a.negate ? 1u << 13 : 0u);
        QueryTile q;
        uint32_t made = 0, round = 0;                           // products with V issued, and key tiles, of all pieces
        bool ok = true;
        const uint64_t q_desc = umma_desc_sw128(smem_s + Sh::oQ + t * Sh::kTile), k_desc = umma_desc_sw128(smem_s + Sh::oRing);
        const uint64_t v_desc = umma_desc_sw128_mn(smem_s + Sh::oRing, Sh::kBlock);
        const uint32_t s_col = tmem + t * kKt, o_col = tmem + Sh::cO + t * D;
        auto full = [&](uint32_t c) { return mbar_wait(bar(Sh::bFull + c % NS), (c / NS) & 1, polls(13)); };
        auto scores = [&](int32_t i) {
            tc_fence_after();
            const uint64_t kd = k_desc + ((ring0 + 2 * i) % NS) * (Sh::kTile >> 4);
            if (elect_one()) {
#pragma unroll
                for (uint32_t kk = 0; kk < D / 16; ++kk) {
                    const uint32_t o = (kk / 4) * (Sh::kBlock >> 4) + (kk % 4) * (32 >> 4);
                    umma_bf16(s_col, q_desc + o, kd + o, idesc_s, kk != 0);
                }
                umma_commit(bar(Sh::bS + t));
            }
            __syncwarp();
        };
        auto release = [&](uint32_t c) {                        // the slot is free once this warp's products so far are done
            if (elect_one()) umma_commit(bar(Sh::bEmpty + c % NS));
            __syncwarp();
        };
        auto q_read = [&]() {                                   // Q may be written once the products so far are done
            if (elect_one()) umma_commit(bar(Sh::bQfree));
            __syncwarp();
        };
        for (uint32_t k = 0; ok && get_item(k); ++k) {
            leave_item(k);
            q = qt[0];
            if (NT == 2 && t == 1) q = qt[NT - 1];
            bool first = true;                                      // no product with V yet: O is written, not added to
            if (kt.n > 0) {
                ok = __all_sync(kFull, mbar_wait(bar(BITS == 16 ? Sh::bQ : Sh::bQh), q_count & 1, polls(13)) && full(ring0));
                if (!ok) break;
                if (kt.seen_by(q, 0)) scores(0);
                release(ring0);
                if (kt.n == 1) q_read();
            }
            for (int32_t i = 0; i < kt.n && ok; ++i) {
                if (NT == 2 && (t == 1 || round > 0)) {
                    ok = __all_sync(kFull, mbar_wait(bar(Sh::bTurn + t), (t == 1 ? round : round - 1) & 1, polls(13)));
                    if (!ok) break;
                }
                ++round;
                if (kt.seen_by(q, i)) {
                    const uint64_t vd = v_desc + ((ring0 + 2 * i + 1) % NS) * (Sh::kTile >> 4);
                    ok = __all_sync(kFull, full(ring0 + 2 * i + 1));
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {              // the weights come in two halves
                        ok = ok && __all_sync(kFull, mbar_wait(bar(Sh::bP + 2 * t + h), made & 1, polls(13)));
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) {
#pragma unroll
                            for (uint32_t kk = h * (kKt / 32); kk < (h + 1) * (kKt / 32); ++kk)
                                umma_ts(o_col, s_col + kk * 8, vd + kk * (2048 >> 4), kIdescO, !first || kk != 0);
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    ++made;
                    first = false;
                }
                release(ring0 + 2 * i + 1);
                if (i + 1 < kt.n) {
                    if (kt.seen_by(q, i + 1)) {
                        ok = __all_sync(kFull, full(ring0 + 2 * i + 2));
                        if (!ok) break;
                        scores(i + 1);
                    }
                    release(ring0 + 2 * i + 2);
                    if (i + 2 == kt.n) q_read();
                }
                if (NT == 2 && lane == 0) mbar_arrive(bar(Sh::bTurn + (t ^ 1)));
                __syncwarp();
            }
            if (!ok) break;
            // (not before the rows' threads have waited for the piece before: a phase that nobody has seen would be lost)
            if (k > 0 && !__all_sync(kFull, mbar_wait(bar(Sh::bRead + t), (k - 1) & 1, polls(13)))) {
                ok = false;
                break;
            }
            if (elect_one()) umma_commit(bar(Sh::bO + t));
            __syncwarp();
            end_item();
        }
        if (!ok) give_up(13);
        if (elect_one()) umma_commit(bar(Sh::bEnd));
        __syncwarp();
        if (!__all_sync(kFull, mbar_wait(bar(Sh::bEnd), 0))) give_up(14);     // tensor memory is given back behind the last product
    } else if (warp == Sh::kSched) {
        // =========================== which piece next ===============================================================
        for (uint32_t k = 0;; ++k) {
            if (!mbar_wait_warp(bar(Sh::bTaken + k % 2), (k / 2 & 1) ^ 1, polls(21))) { give_up(21); break; }
            uint32_t v = 0;
            if (lane == 0) v = (uint32_t)atomicAdd(a.next, 1);
            v = __shfl_sync(kFull, v, 0);
            int4 w0 = make_int4((int32_t)p.B, 0, 0, 0), w1 = make_int4(0, 0, 0, 0);
            if (v < a.count && !*s_abort) {
                w0 = __ldcg(a.plan + (size_t)(v / p.n_kv) * 2);
                w1 = __ldcg(a.plan + (size_t)(v / p.n_kv) * 2 + 1);
            }
            const bool there = (uint32_t)w0.x < p.B;
            const int32_t q0 = w1.y, q_len = w1.z, kv_len = w1.w;
            kt.lo = p.cap;
            kt.hi = 0;
            int32_t lo[NT], hi[NT];                             // what a query tile sees
#pragma unroll
            for (uint32_t t = 0; t < NT; ++t) {
                const int32_t i0 = (int32_t)(((uint32_t)w0.y * NT + t) * a.tt), n = min(max(q_len - i0, 0), (int32_t)a.tt);
                qt[t].p0 = kv_len - q_len + min(i0, q_len);
                qt[t].p1 = qt[t].p0 + n - 1;
                hi[t] = n ? max(min(qt[t].p1 + 1, p.cap), 0) : 0;
                lo[t] = a.window ? min(max(qt[t].p0 - a.window + 1, 0), hi[t]) : 0;
                if (n) {
                    kt.lo = min(kt.lo, lo[t]);
                    kt.hi = max(kt.hi, hi[t]);
                }
            }
            kt.lo = min(kt.lo, kt.hi);
            kt.t_lo = kt.lo / (int32_t)kKt;
            kt.n_sink = a.window ? min((min(a.sinks, kt.hi) + (int32_t)kKt - 1) / (int32_t)kKt, kt.t_lo) : 0;
            kt.n = kt.n_sink + (kt.hi + (int32_t)kKt - 1) / (int32_t)kKt - kt.t_lo;
            if (w0.w > 1) kt.take((uint32_t)w0.z, (uint32_t)w0.w);
            kt.n_first = a.window ? kt.n_sink + max((min(a.sinks, kt.hi) + (int32_t)kKt - 1) / (int32_t)kKt - kt.t_lo, 0) : 0;
#pragma unroll
            for (uint32_t t = 0; t < NT; ++t) {
                qt[t].from = lo[t] / (int32_t)kKt - kt.t_lo + kt.n_sink;
                qt[t].to = qt[t].p1 < qt[t].p0 ? 0 : (hi[t] + (int32_t)kKt - 1) / (int32_t)kKt - kt.t_lo + kt.n_sink;
            }
            if (lane == 0) {
                volatile int32_t *x = s_items + k % 2 * kItemWords;
                x[kSequence] = there ? w0.x : -1;
                x[kHead] = (int32_t)(v % p.n_kv);
                x[kFirstRow] = q0 + (int32_t)((uint32_t)w0.y * NT * a.tt);
                x[kPieces] = w0.w;
                x[kSlot] = w1.x + w0.z;
                x[kTilesAt] = kt.lo;
                x[kTilesAt + 1] = kt.hi;
                x[kTilesAt + 2] = kt.t_lo;
                x[kTilesAt + 3] = kt.n_sink;
                x[kTilesAt + 4] = kt.n;
                x[kTilesAt + 5] = kt.n_first;
#pragma unroll
                for (uint32_t t = 0; t < NT; ++t) {
                    x[kQueriesAt + 4 * t] = qt[t].p0;
                    x[kQueriesAt + 4 * t + 1] = qt[t].p1;
                    x[kQueriesAt + 4 * t + 2] = qt[t].from;
                    x[kQueriesAt + 4 * t + 3] = qt[t].to;
                }
                mbar_arrive(bar(Sh::bItem + k % 2));
            }
            __syncwarp();
            if (!there) break;
        }
    } else if (warp > Sh::kSched) {
        // (warps that fill a warpgroup)
    } else if constexpr (BITS == 16) {
        // =========================== TMA copies ====================================================================
        const uint32_t ids = kKt >> p.page_shift;
        uint32_t issued = 0, queries = 0, kvh = 0;              // copies asked for; the piece's head
        int32_t q_row = 0;                                      // and first token
        bool ok = true;
        auto load_q = [&]() {
            if (q_count && !mbar_wait_warp(bar(Sh::bQfree), (q_count - 1) & 1, polls(22))) return false;
            if (lane == 0) {
                const uint32_t bytes = a.tt * a.group * 128;    // of a block of 64 channels
                mbar_expect_tx(bar(Sh::bQ), NT * NB * bytes);
                for (uint32_t t = 0; t < NT; ++t)
                    for (uint32_t c = 0; c < NB; ++c)
                        tma_load_3d(smem_s + Sh::oQ + t * Sh::kTile + c * Sh::kBlock, &q_map, (int32_t)(c * 64), (int32_t)(kvh * a.group),
                                    q_row + (int32_t)(t * a.tt), bar(Sh::bQ));
            }
            __syncwarp();
            ++queries;
            return true;
        };
        auto row_of = [&](int32_t i) {                          // this lane's page of tile i, as a row of the pool
            const int32_t at = kt.first(i) + (int32_t)(lane << p.page_shift);
            const int32_t id = lane < ids && at < kt.hi ? page_of(p, b, at) : -1;
            return id < 0 ? -(int32_t)kKt : (int32_t)row_index(p, id, kvh, at);
        };
        for (uint32_t k = 0; ok && get_item(k); ++k) {
            kvh = head_of(k);
            q_row = first_row_of(k);
            leave_item(k);
            int32_t next = kt.n > 0 ? row_of(0) : 0;
            for (int32_t i = 0; i < kt.n && ok; ++i) {
                const int32_t r = next;
                if (i + 1 < kt.n) next = row_of(i + 1);
                for (uint32_t kv = 0; kv < 2; ++kv, ++issued) {
                    const uint32_t slot = issued % NS;
                    if (!mbar_wait_warp(bar(Sh::bEmpty + slot), ((issued / NS) & 1) ^ 1, polls(15)) || __any_sync(kFull, *s_abort)) { give_up(15); ok = false; break; }
                    const uint32_t to = bar(Sh::bFull + slot), dst = smem_s + Sh::oRing + slot * Sh::kTile;
                    if (lane == 0) mbar_expect_tx(to, Sh::kTile);
                    __syncwarp();
                    if (lane < ids)
#pragma unroll
                        for (uint32_t c = 0; c < NB; ++c)
                            tma_load_2d(dst + c * Sh::kBlock + (lane << p.page_shift) * 128, kv ? &v_map : &k_map, (int32_t)(c * 64), r, to);
                    __syncwarp();
                    if (i == 0 && kv == 0 && !load_q()) { give_up(22); ok = false; ++issued; break; }
                }
            }
            end_item();
        }
        // Copies under way end before the block does: others may have given up on them, and this warp have left for that.
        for (uint32_t c = issued > NS ? issued - NS : 0; c < issued; ++c) (void)mbar_wait_warp(bar(Sh::bFull + c % NS), (c / NS) & 1);
        if (queries) (void)mbar_wait_warp(bar(Sh::bQ), (queries - 1) & 1);
    } else {
        // =========================== codes to fp16: a thread, or two, per position ==========================================
        constexpr uint32_t G = D / 64;
        constexpr uint32_t PW = Sh::PW, NW = D / 8 / Sh::SPLIT;  // warps; words of a thread
        const uint32_t y = (threadIdx.x - Sh::kProd * 32) % kKt, part = (threadIdx.x - Sh::kProd * 32) / kKt;   // position inside the tile
        const bool first_thread = threadIdx.x == Sh::kProd * 32;
        volatile int32_t *s_scale = reinterpret_cast<volatile int32_t *>(smem + Sh::oBar + Sh::oScale);
        volatile uint32_t *s_largest = reinterpret_cast<volatile uint32_t *>(smem + Sh::oBar + Sh::oLargest);
        volatile int32_t *s_top = reinterpret_cast<volatile int32_t *>(smem + Sh::oBar + Sh::oTop);    // (no register for it in the loop)
        uint32_t issued = 0, queries = 0, kvh = 0;
        int32_t q_row = 0, v_exp;
        bool ok = true;
        // What this thread's position of a tile holds, fetched while the tile before is turned.
        struct Codes {
            uint32_t code[NW], sc[G];
        };
        // Its page as the table has it (looked at when it is there, not when it is asked for); -1 where nobody sees the position.
        auto page_at = [&](int32_t i) {
            if (i >= kt.n) return -1;
            const int32_t at = kt.first(i) + (int32_t)y;
            return at < kt.hi && !(a.window && at < kt.lo && at >= a.sinks)
                       ? __ldg(p.table + (size_t)b * p.table_stride + ((uint32_t)at >> p.page_shift)) : -1;
        };
        auto fetch = [&](Codes &f, int32_t id, int32_t i, uint32_t kv) {
            if ((uint32_t)id >= p.num_pages) return;
            const size_t r = row_index(p, id, kvh, kt.first(i) + (int32_t)y);
            ask_words(f.sc, (kv ? a.vs : a.ks) + r * G);
            ask_words(f.code, reinterpret_cast<const uint32_t *>(kv ? a.v : a.k) + r * (D / 8) + part * NW);
        };
        // (to the end in any case: the warps meet at a barrier)
        auto turn = [&](const Codes &f, int32_t id, int32_t i, uint32_t kv) {
            const uint32_t(&sc)[G] = f.sc;
            const bool there = (uint32_t)id < p.num_pages;
            float big = 0.f;
            if (there)
#pragma unroll
                for (uint32_t g = 0; g < G; ++g) {
                    const float step = lo_bf16(sc[g]), low = hi_bf16(sc[g]);
                    big = fmaxf(big, fmaxf(fabsf(low), fabsf(low + 15.f * step)));
                }
            // the tile's largest exponent
            const uint32_t most = __reduce_max_sync(kFull, (uint32_t)(exponent_of(big) + 200));
            if (lane == 0) s_largest[(issued & 1) * 8 + (warp - Sh::kProd)] = most;
            asm volatile("bar.sync 1, %0;" ::"n"(PW * 32) : "memory");
            int32_t e = 0;
#pragma unroll
            for (uint32_t w = 0; w < PW; ++w) e = max(e, (int32_t)s_largest[(issued & 1) * 8 + w]);
            e -= 200;
            if (kv == 0) e -= 14;                           // below 2^14
            else {
                // from 2^8 to 2^15; where it has to change, below 2^12 again (a tile of zeros changes nothing)
                if (e - v_exp > 15 || (e - v_exp <= 8 && e > -126)) {
                    const int32_t top = max(*s_top, max(e, v_exp + 15));    // no tile so far had more
                    *s_top = top;                               // (the same from every thread, whichever was here before)
                    if (e - v_exp > 15 || top - 80 < v_exp) v_exp = max(e - 12, top - 80);
                }
                e = v_exp;
            }
            const float down = power_of_2(-e / 2), down2 = power_of_2(-e - -e / 2);
            const uint32_t slot = issued % NS, dst = smem_s + Sh::oRing + slot * Sh::kTile + y * 128;
            if (ok && !__all_sync(kFull, mbar_wait(bar(Sh::bEmpty + slot), ((issued / NS) & 1) ^ 1, polls(17)))) {
                give_up(17);
                ok = false;
            }
            if (!ok) return;
            if (first_thread) s_scale[kv * 8 + issued / 2 % 8] = e;
#pragma unroll
            for (uint32_t g = 0; g < G; ++g) {
                const float step = lo_bf16(sc[g]) * down * down2, low = hi_bf16(sc[g]) * down * down2;
                const __half2 step2 = __float2half2_rn(step), low2 = __float2half2_rn(low), base = __float2half2_rn(1024.f);
#pragma unroll
                for (uint32_t c8 = 0; c8 < NW / G; ++c8) {  // a word of the group: eight channels
                    uint32_t o[4] = {0, 0, 0, 0};
                    if (there) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            // fp16 of 1024 + code, the code, and one rounding for what it stands for
                            const uint32_t w = (f.code[c8 * G + g] >> 4 * j & 0x000F000Fu) | 0x64006400u;
                            const __half2 v = __hfma2(__hsub2(*reinterpret_cast<const __half2 *>(&w), base), step2, low2);
                            o[j] = *reinterpret_cast<const uint32_t *>(&v);
                        }
                    }
                    sts_v4(dst + g * Sh::kBlock + ((part * (NW / G) + c8 ^ (y & 7)) << 4), o[0], o[1], o[2], o[3]);
                }
            }
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(Sh::bFull + slot));
        };
        for (uint32_t k = 0;; ++k) {
            if (!all_of<PW * 32>(get_item(k))) break;           // all of these warps go on or none: they meet at a barrier in every tile
            kvh = head_of(k);
            q_row = first_row_of(k);
            leave_item(k);
            v_exp = -1000;                                          // (no tile of V yet)
            *s_top = -126;
            Codes f0, f1;
            int32_t id = page_at(0), id_next = page_at(1);
            if (kt.n > 0) {
                fetch(f0, id, 0, 0);
                if (warp == Sh::kProd) {
                    if (q_count) ok = mbar_wait_warp(bar(Sh::bQfree), (q_count - 1) & 1, polls(22));
                    if (!ok) give_up(22);
                    if (ok && lane == 0) {
                        const uint32_t bytes = a.tt * a.group * 128;
                        mbar_expect_tx(bar(Sh::bQ), NT * NB * bytes);
                        for (uint32_t t = 0; t < NT; ++t)
                            for (uint32_t c = 0; c < NB; ++c)
                                tma_load_3d(smem_s + Sh::oQ + t * Sh::kTile + c * Sh::kBlock, &q_map, (int32_t)(c * 64), (int32_t)(kvh * a.group),
                                            q_row + (int32_t)(t * a.tt), bar(Sh::bQ));
                    }
                    queries += ok;
                    __syncwarp();
                }
            }
            for (int32_t i = 0; i < kt.n; ++i) {
                fetch(f1, id, i, 1);
                turn(f0, id, i, 0);
                ++issued;
                const int32_t id_here = id;
                id = id_next;
                if (i + 1 < kt.n) fetch(f0, id, i + 1, 0);
                id_next = page_at(i + 2);
                turn(f1, id_here, i, 1);
                ++issued;
            }
            end_item();
        }
        if (queries) (void)mbar_wait_warp(bar(Sh::bQ), (queries - 1) & 1);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == Sh::kMma) tmem_dealloc(tmem, 512);
}

// Joins the pieces of an item, kJoinRows rows to a block: D / 4 threads to a row.  In order: the same sum every time.
constexpr uint32_t kJoinRows = 16;
template <int D>
__global__ void __launch_bounds__(256) k_prompt_join(const __grid_constant__ PromptArgs a) {
    constexpr uint32_t NT = PromptShape<D, 16>::NT, kLanes = D / 4, kRows = 256 / kLanes;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t kvh = blockIdx.x % a.p.n_kv;
    const int4 *d = a.cuts + (1 + blockIdx.x / a.p.n_kv) * 2;
    const int32_t cuts = __ldcg(&a.cuts->x);
    const int4 w0 = __ldcg(d), w1 = __ldcg(d + 1);
    if (blockIdx.x / a.p.n_kv >= (uint32_t)cuts) return;
    const uint32_t item = (uint32_t)w0.y, pieces = (uint32_t)w0.w, slot = (uint32_t)w1.x, q_len = (uint32_t)w1.z;
    const int32_t q0 = w1.y;
    for (uint32_t r = blockIdx.y * kJoinRows + threadIdx.x / kLanes; r < (blockIdx.y + 1) * kJoinRows; r += kRows) {
        const uint32_t t = r / 128, tok = r % 128 / a.group, c = threadIdx.x % kLanes * 4;
        const uint32_t at = (item * NT + t) * a.tt + tok;     // the row's token
        if (tok >= a.tt || at >= q_len) continue;
        auto part = [&](uint32_t i) { return ((size_t)(slot + i) * a.p.n_kv + kvh) * (NT * 128) + r; };
        float M = kNone, L = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (uint32_t i0 = 0; i0 < pieces; i0 += 8) {
            float2 ml[8];                                       // asked for together: (max, sum) and outputs
            float4 z[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                ml[i] = make_float2(kNone, 0.f);
                z[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i0 + i < pieces) {
                    ml[i] = __ldcg(reinterpret_cast<const float2 *>(a.ml + part(i0 + i) * 2));
                    z[i] = __ldcg(reinterpret_cast<const float4 *>(a.partial + part(i0 + i) * D + c));
                }
            }
            float most = M;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) most = fmaxf(most, ml[i].x);
            if (most == kNone) continue;
            const float down = M == kNone ? 0.f : ex2(M - most);
            M = most;
            L *= down;
            y.x *= down; y.y *= down; y.z *= down; y.w *= down;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const float e = ml[i].x == kNone ? 0.f : ex2(ml[i].x - M);
                L += e * ml[i].y;
                y.x += e * z[i].x; y.y += e * z[i].y; y.z += e * z[i].z; y.w += e * z[i].w;
            }
        }
        const float inv = M == kNone ? 0.f : 1.f / L;
        *reinterpret_cast<uint2 *>(a.out + (int64_t)(q0 + (int32_t)at) * a.ldo + (size_t)(kvh * a.group + r % 128 % a.group) * D + c) =
            make_uint2(pack_bf16(y.x * inv, y.y * inv), pack_bf16(y.z * inv, y.w * inv));
    }
}

// (of the process; ci_paged_set_wait_limit)
static uint32_t g_prompt_polls = kWaitPolls, g_prompt_at_once = 0;

static size_t prompt_slot_rows(uint32_t head_dim) { return 2 * (size_t)sm_count() * (head_dim == 256 ? 128 : 256); }     // of all slots

PromptPlan prompt_plan(uint32_t head_dim, uint32_t page_size, uint32_t n_kv, const ci_paged_batch *b, uint32_t group, int32_t window,
                       int32_t sinks, uint32_t min_rows, void *workspace) {
    PromptPlan l;
    l.group = group;
    l.per_item = (head_dim == 256 ? 1 : 2) * (128 / group);
    l.min_rows = min_rows;
    l.sms = (uint32_t)sm_count();
    // Lengths are the device's to know: items and pieces as many as there can be, blocks without one leave at once.
    l.may_cut = (uint64_t)b->max_pages * page_size > kFewest * kKt;
    l.count = b->T / l.per_item + b->B + (l.may_cut ? 2 * l.sms / n_kv : 0);
    l.window = window;
    l.sinks = sinks;
    l.cuts = (int4 *)workspace;
    l.pieces = l.cuts + ((size_t)l.sms + 2) * 2;
    return l;
}
size_t prompt_workspace_bytes(uint32_t head_dim, const PromptPlan &l) {
    return (((size_t)l.sms + 2 + l.count) * 2) * sizeof(int4) + prompt_slot_rows(head_dim) * (2 + (size_t)head_dim) * sizeof(float);
}

template <int D, int BITS, bool SHORT>
static int launch_prompt(const PromptArgs &a, const PromptPlan &l, const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm, cudaStream_t s) {
    using Sh = PromptShape<D, BITS>;
    static SmemLimit lim = {};
    if (int rc = ensure_smem_limit(lim, (const void *)k_paged_prompt<D, BITS, SHORT>, Sh::kSmem)) return rc;
    const uint64_t blocks = (uint64_t)l.count * a.p.n_kv;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(blocks < l.sms ? blocks : l.sms));
    cfg.blockDim = dim3(Sh::kThreads);
    cfg.dynamicSmemBytes = Sh::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CI_CUDA(cudaLaunchKernelEx(&cfg, k_paged_prompt<D, BITS, SHORT>, a, qm, km, vm));
    if (!l.may_cut) return CI_OK;
    cfg.gridDim = dim3(l.sms + 1, Sh::NT * 128 / kJoinRows);    // (two pieces at least to a cut item)
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    CI_CUDA(cudaLaunchKernelEx(&cfg, k_prompt_join<D>, a));
    return CI_OK;
}

static int pool_map(CUtensorMap *m, const ci_paged_cache *c, void *base) {
    const cuuint64_t dims[2] = {c->head_dim, (cuuint64_t)c->num_pages * c->n_kv * c->page_size};
    const cuuint64_t strides[1] = {(cuuint64_t)c->head_dim * 2};
    const cuuint32_t box[2] = {64, c->page_size}, one[2] = {1, 1};
    const CUresult r = encode_tiled_fn()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed with code %d", (int)r);
        return CI_E_CUDA;
    }
    return CI_OK;
}

// What launch_paged_prompt asks for, asked before the first kernel of a call is queued.
int check_paged_prompt(const ci_paged_cache *c, const PromptPlan &l) {
    CI_REQUIRE(c->bits == 4 || (uint64_t)c->num_pages * c->n_kv * c->page_size <= 0x7FFFFFFFu, "a pool of more than 2^31 rows");
    CI_REQUIRE((uint64_t)l.count * c->n_kv <= 0x7FFFFFFFu, "too many blocks");
    CI_REQUIRE(encode_tiled_fn() != nullptr, "the driver has no cuTensorMapEncodeTiled");
    return CI_OK;
}

// The pieces of a plan that is there when the kernel runs.  Needs group <= 128.
int launch_paged_prompt(const ci_paged_cache *c, const PagedBatch &p, const PromptPlan &l, const uint16_t *q, int64_t ldq, uint32_t n_q,
                        float scale_log2, uint16_t *out, int64_t ldo, cudaStream_t s) {
    PromptArgs a;
    a.p = p;
    a.k = (const uint8_t *)c->k; a.v = (const uint8_t *)c->v; a.ks = c->k_scale; a.vs = c->v_scale;
    a.group = n_q / c->n_kv;
    a.tt = 128 / a.group;
    a.negate = scale_log2 < 0.f;
    a.window = l.window; a.sinks = l.sinks;
    a.scale_log2 = fmaxf(fabsf(scale_log2), 1e-30f);            // not 0: hidden scores are -inf before they are scaled
    a.out = out; a.ldo = ldo;
    a.plan = l.pieces;
    a.cuts = l.cuts;
    a.next = &l.cuts->y;
    a.count = l.count * p.n_kv;
    a.polls = g_prompt_polls;
    a.at_once = g_prompt_at_once;
    a.ml = (float *)(l.pieces + (size_t)l.count * 2);
    a.partial = a.ml + prompt_slot_rows(c->head_dim) * 2;
    CUtensorMap qm, km, vm;
    memset(&km, 0, sizeof km);
    memset(&vm, 0, sizeof vm);
    const cuuint64_t dims[3] = {c->head_dim, n_q, p.T};
    const cuuint64_t strides[2] = {(cuuint64_t)c->head_dim * 2, (cuuint64_t)ldq * 2};
    const cuuint32_t box[3] = {64, a.group, a.tt}, one[3] = {1, 1, 1};
    const CUresult r = encode_tiled_fn()(&qm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t *>(q), dims, strides, box, one,
                                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed with code %d", (int)r);
        return CI_E_CUDA;
    }
    if (c->bits == 16) {
        if (int rc = pool_map(&km, c, c->k)) return rc;
        if (int rc = pool_map(&vm, c, c->v)) return rc;
    }
    const bool usual = a.polls == kWaitPolls && a.at_once == 0;
    auto launch = [&](auto d) {
        constexpr int D = decltype(d)::value;
        return c->bits == 16 ? (usual ? launch_prompt<D, 16, false>(a, l, qm, km, vm, s) : launch_prompt<D, 16, true>(a, l, qm, km, vm, s))
                             : (usual ? launch_prompt<D, 4, false>(a, l, qm, km, vm, s) : launch_prompt<D, 4, true>(a, l, qm, km, vm, s));
    };
    return c->head_dim == 64    ? launch(std::integral_constant<int, 64>())
           : c->head_dim == 128 ? launch(std::integral_constant<int, 128>())
                                : launch(std::integral_constant<int, 256>());
}

}  // namespace ci

using namespace ci;

extern "C" int ci_paged_status(uint32_t *code, int clear, ci_stream_t stream) {
    void *word = nullptr;
    CI_CUDA(cudaGetSymbolAddress(&word, g_prompt_status));
    return ci_status((uint32_t *)word, code, clear, stream);
}

extern "C" void ci_paged_set_wait_limit(uint32_t polls, uint32_t code) {
    g_prompt_polls = polls ? polls : kWaitPolls;
    g_prompt_at_once = code;
}
