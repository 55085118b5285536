// A paged key/value cache as the kernels see it, and the batch of sequences over it.
//
// Pages of keys and of values are [num_pages, n_kv, page, row] with rows of head_dim bf16, or of head_dim codes of 4 bits
// beside [num_pages, n_kv, page, head_dim / 64] words of (step, lowest), both bf16.  The 32-bit word p of a row of codes
// belongs to group p % G (G = head_dim / 64) and holds channels 8 (p / G) .. + 7 of it, channel i of those in bits
// 4 (i / 2) + 16 (i % 2): two neighbouring channels come out of a word with one shift and one mask, and a lane that
// takes 2 G words in a row has the same channels of every group, as the tensor instructions of the attention want them.
//
// Page ids come from device memory that no host check has seen: an id outside the pool names no page.  Its positions hold
// nothing: they are not written, and no query sees them.
#pragma once
#include "common.cuh"

namespace ci {

constexpr uint32_t kGroup = 64;              // channels that share a step and a lowest value

struct PagedBatch {
    const int32_t *table, *kv_lens, *q_starts;   // q_starts may be null: one new token per sequence
    uint32_t num_pages, page, page_shift, n_kv, table_stride, B, T;
    int32_t cap;                                 // positions that a row of the table can name
};

// How the prompts' kernel (paged_prompt.cu) shares its work, made on the device by k_paged_join, which runs before it.  An item is
// per_item tokens of a sequence for one key/value head.  Items with many more key tiles than others are cut into pieces: no shorter
// than a multiprocessor's share of all tiles where there are no more items than multiprocessors, so that the pieces are not
// more either and run at once (of half a share: 16 sequences of 32 new tokens and 2048 in all 58 us instead of 43, uncut 39; 8 of 32
// over 8000 80 instead of 74, uncut 102); half of that where a multiprocessor has several items anyway (12 sequences of 200 new
// tokens and 300 to 30000 in all, 32 heads of 128 over 8: 454 us, whole shares 621, uncut 618).
// Not shorter than kFewest either: a piece begins with queries and first keys one after the other and ends with k_prompt_join.
// 64 tokens of a sequence of 32000: 59 us, uncut 397.
constexpr uint32_t kKt = 128;                // positions per key tile
constexpr uint32_t kFewest = 4;
struct PromptPlan {
    uint32_t group, per_item, min_rows, sms, count, may_cut;     // min_rows: sequences with as many query rows or fewer are not in it
    int32_t window, sinks;
    int4 *pieces;                            // [count][2]: sequence (B: none), item, piece, pieces; slot of the item's first, q0, q_len, kv_len
    int4 *cuts;                              // [0]: items in several pieces (of each head), 0: blocks count on; [1 + i][2]: the i-th's first piece
};

#ifdef __CUDACC__

struct Seq {
    int32_t q0, q_len, kv_len;                   // first row of the new tokens, their number, all tokens
};

__device__ __forceinline__ Seq load_seq(const PagedBatch &p, uint32_t b) {
    Seq s;
    s.kv_len = max(__ldg(p.kv_lens + b), 0);
    if (p.q_starts == nullptr) {
        s.q0 = (int32_t)b;
        s.q_len = b < p.T ? 1 : 0;
    } else {
        s.q0 = min(max(__ldg(p.q_starts + b), 0), (int32_t)p.T);
        s.q_len = max(min(__ldg(p.q_starts + b + 1), (int32_t)p.T) - s.q0, 0);
    }
    return s;
}

// The page that holds position pos of sequence b, -1 where there is none.
__device__ __forceinline__ int32_t page_of(const PagedBatch &p, uint32_t b, int32_t pos) {
    if (pos < 0 || pos >= p.cap) return -1;
    const int32_t id = __ldg(p.table + (size_t)b * p.table_stride + ((uint32_t)pos >> p.page_shift));
    return (uint32_t)id < p.num_pages ? id : -1;
}

// Index of the row of (page, head, position), in rows.
__device__ __forceinline__ size_t row_index(const PagedBatch &p, int32_t id, uint32_t head, int32_t pos) {
    return (((size_t)id * p.n_kv + head) << p.page_shift) + ((uint32_t)pos & (p.page - 1));
}

// The sequence whose rows t lies in, by a whole warp; B where there is none (rows behind the last sequence).  32 probes a
// round: two rounds for a thousand sequences.
__device__ __forceinline__ uint32_t seq_of(const int32_t *starts, uint32_t B, uint32_t t) {
    const uint32_t lane = lane_id();
    uint32_t lo = 0, n = B + 1;                  // the last entry <= t lies in [lo, lo + n), if there is one
    while (n > 1) {
        const uint32_t step = (n + 31) / 32, i = lo + lane * step;
        const bool below = lane * step < n && __ldg(starts + i) <= (int32_t)t;
        const uint32_t votes = __ballot_sync(kFull, below), hit = votes ? 31 - __clz(votes) : 0;
        n = min(step, n - hit * step);
        lo += hit * step;
    }
    return __ldg(starts + lo) <= (int32_t)t ? lo : B;
}

// Pieces of the prompts' work into l.pieces (all l.count entries), items in several pieces into l.cuts, by `warps` whole warps of which
// this is the first + 0, 1, ...  Lane i of each looks at the i-th share of the sequences.
__device__ __forceinline__ void plan_prompts(const PagedBatch &p, const PromptPlan &l, uint32_t first, uint32_t warps) {
    if (first >= l.count) return;
    const uint32_t B = p.B, lane = lane_id(), per = (B + 31) / 32, b0 = min(lane * per, B), b1 = min(b0 + per, B);
    // items of a sequence and the key tiles of the longest of them, or a few more
    Seq s;
    uint32_t items, tiles, at_b = B;
    auto at = [&](uint32_t b) {
        if (b == at_b) return;
        at_b = b;
        s = load_seq(p, b);
        items = (uint64_t)s.q_len * l.group <= l.min_rows ? 0u : ((uint32_t)s.q_len + l.per_item - 1) / l.per_item;
        uint32_t n = ((uint32_t)min(s.kv_len, p.cap) + kKt - 1) / kKt;
        if (l.window) n = min(n, ((uint32_t)l.sinks + kKt - 1) / kKt + ((uint32_t)l.window + l.per_item) / kKt + 2);    // (below 2^31 each)
        tiles = max(n, 1u);
    };
    float all = 0.f, blocks = 0.f;
    for (uint32_t b = b0; b < b1; ++b) {
        at(b);
        all += (float)items * (float)tiles;
        blocks += (float)items;
    }
    for (int o = 16; o; o >>= 1) {
        all += __shfl_xor_sync(kFull, all, o);
        blocks += __shfl_xor_sync(kFull, blocks, o);
    }
    const float share = all * (float)p.n_kv / (float)l.sms;
    // one more: sums in fp32 may be short of the share by less, where anything is cut (fewer than 2^23 tiles)
    const uint32_t most = max((uint32_t)fminf(blocks * (float)p.n_kv > (float)l.sms ? 0.5f * share : share, 1e9f) + 1, kFewest);
    uint32_t mine = 0, cut = 0;                                  // pieces; slots, and in the upper half cut items
    for (uint32_t b = b0; b < b1; ++b) {
        at(b);
        const uint32_t n = max(tiles / most, 1u);
        mine += items * n;
        if (n > 1) cut += items * n + (items << 16);
    }
    uint32_t end = mine, end_cut = cut;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(kFull, end, o), y = __shfl_up_sync(kFull, end_cut, o);
        if (lane >= (uint32_t)o) {
            end += x;
            end_cut += y;
        }
    }
    if (first == 0 && lane == 31) l.cuts[0] = make_int4((int32_t)(end_cut >> 16), 0, 0, 0);
    for (uint32_t v = first; v < l.count; v += warps) {
        const bool here = end - mine <= v && v < end;
        if (here) {
            uint32_t before = end - mine, slot = end_cut - cut;
            for (uint32_t b = b0; b < b1; ++b) {
                at(b);
                const uint32_t n = max(tiles / most, 1u);
                if (v < before + items * n) {
                    const uint32_t i = (v - before) / n, piece = (v - before) % n;
                    const int4 w0 = make_int4((int32_t)b, (int32_t)(items - 1 - i), (int32_t)piece, (int32_t)n);       // the longest first: they see the most
                    const int4 w1 = make_int4((int32_t)((slot & 0xFFFFu) + i * n), s.q0, s.q_len, s.kv_len);
                    l.pieces[(size_t)v * 2] = w0;
                    l.pieces[(size_t)v * 2 + 1] = w1;
                    if (n > 1 && piece == 0) {
                        int4 *d = l.cuts + (1 + (size_t)(slot >> 16) + i) * 2;
                        d[0] = w0;
                        d[1] = w1;
                    }
                    break;
                }
                before += items * n;
                if (n > 1) slot += items * n + (items << 16);
            }
        }
        if (!__any_sync(kFull, here) && lane == 0) l.pieces[(size_t)v * 2] = make_int4((int32_t)B, 0, 0, 0);
    }
}

// The maximum of a row that has seen nothing, and the least one of a row that has seen scores, though all of them be -infinity or NaN:
// its sum is then 0 or NaN, and the row NaN, as the definition has it.
constexpr float kNone = -INFINITY, kLeast = -3.402823466e38f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lo_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_bf16(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

#endif  // __CUDACC__

int check_paged(const ci_paged_cache *c, const ci_paged_batch *b, PagedBatch &out);
PromptPlan prompt_plan(uint32_t head_dim, uint32_t page_size, uint32_t n_kv, const ci_paged_batch *b, uint32_t group, int32_t window,
                       int32_t sinks, uint32_t min_rows, void *workspace);
size_t prompt_workspace_bytes(uint32_t head_dim, const PromptPlan &l);
int check_paged_prompt(const ci_paged_cache *c, const PromptPlan &l);
int launch_paged_prompt(const ci_paged_cache *c, const PagedBatch &p, const PromptPlan &l, const uint16_t *q, int64_t ldq, uint32_t n_q,
                        float scale_log2, uint16_t *out, int64_t ldo, cudaStream_t s);

}  // namespace ci
