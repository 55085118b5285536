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

__device__ __forceinline__ float lo_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_bf16(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

#endif  // __CUDACC__

int check_paged(const ci_paged_cache *c, const ci_paged_batch *b, PagedBatch &out);
int launch_paged_prompt(const ci_paged_cache *c, const PagedBatch &p, const uint16_t *q, int64_t ldq, uint32_t n_q, int32_t window,
                        int32_t sinks, float scale_log2, uint32_t min_rows, uint16_t *out, int64_t ldo, cudaStream_t s);

}  // namespace ci
