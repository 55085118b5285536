// Attention of new tokens over a paged cache: o_i = sum_j p_ij v_j with p_i = softmax_j(scale q_i . k_j) over the
// positions j <= i that lie in the window (i - j < window) or among the first `sinks`; all of them without a window.
//
// Few queries meet many keys here, so the keys are the long side of the tensor instructions (mma.sync m16n8k16):
//   S^T[16 tokens, 8 queries] = K[16, D] . Q^T[D, 8]        O^T[16 channels, 8 queries] += V^T[16, 16 tokens] . P^T[16, 8]
// Eight queries are the heads that share a key head (and, where a sequence has several new tokens, theirs in turn); keys and
// values go from memory straight into the registers that the instructions read, 16 bytes a lane: a row of K gives a lane
// its k indices in any order as long as Q has the same, a row of V gives channels, and pairs of tokens are put together
// by one byte permute.  P^T comes out of S^T's accumulators by an 8 x 8 transpose between lanes.  Nothing is staged in
// shared memory, no barrier until the warps of a block join their results.
//
// The work of all sequences, key heads and groups of queries is one line of tiles that the blocks share evenly, so that
// one long sequence among short ones, or a single sequence, fills the machine; what a block boundary cuts is joined by
// k_paged_join from (max, sum, output) of the parts.  Lengths are read on the device: a captured call serves any.
//
// What bounds it: in bf16 memory (32 sequences of 1 to 16000 tokens, 251 MB: 49 us, 45 of them this kernel, 5.4 TB/s; it spills in heads
// of 256 alone); heads of 64 and small pages the bytes in flight (67 MB of a window: 18 us of inputs that stay in L2, 22 of others; values
// are asked for where they are used, only keys a tile ahead); 4 bits the instructions that turn codes into operands, 7 for eight keys and
// 11 for eight values beside the permutes, and the latency that 12 warps leave between them (417 MB: 139 us, 3.0 TB/s, integer pipe 60 %
// and issue slots 55 % of the time; four blocks on a multiprocessor 186 us, with one tile at a time 150); a short step its two
// launches and the chain of latencies in each (513 tokens of 32 heads: 10.4 us).
#include "paged.cuh"
#include "ptx.cuh"

namespace ci {

constexpr uint32_t kPaWarps = 4, kPaThreads = kPaWarps * 32;

struct PagedAttnArgs {
    PagedBatch p;
    const uint8_t *k, *v;
    const uint32_t *ks, *vs;
    const uint16_t *q;
    int64_t ldq;                                 // elements between tokens; heads lie D apart
    uint32_t group;
    int32_t window, sinks;                       // window 0: none
    float scale_log2;
    uint32_t max_rows;                           // sequences with more rows (queries x heads of a group) are not this kernel's
    uint16_t *out;
    int64_t ldo;
    int32_t *desc;                               // [blocks][8]: what the join kernel has to do for a block
    float *ml, *partial;                         // [blocks][2][rows][2], [blocks][2][rows][D]
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Rows of queries [RT rt, + RT) of a sequence and the tiles of positions that any of them sees: tile i of `count` starts
// at first(i).
template <int RT, int TILE>
struct Span {
    int32_t p0, p1, hi;                          // positions of the first and last query, end of the visible ones
    int32_t t_lo, n_sink, count;
    __device__ __forceinline__ Span(const PagedAttnArgs &a, const Seq &s, uint32_t rt) {
        const uint32_t rows = (uint32_t)s.q_len * a.group, r0 = rt * RT, r1 = min(rows, r0 + RT) - 1;
        p0 = s.kv_len - s.q_len + (int32_t)(r0 / a.group);
        p1 = s.kv_len - s.q_len + (int32_t)(r1 / a.group);
        hi = max(min(p1 + 1, a.p.cap), 0);
        const int32_t lo = a.window ? min(max(p0 - a.window + 1, 0), hi) : 0;
        t_lo = lo / TILE;
        n_sink = a.window ? min((min(a.sinks, hi) + TILE - 1) / TILE, t_lo) : 0;
        count = n_sink + (hi + TILE - 1) / TILE - t_lo;
    }
    __device__ __forceinline__ int32_t first(int32_t i) const { return (i < n_sink ? i : t_lo + i - n_sink) * TILE; }
};

// What starting on a group of rows and putting its result together costs, in tiles: lengths, queries, page ids, first keys, one
// after the other.  Without it the blocks that get the short sequences of a batch end last (32 sequences of 1 to 16000 tokens, 251 MB:
// 79.2 us with 0, 54.7 with 1, 48.9 with 3, 49.7 with 6).
constexpr uint32_t kItemCost = 3;

// Units of work of a sequence's groups of rows, and the number of those groups.  One group: its own tiles; several: no
// fewer than any of them has.
template <int RT, int TILE>
__device__ __forceinline__ void seq_work(const PagedAttnArgs &a, const Seq &s, uint32_t &groups, uint32_t &units) {
    uint32_t tiles;
    const uint64_t rows = (uint64_t)s.q_len * a.group;
    groups = rows == 0 || rows > a.max_rows ? 0 : (uint32_t)((rows + RT - 1) / RT);
    tiles = 1;
    if (groups == 1) {
        tiles = (uint32_t)max(Span<RT, TILE>(a, s, 0).count, 1);
    } else if (groups > 1) {
        int32_t n = (min(s.kv_len, a.p.cap) + TILE - 1) / TILE;
        if (a.window) n = min(n, (a.sinks + TILE - 1) / TILE + (a.window + (int32_t)((RT - 1) / a.group)) / TILE + 2);
        tiles = (uint32_t)max(n, 1);
    }
    units = tiles + kItemCost;
}

// What a lane holds of 16 tokens: two rows of keys (tokens g and g + 8), four of values (2t, 2t+1, 2t+8, 2t+9).
template <int D, int BITS>
struct Frag;
template <int D>
struct Frag<D, 16> {
    uint4 k[2][D / 32], v[4][D / 64];
};
template <int D>
struct Frag<D, 4> {
    uint32_t k[2][D / 32], v[4][D / 64], ks[2][D / 64], vs[2][D / 64];
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint32_t *p) {
    if (N == 1) w[0] = __ldg(p);
    if (N == 2) { const uint2 x = __ldg(reinterpret_cast<const uint2 *>(p)); w[0] = x.x; w[1] = x.y; }
    if (N >= 4) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p) + i);
            w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
        }
    }
}

constexpr uint32_t kNibbles = 0x000F000Fu, kBase = 0x43004300u;  // bf16 of 128 + c: the code lies in the last four mantissa bits

// Two codes less 8 in bf16.  Values are summed over a whole sequence, where 128 times the sum of the weights would swamp what is
// left of fp32 (outputs of 32000 tokens off by 0.0044 instead of 0.002); the scores' sums are short.
__device__ __forceinline__ uint32_t centred(uint32_t w) {
    const uint32_t x = (w & kNibbles) | kBase;
    uint32_t y;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x43084308u));
    return y;
}

template <int D, int BITS, int NR, int U>
__global__ void __launch_bounds__(kPaThreads, D == 64 ? 4 / NR : D == 128 && NR == 1 ? 3 : 2) k_paged_attention(const __grid_constant__ PagedAttnArgs a) {
    constexpr int RT = 8 * NR, SU = 16 * U, TILE = SU * kPaWarps, G = D / 64, NB = D / 64;
    __shared__ uint64_t s_scan[kPaWarps];
    __shared__ uint64_t s_base;
    __shared__ uint32_t s_b;
    __shared__ float s_m[kPaWarps][RT], s_l[kPaWarps][RT];
    __shared__ __align__(16) float s_o[kPaWarps][RT][D];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t warp = threadIdx.x >> 5, lane = lane_id(), g = lane >> 2, t = lane & 3;
    const PagedBatch &p = a.p;

    // ---- this block's share of the line of tiles --------------------------------------------------------------
    const uint32_t per = (p.B + kPaThreads - 1) / kPaThreads, b0 = min(threadIdx.x * per, p.B), b1 = min(b0 + per, p.B);
    uint64_t mine = 0;
    for (uint32_t b = b0; b < b1; ++b) {
        uint32_t groups, units;
        seq_work<RT, TILE>(a, load_seq(p, b), groups, units);
        mine += (uint64_t)groups * units * p.n_kv;
    }
    uint64_t incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(kFull, incl, o);
        if (lane >= (uint32_t)o) incl += x;
    }
    if (lane == 31) s_scan[warp] = incl;
    if (threadIdx.x == 0) s_b = p.B;
    __syncthreads();
    uint64_t total = 0, before = incl - mine;
    for (uint32_t w = 0; w < kPaWarps; ++w) {
        if (w < warp) before += s_scan[w];
        total += s_scan[w];
    }
    if (threadIdx.x == 0) a.desc[blockIdx.x * 8] = 0;
    const uint64_t blocks = min((uint64_t)gridDim.x, total);    // no block without a tile among those that share an item
    if (blockIdx.x >= blocks) return;
    const uint64_t w0 = total * blockIdx.x / blocks, w1 = total * (blockIdx.x + 1) / blocks;
    if (before <= w0 && w0 < before + mine) {
        for (uint32_t b = b0; b < b1; ++b) {
            uint32_t groups, units;
            seq_work<RT, TILE>(a, load_seq(p, b), groups, units);
            const uint64_t n = (uint64_t)groups * units * p.n_kv;
            if (w0 < before + n) { s_b = b; s_base = before; break; }
            before += n;
        }
    }
    __syncthreads();
    uint32_t b = s_b;
    uint64_t base = s_base;                                     // where sequence b begins in the line

    for (uint64_t w = w0; w < w1;) {
        uint32_t groups, units;
        const Seq s = load_seq(p, b);
        seq_work<RT, TILE>(a, s, groups, units);
        const uint64_t seq_n = (uint64_t)groups * units * p.n_kv;
        if (w >= base + seq_n) {
            base += seq_n;
            ++b;
            continue;
        }
        const uint32_t item = (uint32_t)((w - base) / units), u0 = (uint32_t)((w - base) % units);
        const uint32_t u1 = (uint32_t)min((uint64_t)units, u0 + (w1 - w));
        const uint32_t kvh = item % p.n_kv, rt = item / p.n_kv, rows = (uint32_t)s.q_len * a.group;
        const Span<RT, TILE> sp(a, s, rt);
        const int32_t i0 = max((int32_t)u0 - (int32_t)kItemCost, 0), n_tiles = min((int32_t)u1 - (int32_t)kItemCost, sp.count);

        // ---- queries: the lane's channels of row 8 nr + g --------------------------------------------------------
        uint32_t qf[NR][D / 8];
        int32_t pos[NR][2];                                     // positions of the two rows whose scores this lane gets
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const uint32_t r = rt * RT + nr * 8 + g;
            const uint16_t *src = a.q + (int64_t)(s.q0 + r / a.group) * a.ldq + (size_t)(kvh * a.group + r % a.group) * D;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                uint4 x = make_uint4(0, 0, 0, 0);
                // bf16: chunk t of 32 channels; 4 bits: words 2t and 2t + 1 of the group
                const uint32_t c = BITS == 16 ? i * 32 + t * 8 : (i / 2) * 64 + t * 16 + (i % 2) * 8;
                if (r < rows) x = __ldg(reinterpret_cast<const uint4 *>(src + c));
                qf[nr][4 * i] = x.x; qf[nr][4 * i + 1] = x.y; qf[nr][4 * i + 2] = x.z; qf[nr][4 * i + 3] = x.w;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t rj = rt * RT + nr * 8 + 2 * t + j;
                pos[nr][j] = rj < rows ? s.kv_len - s.q_len + (int32_t)(rj / a.group) : -1;
            }
        }
        float qs[NR][BITS == 4 ? G : 1][2];                     // sums of a row's channels, for the lowest values
        if (BITS == 4) {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    float x = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) x += lo_bf16(qf[nr][8 * gr + i]) + hi_bf16(qf[nr][8 * gr + i]);
                    x += __shfl_xor_sync(kFull, x, 1);
                    x += __shfl_xor_sync(kFull, x, 2);
                    qs[nr][gr][0] = __shfl_sync(kFull, x, 8 * t);
                    qs[nr][gr][1] = __shfl_sync(kFull, x, 8 * t + 4);
                }
        }

        float m[NR][2], l[NR][2], o[NR][NB][4][4], corr[NR][BITS == 4 ? G : 1][2];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            m[nr][0] = m[nr][1] = kLeast;
            l[nr][0] = l[nr][1] = 0.f;
#pragma unroll
            for (int gr = 0; gr < (BITS == 4 ? G : 1); ++gr) corr[nr][gr][0] = corr[nr][gr][1] = 0.f;
#pragma unroll
            for (int x = 0; x < NB * 16; ++x) o[nr][x / 16][x / 4 % 4][x % 4] = 0.f;
        }

        Frag<D, BITS> f[U];
        auto first = [&](int32_t i) { return sp.first(i) + (int32_t)(warp * SU); };
        // Pages of 32 tiles at once, one tile to a lane, and of the 32 after them: no tile waits for its page id.
        auto ask_pages = [&](int32_t i, int32_t (&id)[U]) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int32_t mine = i + (int32_t)lane, tok = mine < n_tiles ? first(mine) + 16 * u : sp.hi;
                id[u] = tok < sp.hi ? __ldg(p.table + (size_t)b * p.table_stride + ((uint32_t)tok >> p.page_shift)) : -1;
            }
        };
        int32_t ids[U], ids_next[U], here[U], page_base = i0;
        uint32_t row[U];                                        // row of the pool of a tile's first token
        auto enter = [&](int32_t i) {                           // tile i is the next to be asked for
            if (i - page_base == 32) {
#pragma unroll
                for (int u = 0; u < U; ++u) ids[u] = ids_next[u];
                page_base = i;
                ask_pages(i + 32, ids_next);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t id = (uint32_t)__shfl_sync(kFull, ids[u], i - page_base);
                here[u] = id < p.num_pages ? 0 : -1;
                row[u] = here[u] ? 0u : ((id * p.n_kv + kvh) << p.page_shift) + ((uint32_t)(first(i) + 16 * u) & (p.page - 1));
            }
        };
        auto load_k = [&]() {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const size_t r = (size_t)row[u] + g;
                    if constexpr (BITS == 16) {
#pragma unroll
                        for (int x = 0; x < D / 32; ++x)
                            f[u].k[j][x] = __ldg(reinterpret_cast<const uint4 *>(a.k + r * D * 2) + j * D + x * 4 + t);      // (8 rows: D chunks)
                    } else {
                        load_words(f[u].k[j], reinterpret_cast<const uint32_t *>(a.k) + r * (D / 8) + t * 2 * G + j * D);
                        load_words(f[u].ks[j], a.ks + r * G + j * 8 * G);
                    }
                }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t r = (size_t)row[u] + 2 * t;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t far = (j & 1) + 8 * (j >> 1);
                    if constexpr (BITS == 16) {
#pragma unroll
                        for (int x = 0; x < NB; ++x)
                            f[u].v[j][x] = __ldg(reinterpret_cast<const uint4 *>(a.v + r * D * 2) + far * (D / 8) + x * 8 + g);
                    } else {
                        load_words(f[u].v[j], reinterpret_cast<const uint32_t *>(a.v) + r * (D / 8) + g * G + far * (D / 8));
                        if (j < 2) load_words(f[u].vs[j], a.vs + ((size_t)row[u] + g + 8 * j) * G);
                    }
                }
            }
        };
        // One tile; all: every row sees all of it, and all of its pages are there.  Pages that are not there were read as page 0.
        auto tile = [&](int32_t i, const bool kAll, const int32_t (&now)[U]) __attribute__((always_inline)) {
            const int32_t tok = first(i);
            // ---- scores ------------------------------------------------------------------------------------------
            float sc[U][NR][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) sc[u][nr][0] = sc[u][nr][1] = sc[u][nr][2] = sc[u][nr][3] = 0.f;
                if constexpr (BITS == 16) {
#pragma unroll
                    for (int x = 0; x < D / 32; ++x) {
                        const uint4 r0 = f[u].k[0][x], r1 = f[u].k[1][x];
                        const uint32_t f0[4] = {r0.x, r1.x, r0.y, r1.y}, f1[4] = {r0.z, r1.z, r0.w, r1.w};
#pragma unroll
                        for (int nr = 0; nr < NR; ++nr) {
                            mma_bf16(sc[u][nr], f0, qf[nr][4 * x], qf[nr][4 * x + 1]);
                            mma_bf16(sc[u][nr], f1, qf[nr][4 * x + 2], qf[nr][4 * x + 3]);
                        }
                    }
                } else {
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        float acc[NR][4] = {};
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t w0r = f[u].k[0][j * G + gr], w1r = f[u].k[1][j * G + gr];
                            const uint32_t f0[4] = {(w0r & kNibbles) | kBase, (w1r & kNibbles) | kBase,
                                                    (w0r >> 4 & kNibbles) | kBase, (w1r >> 4 & kNibbles) | kBase};
                            const uint32_t f1[4] = {(w0r >> 8 & kNibbles) | kBase, (w1r >> 8 & kNibbles) | kBase,
                                                    (w0r >> 12 & kNibbles) | kBase, (w1r >> 12 & kNibbles) | kBase};
#pragma unroll
                            for (int nr = 0; nr < NR; ++nr) {
                                mma_bf16(acc[nr], f0, qf[nr][8 * gr + 4 * j], qf[nr][8 * gr + 4 * j + 1]);
                                mma_bf16(acc[nr], f1, qf[nr][8 * gr + 4 * j + 2], qf[nr][8 * gr + 4 * j + 3]);
                            }
                        }
                        // k = low + step c, and the instructions had 128 + c
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float step = lo_bf16(f[u].ks[j][gr]), low = hi_bf16(f[u].ks[j][gr]) - 128.f * step;
#pragma unroll
                            for (int nr = 0; nr < NR; ++nr) {
                                sc[u][nr][2 * j] += step * acc[nr][2 * j] + low * qs[nr][gr][0];
                                sc[u][nr][2 * j + 1] += step * acc[nr][2 * j + 1] + low * qs[nr][gr][1];
                            }
                        }
                    }
                }
            }
            if (i + 1 < n_tiles) load_k();
            // ---- what is not seen, and the running maximum -------------------------------------------------------
            float mx[NR][2];
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) mx[nr][0] = mx[nr][1] = kNone;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = sc[u][nr][e] * a.scale_log2;
                        if (!kAll) {
                            const int32_t j = tok + 16 * u + (int32_t)g + 8 * (e >> 1), i_pos = pos[nr][e & 1];
                            const bool seen = now[u] == 0 && j <= i_pos && j < sp.hi && (!a.window || j > i_pos - a.window || j < a.sinks);
                            x = seen ? x : kNone;
                        }
                        sc[u][nr][e] = x;
                        mx[nr][e & 1] = fmaxf(mx[nr][e & 1], x);
                    }
            if constexpr (BITS == 16) if (!kAll) {                // 0 times what lies behind a sequence's end need not be 0
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int32_t at = tok + 16 * u + 2 * (int32_t)t + (j & 1) + 8 * (j >> 1);
                        if (now[u] != 0 || at >= sp.hi || (a.window && at <= sp.p0 - a.window && at >= a.sinks))
#pragma unroll
                            for (int x = 0; x < NB; ++x) f[u].v[j][x] = make_uint4(0, 0, 0, 0);
                    }
            }
            bool grown = false;
#pragma unroll
            for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float x = mx[nr][j];
                    x = fmaxf(x, __shfl_xor_sync(kFull, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(kFull, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(kFull, x, 16));
                    mx[nr][j] = fmaxf(x, m[nr][j]);
                    grown |= mx[nr][j] > m[nr][j];
                }
            if (__any_sync(kFull, grown)) {
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float c = ex2(m[nr][j] - mx[nr][j]);
                        m[nr][j] = mx[nr][j];
                        l[nr][j] *= c;
#pragma unroll
                        for (int gr = 0; gr < (BITS == 4 ? G : 0); ++gr) corr[nr][gr][j] *= c;
#pragma unroll
                        for (int x = 0; x < NB * 4; ++x) {
                            o[nr][x / 4][x % 4][j] *= c;
                            o[nr][x / 4][x % 4][2 + j] *= c;
                        }
                    }
            }
            // ---- weights and values ------------------------------------------------------------------------------
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float pr[NR][4];
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        pr[nr][e] = ex2(sc[u][nr][e] - m[nr][e & 1]);
                        l[nr][e & 1] += pr[nr][e];
                    }
                if constexpr (BITS == 16) {
                    // The weights in bf16, the type of the values, which the tensor instructions want alike: half a step of 2^-8
                    // of each, the sums in fp32 (outputs 0.0016 to 0.0021 from 64 bits in the mean, 0.0016 of it their own rounding).
                    uint32_t pb[NR][2];
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr) {
                        pb[nr][0] = transpose8x8(pack_bf16(pr[nr][0], pr[nr][1]));
                        pb[nr][1] = transpose8x8(pack_bf16(pr[nr][2], pr[nr][3]));
                    }
#pragma unroll
                    for (int x = 0; x < NB; ++x) {
                        const uint32_t *v0 = &f[u].v[0][x].x, *v1 = &f[u].v[1][x].x, *v2 = &f[u].v[2][x].x, *v3 = &f[u].v[3][x].x;
#pragma unroll
                        for (int mm = 0; mm < 4; ++mm) {
                            const uint32_t fa[4] = {__byte_perm(v0[mm], v1[mm], 0x5410), __byte_perm(v0[mm], v1[mm], 0x7632),
                                                    __byte_perm(v2[mm], v3[mm], 0x5410), __byte_perm(v2[mm], v3[mm], 0x7632)};
#pragma unroll
                            for (int nr = 0; nr < NR; ++nr) mma_bf16(o[nr][x][mm], fa, pb[nr][0], pb[nr][1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        // v = low + step c = middle + step (c - 8): the step goes with the weight, and what its product loses by
                        // rounding to bf16 counts c - 8 times (outputs 0.0023 from 64 bits in the mean)
                        uint32_t pb[NR][2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float step = lo_bf16(f[u].vs[j][gr]), middle = hi_bf16(f[u].vs[j][gr]) + 8.f * step;
#pragma unroll
                            for (int nr = 0; nr < NR; ++nr) {
                                const float x0 = pr[nr][2 * j], x1 = pr[nr][2 * j + 1];
                                uint32_t y = pack_bf16(x0 * step, x1 * step);
                                if (kAll) {
                                    corr[nr][gr][0] += x0 * middle;
                                    corr[nr][gr][1] += x1 * middle;
                                } else {                        // steps that the row does not see: 0 times them need not be 0
                                    const bool no0 = sc[u][nr][2 * j] == kNone, no1 = sc[u][nr][2 * j + 1] == kNone;
                                    if (no0) y &= 0xFFFF0000u;
                                    if (no1) y &= 0x0000FFFFu;
                                    corr[nr][gr][0] += no0 ? 0.f : x0 * middle;
                                    corr[nr][gr][1] += no1 ? 0.f : x1 * middle;
                                }
                                pb[nr][j] = transpose8x8(y);
                            }
                        }
                        const uint32_t a01 = __byte_perm(f[u].v[0][gr], f[u].v[1][gr], 0x5410);
                        const uint32_t b01 = __byte_perm(f[u].v[0][gr], f[u].v[1][gr], 0x7632);
                        const uint32_t a23 = __byte_perm(f[u].v[2][gr], f[u].v[3][gr], 0x5410);
                        const uint32_t b23 = __byte_perm(f[u].v[2][gr], f[u].v[3][gr], 0x7632);
#pragma unroll
                        for (int mm = 0; mm < 4; ++mm) {
                            const uint32_t fa[4] = {centred(a01 >> 4 * mm), centred(b01 >> 4 * mm), centred(a23 >> 4 * mm), centred(b23 >> 4 * mm)};
#pragma unroll
                            for (int nr = 0; nr < NR; ++nr) mma_bf16(o[nr][gr][mm], fa, pb[nr][0], pb[nr][1]);
                        }
                    }
                }
            }
        };

        if (i0 < n_tiles) {
            ask_pages(i0, ids);
            ask_pages(i0 + 32, ids_next);
            enter(i0);
            load_k();
        }
        for (int32_t i = i0; i < n_tiles; ++i) {
            const int32_t tok = first(i);
            int32_t now[U];
            bool all = tok + SU - 1 <= sp.p0 && (!a.window || tok > sp.p1 - a.window || tok + SU <= a.sinks);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                now[u] = here[u];
                all &= here[u] == 0;
            }
            load_v();
            if (i + 1 < n_tiles) enter(i + 1);
            if (all) tile(i, true, now);
            else tile(i, false, now);
        }

        // ---- the warps' results together -------------------------------------------------------------------------
        __syncthreads();                                        // (the last item's are read)
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float x = l[nr][j];
                x += __shfl_xor_sync(kFull, x, 4);
                x += __shfl_xor_sync(kFull, x, 8);
                x += __shfl_xor_sync(kFull, x, 16);
                if (g == 0) {
                    s_m[warp][nr * 8 + 2 * t + j] = m[nr][j];
                    s_l[warp][nr * 8 + 2 * t + j] = x;
                }
                if constexpr (BITS == 4) {
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        float y = corr[nr][gr][j];
                        y += __shfl_xor_sync(kFull, y, 4);
                        y += __shfl_xor_sync(kFull, y, 8);
                        y += __shfl_xor_sync(kFull, y, 16);
#pragma unroll
                        for (int mm = 0; mm < 4; ++mm) {
                            o[nr][gr][mm][j] += y;
                            o[nr][gr][mm][2 + j] += y;
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < NB; ++x)
#pragma unroll
                    for (int mm = 0; mm < 4; ++mm)
                        *reinterpret_cast<float2 *>(&s_o[warp][nr * 8 + 2 * t + j][x * 64 + 8 * g + 2 * mm]) =
                            make_float2(o[nr][x][mm][j], o[nr][x][mm][2 + j]);
            }
        __syncthreads();
        // Whether a row sees a position of these tiles: asked where it has no weight.
        auto sees = [&](uint32_t row) {
            const int32_t at = s.kv_len - s.q_len + (int32_t)(row / a.group);
            for (int32_t i = i0; i < n_tiles; ++i)
                for (int32_t j0 = sp.first(i), k = 0; k < TILE / 16; ++k, j0 += 16)
                    if (j0 <= at && j0 < sp.hi && (!a.window || min(j0 + 15, at) > at - a.window || j0 < a.sinks) && page_of(p, b, j0) >= 0) return true;
            return false;
        };
        const bool whole = u0 == 0 && u1 == units;
        const uint32_t slot = blockIdx.x * 2 + (u0 == 0 ? 1 : 0);   // the part that begins an item, or one that goes on with it
        for (uint32_t x = threadIdx.x; x < RT * D / 4; x += kPaThreads) {
            const uint32_t r = x / (D / 4), c = x % (D / 4) * 4, row = rt * RT + r;
            float M = kLeast, L = 0.f;
#pragma unroll
            for (uint32_t w4 = 0; w4 < kPaWarps; ++w4) M = fmaxf(M, s_m[w4][r]);
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (uint32_t w4 = 0; w4 < kPaWarps; ++w4) {
                if (s_l[w4][r] == 0.f) continue;                // (values that the row does not see may have left a NaN)
                const float e = ex2(s_m[w4][r] - M);
                const float4 z = *reinterpret_cast<const float4 *>(&s_o[w4][r][c]);
                L += e * s_l[w4][r];
                y.x += e * z.x; y.y += e * z.y; y.z += e * z.z; y.w += e * z.w;
            }
            if (L == 0.f && !(row < rows && sees(row))) M = kNone;
            if (whole) {
                if (row < rows) {
                    const float inv = M == kNone ? 0.f : 1.f / L;
                    *reinterpret_cast<uint2 *>(a.out + (int64_t)(s.q0 + row / a.group) * a.ldo + (size_t)(kvh * a.group + row % a.group) * D + c) =
                        make_uint2(pack_bf16(y.x * inv, y.y * inv), pack_bf16(y.z * inv, y.w * inv));
                }
            } else {
                *reinterpret_cast<float4 *>(a.partial + ((size_t)slot * RT + r) * D + c) = y;
                if (c == 0) *reinterpret_cast<float2 *>(a.ml + ((size_t)slot * RT + r) * 2) = make_float2(M, L);
            }
        }
        if (u0 == 0 && !whole && threadIdx.x == 0) {            // this block begins an item that others end
            const uint64_t last = base + (uint64_t)(item + 1) * units - 1;
            const uint64_t owner = ((last + 1) * blocks - 1) / total;
            int32_t *d = a.desc + blockIdx.x * 8;
            d[0] = (int32_t)(owner - blockIdx.x + 1);
            d[1] = s.q0;
            d[2] = (int32_t)rows;
            d[3] = (int32_t)(rt * RT);
            d[4] = (int32_t)kvh;
        }
        w += u1 - u0;
    }
}

// Joins the parts of an item that several blocks had: block c has the item that block c of the attention began, all rows at once, if
// that has few parts.  Items of many parts are few, and the blocks share their rows: a block per row, its threads over the
// parts (a step of 5 sequences of 20000 tokens, eight heads of 256 over one, 59 parts each: 36.4 us, 42.2 without).  Everything in a
// fixed order: the same sum every time.
constexpr int32_t kFewParts = 16, kAtOnce = 8;

template <int D, int RT>
__global__ void __launch_bounds__(256) k_paged_join(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ PromptPlan plan) {
    constexpr uint32_t kLanes = D / 4, kShares = 256 / kLanes;  // threads of a row, and such rows of threads
    __shared__ __align__(16) float4 s_y[kShares][kLanes];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    auto slot = [&](uint32_t c, int32_t i) { return (size_t)(c + i) * 2 + (i == 0 ? 1 : 0); };
    auto store = [&](const int4 &head, int32_t kvh, uint32_t row, uint32_t c, const float4 &y, float inv) {
        *reinterpret_cast<uint2 *>(a.out + (int64_t)(head.y + (int32_t)(row / a.group)) * a.ldo + (size_t)(kvh * a.group + row % a.group) * D + c) =
            make_uint2(pack_bf16(y.x * inv, y.y * inv), pack_bf16(y.z * inv, y.w * inv));
    };
    uint32_t rows_here = 0;                                     // of items of many parts: a bit per row
    {
        int32_t n[RT];
#pragma unroll
        for (uint32_t k = 0; k < RT; ++k) n[k] = __ldcg(a.desc + (blockIdx.x + k * gridDim.x) / RT * 8);
#pragma unroll
        for (uint32_t k = 0; k < RT; ++k) rows_here |= n[k] > kFewParts ? 1u << k : 0u;
    }
    if (plan.count) plan_prompts(a.p, plan, blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8);
    const int32_t *d = a.desc + blockIdx.x * 8;
    const int4 head = __ldcg(reinterpret_cast<const int4 *>(d));
    if (head.x > 0 && head.x <= kFewParts) {
        const int32_t parts = head.x, kvh = __ldcg(d + 4);
#pragma unroll 1
        for (uint32_t x = threadIdx.x; x < RT * kLanes; x += 256) {
            const uint32_t r = x / kLanes, c = x % kLanes * 4, row = (uint32_t)head.w + r;
            if ((int32_t)row >= head.z) continue;
            float M = kNone, L = 0.f;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int32_t i0 = 0; i0 < parts; i0 += kAtOnce) {
                float2 ml[kAtOnce];                             // asked for together: (max, sum) and outputs
                float4 z[kAtOnce];
#pragma unroll
                for (int32_t i = 0; i < kAtOnce; ++i) {
                    ml[i] = make_float2(kNone, 0.f);
                    z[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (i0 + i < parts) {
                        ml[i] = __ldcg(reinterpret_cast<const float2 *>(a.ml + (slot(blockIdx.x, i0 + i) * RT + r) * 2));
                        z[i] = __ldcg(reinterpret_cast<const float4 *>(a.partial + (slot(blockIdx.x, i0 + i) * RT + r) * D + c));
                    }
                }
                float most = M;
#pragma unroll
                for (int32_t i = 0; i < kAtOnce; ++i) most = fmaxf(most, ml[i].x);
                if (most == kNone) continue;
                const float down = M == kNone ? 0.f : ex2(M - most);
                M = most;
                L *= down;
                y.x *= down; y.y *= down; y.z *= down; y.w *= down;
#pragma unroll
                for (int32_t i = 0; i < kAtOnce; ++i) {
                    const float e = ml[i].x == kNone ? 0.f : ex2(ml[i].x - M);
                    L += e * ml[i].y;
                    y.x += e * z[i].x; y.y += e * z[i].y; y.z += e * z[i].z; y.w += e * z[i].w;
                }
            }
            store(head, kvh, row, c, y, M == kNone ? 0.f : 1.f / L);
        }
    }
    for (; rows_here; rows_here &= rows_here - 1) {
        const uint32_t u = blockIdx.x + (__ffs(rows_here) - 1) * gridDim.x, c = u / RT, r = u % RT;
        const int4 h = __ldcg(reinterpret_cast<const int4 *>(a.desc + c * 8));
        const uint32_t row = (uint32_t)h.w + r;
        if ((int32_t)row >= h.z) continue;
        const int32_t parts = h.x, kvh = __ldcg(a.desc + c * 8 + 4);
        const uint32_t lane = lane_id();
        float M = kNone, L = 0.f;                               // in every warp: lane l has parts l, l + 32, ...
        const float2 mine = (int32_t)lane < parts ? __ldcg(reinterpret_cast<const float2 *>(a.ml + (slot(c, lane) * RT + r) * 2)) : make_float2(kNone, 0.f);
        M = mine.x;
#pragma unroll 4
        for (int32_t i = lane + 32; i < parts; i += 32) M = fmaxf(M, __ldcg(a.ml + (slot(c, i) * RT + r) * 2));
        for (uint32_t o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(kFull, M, o));
        const float safe = M == kNone ? 0.f : M;
        L = mine.x == kNone ? 0.f : ex2(mine.x - safe) * mine.y;
#pragma unroll 4
        for (int32_t i = lane + 32; i < parts; i += 32) {
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(a.ml + (slot(c, i) * RT + r) * 2));
            L += ml.x == kNone ? 0.f : ex2(ml.x - safe) * ml.y;
        }
        for (uint32_t o = 16; o; o >>= 1) L += __shfl_xor_sync(kFull, L, o);
        const uint32_t at = threadIdx.x % kLanes, share = threadIdx.x / kLanes;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int32_t i = share; i < parts; i += kShares) {
            const float m = __ldcg(a.ml + (slot(c, i) * RT + r) * 2);
            const float4 z = __ldcg(reinterpret_cast<const float4 *>(a.partial + (slot(c, i) * RT + r) * D + at * 4));
            const float e = m == kNone ? 0.f : ex2(m - safe);
            y.x += e * z.x; y.y += e * z.y; y.z += e * z.z; y.w += e * z.w;
        }
        __syncthreads();                                        // (the last row's are read)
        s_y[share][at] = y;
        __syncthreads();
        if (threadIdx.x < kLanes) {
#pragma unroll
            for (uint32_t j = 1; j < kShares; ++j) {
                const float4 z = s_y[j][at];
                y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
            }
            store(h, kvh, row, at * 4, y, M == kNone ? 0.f : 1.f / L);
        }
    }
}

constexpr uint32_t kPaMaxRows = 16;              // widest group of query rows of any variant
// Query rows of a sequence and key head up to which this kernel has them.  24 drawn batches of 6 to 120 rows over 250 to 12000
// tokens: up to 32 rows 8 % slower in the mean, 16 21 %, 8 31 %; 128 13 % faster (0.44 to 1.01 of the time).
constexpr uint32_t kPaRows = 64;
constexpr uint32_t kPaMaxResident = 4;           // blocks of a multiprocessor that the workspace has room for

// As many blocks as fit on the device at once: a block more would start when the others have ended.
static int resident_blocks(const void *kernel, uint32_t &blocks) {
    int n = 0;
    CI_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, (int)kPaThreads, 0));
    blocks = n < 1 ? 1u : n > (int)kPaMaxResident ? kPaMaxResident : (uint32_t)n;
    return CI_OK;
}

template <int D, int BITS, int NR>
static int launch_attention(const PagedAttnArgs &a, const PromptPlan &plan, cudaStream_t s) {
    // 4 bits: two tiles of 16 tokens at once; heads of 256 have no registers for that (32 sequences of 100 to 700 tokens 22.4 us with
    // two, 17.8 with one; four of 38000 86.5 and 87.5).  bf16 heads of 64: 23.4 us with two where one takes 18.1.
    constexpr int U = BITS == 4 && D < 256 ? 2 : 1;
    static uint32_t resident = 0;
    if (resident == 0)
        if (int rc = resident_blocks((const void *)k_paged_attention<D, BITS, NR, U>, resident)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((uint32_t)sm_count() * resident);
    cfg.blockDim = dim3(kPaThreads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CI_CUDA(cudaLaunchKernelEx(&cfg, k_paged_attention<D, BITS, NR, U>, a));
    cfg.blockDim = dim3(256);
    CI_CUDA(cudaLaunchKernelEx(&cfg, k_paged_join<D, 8 * NR>, a, plan));
    return CI_OK;
}

template <int D>
static int launch_attention_bits(const PagedAttnArgs &a, const PromptPlan &plan, uint32_t bits, bool wide, cudaStream_t s) {
    if constexpr (D <= 128) {
        if (wide) return bits == 16 ? launch_attention<D, 16, 2>(a, plan, s) : launch_attention<D, 4, 2>(a, plan, s);
    }
    return bits == 16 ? launch_attention<D, 16, 1>(a, plan, s) : launch_attention<D, 4, 1>(a, plan, s);
}

static size_t few_bytes(uint32_t head_dim) {
    const size_t blocks = (size_t)sm_count() * kPaMaxResident;
    return blocks * 8 * sizeof(int32_t) + blocks * 2 * kPaMaxRows * (2 + (size_t)head_dim) * sizeof(float);
}
static uint64_t longest_of(const ci_paged_batch *b, uint32_t max_q_len) {
    return b->q_starts == nullptr ? 1 : max_q_len && max_q_len < b->T ? max_q_len : b->T;
}
// Sequences of many new tokens go to the tensor cores' kernel, the others to this one; both look at every sequence.
static bool has_prompts(const ci_paged_batch *b, uint32_t group, uint32_t max_q_len) {
    return b->q_starts != nullptr && longest_of(b, max_q_len) * group > kPaRows && group <= 128;
}

}  // namespace ci

using namespace ci;

extern "C" {

size_t ci_paged_attention_workspace_bytes(const ci_paged_cache *c, const ci_paged_batch *batch, uint32_t n_q, uint32_t max_q_len) {
    if (c == nullptr || batch == nullptr || c->n_kv == 0) return 0;
    const size_t few = few_bytes(c->head_dim);
    const uint32_t group = n_q / c->n_kv;
    if (group == 0 || !has_prompts(batch, group, max_q_len)) return few;
    return few + prompt_workspace_bytes(c->head_dim, prompt_plan(c->head_dim, c->page_size, c->n_kv, batch, group, 0, 0, kPaRows, nullptr));
}

int ci_paged_attention(const ci_paged_cache *c, const ci_paged_batch *batch, const uint16_t *d_q, int64_t ldq, uint32_t n_q,
                       uint32_t max_q_len, uint32_t window, uint32_t sinks, float scale, void *d_workspace, size_t workspace_bytes,
                       uint16_t *d_out, int64_t ldo, ci_stream_t stream) {
    PagedAttnArgs a;
    if (int rc = check_paged(c, batch, a.p)) return rc;
    CI_REQUIRE(d_q && d_out, "null pointer");
    CI_REQUIRE(n_q > 0 && n_q <= 65535 && n_q % c->n_kv == 0, "%u query heads over %u key/value heads", n_q, c->n_kv);
    CI_REQUIRE(((reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_out)) & 15u) == 0 && ldq % 8 == 0 && ldo % 8 == 0,
               "queries and output must be 16-byte aligned");
    CI_REQUIRE((uint64_t)a.p.T * n_q <= 0x7FFFFFFFu, "%u tokens of %u query heads", a.p.T, n_q);
    CI_REQUIRE(isfinite(scale * 1.4427f), "a scale of %g", scale);
    if (a.p.T == 0 || a.p.B == 0) return CI_OK;
    CI_REQUIRE(d_workspace != nullptr && (reinterpret_cast<uintptr_t>(d_workspace) & 15u) == 0, "attention needs an aligned workspace");
    const size_t need = ci_paged_attention_workspace_bytes(c, batch, n_q, max_q_len);
    if (workspace_bytes < need) {
        set_error("attention workspace of %zu bytes, %zu needed", workspace_bytes, need);
        return CI_E_WORKSPACE;
    }
    a.k = (const uint8_t *)c->k; a.v = (const uint8_t *)c->v; a.ks = c->k_scale; a.vs = c->v_scale;
    a.q = d_q;
    a.ldq = ldq;
    a.group = n_q / c->n_kv;
    constexpr uint32_t kFar = 1u << 30;                         // further than any position lies
    a.window = (int32_t)(window >= kFar ? 0 : window);
    a.sinks = (int32_t)(sinks >= kFar ? kFar : sinks);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.out = d_out;
    a.ldo = ldo;
    const size_t blocks = (size_t)sm_count() * kPaMaxResident;
    a.desc = (int32_t *)d_workspace;
    a.ml = (float *)(a.desc + blocks * 8);
    a.partial = a.ml + blocks * 2 * kPaMaxRows * 2;
    const bool prompts = has_prompts(batch, a.group, max_q_len);
    a.max_rows = prompts ? kPaRows : 0xFFFFFFFFu;
    PromptPlan plan = {};
    if (prompts) {
        plan = prompt_plan(c->head_dim, c->page_size, c->n_kv, batch, a.group, a.window, a.sinks, kPaRows, (uint8_t *)d_workspace + few_bytes(c->head_dim));
        if (int rc = check_paged_prompt(c, plan)) return rc;
    }
    const bool wide = longest_of(batch, max_q_len) * a.group > 8;
    cudaStream_t s = (cudaStream_t)stream;
    const int rc = c->head_dim == 64    ? launch_attention_bits<64>(a, plan, c->bits, wide, s)
                   : c->head_dim == 128 ? launch_attention_bits<128>(a, plan, c->bits, wide, s)
                                        : launch_attention_bits<256>(a, plan, c->bits, wide, s);
    if (rc != CI_OK || !prompts) return rc;
    return launch_paged_prompt(c, a.p, plan, d_q, ldq, n_q, a.scale_log2, d_out, ldo, s);
}

}  // extern "C"
