// New tokens into a paged cache, and a cache's rows back out of it.
#include "paged.cuh"

namespace ci {

int check_paged(const ci_paged_cache *c, const ci_paged_batch *b, PagedBatch &o) {
    CI_REQUIRE(c && b, "null descriptor");
    CI_REQUIRE(c->k && c->v, "null pages");
    CI_REQUIRE(c->bits == 16 || c->bits == 4, "a cache of %u bits; 16 or 4", c->bits);
    CI_REQUIRE(c->bits == 16 || (c->k_scale && c->v_scale), "a cache of 4 bits needs its steps and lowest values");
    CI_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "head dimension %u must be 64, 128 or 256", c->head_dim);
    CI_REQUIRE(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128,
               "pages of %u tokens; 16, 32, 64 or 128", c->page_size);
    CI_REQUIRE(c->num_pages > 0 && c->num_pages <= 0x7FFFFFFFu && c->n_kv > 0 && c->n_kv <= 65535, "empty or too large a cache");
    CI_REQUIRE((uint64_t)c->num_pages * c->n_kv * c->page_size <= 0xFFFFFF00u, "a pool of more than 2^32 rows");
    CI_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) | reinterpret_cast<uintptr_t>(c->k_scale) |
                 reinterpret_cast<uintptr_t>(c->v_scale)) & 15u) == 0, "pages must be 16-byte aligned");
    CI_REQUIRE(b->B == 0 || ((b->block_table || b->max_pages == 0) && b->kv_lens), "null block table or lengths");
    CI_REQUIRE(b->B <= (1u << 20) && b->T <= (1u << 30), "%u sequences with %u new tokens", b->B, b->T);
    CI_REQUIRE((uint64_t)b->max_pages * c->page_size <= (1u << 30), "a block table of %u pages of %u tokens", b->max_pages, c->page_size);
    CI_REQUIRE(b->table_stride >= b->max_pages, "block table rows of %u pages %u apart", b->max_pages, b->table_stride);
    o.table = b->block_table;
    o.kv_lens = b->kv_lens;
    o.q_starts = b->q_starts;
    o.num_pages = c->num_pages;
    o.page = c->page_size;
    o.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    o.n_kv = c->n_kv;
    o.table_stride = b->table_stride;
    o.B = b->B;
    o.T = b->T;
    o.cap = (int32_t)(b->max_pages * c->page_size);
    return CI_OK;
}

struct AppendArgs {
    PagedBatch p;
    const uint16_t *q, *k, *v, *cos_t, *sin_t;
    int64_t ldq, ldk, ldv;
    uint32_t n_q, table_len, vec, parts;
    uint16_t *q_out;
    uint8_t *kc, *vc;
    uint32_t *ks, *vs;
};

// Eight neighbouring channels; vec: the address is 16-byte aligned.
__device__ __forceinline__ uint4 load8(const uint16_t *p, uint32_t vec) {
    if (vec) return __ldg(reinterpret_cast<const uint4 *>(p));
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __ldg(p + 2 * j) | (uint32_t)__ldg(p + 2 * j + 1) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void unpack(const uint4 &v, float (&f)[8]) {
    f[0] = lo_bf16(v.x); f[1] = hi_bf16(v.x); f[2] = lo_bf16(v.y); f[3] = hi_bf16(v.y);
    f[4] = lo_bf16(v.z); f[5] = hi_bf16(v.z); f[6] = lo_bf16(v.w); f[7] = hi_bf16(v.w);
}
__device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}

// The (step, lowest) of a group from its extremes.  NaN among the values: fminf and fmaxf pass it over, so it is handed on in
// `bad` and makes the group NaN.
__device__ __forceinline__ uint32_t scale_word(float lo, float hi, bool bad) {
    const float step = bad ? __uint_as_float(0x7FC00000u) : __fdiv_rn(__fsub_rn(hi, lo), 15.f);
    return pack_bf16(step, lo);
}
// Eight codes round((x - lowest) / step).  The quotient by a reciprocal is within 2^-18 of the division's, which decides but next to
// a half; there the division itself is made.  (max - lowest) / step is below 15.5, the step being off by 2^-8 at most: no code
// needs a limit.
__device__ __forceinline__ uint32_t code_word(const float (&f)[8], uint32_t scale) {
    const float step = lo_bf16(scale), low = hi_bf16(scale), inv = __frcp_rn(step);
    constexpr float kRound = 12582912.f;                        // 1.5 * 2^23: the sum's last bits are the rounded quotient
    if (!(step > 0.f && step < 3.3e38f && inv < 3.3e38f)) {     // one value, none that is finite, or one whose reciprocal is not
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = step > 0.f ? rintf(__fdiv_rn(__fsub_rn(f[i], low), step)) : 0.f;
            w |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * (i / 2) + 16 * (i % 2));
        }
        return w;
    }
    uint32_t w = 0;
    bool near_half = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = __fsub_rn(f[i], low) * inv, r = __fadd_rn(q, kRound);
        near_half |= fabsf(fabsf(q - __fsub_rn(r, kRound)) - 0.5f) < 1e-5f;
        w |= (__float_as_uint(r) & 15u) << (4 * (i / 2) + 16 * (i % 2));
    }
    if (near_half) {
        w = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w |= (__float_as_uint(__fadd_rn(__fdiv_rn(__fsub_rn(f[i], low), step), kRound)) & 15u) << (4 * (i / 2) + 16 * (i % 2));
    }
    return w;
}

// A warp's token and the share of its heads that it has: tokens of few have several warps.
struct TokenPart {
    uint32_t t, part;
    __device__ __forceinline__ explicit TokenPart(uint32_t parts) {
        const uint32_t w = blockIdx.x * 8 + (threadIdx.x >> 5);
        t = w / parts;
        part = w % parts;
    }
};

// A warp has a token, or a share of its heads: its sequence, place, page and angles are looked up once for all of them.  A head takes
// D / 16 lanes: a lane has eight channels of its lower half and the eight that are rotated with them.  Groups of 64 channels
// lie in eight lanes (four of them, both halves, for D = 64).  Two rounds of heads are in flight.  7100 tokens of 32 + 8 + 8
// heads of 128: 35 us, 5.1 TB/s: memory.  Into 4 bits, 8500 tokens: 53 us, 2.8 TB/s, neither memory nor a pipe (integers 40 %, issue slots
// 57 %): latency, with three blocks of 80 registers on a multiprocessor (two take 58).  The angles are 32 of those registers in fp32; all
// variants spill 28 to 44 bytes a thread.
template <int D, int BITS>
__global__ void __launch_bounds__(256, BITS == 16 ? 4 : 3) k_rope_append(const __grid_constant__ AppendArgs a) {
    constexpr uint32_t LANES = D / 16, G = D / kGroup, PER = 32 / LANES, FLIGHT = 2;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const TokenPart tp(a.parts);
    const uint32_t t = tp.t, lane = lane_id();
    if (t >= a.p.T) return;
    const uint32_t b = a.p.q_starts ? seq_of(a.p.q_starts, a.p.B, t) : t;
    if (b >= a.p.B) return;                                     // behind the last sequence
    const Seq s = load_seq(a.p, b);
    const int32_t pos = s.kv_len - s.q_len + ((int32_t)t - s.q0);
    const bool there = pos >= 0 && (uint32_t)pos < a.table_len;
    const uint32_t c = (lane % LANES) * 8, n_kv = a.p.n_kv, heads = a.n_q + 2 * n_kv;
    const int32_t id = there ? page_of(a.p, b, pos) : -1;
    const uint32_t row0 = id >= 0 ? (uint32_t)row_index(a.p, id, 0, pos) : 0;       // head 0's; the others' lie a page apart
    float c0[8], c1[8], s0[8], s1[8];
    if (there) {
        const uint16_t *ct = a.cos_t + (size_t)pos * D + c, *st = a.sin_t + (size_t)pos * D + c;
        unpack(load8(ct, a.vec), c0);
        unpack(load8(ct + D / 2, a.vec), c1);
        unpack(load8(st, a.vec), s0);
        unpack(load8(st + D / 2, a.vec), s1);
    }
    for (uint32_t first = tp.part * PER; first < heads; first += a.parts * PER * FLIGHT) {
        uint4 xl[FLIGHT], xh[FLIGHT];
#pragma unroll
        for (uint32_t k = 0; k < FLIGHT; ++k) {
            const uint32_t unit = first + k * a.parts * PER + lane / LANES;
            xl[k] = xh[k] = make_uint4(0, 0, 0, 0);
            if (unit < heads && there) {
                const uint32_t head = unit < a.n_q ? unit : unit < a.n_q + n_kv ? unit - a.n_q : unit - a.n_q - n_kv;
                const uint16_t *src = (unit < a.n_q ? a.q + (int64_t)t * a.ldq : unit < a.n_q + n_kv ? a.k + (int64_t)t * a.ldk : a.v + (int64_t)t * a.ldv) + head * D + c;
                xl[k] = load8(src, a.vec);
                xh[k] = load8(src + D / 2, a.vec);
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < FLIGHT; ++k) {
            const uint32_t unit = first + k * a.parts * PER + lane / LANES;
            if (first + k * a.parts * PER >= heads) break;      // (the whole warp)
            const bool live = unit < heads, is_q = unit < a.n_q, is_v = unit >= a.n_q + n_kv;
            const uint32_t head = is_q ? unit : is_v ? unit - a.n_q - n_kv : unit - a.n_q;
            uint4 wl = xl[k], wh = xh[k];
            if (!is_v && there) {
                float lo[8], hi[8];
                unpack(wl, lo);
                unpack(wh, hi);
#pragma unroll
                for (int i = 0; i < 8; ++i) {                   // products of two bf16 are exact in fp32: one rounding each
                    const float x = lo[i], y = hi[i];
                    lo[i] = x * c0[i] - y * s0[i];
                    hi[i] = y * c1[i] + x * s1[i];
                }
                wl = pack(lo);
                wh = pack(hi);
            }
            if (live && is_q) {
                uint4 *dst = reinterpret_cast<uint4 *>(a.q_out + ((size_t)t * a.n_q + head) * D + c);
                dst[0] = wl;
                dst[D / 16] = wh;
            }
            const bool keep = live && !is_q && id >= 0;
            const size_t row = (size_t)row0 + (keep ? head << a.p.page_shift : 0);
            if (BITS == 16) {
                if (!keep) continue;
                uint4 *dst = reinterpret_cast<uint4 *>((is_v ? a.vc : a.kc) + (row * D + c) * 2);
                dst[0] = wl;
                dst[D / 16] = wh;
            } else {
                if (!__any_sync(kFull, keep)) continue;
                float lo[8], hi[8];
                unpack(wl, lo);                                 // the cache in bf16 and the one in 4 bits hold the same keys
                unpack(wh, hi);
                float mn[2] = {lo[0], hi[0]}, mx[2] = {lo[0], hi[0]};
                bool bad[2] = {false, false};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    mn[0] = fminf(mn[0], lo[i]); mx[0] = fmaxf(mx[0], lo[i]); bad[0] |= lo[i] != lo[i];
                    mn[1] = fminf(mn[1], hi[i]); mx[1] = fmaxf(mx[1], hi[i]); bad[1] |= hi[i] != hi[i];
                }
                if (G == 1) {
                    mn[0] = mn[1] = fminf(mn[0], mn[1]);
                    mx[0] = mx[1] = fmaxf(mx[0], mx[1]);
                    bad[0] = bad[1] = bad[0] | bad[1];
                }
                constexpr uint32_t SPAN = G == 1 ? 4 : 8;       // lanes of a group
                uint32_t scale[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (G == 1 && h == 1) { scale[1] = scale[0]; break; }
                    for (uint32_t o = SPAN / 2; o; o >>= 1) {
                        mn[h] = fminf(mn[h], __shfl_xor_sync(kFull, mn[h], o));
                        mx[h] = fmaxf(mx[h], __shfl_xor_sync(kFull, mx[h], o));
                    }
                    const uint32_t votes = __ballot_sync(kFull, bad[h]), mask = (SPAN == 8 ? 0xFFu : 0xFu) << (lane & ~(SPAN - 1));
                    scale[h] = scale_word(mn[h], mx[h], votes & mask);
                }
                if (!keep) continue;
                uint32_t *dst = reinterpret_cast<uint32_t *>(is_v ? a.vc : a.kc) + row * (D / 8);
                uint32_t *sc = (is_v ? a.vs : a.ks) + row * G;
                const uint32_t g0 = G == 1 ? 0 : c / kGroup, g1 = G == 1 ? 0 : g0 + G / 2;
                const uint32_t w0 = c % kGroup / 8, w1 = G == 1 ? w0 + 4 : w0;
                dst[w0 * G + g0] = code_word(lo, scale[0]);
                dst[w1 * G + g1] = code_word(hi, scale[1]);
                if (c % kGroup == 0) {
                    sc[g0] = scale[0];
                    if (G > 1) sc[g1] = scale[1];
                }
            }
        }
    }
}

struct GatherArgs {
    PagedBatch p;
    const uint8_t *kc, *vc;
    const uint32_t *ks, *vs;
    uint16_t *k_out, *v_out;
    uint32_t parts;
};

// Rows of a cache as bf16, a token, or a share of its heads, per warp: a row takes D / 8 lanes, 16 bytes to each; positions without a page
// give zeros.  23 thousand tokens of 8 heads of 128 out of 4 bits, 123 MB: 33 us, 3.8 TB/s (integers 54 %, issue slots 57 %, loads
// under way); 8 thousand out of bf16, 69 MB that stay in L2: 9 us.
template <int D, int BITS>
__global__ void __launch_bounds__(256) k_paged_gather(const __grid_constant__ GatherArgs a) {
    constexpr uint32_t LANES = D / 8, G = D / kGroup, PER = 32 / LANES;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const TokenPart tp(a.parts);
    const uint32_t t = tp.t, lane = lane_id(), c8 = lane % LANES, n_kv = a.p.n_kv;
    if (t >= a.p.T) return;
    const uint32_t b = a.p.q_starts ? seq_of(a.p.q_starts, a.p.B, t) : t;
    if (b >= a.p.B) return;
    const Seq s = load_seq(a.p, b);
    const int32_t pos = s.kv_len - s.q_len + ((int32_t)t - s.q0), id = page_of(a.p, b, pos);
    const uint32_t row0 = id >= 0 ? (uint32_t)row_index(a.p, id, 0, pos) : 0;
#pragma unroll 4
    for (uint32_t unit = tp.part * PER + lane / LANES; unit < 2 * n_kv; unit += a.parts * PER) {
        const bool is_v = unit >= n_kv;
        const uint32_t head = is_v ? unit - n_kv : unit;
        uint4 o = make_uint4(0, 0, 0, 0);
        if (id >= 0) {
            const size_t row = (size_t)row0 + (head << a.p.page_shift);
            if (BITS == 16) {
                o = __ldg(reinterpret_cast<const uint4 *>((is_v ? a.vc : a.kc) + row * D * 2) + c8);
            } else {
                const uint32_t g = c8 / 8, w = __ldg(reinterpret_cast<const uint32_t *>(is_v ? a.vc : a.kc) + row * (D / 8) + (c8 % 8) * G + g);
                const uint32_t sc = __ldg((is_v ? a.vs : a.ks) + row * G + g);
                const float step = lo_bf16(sc), low = hi_bf16(sc);
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {                   // the code where it lies in the mantissa of 2^23, and the step by as much less
                    const int at = 4 * (i / 2);
                    const float c = __uint_as_float(((i % 2 ? w >> 16 : w) & 15u << at) | 0x4B000000u) - 8388608.f;
                    f[i] = step * (1.f / (1 << at)) * c + low;  // all exact but the sum
                }
                o = pack(f);
            }
        }
        *reinterpret_cast<uint4 *>((is_v ? a.v_out : a.k_out) + ((size_t)t * n_kv + head) * D + c8 * 8) = o;
    }
}

// Warps per token: one where there are tokens enough for 16 to a multiprocessor, at most one for each round of heads.
static uint32_t warps_per_token(uint32_t T, uint32_t rounds) {
    const uint32_t want = ((uint32_t)sm_count() * 16 + T - 1) / T;
    return want < 1 ? 1 : want > rounds ? rounds : want;
}

template <typename Args>
static int launch_tokens(void (*kernel)(Args), const Args &args, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((uint64_t)args.p.T * args.parts + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CI_CUDA(cudaLaunchKernelEx(&cfg, kernel, args));
    return CI_OK;
}

}  // namespace ci

using namespace ci;

extern "C" {

int ci_rope_paged_append(const ci_paged_cache *c, const ci_paged_batch *batch, const uint16_t *d_q, int64_t ldq, const uint16_t *d_k,
                         int64_t ldk, const uint16_t *d_v, int64_t ldv, uint32_t n_q, const uint16_t *d_cos, const uint16_t *d_sin,
                         uint32_t table_len, uint16_t *d_q_out, ci_stream_t stream) {
    AppendArgs a;
    if (int rc = check_paged(c, batch, a.p)) return rc;
    CI_REQUIRE(d_q && d_k && d_v && d_cos && d_sin && d_q_out, "null pointer");
    CI_REQUIRE(n_q > 0 && n_q <= 65535, "%u query heads", n_q);
    CI_REQUIRE((reinterpret_cast<uintptr_t>(d_q_out) & 15u) == 0, "the rotated queries must be 16-byte aligned");
    if (a.p.T == 0 || a.p.B == 0) return CI_OK;
    a.q = d_q; a.k = d_k; a.v = d_v; a.cos_t = d_cos; a.sin_t = d_sin;
    a.ldq = ldq; a.ldk = ldk; a.ldv = ldv;
    a.n_q = n_q;
    a.table_len = table_len;
    a.q_out = d_q_out;
    a.kc = (uint8_t *)c->k; a.vc = (uint8_t *)c->v; a.ks = c->k_scale; a.vs = c->v_scale;
    a.vec = ((reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v) |
              reinterpret_cast<uintptr_t>(d_cos) | reinterpret_cast<uintptr_t>(d_sin)) & 15u) == 0 &&
            ldq % 8 == 0 && ldk % 8 == 0 && ldv % 8 == 0;
    void (*kernel)(AppendArgs) =
        c->bits == 16 ? (c->head_dim == 64 ? k_rope_append<64, 16> : c->head_dim == 128 ? k_rope_append<128, 16> : k_rope_append<256, 16>)
                      : (c->head_dim == 64 ? k_rope_append<64, 4> : c->head_dim == 128 ? k_rope_append<128, 4> : k_rope_append<256, 4>);
    const uint32_t per = 512 / c->head_dim;                     // heads of a round
    a.parts = warps_per_token(a.p.T, (n_q + 2 * c->n_kv + per - 1) / per);
    return launch_tokens(kernel, a, (cudaStream_t)stream);
}

int ci_paged_gather(const ci_paged_cache *c, const ci_paged_batch *batch, uint16_t *d_k, uint16_t *d_v, ci_stream_t stream) {
    GatherArgs a;
    if (int rc = check_paged(c, batch, a.p)) return rc;
    CI_REQUIRE(d_k && d_v && ((reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v)) & 15u) == 0,
               "gathered rows need 16-byte aligned room");
    if (a.p.T == 0 || a.p.B == 0) return CI_OK;
    a.kc = (const uint8_t *)c->k; a.vc = (const uint8_t *)c->v; a.ks = c->k_scale; a.vs = c->v_scale;
    a.k_out = d_k; a.v_out = d_v;
    void (*kernel)(GatherArgs) =
        c->bits == 16 ? (c->head_dim == 64 ? k_paged_gather<64, 16> : c->head_dim == 128 ? k_paged_gather<128, 16> : k_paged_gather<256, 16>)
                      : (c->head_dim == 64 ? k_paged_gather<64, 4> : c->head_dim == 128 ? k_paged_gather<128, 4> : k_paged_gather<256, 4>);
    const uint32_t per = 256 / c->head_dim;
    a.parts = warps_per_token(a.p.T, (2 * c->n_kv + per - 1) / per);
    return launch_tokens(kernel, a, (cudaStream_t)stream);
}

}  // extern "C"
