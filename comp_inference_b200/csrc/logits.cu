// What a sampler does to logits before it picks a token, in one pass over them: penalties for tokens that have been,
// biases, and a mask of the tokens that may come.
//
//   x -> x / r where x > 0, x * r elsewhere, for tokens of the history (prompt and generated)
//   x -> x - f * count - p * (count > 0), count over the generated part
//   x -> x + the sum of the token's biases;  -inf where its mask bit is 0
//
// A block has CHUNK tokens of one row: it asks for its logits, counts the history's tokens of that range in shared memory
// meanwhile, and then changes and writes the logits, eight to a load.  Tokens in neither history nor biases are most: one word in
// shared memory says so, and where a token's biases lie.  Rows of any vocabulary start on any even address; a block's range starts where
// 16-byte accesses do, and what sticks out in front and behind is taken apart.  64 rows of 131072 with histories up to 4096 tokens, 32
// biases and a mask: 14.2 us, 2.5 TB/s of an L2-resident 35 MB.  Its 1088 blocks go through loads, counts and stores one after the other,
// in 1.8 rounds of what fits on the device, and issue slots are 73 % busy (with histories of 2048 in every row): clearing and
// reading a word per token, and the history gone through by each of a row's 17 blocks.  One row of 32000: 5.4 us, the launch.
#include "paged.cuh"

namespace ci {

constexpr uint32_t kBiases = 512;            // of a row that are kept in shared memory; more than that are read again
// A token's word: seen; biased; kBiases less its first bias's place among the kept ones, or 0; how often it was generated.
constexpr uint32_t kSeen = 1u << 31, kBiased = 1u << 30, kPlace = 20, kCount = (1u << kPlace) - 1;
static_assert(kBiases < 1u << (30 - kPlace), "room for a place");

struct LogitArgs {
    const uint16_t *in;
    uint16_t *out;
    int64_t ldi, ldo, ld_tokens, ld_mask, ld_bias;
    uint32_t V, L, n_bias, vec;              // vec: rows of in and out start at the same place of a 16-byte word
    const int64_t *tokens, *bias_ids;
    const int32_t *lens, *prompt_lens;
    const float *repetition, *presence, *frequency, *bias;
    const uint32_t *mask;
};

template <uint32_t CHUNK, uint32_t THREADS>
__global__ void __launch_bounds__(THREADS) k_adjust_logits(const __grid_constant__ LogitArgs a) {
    constexpr uint32_t LOADS = CHUNK / (THREADS * 8);
    __shared__ __align__(16) uint32_t s_word[CHUNK];
    __shared__ int32_t s_at[kBiases];            // places of the biases in this range, -1: elsewhere
    __shared__ float s_bias[kBiases];
    __shared__ uint8_t s_more[kBiases];          // the token of this bias has others behind it
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t b = blockIdx.y;
    const uint16_t *in = a.in + (int64_t)b * a.ldi;
    uint16_t *out = a.out + (int64_t)b * a.ldo;
    // token v0 + i has word i; the first block's first `pre` tokens lie in front of the row
    const int64_t v0 = (int64_t)blockIdx.x * CHUNK - (int64_t)((reinterpret_cast<uintptr_t>(in) & 15u) / 2);
    const uint32_t n0 = v0 < 0 ? (uint32_t)-v0 : 0u, n1 = (uint32_t)max(min((int64_t)CHUNK, (int64_t)a.V - v0), (int64_t)0);
    in += v0;
    out += v0;
    const uint32_t *mask = a.mask ? a.mask + (int64_t)b * a.ld_mask : nullptr;
    uint4 x[LOADS];
    uint32_t bits[LOADS];
#pragma unroll
    for (uint32_t k = 0; k < LOADS; ++k) {
        const uint32_t i = (k * THREADS + threadIdx.x) * 8;
        x[k] = make_uint4(0, 0, 0, 0);
        bits[k] = 0xFFu;
        if (i >= n1) continue;
        if (i >= n0 && i + 8 <= n1) {
            x[k] = *reinterpret_cast<const uint4 *>(in + i);
        } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
                if (i + j >= n0 && i + j < n1) w[j / 2] |= (uint32_t)in[i + j] << (16 * (j % 2));
            x[k] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (mask) {
            const uint32_t v = i < n0 ? 0u : (uint32_t)(v0 + i), low = i < n0 ? n0 - i : 0u;
            uint32_t m = __ldg(mask + v / 32) >> (v % 32);
            if (v % 32 > 24 && v / 32 + 1 < (a.V + 31) / 32) m |= __ldg(mask + v / 32 + 1) << (32 - v % 32);
            bits[k] = m << low;
        }
    }
    const float r = a.repetition ? __ldg(a.repetition + b) : 1.f, f = a.frequency ? __ldg(a.frequency + b) : 0.f;
    const float p = a.presence ? __ldg(a.presence + b) : 0.f;
    // Lengths and the first biases are asked for now too.
    const uint32_t n_bias = min(a.n_bias, kBiases);
    const int64_t *bias_ids = a.bias_ids + (int64_t)b * a.ld_bias;
    const float *bias = a.bias + (int64_t)b * a.ld_bias;
    const int64_t *tok = a.tokens + (int64_t)b * a.ld_tokens;
    int64_t id0 = -1;
    float bias0 = 0.f;
    uint32_t len = 0, prompt = 0;
    if (a.tokens) {
        len = (uint32_t)min(max(__ldg(a.lens + b), 0), (int32_t)a.L);
        prompt = a.prompt_lens ? (uint32_t)max(__ldg(a.prompt_lens + b), 0) : 0;
    }
    if (threadIdx.x < n_bias) {
        id0 = __ldg(bias_ids + threadIdx.x);
        bias0 = __ldg(bias + threadIdx.x);
    }
    for (uint32_t i = threadIdx.x; i < CHUNK / 4; i += THREADS) reinterpret_cast<uint4 *>(s_word)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    auto place = [&](int64_t id) { return (uint64_t)id < a.V ? (uint64_t)(id - v0) : ~0ull; };
    for (uint32_t i = threadIdx.x; i < n_bias; i += THREADS) {
        const uint64_t at = place(i == threadIdx.x ? id0 : __ldg(bias_ids + i));
        if (at < CHUNK) atomicMax(&s_word[at], kBiased | (kBiases - i) << kPlace);      // the first one's place is the largest
        s_at[i] = at < CHUNK ? (int32_t)at : -1;
        s_bias[i] = i == threadIdx.x ? bias0 : __ldg(bias + i);
        s_more[i] = 0;
    }
    if (a.n_bias) __syncthreads();
    if (a.tokens) {
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < len; i += THREADS) {
            const uint64_t at = place(__ldg(tok + i));
            if (at < CHUNK) {
                atomicOr(&s_word[at], kSeen);
                if (i >= prompt) atomicAdd(&s_word[at], 1u);
            }
        }
    }
    auto first_bias = [&](uint32_t word) { return kBiases - (word >> kPlace & 1023u); };        // kBiases: none of the kept ones
    bool again = false;                                         // a token has several biases
    for (uint32_t i = threadIdx.x; i < n_bias; i += THREADS)
        if (s_at[i] >= 0) {
            const uint32_t first = first_bias(*(volatile uint32_t *)&s_word[s_at[i]]);
            if (first != i) {
                s_more[first] = 1;
                again = true;
            }
        }
    for (uint32_t i = kBiases + threadIdx.x; i < a.n_bias; i += THREADS) {
        const uint64_t at = place(__ldg(bias_ids + i));
        if (at < CHUNK) atomicOr(&s_word[at], kBiased);
    }
    if (__syncthreads_or(again)) {
        for (uint32_t i = threadIdx.x; i < n_bias; i += THREADS)
            if (s_more[i]) {                                    // in order: the same sum every time
                const int32_t at = s_at[i];
                float sum = s_bias[i];
#pragma unroll 8
                for (uint32_t k = i + 1; k < n_bias; ++k) sum = s_at[k] == at ? sum + s_bias[k] : sum;
                s_bias[i] = sum;                                // (no other thread reads it for its own sum)
            }
        __syncthreads();
    }
    auto one = [&](float y, uint32_t i) {
        const uint32_t w = s_word[i], count = w & kCount;
        if (w) {
            if (a.repetition && (w & kSeen)) y = y > 0.f ? __fdiv_rn(y, r) : y * r;
            if (count) y = y - f * (float)count - p;
            if (w & kBiased) {
                const uint32_t first = first_bias(w);
                float sum = first < kBiases ? s_bias[first] : 0.f;
                for (uint32_t k = kBiases; k < a.n_bias; ++k)
                    if (place(__ldg(bias_ids + k)) == i) sum += __ldg(bias + k);
                y += sum;
            }
        }
        return y;
    };
#pragma unroll
    for (uint32_t k = 0; k < LOADS; ++k) {
        const uint32_t i = (k * THREADS + threadIdx.x) * 8;
        if (i >= n1) continue;
        const uint4 c0 = *reinterpret_cast<const uint4 *>(s_word + i), c1 = *reinterpret_cast<const uint4 *>(s_word + i + 4);
        const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
        uint32_t y[4] = {w[0], w[1], w[2], w[3]};
        if (c0.x | c0.y | c0.z | c0.w | c1.x | c1.y | c1.z | c1.w) {
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = pack_bf16(one(lo_bf16(w[j]), i + 2 * j), one(hi_bf16(w[j]), i + 2 * j + 1));
        }
        if (mask) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!(bits[k] >> 2 * j & 1)) y[j] = (y[j] & 0xFFFF0000u) | 0xFF80u;
                if (!(bits[k] >> (2 * j + 1) & 1)) y[j] = (y[j] & 0x0000FFFFu) | 0xFF800000u;
            }
        }
        if (a.vec && i >= n0 && i + 8 <= n1) {
            *reinterpret_cast<uint4 *>(out + i) = make_uint4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
                if (i + j >= n0 && i + j < n1) out[i + j] = (uint16_t)(y[j / 2] >> (16 * (j % 2)));
        }
    }
}

// Blocks of 8192 tokens where that fills the device: the history is gone through once per block.  Else of 2048.
template <uint32_t CHUNK, uint32_t THREADS>
static int launch_adjust(const LogitArgs &a, uint32_t B, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((uint64_t)a.V + 7 + CHUNK - 1) / CHUNK), B);         // (up to seven tokens in front of a row)
    cfg.blockDim = dim3(THREADS);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CI_CUDA(cudaLaunchKernelEx(&cfg, k_adjust_logits<CHUNK, THREADS>, a));
    return CI_OK;
}

}  // namespace ci

using namespace ci;

extern "C" int ci_adjust_logits(const ci_logit_adjust *d, ci_stream_t stream) {
    CI_REQUIRE(d && d->d_in && d->d_out, "null pointer");
    CI_REQUIRE(d->V > 0 && d->V <= 0x7FFFFFFFu && d->ld_in >= (int64_t)d->V && d->ld_out >= (int64_t)d->V, "row stride smaller than the vocabulary");
    CI_REQUIRE(d->B <= 65535, "%u rows of logits", d->B);
    CI_REQUIRE(((reinterpret_cast<uintptr_t>(d->d_in) | reinterpret_cast<uintptr_t>(d->d_out)) & 1u) == 0, "logits on an odd address");
    CI_REQUIRE(d->L == 0 || d->d_tokens == nullptr || (d->d_lens && d->ld_tokens >= (int64_t)d->L), "a history needs its lengths");
    CI_REQUIRE(d->L <= kCount, "a history of %u tokens", d->L);
    CI_REQUIRE(d->n_bias == 0 || (d->d_bias_ids && d->d_bias && d->ld_bias >= (int64_t)d->n_bias), "biases need their tokens and values");
    CI_REQUIRE(d->d_mask == nullptr || d->ld_mask >= ((int64_t)d->V + 31) / 32, "mask rows shorter than the vocabulary");
    if (d->B == 0) return CI_OK;
    LogitArgs a;
    a.in = d->d_in; a.out = d->d_out;
    a.ldi = d->ld_in; a.ldo = d->ld_out; a.ld_tokens = d->ld_tokens; a.ld_mask = d->ld_mask; a.ld_bias = d->ld_bias;
    a.V = d->V; a.L = d->L; a.n_bias = d->n_bias;
    a.tokens = d->L ? d->d_tokens : nullptr; a.bias_ids = d->d_bias_ids;
    a.lens = d->d_lens; a.prompt_lens = d->d_prompt_lens;
    a.repetition = d->d_repetition; a.presence = d->d_presence; a.frequency = d->d_frequency; a.bias = d->d_bias;
    a.mask = d->d_mask;
    a.vec = ((reinterpret_cast<uintptr_t>(d->d_in) ^ reinterpret_cast<uintptr_t>(d->d_out)) & 15u) == 0 && (d->ld_in - d->ld_out) % 8 == 0;
    cudaStream_t s = (cudaStream_t)stream;
    return ((uint64_t)d->V + 8191) / 8192 * d->B >= (uint32_t)sm_count() ? launch_adjust<8192, 512>(a, d->B, s)
                                                                          : launch_adjust<2048, 256>(a, d->B, s);
}
