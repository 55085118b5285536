// What a sampler does to logits before it picks a token, in one pass over them: penalties for tokens that have been,
// biases, and a mask of the tokens that may come.
//
//   x -> x / r where x > 0, x * r elsewhere, for tokens of the history (prompt and generated)
//   x -> x - f * count - p * (count > 0), count over the generated part
//   x -> x + the sum of the token's biases;  -inf where its mask bit is 0
//
// A block has kChunk tokens of one row: it asks for its logits, counts the history's tokens of that range in shared memory
// meanwhile (bit 31: seen, bit 30: has a bias), and then changes and writes the logits, eight to a load.  Tokens in neither are
// most: one word in shared memory says so.  64 rows of 131072 with histories up to 4096 tokens, 32 biases and a mask: ZZZZ.
#include "paged.cuh"

namespace ci {

constexpr uint32_t kChunk = 8192, kLogitThreads = 512, kLogitLoads = kChunk / (kLogitThreads * 8);
constexpr uint32_t kBiases = 512;
constexpr uint32_t kSeen = 1u << 31, kBiased = 1u << 30;

struct LogitArgs {
    const uint16_t *in;
    uint16_t *out;
    int64_t ldi, ldo, ld_tokens, ld_mask, ld_bias;
    uint32_t V, L, n_bias, vec;
    const int64_t *tokens, *bias_ids;
    const int32_t *lens, *prompt_lens;
    const float *repetition, *presence, *frequency, *bias;
    const uint32_t *mask;
};

__global__ void __launch_bounds__(kLogitThreads) k_adjust_logits(const __grid_constant__ LogitArgs a) {
    __shared__ __align__(16) uint32_t s_count[kChunk];
    __shared__ int32_t s_at[kBiases];            // places of the biases in this range, -1: elsewhere
    __shared__ float s_bias[kBiases];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t b = blockIdx.y, v0 = blockIdx.x * kChunk, n = min(kChunk, a.V - v0);
    const uint16_t *in = a.in + (int64_t)b * a.ldi + v0;
    uint16_t *out = a.out + (int64_t)b * a.ldo + v0;
    const uint32_t *mask = a.mask ? a.mask + (int64_t)b * a.ld_mask + v0 / 32 : nullptr;
    uint4 x[kLogitLoads];
    uint32_t bits[kLogitLoads];
#pragma unroll
    for (uint32_t k = 0; k < kLogitLoads; ++k) {
        const uint32_t i = (k * kLogitThreads + threadIdx.x) * 8;
        x[k] = make_uint4(0, 0, 0, 0);
        bits[k] = 0xFFu;
        if (a.vec && i < n) {
            x[k] = *reinterpret_cast<const uint4 *>(in + i);
            if (mask) bits[k] = __ldg(mask + i / 32) >> (i % 32);
        }
    }
    const bool history = a.tokens != nullptr;
    const float r = a.repetition ? __ldg(a.repetition + b) : 1.f, f = a.frequency ? __ldg(a.frequency + b) : 0.f;
    const float p = a.presence ? __ldg(a.presence + b) : 0.f;
    for (uint32_t i = threadIdx.x; i < kChunk / 4; i += kLogitThreads) reinterpret_cast<uint4 *>(s_count)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (history) {
        const uint32_t len = (uint32_t)min(max(__ldg(a.lens + b), 0), (int32_t)a.L);
        const uint32_t prompt = a.prompt_lens ? (uint32_t)min(max(__ldg(a.prompt_lens + b), 0), (int32_t)len) : 0;
        const int64_t *tok = a.tokens + (int64_t)b * a.ld_tokens;
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < len; i += kLogitThreads) {
            const uint64_t at = (uint64_t)__ldg(tok + i) - v0;
            if (at < n) {
                atomicOr(&s_count[at], kSeen);
                if (i >= prompt) atomicAdd(&s_count[at], 1u);
            }
        }
    }
    const uint32_t n_bias = min(a.n_bias, kBiases);             // kept in shared memory; more than that are read again
    for (uint32_t i = threadIdx.x; i < a.n_bias; i += kLogitThreads) {
        const uint64_t at = (uint64_t)__ldg(a.bias_ids + (int64_t)b * a.ld_bias + i) - v0;
        if (at < n) atomicOr(&s_count[at], kBiased);
        if (i < kBiases) {
            s_at[i] = at < n ? (int32_t)at : -1;
            s_bias[i] = __ldg(a.bias + (int64_t)b * a.ld_bias + i);
        }
    }
    __syncthreads();
    auto one = [&](float y, uint32_t i, uint32_t allowed) {
        const uint32_t c = s_count[i], count = c & (kBiased - 1);
        if (c) {
            if (a.repetition && (c & kSeen)) y = y > 0.f ? __fdiv_rn(y, r) : y * r;
            if (count) y = y - f * (float)count - p;
            if (c & kBiased) {                                  // in order: the same sum every time
                float sum = 0.f;
                for (uint32_t k = 0; k < n_bias; ++k)
                    if (s_at[k] == (int32_t)i) sum += s_bias[k];
                for (uint32_t k = kBiases; k < a.n_bias; ++k)
                    if ((uint64_t)__ldg(a.bias_ids + (int64_t)b * a.ld_bias + k) - v0 == i) sum += __ldg(a.bias + (int64_t)b * a.ld_bias + k);
                y += sum;
            }
        }
        return allowed ? y : -INFINITY;
    };
    if (a.vec) {
#pragma unroll
        for (uint32_t k = 0; k < kLogitLoads; ++k) {
            const uint32_t i = (k * kLogitThreads + threadIdx.x) * 8;
            if (i >= n) continue;
            const uint4 c0 = *reinterpret_cast<const uint4 *>(s_count + i), c1 = *reinterpret_cast<const uint4 *>(s_count + i + 4);
            const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
            uint32_t y[4] = {w[0], w[1], w[2], w[3]};
            if (c0.x | c0.y | c0.z | c0.w | c1.x | c1.y | c1.z | c1.w) {
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = pack_bf16(one(lo_bf16(w[j]), i + 2 * j, 1), one(hi_bf16(w[j]), i + 2 * j + 1, 1));
            }
            if (mask) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!(bits[k] >> 2 * j & 1)) y[j] = (y[j] & 0xFFFF0000u) | 0xFF80u;
                    if (!(bits[k] >> (2 * j + 1) & 1)) y[j] = (y[j] & 0x0000FFFFu) | 0xFF800000u;
                }
            }
            *reinterpret_cast<uint4 *>(out + i) = make_uint4(y[0], y[1], y[2], y[3]);
        }
    } else {
        for (uint32_t i = threadIdx.x; i < n; i += kLogitThreads)
            out[i] = float_to_bf16_bits(one(lo_bf16(in[i]), i, mask ? __ldg(mask + i / 32) >> (i % 32) & 1 : 1));
    }
}

}  // namespace ci

using namespace ci;

extern "C" int ci_adjust_logits(const ci_logit_adjust *d, ci_stream_t stream) {
    CI_REQUIRE(d && d->d_in && d->d_out, "null pointer");
    CI_REQUIRE(d->V > 0 && d->V <= 0x7FFFFFFFu && d->ld_in >= (int64_t)d->V && d->ld_out >= (int64_t)d->V, "row stride smaller than the vocabulary");
    CI_REQUIRE(d->B <= 65535, "%u rows of logits", d->B);
    CI_REQUIRE(d->L == 0 || d->d_tokens == nullptr || (d->d_lens && d->ld_tokens >= (int64_t)d->L), "a history needs its lengths");
    CI_REQUIRE(d->L < kBiased, "a history of %u tokens", d->L);
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
    a.vec = d->V % 8 == 0 && d->ld_in % 8 == 0 && d->ld_out % 8 == 0 &&
            ((reinterpret_cast<uintptr_t>(d->d_in) | reinterpret_cast<uintptr_t>(d->d_out)) & 15u) == 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((d->V + kChunk - 1) / kChunk, d->B);
    cfg.blockDim = dim3(kLogitThreads);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CI_CUDA(cudaLaunchKernelEx(&cfg, k_adjust_logits, a));
    return CI_OK;
}
