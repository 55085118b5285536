// What a sampler does to logits before it picks a token, in one pass over them: penalties for tokens that have been,
// biases, and a mask of the tokens that may come.
//
//   x -> x / r where x > 0, x * r elsewhere, for tokens of the history (prompt and generated)
//   x -> x - f * count - p * (count > 0), count over the generated part
//   x -> x + the sum of the token's biases;  -inf where its mask bit is 0
//
// A block has kChunk tokens of one row: it counts the history's tokens of that range in shared memory (bit 31: seen),
// adds up the biases there, and then reads, changes and writes the logits, eight to a load.
#include "paged.cuh"

namespace ci {

constexpr uint32_t kChunk = 4096;

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

__global__ void __launch_bounds__(256) k_adjust_logits(const __grid_constant__ LogitArgs a) {
    __shared__ uint32_t s_count[kChunk];
    __shared__ float s_bias[kChunk];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t b = blockIdx.y, v0 = blockIdx.x * kChunk, n = min(kChunk, a.V - v0);
    const bool history = a.tokens != nullptr, biases = a.n_bias != 0;
    for (uint32_t i = threadIdx.x; i < kChunk; i += 256) {
        s_count[i] = 0;
        s_bias[i] = 0.f;
    }
    __syncthreads();
    if (history) {
        const uint32_t len = (uint32_t)min(max(a.lens[b], 0), (int32_t)a.L);
        const uint32_t prompt = a.prompt_lens ? (uint32_t)min(max(a.prompt_lens[b], 0), (int32_t)len) : 0;
        const int64_t *tok = a.tokens + (int64_t)b * a.ld_tokens;
        for (uint32_t i = threadIdx.x; i < len; i += 256) {
            const uint64_t at = (uint64_t)__ldg(tok + i) - v0;
            if (at >= n) continue;
            if (i >= prompt) atomicAdd(&s_count[at], 1u);
            atomicOr(&s_count[at], 0x80000000u);
        }
    }
    if (biases && threadIdx.x == 0) {                           // in order: the same sum every time
        for (uint32_t i = 0; i < a.n_bias; ++i) {
            const uint64_t at = (uint64_t)a.bias_ids[(int64_t)b * a.ld_bias + i] - v0;
            if (at < n) s_bias[at] += a.bias[(int64_t)b * a.ld_bias + i];
        }
    }
    __syncthreads();
    const float r = a.repetition ? a.repetition[b] : 1.f, f = a.frequency ? a.frequency[b] : 0.f, p = a.presence ? a.presence[b] : 0.f;
    const uint16_t *in = a.in + (int64_t)b * a.ldi + v0;
    uint16_t *out = a.out + (int64_t)b * a.ldo + v0;
    auto one = [&](float x, uint32_t i, uint32_t allowed) {
        const uint32_t c = s_count[i], count = c & 0x7FFFFFFFu;
        if (c) {
            if (a.repetition) x = x > 0.f ? __fdiv_rn(x, r) : x * r;
            if (count) x = x - f * (float)count - p;
        }
        if (biases) x += s_bias[i];
        return allowed ? x : -INFINITY;
    };
    const uint32_t *mask = a.mask ? a.mask + (int64_t)b * a.ld_mask + v0 / 32 : nullptr;
    if (a.vec) {
        for (uint32_t i = threadIdx.x * 8; i < n; i += 2048) {
            const uint4 w = *reinterpret_cast<const uint4 *>(in + i);
            const uint32_t bits = mask ? __ldg(mask + i / 32) >> (i % 32) : 0xFFu;
            const uint32_t x[4] = {w.x, w.y, w.z, w.w};
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                y[j] = pack_bf16(one(lo_bf16(x[j]), i + 2 * j, bits >> 2 * j & 1), one(hi_bf16(x[j]), i + 2 * j + 1, bits >> (2 * j + 1) & 1));
            *reinterpret_cast<uint4 *>(out + i) = make_uint4(y[0], y[1], y[2], y[3]);
        }
    } else {
        for (uint32_t i = threadIdx.x; i < n; i += 256)
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
    CI_REQUIRE(d->L <= 0x7FFFFFFFu, "a history of %u tokens", d->L);
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
    cfg.blockDim = dim3(256);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CI_CUDA(cudaLaunchKernelEx(&cfg, k_adjust_logits, a));
    return CI_OK;
}
