// Verification of drafted tokens against the target's probabilities.
#include <cuda_runtime.h>

#include <math.h>

#include "common.cuh"
#include "host.hpp"

namespace esp {
namespace {

struct VerifyParams {
    const void* logits;
    const void* draft_probs;
    const int *starts, *drafts;
    const float *uniform, *noise, *temperature;
    int *tokens, *accepted;
    float* probs;
    long long stride, rows, n_drafts, probs_stride, noise_stride;
    int dtype, probs_dtype, vocab, max_drafts;
};

__device__ __forceinline__ float load1(const void* p, int dtype, size_t i) {
    if (dtype == F32) return static_cast<const float*>(p)[i];
    if (dtype == BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}

// A logit as the softmax takes it: NaN is a token ruled out, and -0 is 0 (equal logits are a tie).
__device__ __forceinline__ float logit(const VerifyParams& p, size_t row, int v) {
    const float l = load1(p.logits, p.dtype, row * p.stride + v);
    return l == l ? l + 0.0f : -INFINITY;
}

// exp((l - m) / T) with m the row's largest logit: 1 at the largest, also where that is +inf (the row's mass is then
// shared by its infinite logits) and 0 at -inf.
__device__ __forceinline__ float weight(float l, float m, float inv_t) {
    return l == m ? 1.0f : expf((l - m) * inv_t);
}

// Order-preserving key of a non-negative score with the lowest id first among equals; 0 is no candidate.
__device__ __forceinline__ unsigned long long score_key(float s, int v) {
    return (static_cast<unsigned long long>(__float_as_uint(s)) << 32) | (0xffffffffu - static_cast<unsigned>(v));
}
__device__ __forceinline__ int key_id(unsigned long long k) { return static_cast<int>(0xffffffffu - static_cast<unsigned>(k)); }
// The same for any float: the sign bit flipped for positives, all bits for negatives.
__device__ __forceinline__ unsigned long long logit_key(float l, int v) {
    const unsigned u = __float_as_uint(l);
    return (static_cast<unsigned long long>(u & 0x80000000u ? ~u : u | 0x80000000u) << 32) |
           (0xffffffffu - static_cast<unsigned>(v));
}
__device__ __forceinline__ float key_logit(unsigned long long k) {
    const unsigned u = static_cast<unsigned>(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

constexpr int THREADS = 1024;

template <typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, T* scratch, Op op) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, m));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[0];
    for (int w = 1; w < THREADS / 32; ++w) v = op(v, scratch[w]);
    return v;
}

// A CTA a request: rows in order until a drafted token falls.
__global__ void __launch_bounds__(THREADS) verify_kernel(VerifyParams p) {
    __shared__ unsigned long long scratch[THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x, V = p.vocab, width = p.max_drafts + 1;
    const auto max64 = [](unsigned long long a, unsigned long long c) { return a > c ? a : c; };
    const auto add = [](float a, float c) { return a + c; };
    const long long at = p.starts[b], first = at + b;
    const long long k_all = static_cast<long long>(p.starts[b + 1]) - at;
    const bool fits = at >= 0 && k_all >= 0 && at + k_all <= p.n_drafts && first + k_all < p.rows;
    const int k = static_cast<int>(min(k_all, static_cast<long long>(p.max_drafts)));
    float t = p.temperature ? p.temperature[b] : 1.0f;
    const bool greedy = !(t > 0.0f);
    const float inv_t = greedy ? 1.0f : 1.0f / fminf(fmaxf(t, 1e-30f), 1e30f);

    int n = 0, token = -1;
    float token_p = 0.0f;
    for (int i = 0; fits && i <= k; ++i) {
        const size_t row = first + i;
        unsigned long long key = 0;
        for (int v = threadIdx.x; v < V; v += THREADS) key = max64(key, logit_key(logit(p, row, v), v));
        key = block_reduce(key, scratch, max64);
        const float m = key_logit(key);
        const int best = key_id(key);
        n = i;
        if (m == -INFINITY) break;      // nothing left to choose from
        float z = 0.0f;
        for (int v = threadIdx.x; v < V; v += THREADS) z += weight(logit(p, row, v), m, inv_t);
        z = block_reduce(z, reinterpret_cast<float*>(scratch), add);

        int d = -1;
        float pd = 0.0f;
        if (i < k) {
            d = p.drafts[at + i];
            if (d < 0 || d >= V) d = -1;
            else pd = weight(logit(p, row, d), m, inv_t) / z;
            bool stands = false;
            if (d >= 0) {
                const float q = p.draft_probs ? load1(p.draft_probs, p.probs_dtype, (at + i) * p.probs_stride + d) : 1.0f;
                stands = greedy ? d == best : p.uniform[at + i] * q < pd;
            }
            if (stands) {
                if (threadIdx.x == 0) {
                    p.tokens[static_cast<size_t>(b) * width + i] = d;
                    p.probs[static_cast<size_t>(b) * width + i] = pd;
                }
                continue;
            }
        }
        token = best;
        if (!greedy) {
            const bool fell = i < k;
            unsigned long long won = 0;
            for (int v = threadIdx.x; v < V; v += THREADS) {
                float w = weight(logit(p, row, v), m, inv_t) / z;
                if (fell) {
                    if (p.draft_probs) w -= load1(p.draft_probs, p.probs_dtype, (at + i) * p.probs_stride + v);
                    else if (v == d) w = 0.0f;
                }
                if (w > 0.0f) {
                    const float s = w / p.noise[b * p.noise_stride + v];
                    if (s >= 0.0f) won = max64(won, score_key(s, v));
                }
            }
            won = block_reduce(won, scratch, max64);
            if (won) token = key_id(won);
        }
        token_p = weight(logit(p, row, token), m, inv_t) / z;
        break;
    }
    if (threadIdx.x == 0) p.accepted[b] = n;
    for (int i = n + threadIdx.x; i < width; i += THREADS) {
        p.tokens[static_cast<size_t>(b) * width + i] = i == n ? token : -1;
        p.probs[static_cast<size_t>(b) * width + i] = i == n ? token_p : 0.0f;
    }
}

bool known_dtype(int t) { return t == F16 || t == BF16 || t == F32; }

}  // namespace
}  // namespace esp

extern "C" int esp_verify(const void* logits, int dtype, long long stride, long long rows, int vocab, const int* starts,
                          int requests, const int* drafts, const float* uniform, long long n_drafts,
                          const void* draft_probs, int probs_dtype, long long probs_stride, const float* noise,
                          long long noise_stride, const float* temperature, int max_drafts, int* tokens, int* accepted,
                          float* probs, void* stream) {
    using namespace esp;
    ESP_REQUIRE(known_dtype(dtype), ESP_ERR_INVALID, "esp_verify: unknown logits dtype %d", dtype);
    ESP_REQUIRE(requests >= 0 && rows >= 0 && n_drafts >= 0 && max_drafts >= 0, ESP_ERR_INVALID,
                "esp_verify: negative size");
    ESP_REQUIRE(vocab >= 1, ESP_ERR_INVALID, "esp_verify: vocabulary of %d", vocab);
    if (requests == 0) return ok();
    ESP_REQUIRE(logits && starts && noise && tokens && accepted && probs, ESP_ERR_INVALID, "esp_verify: null pointer");
    ESP_REQUIRE(n_drafts == 0 || (drafts && uniform), ESP_ERR_INVALID, "esp_verify: drafted tokens without a pointer");
    ESP_REQUIRE(!draft_probs || known_dtype(probs_dtype), ESP_ERR_INVALID, "esp_verify: unknown draft_probs dtype %d",
                probs_dtype);
    const VerifyParams p{logits, draft_probs, starts, drafts, uniform, noise, temperature, tokens, accepted, probs,
                         stride, rows, n_drafts, probs_stride, noise_stride, dtype, probs_dtype, vocab, max_drafts};
    if (const int rc = launch(verify_kernel, dim3(static_cast<unsigned>(requests)), dim3(THREADS), 0, stream, true, p))
        return rc;
    return ok();
}
