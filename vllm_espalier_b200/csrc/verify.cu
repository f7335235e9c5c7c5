// Verification of drafted tokens against the target's probabilities.
#include <cuda_runtime.h>

#include <limits.h>
#include <math.h>

#include <type_traits>

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

__device__ __forceinline__ float f32(float v) { return v; }
__device__ __forceinline__ float f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float f32(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr float LOG2E = 1.4426950408889634f;

// exp((l - m) / T) as 2^((l - m) c), c = log2(e) / T: 1 at the row's largest logit m, also where that is +inf (the row's
// mass is then shared by its infinite logits), 0 for -inf and NaN.
__device__ __forceinline__ float weight(float l, float m, float c) {
    return l == m ? 1.0f : ex2(fmaxf((l - m) * c, -200.0f));
}

// Order-preserving key of a non-negative score with the lowest id first among equals; 0 is no candidate.
__device__ __forceinline__ unsigned long long score_key(float s, int v) {
    return (static_cast<unsigned long long>(__float_as_uint(s) & 0x7fffffffu) << 32) | (0xffffffffu - static_cast<unsigned>(v));
}
__device__ __forceinline__ int key_id(unsigned long long k) { return static_cast<int>(0xffffffffu - static_cast<unsigned>(k)); }

// What is known of a part of a row: the largest logit, the sum of the weights against it, the lowest place of it (only
// where places are asked for).
struct alignas(16) Part {
    float m, z;
    int at, unused;
};

__device__ __forceinline__ Part joined(Part a, Part b, float c) {
    const float m = fmaxf(a.m, b.m);
    const float z = (a.m == m ? a.z : a.z * ex2((a.m - m) * c)) + (b.m == m ? b.z : b.z * ex2((b.m - m) * c));
    return {m, z, a.m == b.m ? min(a.at, b.at) : a.m > b.m ? a.at : b.at, 0};
}

// The join of the CTA's threads, in thread 0 (a barrier inside).
__device__ __forceinline__ Part block_part(Part t, float c, bool places, Part* warps) {
    float m = t.m;
#pragma unroll
    for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    float z = t.m == m ? t.z : t.z * ex2((t.m - m) * c);
#pragma unroll
    for (int k = 16; k; k >>= 1) z += __shfl_xor_sync(0xffffffffu, z, k);
    int at = 0;
    if (places) at = __reduce_min_sync(0xffffffffu, t.m == m ? t.at : INT_MAX);
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = {m, z, at, 0};
    __syncthreads();
    t = {-INFINITY, 0.0f, INT_MAX, 0};
    if (threadIdx.x < 32) {
        if (threadIdx.x < WARPS) t = warps[threadIdx.x];
#pragma unroll
        for (int k = WARPS / 2; k; k >>= 1)
            t = joined(t, {__shfl_xor_sync(0xffffffffu, t.m, k), __shfl_xor_sync(0xffffffffu, t.z, k),
                           __shfl_xor_sync(0xffffffffu, t.at, k), 0}, c);
    }
    return t;
}

template <typename T>
struct alignas(16) Pack {
    T e[16 / sizeof(T)];
};

// This thread's share of the part [lo, hi) of a row, in one pass. The thread keeps the largest logit m that it has met
// and the sum of 2^(l c - mc) with mc = m c rounded; a larger m rescales the sum by 2^(mc - mc'). The rounding of mc is
// taken out once, at the end (2^(mc - m c)), so a logit costs one fma and one exponential. For c in [1e-6, 1e6], where a
// logit below FLOOR weighs nothing beside one above it. A row with NaN, +inf, an m c that overflows or nothing above
// FLOOR comes out with a sum that is NaN, infinite or 0, which the caller sees and takes careful_part instead.
constexpr float FLOOR = -1e30f;
template <typename T>
__device__ __forceinline__ Part fast_part(const T* row, int lo, int hi, float c, bool places) {
    constexpr int N = 16 / sizeof(T), UNROLL = 4;
    float m = FLOOR, mc = 0.0f, z = 0.0f;
    int first = -1;         // where the pack starts among whose logits the largest was first met
    const auto take = [&](const Pack<T>& k, int v) {
        float l[N], top = -INFINITY;
#pragma unroll
        for (int e = 0; e < N; ++e) top = fmaxf(top, l[e] = f32(k.e[e]));
        if (top > m) {
            const float next = top * c;
            z = first < 0 ? 0.0f : z * ex2(mc - next);
            m = top, mc = next, first = v;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) z += ex2(fmaf(l[e], c, -mc));
    };
    // 16-byte loads from the first boundary on, the ends one by one
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row + lo) % 16 / sizeof(T));
    const int head = min(hi, lo + (off ? N - off : 0)), packs = (hi - head) / N, tail = head + packs * N;
    const auto single = [&](int v) {
        const float l = f32(row[v]);
        if (l > m) {
            const float next = l * c;
            z = first < 0 ? 0.0f : z * ex2(mc - next);
            m = l, mc = next, first = v;
        }
        z += ex2(fmaf(l, c, -mc));
    };
    // before the packs, so that a thread meets its places in order
    if (lo + static_cast<int>(threadIdx.x) < head) single(lo + threadIdx.x);
    int i = threadIdx.x;
    for (; i + (UNROLL - 1) * THREADS < packs; i += UNROLL * THREADS) {
        Pack<T> k[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) k[u] = *reinterpret_cast<const Pack<T>*>(row + head + (i + u * THREADS) * N);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) take(k[u], head + (i + u * THREADS) * N);
    }
    for (; i < packs; i += THREADS) take(*reinterpret_cast<const Pack<T>*>(row + head + i * N), head + i * N);
    if (tail + static_cast<int>(threadIdx.x) < hi) single(tail + threadIdx.x);
    if (first >= 0) z *= ex2(-fmaf(m, c, -mc));
    int at = first;
    if (places && first >= 0)
        while (f32(row[at]) != m) ++at;     // met: a logit of the pack at `first` equals m
    return {m, z, first < 0 ? INT_MAX : at, 0};
}

// The same for any row: NaN counts as -inf, weights as weight() has them. The whole CTA's part, in every thread.
template <typename T>
__device__ __noinline__ Part careful_part(const T* row, int lo, int hi, float c, Part* warps) {
    Part t = {-INFINITY, 0.0f, INT_MAX, 0};
    for (int v = lo + threadIdx.x; v < hi; v += THREADS) {
        const float l = f32(row[v]);
        if (l > t.m) t = {l, 0.0f, v, 0};
    }
    __shared__ Part all;
    t = block_part(t, c, true, warps);      // no sums yet: only the largest and its place
    if (threadIdx.x == 0) all = t;
    __syncthreads();
    t = all;
    float z = 0.0f;
    if (t.m > -INFINITY)
        for (int v = lo + threadIdx.x; v < hi; v += THREADS) z += weight(f32(row[v]), t.m, c);
    const Part sum = block_part({0.0f, z, 0, 0}, c, false, warps);
    if (threadIdx.x == 0) all.z = sum.z;
    __syncthreads();
    t = all;
    __syncthreads();
    return t;
}

// Every CTA of the cluster gives its part (of thread 0) and gets the row's, joined in the order of the ranks: one cluster
// barrier. `slot` is written again only after another barrier of the cluster.
__device__ __forceinline__ Part cluster_part(Part mine, float c, Part* slot, int ctas) {
    if (threadIdx.x == 0) *slot = mine;
    cluster_sync_all();
    Part t = {-INFINITY, 0.0f, INT_MAX, 0};
    for (int r = 0; r < ctas; ++r) {
        const float4 q = ld_cluster_f4(slot, r);
        t = joined(t, {q.x, q.y, __float_as_int(q.z), 0}, c);
    }
    return t;
}

struct NoProbs {};      // the drafter chose its token outright
template <typename Q>
__device__ __forceinline__ float draft_prob(const Q* q, long long i) {
    if constexpr (std::is_same_v<Q, NoProbs>) return 1.0f;
    else return f32(q[i]);
}

// A cluster of `ctas` CTAs a request, each with its part of the vocabulary: rows in order until a drafted token falls.
// Every CTA reads the same parts and so takes the same decisions.
template <typename T, typename Q>
__global__ void __launch_bounds__(THREADS, 2) verify_kernel(VerifyParams p, int ctas) {
    __shared__ Part warps[WARPS], parts[5];      // parts: two rows' in turn, two careful ones', the last resort's
    __shared__ alignas(16) unsigned long long best_key[2];
    constexpr bool ONE_HOT = std::is_same_v<Q, NoProbs>;
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x / ctas, rank = blockIdx.x % ctas, V = p.vocab, width = p.max_drafts + 1;
    const int share = (V + 8 * ctas - 1) / (8 * ctas) * 8, lo = min(V, rank * share), hi = min(V, lo + share);
    const bool writes = rank == 0 && threadIdx.x == 0;
    const long long at = p.starts[b], first = at + b;
    const long long k_all = static_cast<long long>(p.starts[b + 1]) - at;
    const bool fits = at >= 0 && k_all >= 0 && at + k_all <= p.n_drafts && first + k_all < p.rows;
    const int k = static_cast<int>(min(k_all, static_cast<long long>(p.max_drafts)));
    const float t = p.temperature ? p.temperature[b] : 1.0f;
    const bool greedy = !(t > 0.0f);
    const float c = greedy ? LOG2E : LOG2E / fminf(fmaxf(t, 1e-30f), 1e30f);
    int* tokens = p.tokens + static_cast<size_t>(b) * width;
    float* probs = p.probs + static_cast<size_t>(b) * width;

    int n = 0, token = -1;
    float token_p = 0.0f;
    for (int i = 0; fits && i <= k; ++i) {
        const T* row = static_cast<const T*>(p.logits) + (first + i) * p.stride;
        const Q* q = static_cast<const Q*>(p.draft_probs) + (ONE_HOT ? 0 : (at + i) * p.probs_stride);
        int d = -1;
        float ld = 0.0f, qd = 0.0f, u = 0.0f;
        if (i < k) {
            d = p.drafts[at + i];
            if (d < 0 || d >= V) d = -1;
            else ld = f32(row[d]), qd = draft_prob(q, d), u = p.uniform[at + i];
        }
        n = i;
        Part all = {-INFINITY, 0.0f, INT_MAX, 0};
        if (c >= 1e-6f && c <= 1e6f)
            all = cluster_part(block_part(fast_part(row, lo, hi, c, greedy), c, greedy, warps), c, &parts[i & 1], ctas);
        if (!(all.z > 0.0f && all.z < INFINITY)) {
            all = cluster_part(careful_part(row, lo, hi, c, warps), c, &parts[2 + (i & 1)], ctas);
            if (all.m == -INFINITY) break;      // nothing left to choose from
        }
        const float m = all.m, inv_z = 1.0f / all.z;
        const float pd = d >= 0 ? weight(ld, m, c) * inv_z : 0.0f;
        if (d >= 0 && (greedy ? d == all.at : u * qd < pd)) {
            if (writes) tokens[i] = d, probs[i] = pd;
            continue;
        }
        if (greedy) {
            token = all.at;
            token_p = inv_z;
            break;
        }
        // The race: the largest w / noise, the lowest id among equals.
        const float* noise = p.noise + b * p.noise_stride;
        const bool fell = i < k;
        unsigned long long key = 0;
        {
            float top = -1.0f;
            int id = 0;
            for (int v = lo + threadIdx.x; v < hi; v += THREADS) {
                float w = weight(f32(row[v]), m, c) * inv_z;
                if (fell) {
                    if (ONE_HOT) w = v == d ? 0.0f : w;
                    else w -= draft_prob(q, v);
                }
                const float score = __fdividef(w, noise[v]);
                if (w > 0.0f && score > top) top = score, id = v;
            }
            if (top >= 0.0f) key = score_key(top, id);
        }
#pragma unroll
        for (int j = 16; j; j >>= 1) {
            const unsigned long long o = __shfl_xor_sync(0xffffffffu, key, j);
            key = o > key ? o : key;
        }
        unsigned long long* keys = reinterpret_cast<unsigned long long*>(warps);
        if ((threadIdx.x & 31) == 0) keys[threadIdx.x >> 5] = key;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < WARPS; ++w) key = keys[w] > key ? keys[w] : key;
            best_key[0] = key;
        }
        cluster_sync_all();
        key = 0;
        for (int r = 0; r < ctas; ++r) {
            const float4 o = ld_cluster_f4(best_key, r);
            const unsigned long long other =
                static_cast<unsigned long long>(__float_as_uint(o.y)) << 32 | __float_as_uint(o.x);
            key = other > key ? other : key;
        }
        if (key) {
            token = key_id(key);
        } else {        // no weight left: the target's likeliest token
            all = cluster_part(careful_part(row, lo, hi, c, warps), c, &parts[4], ctas);
            token = all.at;
        }
        token_p = weight(f32(row[token]), m, c) * inv_z;
        break;
    }
    if (writes) p.accepted[b] = n;
    if (rank == 0)
        for (int i = n + threadIdx.x; i < width; i += THREADS) {
            tokens[i] = i == n ? token : -1;
            probs[i] = i == n ? token_p : 0.0f;
        }
    cluster_sync_all();     // no CTA leaves while another may read its shared memory
}

// CTAs a request, by the vocabulary alone, so that a row's sums do not depend on the batch.
int cluster_ctas(int vocab) { return vocab > 32768 ? 8 : vocab > 16384 ? 4 : vocab > 8192 ? 2 : 1; }

template <typename T>
auto kernel_of(bool given, int probs_dtype) {
    if (!given) return verify_kernel<T, NoProbs>;
    if (probs_dtype == F32) return verify_kernel<T, float>;
    return probs_dtype == BF16 ? verify_kernel<T, __nv_bfloat16> : verify_kernel<T, __half>;
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
    const auto kernel = dtype == F32    ? kernel_of<float>(draft_probs, probs_dtype)
                        : dtype == BF16 ? kernel_of<__nv_bfloat16>(draft_probs, probs_dtype)
                                        : kernel_of<__half>(draft_probs, probs_dtype);
    const int ctas = cluster_ctas(vocab);
    ESP_REQUIRE(requests <= INT_MAX / ctas, ESP_ERR_INVALID, "esp_verify: %d requests", requests);
    if (const int rc = launch_cluster(kernel, dim3(static_cast<unsigned>(requests * ctas)), dim3(THREADS), 0, stream, true,
                                      ctas, p, ctas))
        return rc;
    return ok();
}
