// Low-rank adapters of many requests at once beside a shared projection.
#include <cuda_runtime.h>

#include "common.cuh"
#include "host.hpp"

namespace esp {
namespace {

struct AdaptParams {
    esp_adapters_t ad;
    const void *x, *y;
    const int* ids;
    void* out;
    long long x_stride, y_stride, out_stride;
    int n;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// A CTA a row: the rank products by a warp each, then a column a thread.
template <typename T>
__global__ void adapt_kernel(AdaptParams p) {
    extern __shared__ float u[];        // [n_mats][rank]
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, slot = p.ids[t], lane = threadIdx.x & 31, cap = p.ad.rank, K = p.ad.k;
    const T* x = static_cast<const T*>(p.x) + t * p.x_stride;
    const T* y = static_cast<const T*>(p.y) + t * p.y_stride;
    T* out = static_cast<T*>(p.out) + t * p.out_stride;
    int rank = 0;
    if (slot >= 0 && slot < p.ad.slots) rank = p.ad.ranks ? min(max(p.ad.ranks[slot], 0), cap) : cap;
    const float scale = rank && p.ad.scales ? p.ad.scales[slot] : 1.0f;
    for (int j = threadIdx.x >> 5; j < p.ad.n_mats * cap; j += blockDim.x >> 5) {
        if (j % cap >= rank) continue;
        const T* a = static_cast<const T*>(p.ad.a) + (static_cast<size_t>(slot) * p.ad.n_mats * cap + j) * K;
        float s = 0.0f;
        for (int i = lane; i < K; i += 32) s = fmaf(to_f32(x[i]), to_f32(a[i]), s);
#pragma unroll
        for (int m = 16; m; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        if (lane == 0) u[j] = s;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.n; c += blockDim.x) {
        float s = 0.0f;
        if (rank) {
            int m = 0;
            for (int edge = p.ad.widths[0]; c >= edge; edge += p.ad.widths[++m]) {}
            const T* b = static_cast<const T*>(p.ad.b) + (static_cast<size_t>(slot) * p.n + c) * cap;
            for (int j = 0; j < rank; ++j) s = fmaf(u[m * cap + j], to_f32(b[j]), s);
        }
        out[c] = rank ? from_f32<T>(fmaf(scale, s, to_f32(y[c]))) : y[c];
    }
}

constexpr int MAX_SLOTS = 4096;

}  // namespace
}  // namespace esp

extern "C" size_t esp_adapt_ws_bytes(int, int) { return 0; }

extern "C" int esp_adapt(const esp_adapters_t* ad, const void* x, long long x_stride, const void* y, long long y_stride,
                         const int* ids, int t_rows, void* out, long long out_stride, void* ws, size_t ws_bytes,
                         void* stream) {
    using namespace esp;
    ESP_REQUIRE(ad, ESP_ERR_INVALID, "esp_adapt: adapters are NULL");
    ESP_REQUIRE(ad->dtype == F16 || ad->dtype == BF16, ESP_ERR_INVALID, "esp_adapt: adapters must be fp16 or bf16");
    ESP_REQUIRE(ad->slots >= 1 && ad->slots <= MAX_SLOTS && ad->n_mats >= 1 && ad->n_mats <= 4, ESP_ERR_INVALID,
                "esp_adapt: %d slots of %d matrices (1..%d slots, 1..4 matrices)", ad->slots, ad->n_mats, MAX_SLOTS);
    ESP_REQUIRE(ad->rank >= 8 && ad->rank <= 128 && ad->rank % 8 == 0, ESP_ERR_INVALID,
                "esp_adapt: rank %d is not a multiple of 8 in 8..128", ad->rank);
    ESP_REQUIRE(ad->k >= 8 && ad->k % 8 == 0, ESP_ERR_INVALID, "esp_adapt: k %d is not a multiple of 8", ad->k);
    long long n = 0;
    for (int m = 0; m < ad->n_mats; ++m) {
        ESP_REQUIRE(ad->widths[m] >= 8 && ad->widths[m] % 8 == 0, ESP_ERR_INVALID,
                    "esp_adapt: width %d is not a multiple of 8", ad->widths[m]);
        n += ad->widths[m];
    }
    ESP_REQUIRE(n < (1ll << 31), ESP_ERR_INVALID, "esp_adapt: %lld columns", n);
    ESP_REQUIRE(t_rows >= 0, ESP_ERR_INVALID, "esp_adapt: %d rows", t_rows);
    if (t_rows == 0) return ok();
    ESP_REQUIRE(ad->a && ad->b && x && y && ids && out, ESP_ERR_INVALID, "esp_adapt: null pointer");
    ESP_REQUIRE(aligned(ad->a, 16) && aligned(ad->b, 16) && aligned(x, 16) && aligned(y, 16) && aligned(out, 16) &&
                    x_stride % 8 == 0 && y_stride % 8 == 0 && out_stride % 8 == 0,
                ESP_ERR_INVALID, "esp_adapt: rows and weights must be 16-byte aligned");
    const size_t need = esp_adapt_ws_bytes(t_rows, ad->slots);
    ESP_REQUIRE(need == 0 || (ws && aligned(ws, 16) && ws_bytes >= need), ESP_ERR_SCRATCH,
                "esp_adapt: workspace of %zu bytes, %zu needed (16-byte aligned)", ws ? ws_bytes : 0, need);
    const AdaptParams p{*ad, x, y, ids, out, x_stride, y_stride, out_stride, static_cast<int>(n)};
    const auto kernel = ad->dtype == F16 ? adapt_kernel<__half> : adapt_kernel<__nv_bfloat16>;
    if (const int rc = launch(kernel, dim3(t_rows), dim3(256), sizeof(float) * ad->n_mats * ad->rank, stream, true, p))
        return rc;
    return ok();
}
