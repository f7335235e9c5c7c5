// The norms, gate and residual add between two blocks of a decoder, in one pass over the rows.
#include <cuda_runtime.h>

#include <math.h>

#include "common.cuh"
#include "host.hpp"

namespace esp {
namespace {

struct NormParams {
    esp_block_norm_op_t op;
    const void *x, *x2, *residual, *gate;
    void *r_out, *h_out;
    long long x_stride, x2_stride, residual_stride, gate_stride, r_out_stride, h_out_stride;
    int x_dtype, r_dtype, gate_kind, gate_dtype;
};

__device__ __forceinline__ float load1(const void* p, int dtype, size_t i) {
    if (dtype == F32) return static_cast<const float*>(p)[i];
    if (dtype == BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store1(void* p, int dtype, size_t i, float v) {
    if (dtype == F32) static_cast<float*>(p)[i] = v;
    else if (dtype == BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

__device__ __forceinline__ float activation(float g, int act) {
    if (act == ESP_ACT_SIGMOID) return 1.0f / (1.0f + expf(-g));
    if (act == ESP_ACT_TANH) return tanhf(g);
    return g;
}

// The sum of v over the CTA, in every thread (scratch: 32 floats, reused by the next call after its first barrier).
__device__ __forceinline__ float block_sum(float v, float* scratch) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    for (unsigned w = 0; w < (blockDim.x + 31) / 32; ++w) s += scratch[w];
    return s;
}

// Mean (layer norm) and reciprocal root of the second moment of a row held in shared memory.
__device__ __forceinline__ void moments(const float* row, int d, int kind, float eps, float* scratch, float& mean,
                                        float& inv) {
    mean = 0.0f;
    if (kind == ESP_NORM_LAYER) {
        float s = 0.0f;
        for (int i = threadIdx.x; i < d; i += blockDim.x) s += row[i];
        mean = block_sum(s, scratch) / d;
    }
    float q = 0.0f;
    for (int i = threadIdx.x; i < d; i += blockDim.x) q += (row[i] - mean) * (row[i] - mean);
    inv = rsqrtf(block_sum(q, scratch) / d + eps);
}

__device__ __forceinline__ float affine(float v, const NormParams& p, const void* w, const void* b, int i) {
    if (w) v *= p.op.weight_offset + load1(w, p.op.w_dtype, i);
    return b ? v + load1(b, p.op.w_dtype, i) : v;
}

// Any width, alignment and type: a CTA a row, the row in shared memory as fp32.
__global__ void block_norm_kernel(NormParams p) {
    extern __shared__ float row[];
    __shared__ float scratch[32];
    pdl_launch_dependents();
    pdl_wait();
    const size_t t = blockIdx.x;
    const int d = p.op.d;
    for (int i = threadIdx.x; i < d; i += blockDim.x) {
        float v = load1(p.x, p.x_dtype, t * p.x_stride + i);
        if (p.x2) v += load1(p.x2, p.x_dtype, t * p.x2_stride + i);
        row[i] = v;
    }
    float mean = 0.0f, inv = 1.0f;
    if (p.op.post) moments(row, d, p.op.post, p.op.eps, scratch, mean, inv);
    float scale = p.op.block_scale;
    if (p.gate_kind == ESP_GATE_ROW) scale *= activation(load1(p.gate, p.gate_dtype, t * p.gate_stride), p.op.gate_act);
    for (int i = threadIdx.x; i < d; i += blockDim.x) {
        float v = row[i];
        if (p.op.post) v = affine((v - mean) * inv, p, p.op.post_w, p.op.post_b, i);
        if (p.gate_kind == ESP_GATE_CHANNEL) v *= activation(load1(p.gate, p.gate_dtype, i), p.op.gate_act);
        if (p.gate_kind == ESP_GATE_ELEMENT)
            v *= activation(load1(p.gate, p.gate_dtype, t * p.gate_stride + i), p.op.gate_act);
        v *= scale;
        if (p.residual) v = fmaf(p.op.residual_scale, load1(p.residual, p.r_dtype, t * p.residual_stride + i), v);
        row[i] = v;
        if (p.r_out) store1(p.r_out, p.r_dtype, t * p.r_out_stride + i, v);
    }
    if (!p.op.pre) return;
    moments(row, d, p.op.pre, p.op.eps, scratch, mean, inv);
    for (int i = threadIdx.x; i < d; i += blockDim.x)
        store1(p.h_out, p.x_dtype, t * p.h_out_stride + i, affine((row[i] - mean) * inv, p, p.op.pre_w, p.op.pre_b, i));
}

constexpr int MAX_D = 49152;   // the row as fp32 in shared memory: 192 KB
bool known_dtype(int t) { return t == F16 || t == BF16 || t == F32; }

}  // namespace
}  // namespace esp

extern "C" int esp_block_norm(const esp_block_norm_op_t* op, const void* x, long long x_stride, const void* x2,
                              long long x2_stride, int x_dtype, const void* residual, long long residual_stride,
                              int r_dtype, const void* gate, int gate_kind, int gate_dtype, long long gate_stride,
                              void* r_out, long long r_out_stride, void* h_out, long long h_out_stride,
                              long long rows, void* stream) {
    using namespace esp;
    ESP_REQUIRE(op, ESP_ERR_INVALID, "esp_block_norm: op is NULL");
    ESP_REQUIRE(op->d >= 1 && op->d <= MAX_D, ESP_ERR_INVALID, "esp_block_norm: d %d outside 1..%d", op->d, MAX_D);
    ESP_REQUIRE(op->post >= ESP_NORM_NONE && op->post <= ESP_NORM_LAYER && op->pre >= ESP_NORM_NONE &&
                    op->pre <= ESP_NORM_LAYER && op->gate_act >= ESP_ACT_NONE && op->gate_act <= ESP_ACT_TANH,
                ESP_ERR_INVALID, "esp_block_norm: unknown norm or gate activation");
    ESP_REQUIRE(known_dtype(x_dtype) && known_dtype(r_dtype) && known_dtype(op->w_dtype), ESP_ERR_INVALID,
                "esp_block_norm: unknown dtype");
    ESP_REQUIRE(rows >= 0 && rows < (1ll << 31), ESP_ERR_INVALID, "esp_block_norm: %lld rows", rows);
    if (rows == 0) return ok();
    ESP_REQUIRE(x, ESP_ERR_INVALID, "esp_block_norm: x is NULL");
    ESP_REQUIRE(gate_kind >= ESP_GATE_NONE && gate_kind <= ESP_GATE_ELEMENT, ESP_ERR_INVALID,
                "esp_block_norm: unknown gate kind %d", gate_kind);
    ESP_REQUIRE((gate_kind == ESP_GATE_NONE) == (gate == nullptr), ESP_ERR_INVALID,
                "esp_block_norm: the gate pointer and its kind disagree");
    ESP_REQUIRE(gate_kind == ESP_GATE_NONE || known_dtype(gate_dtype), ESP_ERR_INVALID,
                "esp_block_norm: unknown gate dtype");
    ESP_REQUIRE((op->pre == ESP_NORM_NONE) == (h_out == nullptr), ESP_ERR_INVALID,
                "esp_block_norm: h_out and the norm before the next block disagree");
    ESP_REQUIRE(r_out || h_out, ESP_ERR_INVALID, "esp_block_norm: no output");
    NormParams p{*op, x, x2, residual, gate, r_out, h_out, x_stride, x2_stride, residual_stride, gate_stride,
                 r_out_stride, h_out_stride, x_dtype, r_dtype, gate_kind, gate_dtype};
    const size_t smem = static_cast<size_t>(op->d) * 4;
    if (const int rc = allow_smem(block_norm_kernel, smem)) return rc;
    if (const int rc = launch(block_norm_kernel, dim3(static_cast<unsigned>(rows)), dim3(op->d <= 4096 ? 256 : 1024), smem,
                              stream, true, p))
        return rc;
    return ok();
}
