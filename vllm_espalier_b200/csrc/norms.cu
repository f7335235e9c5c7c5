// The norms, gate and residual add between two blocks of a decoder, in one pass over the rows:
//   v = x (+ x2);  p = post(v);  r = a residual + b act(gate) p;  h = pre(r)
// all in fp32 from the inputs to one rounding an output. A layer norm takes its mean off the values it holds before it sums
// their squares, so a large mean costs no digits.
//
// Bytes bound it: each input read once, each output written once, about 40 instructions a value. Four forms:
//   block_norm_ring     many rows: bulk copies keep eight rows of a CTA on their way, whatever registers the threads hold.
//                       16384 x 2048 (two bf16 inputs, fp32 stream, row gate): 76 us = 6.1 TB/s, 95% of a plain copy; without
//                       the extras 50 us (83%: five barriers' and shuffles' latency a row begins to show)
//   block_norm_rows     up to a row a place on the GPU: the row in registers. One row 2.0 us, 32 rows 2.4 us: launch, one
//                       memory round trip, two reductions
//   block_norm_shifted  16-bit rows on any boundary, any width: 1023 x 2047, layer norms, a gate an element: 11 us against
//                       22 us with scalar loads, 3.2 us of bytes; its two layer norms' four reductions a row bound it
//   block_norm_kernel   what fits none of these (rows past 8192 columns, unusual mixes of types)
#include <cuda_runtime.h>

#include <math.h>

#include <algorithm>
#include <type_traits>

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

// sigmoid(g) = n / (1 + a) with a = exp(-|g|) and n = 1, or a for a negative g. a = 2^t (1 + r ln 2): t the rounded product
// |g| log2(e), r what the rounding and log2(e)'s own left out. From |g| = 104 on a negative g's rounds to 0. NaN stays NaN.
// At most 2.6 units of fp32 off (4 million values of g from -87 to 30).
__device__ __forceinline__ float sigmoid(float g) {
    constexpr float LOG2E = 1.44269502f, LOG2E_REST = 1.92596303e-8f, LN2 = 0.693147182f;
    float x, e, inv;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(fabsf(g)), "f"(104.0f));
    const float t = x * -LOG2E, r = fmaf(x, -LOG2E_REST, fmaf(x, -LOG2E, -t));
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(t));
    const float a = fmaf(e, r * LN2, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(1.0f + a));
    return (g < 0.0f ? a : 1.0f) * inv;
}

// SHORT, where both outputs are 16-bit: without r. That is up to (|g| + 4) 2^-24 of it off, at |g| = 88 a 40th of fp16's own
// rounding (and 0 below 2^-126). 8192 x 2048, a gate a value, all bf16: 43 us so, 47 with r, 50 by expf and a division.
template <bool SHORT = false>
__device__ __forceinline__ float activation(float g, int act) {
    if (act == ESP_ACT_SIGMOID) return SHORT ? __fdividef(1.0f, 1.0f + __expf(-g)) : sigmoid(g);
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

// Any width, alignment and mix of types: a CTA a row, the row in shared memory as fp32.
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

// ---------------------------------------------------------------------------------------------------------------
// The row in registers: thread i of NT holds VPT groups of VEC consecutive columns, group j at column (j NT + i) VEC.
// Every input of the row is asked for before the first sum, so a row costs one memory round trip, its reductions (one
// barrier each) and the stores. VEC 8: 16-byte loads, the weights asked for with the rest; VEC 1: any width and
// alignment, a register a value, so the weights (and always the biases) are read where they are used.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int VEC>
struct alignas(VEC * sizeof(T) >= 16 ? 16 : sizeof(T)) Group {
    T e[VEC];
};

__device__ __forceinline__ float f32(float v) { return v; }
__device__ __forceinline__ float f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// A group rounded to its type, two values an instruction where there are two.
template <int VEC>
__device__ __forceinline__ void rounded(const float (&v)[VEC], Group<float, VEC>& g) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) g.e[e] = v[e];
}
template <int VEC>
__device__ __forceinline__ void rounded(const float (&v)[VEC], Group<__half, VEC>& g) {
    if constexpr (VEC == 1) g.e[0] = __float2half_rn(v[0]);
    else
#pragma unroll
        for (int e = 0; e < VEC; e += 2) *reinterpret_cast<__half2*>(&g.e[e]) = __floats2half2_rn(v[e], v[e + 1]);
}
template <int VEC>
__device__ __forceinline__ void rounded(const float (&v)[VEC], Group<__nv_bfloat16, VEC>& g) {
    if constexpr (VEC == 1) g.e[0] = __float2bfloat16_rn(v[0]);
    else
#pragma unroll
        for (int e = 0; e < VEC; e += 2)
            *reinterpret_cast<__nv_bfloat162*>(&g.e[e]) = __floats2bfloat162_rn(v[e], v[e + 1]);
}

template <typename T, int VEC>
__device__ __forceinline__ void fetch(Group<T, VEC>& g, const void* base, size_t i) {
    g = *reinterpret_cast<const Group<T, VEC>*>(static_cast<const T*>(base) + i);
}

// Eight 16-bit values from any 2-byte boundary on, `n` of them the row's (the rest come out as anything): the 16-byte blocks
// that hold them (each has a byte of the row, so it is mapped memory) and a shift, the same for all of a row's groups.
template <typename T>
__device__ __forceinline__ void fetch_shifted(Group<T, 8>& g, const void* base, size_t i, int n) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(static_cast<const T*>(base) + i);
    const int s = a % 16;
    const uint4* from = reinterpret_cast<const uint4*>(a - s);
    uint4 lo = from[0], hi = {0, 0, 0, 0};
    if (s && 16 < s + 2 * n) hi = from[1];
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (s & 4)
#pragma unroll
        for (int k = 0; k < 7; ++k) w[k] = w[k + 1];
    if (s & 8)
#pragma unroll
        for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
    if (s & 2)
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
    g = *reinterpret_cast<const Group<T, 8>*>(w);
}

// The other way round, by all lanes of a warp with consecutive groups (n <= 0: none): a lane stores the 16-byte block in
// which its group starts, with the end of the group before it from its neighbour; at the ends of the warp and of the row
// the pieces of a block go one by one.
template <typename T>
__device__ __forceinline__ void store_shifted(const Group<T, 8>& g, void* base, size_t i, int n) {
    T* to = static_cast<T*>(base) + i;
    const int s = reinterpret_cast<uintptr_t>(to) % 16, lane = threadIdx.x & 31, first = (16 - s) / 2;   // of the group's in its block
    const uint32_t* o = reinterpret_cast<const uint32_t*>(&g);
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __shfl_up_sync(0xffffffffu, o[k], 1), w[k + 4] = o[k];
    const int next = __shfl_down_sync(0xffffffffu, n, 1);
    if (n <= 0) return;
    const bool block = s == 0 ? n == 8 : lane > 0 && n >= first;
    if (block) {
        const int skip = 16 - s;        // bytes of the two groups before the block
        if (s == 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = w[k + 4];
        } else {
            if (skip & 4)
#pragma unroll
                for (int k = 0; k < 7; ++k) w[k] = w[k + 1];
            if (skip & 8)
#pragma unroll
                for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
            if (skip & 2)
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(to) - s) = {w[0], w[1], w[2], w[3]};
    }
    // one by one: what is before the next block where this lane stored none, and what is in it where no lane stores that
    const bool followed = lane < 31 && next >= first;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n && (e < first ? !block : !followed)) to[e] = g.e[e];
}

// The sum over the CTA with one barrier; `scratch` (a word a warp) is this reduction's own.
template <int NT>
__device__ __forceinline__ float rows_sum(float v, float* scratch) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if (NT == 32) return v;
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    float4 s = *reinterpret_cast<const float4*>(scratch);       // NT is a multiple of 128
#pragma unroll
    for (int w = 4; w < NT / 32; w += 4) {
        const float4 u = *reinterpret_cast<const float4*>(scratch + w);
        s.x += u.x, s.y += u.y, s.z += u.z, s.w += u.w;
    }
    return (s.x + s.y) + (s.z + s.w);
}

template <bool SHIFT, typename T, int VEC>
__device__ __forceinline__ void fetch_any(Group<T, VEC>& g, const void* base, int c, int d) {
    if constexpr (SHIFT) {
        if (c < d) fetch_shifted(g, base, c, d - c);
    } else {
        fetch(g, base, c);
    }
}

// A group's values from the n-th on become 0.
template <int VEC>
__device__ __forceinline__ void zero_from(float (&v)[VEC], int n) {
    if (n < VEC)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (e >= n) v[e] = 0.0f;
}

// v becomes (v - mean) for a layer norm; inv the reciprocal root of its second moment. Columns past d hold 0 in v.
template <int NT, int VEC, int VPT>
__device__ __forceinline__ float rows_moments(float (&v)[VPT][VEC], int d, int kind, float eps, float (*scratch)[32]) {
    if (kind == ESP_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += v[j][e];
        const float mean = rows_sum<NT>(s, scratch[0]) / d;
#pragma unroll
        for (int j = 0; j < VPT; ++j)
            if ((j * NT + static_cast<int>(threadIdx.x)) * VEC < d) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[j][e] -= mean;
                if (VEC > 1) zero_from(v[j], d - (j * NT + static_cast<int>(threadIdx.x)) * VEC);
            }
    }
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) q = fmaf(v[j][e], v[j][e], q);
    return rsqrtf(rows_sum<NT>(q, scratch[1]) / d + eps);
}

// A row's inputs as a thread gets at them, group j at column c: held in registers, or read where they are used out of a
// stage of shared memory (x, x2, gate, residual one after another).
template <typename TX, typename TR, int VEC, int VPT>
struct InRegisters {
    Group<TX, VEC> x_[VPT], x2_[VPT], gate_[VPT];
    Group<TR, VEC> res_[VPT];
    __device__ __forceinline__ Group<TX, VEC> x(int j, int) const { return x_[j]; }
    __device__ __forceinline__ Group<TX, VEC> x2(int j, int) const { return x2_[j]; }
    __device__ __forceinline__ Group<TX, VEC> gate(int j, int) const { return gate_[j]; }
    __device__ __forceinline__ Group<TR, VEC> res(int j, int) const { return res_[j]; }
};
template <typename TX, typename TR, int VEC>
struct InStage {
    const unsigned char *x_, *x2_, *gate_, *res_;     // gate_: a row's, or the channels' in global memory
    template <typename T>
    static __device__ __forceinline__ Group<T, VEC> get(const unsigned char* p, int c) {
        return *reinterpret_cast<const Group<T, VEC>*>(p + c * sizeof(T));
    }
    __device__ __forceinline__ Group<TX, VEC> x(int, int c) const { return get<TX>(x_, c); }
    __device__ __forceinline__ Group<TX, VEC> x2(int, int c) const { return get<TX>(x2_, c); }
    __device__ __forceinline__ Group<TX, VEC> gate(int, int c) const { return get<TX>(gate_, c); }
    __device__ __forceinline__ Group<TR, VEC> res(int, int c) const { return get<TR>(res_, c); }
};
template <typename TW, int VEC, int VPT>
struct RowWeights {
    Group<TW, VEC> post_w[VPT], pre_w[VPT];
};

__device__ __forceinline__ bool gated(const NormParams& p) {
    return p.gate_kind == ESP_GATE_ELEMENT || p.gate_kind == ESP_GATE_CHANNEL;
}

template <typename TW, int VEC>
__device__ __forceinline__ void scale_by(float (&a)[VEC], const Group<TW, VEC>& w, float offset) {
    if (offset != 0.0f) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[e] *= offset + f32(w.e[e]);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[e] *= f32(w.e[e]);
    }
}

template <typename TW, int VEC, int NT, int VPT>
__device__ __forceinline__ void fetch_weights(RowWeights<TW, VEC, VPT>& w, const NormParams& p) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = (j * NT + static_cast<int>(threadIdx.x)) * VEC;
        if (c < p.op.d && p.op.post_w) fetch(w.post_w[j], p.op.post_w, c);
        if (c < p.op.d && p.op.pre_w) fetch(w.pre_w[j], p.op.pre_w, c);
    }
}

// Row t from its inputs to its outputs. Each term is a branch of the whole group, not of each value. WEIGHTS: the weights
// are in `w`, otherwise they are read where they are used.
template <typename TX, typename TR, typename TW, int VEC, int NT, int VPT, bool WEIGHTS, bool SHIFT = false, typename In>
__device__ __forceinline__ void norm_row(const NormParams& p, size_t t, const In& in, RowWeights<TW, VEC, VPT>& w,
                                         float (*scratch)[32]) {
    const int d = p.op.d;
    float scale = p.op.block_scale;
    if (p.gate_kind == ESP_GATE_ROW) scale *= activation(load1(p.gate, p.gate_dtype, t * p.gate_stride), p.op.gate_act);
    float v[VPT][VEC];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = (j * NT + static_cast<int>(threadIdx.x)) * VEC;
        if (c < d) {
            const Group<TX, VEC> x = in.x(j, c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[j][e] = f32(x.e[e]);
            if (p.x2) {
                const Group<TX, VEC> x2 = in.x2(j, c);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[j][e] += f32(x2.e[e]);
            }
            if (SHIFT) zero_from(v[j], d - c);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[j][e] = 0.0f;
        }
    }
    const float inv = p.op.post ? rows_moments<NT, VEC, VPT>(v, d, p.op.post, p.op.eps, scratch) : 1.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = (j * NT + static_cast<int>(threadIdx.x)) * VEC;
        if (!SHIFT && c >= d) continue;
        float(&a)[VEC] = v[j];
        if (p.op.post)
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] *= inv;
        if (p.op.post_w) {
            if (!WEIGHTS) fetch(w.post_w[j], p.op.post_w, c);
            scale_by(a, w.post_w[j], p.op.weight_offset);
        }
        if (p.op.post_b) {
            Group<TW, VEC> b;
            fetch_any<SHIFT>(b, p.op.post_b, c, d);
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] += f32(b.e[e]);
        }
        if (gated(p)) {
            const Group<TX, VEC> gate = in.gate(j, c);
            float g[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) g[e] = f32(gate.e[e]);
            if (p.op.gate_act != ESP_ACT_NONE)
#pragma unroll
                for (int e = 0; e < VEC; ++e) g[e] = activation<sizeof(TX) == 2 && sizeof(TR) == 2>(g[e], p.op.gate_act);
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] *= g[e];
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[e] *= scale;
        if (p.residual) {
            const Group<TR, VEC> res = in.res(j, c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] = fmaf(p.op.residual_scale, f32(res.e[e]), a[e]);
        }
        if (SHIFT) zero_from(a, d - c);
        if (p.r_out) {
            Group<TR, VEC> r;
            rounded(a, r);
            if constexpr (SHIFT) store_shifted(r, p.r_out, t * p.r_out_stride + c, min(8, d - c));
            else *reinterpret_cast<Group<TR, VEC>*>(static_cast<TR*>(p.r_out) + t * p.r_out_stride + c) = r;
        }
    }
    if (!p.op.pre) return;
    const float inv2 = rows_moments<NT, VEC, VPT>(v, d, p.op.pre, p.op.eps, scratch + 2);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = (j * NT + static_cast<int>(threadIdx.x)) * VEC;
        if (!SHIFT && c >= d) continue;
        float(&a)[VEC] = v[j];
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[e] *= inv2;
        if (p.op.pre_w) {
            if (!WEIGHTS) fetch(w.pre_w[j], p.op.pre_w, c);
            scale_by(a, w.pre_w[j], p.op.weight_offset);
        }
        if (p.op.pre_b) {
            Group<TW, VEC> b;
            fetch_any<SHIFT>(b, p.op.pre_b, c, d);
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] += f32(b.e[e]);
        }
        Group<TX, VEC> h;
        rounded(a, h);
        if constexpr (SHIFT) store_shifted(h, p.h_out, t * p.h_out_stride + c, min(8, d - c));
        else *reinterpret_cast<Group<TX, VEC>*>(static_cast<TX*>(p.h_out) + t * p.h_out_stride + c) = h;
    }
}

template <typename TX, typename TR, typename TW, int VEC, int NT, int VPT>
__global__ void __launch_bounds__(NT) block_norm_rows(NormParams p) {
    __shared__ __align__(16) float scratch[4][32];
    pdl_launch_dependents();
    pdl_wait();
    const size_t t = blockIdx.x;
    InRegisters<TX, TR, VEC, VPT> in;
    RowWeights<TW, VEC, VPT> w;
    const size_t gate_at = p.gate_kind == ESP_GATE_ELEMENT ? t * p.gate_stride : 0;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = (j * NT + static_cast<int>(threadIdx.x)) * VEC;
        if (c >= p.op.d) continue;
        fetch(in.x_[j], p.x, t * p.x_stride + c);
        if (p.x2) fetch(in.x2_[j], p.x2, t * p.x2_stride + c);
        if (p.residual) fetch(in.res_[j], p.residual, t * p.residual_stride + c);
        if (gated(p)) fetch(in.gate_[j], p.gate, gate_at + c);
    }
    if constexpr (VEC > 1) fetch_weights<TW, VEC, NT, VPT>(w, p);
    norm_row<TX, TR, TW, VEC, NT, VPT, (VEC > 1)>(p, t, in, w, scratch);
}

// 16-bit rows of any width and alignment by 16-byte loads and stores all the same: each group of eight shifted into place.
// Same columns a thread as block_norm_rows with VEC 8.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) block_norm_shifted(NormParams p) {
    __shared__ __align__(16) float scratch[4][32];
    pdl_launch_dependents();
    pdl_wait();
    const size_t t = blockIdx.x;
    InRegisters<T, T, 8, 1> in;
    RowWeights<T, 8, 1> w;
    const int c = threadIdx.x * 8, n = p.op.d - c;
    if (n > 0) {
        fetch_shifted(in.x_[0], p.x, t * p.x_stride + c, n);
        if (p.x2) fetch_shifted(in.x2_[0], p.x2, t * p.x2_stride + c, n);
        if (p.residual) fetch_shifted(in.res_[0], p.residual, t * p.residual_stride + c, n);
        if (gated(p)) fetch_shifted(in.gate_[0], p.gate, (p.gate_kind == ESP_GATE_ELEMENT ? t * p.gate_stride : 0) + c, n);
        if (p.op.post_w) fetch_shifted(w.post_w[0], p.op.post_w, c, n);
        if (p.op.pre_w) fetch_shifted(w.pre_w[0], p.op.pre_w, c, n);
    }
    norm_row<T, T, T, 8, NT, 1, true, true>(p, t, in, w, scratch);
}

// ---------------------------------------------------------------------------------------------------------------
// Many rows: a CTA walks its rows (blockIdx, + gridDim, ...), the next STAGES rows' inputs on their way into a ring of
// shared memory by bulk copies (one thread asks, an mbarrier a stage counts the bytes), so the copies in flight do not
// depend on how many registers the threads hold, and the weights stay in registers over the rows. Same columns a
// thread and same sums as block_norm_rows, so the same bits.
// ---------------------------------------------------------------------------------------------------------------
constexpr int MAX_STAGES = 8;
constexpr int RING_BYTES = 227 * 1024;          // an SM's shared memory for its CTAs' rings
constexpr int RING_FIXED = 4 * 1024;            // of it, a CTA's barriers, scratch and the 1 KB the system keeps, rounded up
// CTAs an SM: 1024 threads of them at 64 registers each (a thread with two groups needs twice that).
constexpr int ring_ctas(int threads, int groups) { return groups > 1 ? 1 : threads >= 64 ? 1024 / threads : 16; }

template <typename TX, typename TR, typename TW, int NT, int VPT>
__global__ void __launch_bounds__(NT, ring_ctas(NT, VPT)) block_norm_ring(NormParams p, unsigned rows, int stages) {
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ __align__(8) uint64_t full[MAX_STAGES];
    __shared__ __align__(16) float scratch[2][4][32];
    constexpr int VEC = 8;
    const int d = p.op.d, tid = threadIdx.x;
    const uint32_t bx = d * sizeof(TX), br = d * sizeof(TR);
    const bool gate_rows = p.gate_kind == ESP_GATE_ELEMENT;
    const uint32_t stage_bytes = bx * (1 + (p.x2 != nullptr) + gate_rows) + (p.residual ? br : 0);
    if (tid == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
    }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();
    const auto request = [&](unsigned row, int s) {         // thread 0
        uint32_t to = smem_addr(ring) + s * stage_bytes;
        mbar_arrive_expect_tx(&full[s], stage_bytes);
        bulk_g2s(to, static_cast<const TX*>(p.x) + row * p.x_stride, bx, &full[s]);
        to += bx;
        if (p.x2) bulk_g2s(to, static_cast<const TX*>(p.x2) + row * p.x2_stride, bx, &full[s]), to += bx;
        if (gate_rows) bulk_g2s(to, static_cast<const TX*>(p.gate) + row * p.gate_stride, bx, &full[s]), to += bx;
        if (p.residual) bulk_g2s(to, static_cast<const TR*>(p.residual) + row * p.residual_stride, br, &full[s]);
    };
    // (unsigned: rows end below 2^31, and a row past the last by less than MAX_STAGES grids is still none)
    const unsigned step = gridDim.x;
    if (tid == 0)
        for (int s = 0; s < stages && blockIdx.x + s * step < rows; ++s) request(blockIdx.x + s * step, s);
    RowWeights<TW, VEC, VPT> w;
    fetch_weights<TW, VEC, NT, VPT>(w, p);
    int s = 0, phase = 0, parity = 0;
    for (unsigned row = blockIdx.x; row < rows; row += step) {
        // A wait that gave up ends the CTA, all threads together, after a bounded wait for the copies still on their way.
        if (!__syncthreads_and(mbar_wait(&full[s], phase))) {
            if (tid == 0)
                for (int k = 0; k < stages; ++k) mbar_wait(&full[k], k < s ? phase ^ 1 : phase);
            return;
        }
        // that barrier also ends the row before: its stage can be filled again
        if (tid == 0 && row != blockIdx.x) {
            const unsigned next = row + (stages - 1) * step;
            if (next < rows) request(next, (s ? s : stages) - 1);
        }
        InStage<TX, TR, VEC> in;
        in.x_ = ring + s * stage_bytes;
        in.x2_ = in.x_ + bx;
        in.gate_ = gate_rows ? in.x2_ + (p.x2 ? bx : 0) : static_cast<const unsigned char*>(p.gate);
        in.res_ = in.x_ + stage_bytes - br;
        norm_row<TX, TR, TW, VEC, NT, VPT, true>(p, row, in, w, scratch[parity]);
        parity ^= 1;
        if (++s == stages) s = 0, phase ^= 1;
    }
}

constexpr int MAX_D = 49152;   // the row as fp32 in shared memory: 192 KB
bool known_dtype(int t) { return t == F16 || t == BF16 || t == F32; }

// Whether every row of a tensor starts on a 16-byte boundary (NULL: nothing to load).
bool vector_rows(const void* p, int dtype, long long stride) {
    return !p || (aligned(p, 16) && stride % (dtype == F32 ? 4 : 8) == 0);
}

struct RowsKernel {
    void (*run)(NormParams) = nullptr;
    void (*ring)(NormParams, unsigned, int) = nullptr;
    int threads = 0, ctas = 0;      // of a CTA; CTAs of the ring's kernel an SM
};

template <typename TX, typename TR, typename TW, int VEC, int NT, int VPT>
RowsKernel rows_instance() {
    if constexpr (VEC == 8)
        return {block_norm_rows<TX, TR, TW, VEC, NT, VPT>, block_norm_ring<TX, TR, TW, NT, VPT>, NT, ring_ctas(NT, VPT)};
    else return {block_norm_rows<TX, TR, TW, VEC, NT, VPT>, nullptr, NT, 0};
}

// The registers' kernel for this width, none where the row does not fit: the threads a row needs for one group each
// (two at most), so that a row's order of summation depends on its width and whether vector loads fit, not on the
// number of rows.
template <typename TX, typename TR, typename TW>
RowsKernel rows_kernel(int d, bool vec) {
    if (vec) {
        if (d <= 256) return rows_instance<TX, TR, TW, 8, 32, 1>();
        if (d <= 1024) return rows_instance<TX, TR, TW, 8, 128, 1>();
        if (d <= 2048) return rows_instance<TX, TR, TW, 8, 256, 1>();
        if (d <= 4096) return rows_instance<TX, TR, TW, 8, 512, 1>();
        if (d <= 8192) return rows_instance<TX, TR, TW, 8, 512, 2>();
        return {};
    }
    if constexpr (sizeof(TX) == 2 && std::is_same_v<TX, TR> && std::is_same_v<TX, TW>) {
        if (d <= 1024) return {block_norm_shifted<TX, 128>, nullptr, 128, 0};
        if (d <= 2048) return {block_norm_shifted<TX, 256>, nullptr, 256, 0};
        if (d <= 4096) return {block_norm_shifted<TX, 512>, nullptr, 512, 0};
        if (d <= 8192) return {block_norm_shifted<TX, 1024>, nullptr, 1024, 0};
    }
    if (d <= 2048) return rows_instance<TX, TR, TW, 1, 512, 4>();
    if (d <= 8192) return rows_instance<TX, TR, TW, 1, 1024, 8>();
    return {};
}

template <typename TX>
RowsKernel rows_kernel(const NormParams& p, bool vec) {
    const bool r32 = p.r_dtype == F32, w32 = p.op.w_dtype == F32;
    if (r32 && w32) return rows_kernel<TX, float, float>(p.op.d, vec);
    if constexpr (!std::is_same_v<TX, float>) {
        if (r32) return rows_kernel<TX, float, TX>(p.op.d, vec);
        if (w32) return rows_kernel<TX, TX, float>(p.op.d, vec);
        return rows_kernel<TX, TX, TX>(p.op.d, vec);
    }
    return {};
}

// The kernel for a call: the registers' one where its types are those a model mixes (x's own or fp32 for the stream and
// for the weights, x's own for a gate of more than a value a row), none otherwise.
RowsKernel rows_kernel(const NormParams& p) {
    const auto fits = [&](int dtype) { return dtype == p.x_dtype || dtype == F32; };
    const bool gated = p.gate_kind == ESP_GATE_CHANNEL || p.gate_kind == ESP_GATE_ELEMENT;
    if (!fits(p.r_dtype) || !fits(p.op.w_dtype) || (gated && p.gate_dtype != p.x_dtype)) return {};
    const bool vec = p.op.d % 8 == 0 && vector_rows(p.x, p.x_dtype, p.x_stride) &&
                     vector_rows(p.x2, p.x_dtype, p.x2_stride) &&
                     vector_rows(p.residual, p.r_dtype, p.residual_stride) &&
                     (!gated || vector_rows(p.gate, p.gate_dtype, p.gate_kind == ESP_GATE_ELEMENT ? p.gate_stride : 0)) &&
                     vector_rows(p.r_out, p.r_dtype, p.r_out_stride) && vector_rows(p.h_out, p.x_dtype, p.h_out_stride) &&
                     vector_rows(p.op.post_w, p.op.w_dtype, 0) && vector_rows(p.op.post_b, p.op.w_dtype, 0) &&
                     vector_rows(p.op.pre_w, p.op.w_dtype, 0) && vector_rows(p.op.pre_b, p.op.w_dtype, 0);
    if (p.x_dtype == BF16) return rows_kernel<__nv_bfloat16>(p, vec);
    if (p.x_dtype == F16) return rows_kernel<__half>(p, vec);
    return rows_kernel<float>(p, vec);
}

// Bytes of one row's inputs (a stage of the ring).
int row_bytes(const NormParams& p) {
    const int x = p.x_dtype == F32 ? 4 : 2, r = p.r_dtype == F32 ? 4 : 2;
    return p.op.d * (x * (1 + (p.x2 != nullptr) + (p.gate_kind == ESP_GATE_ELEMENT)) + (p.residual ? r : 0));
}

}  // namespace
}  // namespace esp

ESP_DEFINE_STATUS_READER(norms)

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
    if (const RowsKernel k = rows_kernel(p); k.run) {
        const int stages = k.ring ? std::min(MAX_STAGES, (RING_BYTES / k.ctas - RING_FIXED) / row_bytes(p)) : 0;
        // The ring where the rows outnumber its CTAs. 2048 wide bf16, ring / a CTA a row: 64 rows 3.1 / 2.7 us, 592 3.7 / 3.6,
        // 1184 5.9 / 5.9, 8192 34 / 37; 4096 wide with a fp32 stream: 148 rows 4.3 / 3.4 us, 1200 15.4 / 16.7, 4096 41 / 52.
        if (rows > static_cast<long long>(k.ctas) * device_sms() && stages >= 2) {
            const int smem = stages * row_bytes(p);
            if (const int rc = allow_any_smem(k.ring, smem)) return rc;
            if (const int rc = launch(k.ring, dim3(k.ctas * device_sms()), dim3(k.threads), smem, stream, true, p,
                                      static_cast<unsigned>(rows), stages))
                return rc;
            return ok();
        }
        if (const int rc = launch(k.run, dim3(static_cast<unsigned>(rows)), dim3(k.threads), 0, stream, true, p)) return rc;
        return ok();
    }
    const size_t smem = static_cast<size_t>(op->d) * 4;
    if (const int rc = allow_any_smem(block_norm_kernel, smem)) return rc;
    if (const int rc = launch(block_norm_kernel, dim3(static_cast<unsigned>(rows)), dim3(op->d <= 4096 ? 256 : 1024), smem,
                              stream, true, p))
        return rc;
    return ok();
}
