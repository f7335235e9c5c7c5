// Low-rank adapters of many requests at once beside a shared projection.
//
// out[t] = y[t] + scale (x[t] A^T) B^T. Rows are grouped by adapter into tiles; a cluster of CTAs takes a tile. Each CTA
// multiplies its share of k (u = x A^T, partial), the partial sums meet in distributed shared memory (each CTA joins its
// share of the tile's rows and stores them into all), and each CTA multiplies u by its share of the columns of B and adds y.
// Both products are m16n8k16 matrix instructions. The contraction index may be taken in any order as long as both operands
// agree, so a lane loads eight consecutive values (16 bytes) of a row and uses them as the fragments of two instructions.
//
// The sum over k has one order for every batch: eight segments of k, each in ascending order in one accumulator, joined as
// a balanced tree ((0 + 1) + (2 + 3)) + ((4 + 5) + (6 + 7)), whichever CTA has which. So a row's bits do not depend on the
// tile's size or on the rows beside it.
//
// The products are small (rank 16: 35 flops a byte), so bytes bound a large batch and latency a small one. mma.sync and not
// tcgen05: the tensor pipe is 7 to 20% busy, u is born in registers and goes back into them, and both paths share one order
// of summation. Measured (q | k | v of 2048 -> 5120, bf16, rank 16 unless said): one token 5.9 us (ids, one round trip to A,
// two cluster barriers, one to B and y), 48 rows of 64 adapters of rank 32 14 us, 8192 rows of 12 prompts 61 us = 3.3 TB/s
// (52% of a plain copy; plan 4 us, the rest is stage hand-overs), 3001 rows at rank 64 81 us (15%: the parts that hold u in
// fp32 treble the second product, and sums or parts and the ring leave one CTA an SM).
#include <cuda_runtime.h>

#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "host.hpp"

namespace esp {
namespace {

constexpr int SEGMENTS = 8, MAX_SLOTS = 4096;
// Up to this many rows every CTA finds its tile's rows itself, above it a launch of its own does: 17 / 32 / 48 / 64 rows 8.0 /
// 8.2 / 9.1 / 10.7 us so, 10.3 / 11.2 / 11.2 / 11.4 with the plan.
constexpr int NO_PLAN = 64;

struct AdaptParams {
    esp_adapters_t ad;
    const void *x, *y;
    const int* ids;
    void* out;
    const int* plan;        // tiles, then rows (above NO_PLAN rows)
    long long x_stride, y_stride, out_stride;
    int rows, n, max_tiles;
};

// A tile of the plan: its adapter (-1: none), where its rows start in the list of rows, how many there are.
struct Tile {
    int slot, first, count, unused;
};

__device__ __forceinline__ int slot_of(const AdaptParams& p, int t) {
    const int id = p.ids[t];
    return id >= 0 && id < p.ad.slots ? id : -1;
}

// ---------------------------------------------------------------------------------------------------------------
// The plan: rows sorted by adapter and cut into tiles, by one CTA. Places within an adapter are taken by atomics, so the
// order of a tile's rows may change from run to run; no row's result depends on it.
// ---------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(1024) plan_kernel(AdaptParams p, Tile* tiles, int* rows, int m) {
    extern __shared__ int count[];      // [slots + 1]: the rows of a slot, then where its next row goes; last: no adapter
    __shared__ int warp_rows[32], warp_tiles[32], base_rows, base_tiles;
    pdl_launch_dependents();
    pdl_wait();
    const int slots = p.ad.slots + 1, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int s = tid; s < slots; s += 1024) count[s] = 0;
    if (tid == 0) base_rows = base_tiles = 0;
    __syncthreads();
    // PER rows a thread at once, 1024 apart: their ids are on the way together
    constexpr int PER = 8;
    int ids[PER];
    const auto load = [&](int t0) {
#pragma unroll
        for (int i = 0; i < PER; ++i) ids[i] = t0 + i * 1024 + tid < p.rows ? slot_of(p, t0 + i * 1024 + tid) : -2;
    };
    for (int t0 = 0; t0 < p.rows; t0 += PER * 1024) {
        load(t0);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (t0 + i * 1024 >= p.rows) break;
            const unsigned same = __match_any_sync(0xffffffffu, ids[i]);
            if (ids[i] >= -1 && lane == __ffs(same) - 1) atomicAdd(&count[ids[i] < 0 ? slots - 1 : ids[i]], __popc(same));
        }
    }
    __syncthreads();
    // exclusive sums over the slots of their rows and tiles, 1024 slots a round
    for (int s0 = 0; s0 < slots; s0 += 1024) {
        const int s = s0 + tid, c = s < slots ? count[s] : 0, n = (c + m - 1) / m;
        int sum_c = c, sum_n = n;
#pragma unroll
        for (int k = 1; k < 32; k <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, sum_c, k), b = __shfl_up_sync(0xffffffffu, sum_n, k);
            if (lane >= k) sum_c += a, sum_n += b;
        }
        if (lane == 31) warp_rows[warp] = sum_c, warp_tiles[warp] = sum_n;
        __syncthreads();
        if (warp == 0) {
            int a = warp_rows[lane], b = warp_tiles[lane];
#pragma unroll
            for (int k = 1; k < 32; k <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, a, k), v = __shfl_up_sync(0xffffffffu, b, k);
                if (lane >= k) a += u, b += v;
            }
            warp_rows[lane] = a, warp_tiles[lane] = b;
        }
        __syncthreads();
        const int at = base_rows + sum_c - c + (warp ? warp_rows[warp - 1] : 0);
        const int tile = base_tiles + sum_n - n + (warp ? warp_tiles[warp - 1] : 0);
        for (int i = 0; i < n; ++i)
            tiles[tile + i] = {s == slots - 1 ? -1 : s, at + i * m, min(m, c - i * m), 0};
        if (s < slots) count[s] = at;
        __syncthreads();
        if (tid == 0) base_rows += warp_rows[31], base_tiles += warp_tiles[31];
        __syncthreads();
    }
    for (int i = base_tiles + tid; i < p.max_tiles; i += 1024) tiles[i] = {-1, 0, 0, 0};
    for (int t0 = 0; t0 < p.rows; t0 += PER * 1024) {
        if (p.rows > PER * 1024) load(t0);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (t0 + i * 1024 >= p.rows) break;
            const unsigned same = __match_any_sync(0xffffffffu, ids[i]);
            const int leader = __ffs(same) - 1;
            int at = 0;
            if (ids[i] >= -1 && lane == leader) at = atomicAdd(&count[ids[i] < 0 ? slots - 1 : ids[i]], __popc(same));
            at = __shfl_sync(0xffffffffu, at, leader);
            if (ids[i] >= -1) rows[at + __popc(same & ((1u << lane) - 1))] = t0 + i * 1024 + tid;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Matrix fragments
// ---------------------------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float2 unpack(uint32_t v, __half) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
__device__ __forceinline__ float2 unpack(uint32_t v, __nv_bfloat16) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}
__device__ __forceinline__ uint32_t pack(float a, float b, __half) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// ---------------------------------------------------------------------------------------------------------------
// What both kernels below share. Inner columns of a tile: RP = 16 RANK16 a matrix (the capacity in steps of 16), u of all
// matrices side by side.
// ---------------------------------------------------------------------------------------------------------------
// u's parts of 16 bits each, which add up to it: three of bf16's 8 bits hold an fp32 sum's 24, two of fp16's 11 with their
// rounding to nearest miss at most its last one.
template <typename T>
constexpr int PARTS = std::is_same_v<T, __half> ? 2 : 3;

// Elements between rows of u's parts: 64 bytes past a multiple of 128, so that the eight lanes of a quarter load meet
// every bank once.
__host__ __device__ constexpr int u_stride(int cols) { return cols + (192 - cols * 2 % 128) % 128 / 2; }

// Shared memory of a tile: sums [M][cols] fp32 of this CTA, then (or over them) u's parts [PARTS][M][stride] and, of fp16, the
// factors [M][4] of a row's matrices.
template <typename T>
struct Inner {
    float* sums;
    T* part;
    float* factor;
    int cols, stride, part_size;        // elements from a row and from a part to the next
    __device__ __forceinline__ Inner(unsigned char* at, int m, int cols_, bool over)
        : cols(cols_), stride(u_stride(cols_)), part_size(m * stride) {
        sums = reinterpret_cast<float*>(at);
        part = reinterpret_cast<T*>(over ? sums : sums + m * cols);
        factor = reinterpret_cast<float*>(part + PARTS<T> * part_size);
    }
};
constexpr int sums_bytes(int m, int cols) { return m * cols * 4; }
constexpr int parts_bytes(int m, int cols, int parts) { return m * (parts * u_stride(cols) * 2 + (parts == 2 ? 16 : 0)); }

// The adapter of a slot: its rank in whole steps of 8 (0: nothing to add), its matrices.
template <typename T>
struct Adapter {
    const T *a, *b;
    int r8, tiles_a_mat, n_tiles, cap, k;     // n8 tiles of inner columns: a matrix, all
    __device__ __forceinline__ Adapter(const AdaptParams& p, int slot) : r8(0), cap(p.ad.rank), k(p.ad.k) {
        if (slot >= 0) r8 = p.ad.ranks ? (min(max(p.ad.ranks[slot], 0), cap) + 7) / 8 * 8 : cap;
        tiles_a_mat = r8 / 8, n_tiles = p.ad.n_mats * tiles_a_mat;
        const size_t s = slot < 0 ? 0 : slot;
        a = static_cast<const T*>(p.ad.a) + s * p.ad.n_mats * cap * k;
        b = static_cast<const T*>(p.ad.b) + s * p.n * cap;
    }
    __device__ __forceinline__ const T* a_row(int t, int r) const {        // row r of tile t of A
        const int m = t / tiles_a_mat;
        return a + (static_cast<size_t>(m) * cap + (t - m * tiles_a_mat) * 8 + r) * k;
    }
    template <int RP>
    __device__ __forceinline__ int column(int t) const {                   // the tile's first column in sums and u
        const int m = t / tiles_a_mat;
        return m * RP + (t - m * tiles_a_mat) * 8;
    }
};

// A block of 32 columns of the output (never across matrices): its matrix, first column, and how many columns are left of
// the matrix from there on.
struct Block {
    int m, col, left;
};
__device__ __forceinline__ Block block_at(const AdaptParams& p, int b) {
    int col = 0;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const int w = p.ad.widths[m], n = (w + 31) / 32;
        if (m == p.ad.n_mats - 1 || b < n) return {m, col + b * 32, w - b * 32};
        b -= n, col += w;
    }
    return {0, 0, 0};
}
__device__ __forceinline__ int block_count(const AdaptParams& p) {
    int n = 0;
#pragma unroll
    for (int m = 0; m < 4; ++m)
        if (m < p.ad.n_mats) n += (p.ad.widths[m] + 31) / 32;
    return n;
}

__device__ __forceinline__ int segment_at(int blocks, int s) { return blocks * s / SEGMENTS; }     // its first block of 32 k

// Rows without an adapter: y itself, this CTA's share of the columns.
template <typename T>
__device__ __forceinline__ void copy_rows(const AdaptParams& p, const int* tile_rows, int count, int rank, int ctas, int warps) {
    if (p.out == p.y && p.out_stride == p.y_stride) return;
    const int from = p.n / 8 * rank / ctas, to = p.n / 8 * (rank + 1) / ctas;
    for (int r = threadIdx.x / 32; r < count; r += warps)
        for (int c = from + threadIdx.x % 32; c < to; c += 32)
            reinterpret_cast<uint4*>(static_cast<T*>(p.out) + tile_rows[r] * p.out_stride)[c] =
                reinterpret_cast<const uint4*>(static_cast<const T*>(p.y) + tile_rows[r] * p.y_stride)[c];
}

// The cluster's sums of one row (a warp), joined as the tree over the segments: a lane's columns 2 lane + 64 i and the next.
template <typename T, int RANK16, int CTAS>
__device__ __forceinline__ void join_row(const Inner<T>& u, int r, int r8, float2 (&v)[RANK16]) {
    constexpr int RP = RANK16 * 16;
#pragma unroll
    for (int i = 0; i < RANK16; ++i) {
        const int c = threadIdx.x % 32 * 2 + i * 64;
        v[i] = {0.0f, 0.0f};
        if (c < u.cols && c % RP < r8) {
            float2 o[CTAS];
#pragma unroll
            for (int w = 0; w < CTAS; ++w) o[w] = ld_cluster_f2(u.sums + r * u.cols + c, w);
#pragma unroll
            for (int n = 1; n < CTAS; n *= 2)
#pragma unroll
                for (int w = 0; w < CTAS; w += 2 * n) o[w].x += o[w + n].x, o[w].y += o[w + n].y;
            v[i] = o[0];
        }
    }
}

// Store it into every CTA as its parts, so that the second product holds it in fp32 as the sum had it. For fp16 the values of
// each matrix are first scaled by a power of two that brings the row's largest to [2^14, 2^15): one of 2^-15 of that or more
// keeps its 24 bits, a smaller one is held to 2^-39 of the largest. The matrix's factor comes back with the adapter's scale.
template <typename T, int RANK16, int CTAS>
__device__ __forceinline__ void store_row(const Inner<T>& u, int r, const float2 (&v)[RANK16], float scale) {
    constexpr int RP = RANK16 * 16;
    const int lane = threadIdx.x % 32;
    float up[RANK16];
    if constexpr (std::is_same_v<T, __half>) {
        float top[RANK16];      // of a lane's columns, then of their matrix: RP / 2 lanes of an i, or two i of all lanes
#pragma unroll
        for (int i = 0; i < RANK16; ++i) top[i] = fmaxf(fabsf(v[i].x), fabsf(v[i].y));
#pragma unroll
        for (int i = 0; i < RANK16; ++i) {
            if (RANK16 == 8 && i % 2 == 0) top[i] = fmaxf(top[i], top[(i + 1) % RANK16]);
            if (RANK16 == 8 && i % 2) {
                top[i] = top[i - 1];
                continue;
            }
#pragma unroll
            for (int k = RP < 64 ? RP / 4 : 16; k; k >>= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], k));
        }
#pragma unroll
        for (int i = 0; i < RANK16; ++i) {
            const int c = lane * 2 + i * 64, to = c % RP / 2;
            const int e = max(static_cast<int>(__float_as_uint(top[i]) >> 23) - 127 - 14, -113);
            up[i] = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            if (c < u.cols && to < CTAS)
                st_cluster_u32(u.factor + r * 4 + c / RP, to,
                               __float_as_uint(scale * __uint_as_float(static_cast<uint32_t>(127 + e) << 23)));
        }
    }
#pragma unroll
    for (int i = 0; i < RANK16; ++i) {
        const int c = lane * 2 + i * 64;
        if (c >= u.cols) continue;
        float a = v[i].x, b = v[i].y;
        if constexpr (std::is_same_v<T, __half>) a *= up[i], b *= up[i];
#pragma unroll
        for (int k = 0; k < PARTS<T>; ++k) {
            const uint32_t bits = pack(a, b, T());
            const float2 back = unpack(bits, T());
            // (an infinite part leaves nothing to the others)
            a = isinf(back.x) ? 0.0f : a - back.x, b = isinf(back.y) ? 0.0f : b - back.y;
#pragma unroll
            for (int w = 0; w < CTAS; ++w) st_cluster_u32(u.part + k * u.part_size + r * u.stride + c, w, bits);
        }
    }
}

// What row r's sums over u of matrix m are multiplied by.
template <typename T>
__device__ __forceinline__ float factor_of(const Inner<T>& u, int r, int m, float scale) {
    if constexpr (std::is_same_v<T, __half>) return u.factor[r * 4 + m];
    else return scale;
}

// The fragments of u's steps s and s + 1 of a lane's two rows (g and g + 8 from `u` on).
template <int RANK16, typename T>
__device__ __forceinline__ void u_fragments(const T* u, int stride, int s, int q, uint32_t (&f)[2][4]) {
    if constexpr (RANK16 == 1) {
        const uint2 a = *reinterpret_cast<const uint2*>(u + q * 4), b = *reinterpret_cast<const uint2*>(u + 8 * stride + q * 4);
        f[0][0] = a.x, f[0][1] = b.x, f[0][2] = a.y, f[0][3] = b.y;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(u + s * 16 + q * 8);
        const uint4 b = *reinterpret_cast<const uint4*>(u + 8 * stride + s * 16 + q * 8);
        f[0][0] = a.x, f[0][1] = b.x, f[0][2] = a.y, f[0][3] = b.y;
        f[1][0] = a.z, f[1][1] = b.z, f[1][2] = a.w, f[1][3] = b.w;
    }
}

// u times a block of B into acc. The four n8 tiles of a block take columns so that a lane ends up with eight consecutive
// ones: tile j's column c is 8 (c / 2) + 2 j + c % 2 of the block; w(j, s) gives the lane's values of B's row for its
// column g of tile j (eight of steps s and s + 1; four of the one step of RANK16 1). The order of the products that meet in
// a value: two steps of the first part, of the second, ..., the next two steps.
template <typename T, int RANK16, typename W>
__device__ __forceinline__ void second_product(float (&acc)[4][4], const Inner<T>& u, int at, int r8, int q, W w) {
#pragma unroll
    for (int s = 0; s < RANK16; s += 2) {
        if (s * 16 >= r8) break;
        uint4 k[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = w(j, s);
#pragma unroll
        for (int i = 0; i < PARTS<T>; ++i) {
            uint32_t f[2][4];
            u_fragments<RANK16>(u.part + i * u.part_size + at, u.stride, s, q, f);
#pragma unroll
            for (int j = 0; j < 4; ++j) mma<T>(acc[j], f[0], k[j].x, k[j].y);
            if constexpr (RANK16 > 1)
#pragma unroll
                for (int j = 0; j < 4; ++j) mma<T>(acc[j], f[1], k[j].z, k[j].w);
        }
    }
}

// Eight values of y plus f times a row of acc (e: 0 or 2, its first element), rounded once.
template <typename T>
__device__ __forceinline__ uint4 added(const uint4& y, const float (&acc)[4][4], int e, float f) {
    uint4 o;
    const uint32_t* from = &y.x;
    uint32_t* to = &o.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 v = unpack(from[j], T());
        to[j] = pack(fmaf(f, acc[j][e], v.x), fmaf(f, acc[j][e + 1], v.y), T());
    }
    return o;
}

// ---------------------------------------------------------------------------------------------------------------
// Few rows an adapter: tiles of 16 rows, eight CTAs of eight warps, operands straight from global memory, the loads of many
// blocks of k asked for before the first product.
// ---------------------------------------------------------------------------------------------------------------
constexpr int FEW_ROWS = 16, FEW_WARPS = 8, FEW_CTAS = 8;

template <typename T, int RANK16>
__global__ void __launch_bounds__(FEW_WARPS * 32, 2) adapt_few(AdaptParams p) {
    constexpr int M = FEW_ROWS, WARPS = FEW_WARPS, THREADS = WARPS * 32, RP = RANK16 * 16;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int tile_rows[M];
    __shared__ int tile_slot, tile_count, found;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    const int rank = blockIdx.x % FEW_CTAS, tile = blockIdx.x / FEW_CTAS;
    const Inner<T> u(smem, M, p.ad.n_mats * RP, false);
    pdl_launch_dependents();
    pdl_wait();

    // The tile's adapter and rows.
    if (p.plan) {
        const Tile mine = reinterpret_cast<const Tile*>(p.plan)[tile];
        if (mine.count == 0) return;        // (the whole cluster: one tile)
        const int* rows = p.plan + 4 * p.max_tiles + mine.first;
        if (tid < M) tile_rows[tid] = tid < mine.count ? rows[tid] : -1;
        if (tid == 0) tile_slot = mine.slot, tile_count = mine.count;
    } else {
        // Tile j is row j's if the rows of its adapter before it fill whole tiles; it takes the next M of them.
        const int slot = slot_of(p, tile);
        if (tid < M) tile_rows[tid] = -1;
        if (tid == 0) tile_slot = slot;
        __syncthreads();
        if (warp == 0) {
            int before = 0, taken = 0;
            for (int t0 = 0; t0 < p.rows; t0 += 32) {
                const int t = t0 + lane;
                const unsigned same = __ballot_sync(0xffffffffu, t < p.rows && slot_of(p, t) == slot);
                const unsigned from = tile <= t0 ? 0xffffffffu : tile >= t0 + 32 ? 0u : ~0u << (tile - t0);
                before += __popc(same & ~from);
                const int at = taken + __popc(same & from & ((1u << lane) - 1));
                if ((same & from) >> lane & 1 && at < M) tile_rows[at] = t;
                taken += __popc(same & from);
            }
            if (lane == 0) tile_count = min(taken, M), found = before % M == 0;
        }
        __syncthreads();
        if (!found) return;
    }
    __syncthreads();
    const int slot = tile_slot, count = tile_count;
    const Adapter<T> ad(p, slot);
    if (ad.r8 == 0) return copy_rows<T>(p, tile_rows, count, rank, FEW_CTAS, WARPS);
    const T* x = static_cast<const T*>(p.x);
    const T* y = static_cast<const T*>(p.y);
    T* out = static_cast<T*>(p.out);
    const int blocks = block_count(p), block_lo = blocks * rank / FEW_CTAS, block_hi = blocks * (rank + 1) / FEW_CTAS;
    if (block_lo < block_hi) {      // what the second product will read, into L2 meanwhile
        const Block a = block_at(p, block_lo), z = block_at(p, block_hi - 1);
        const int columns = z.col + min(z.left, 32) - a.col;
        if (tid < count) prefetch_l2(y + tile_rows[tid] * p.y_stride + a.col, columns * sizeof(T));
        if (tid == THREADS - 1)
            prefetch_l2(ad.b + static_cast<size_t>(a.col) * ad.cap, static_cast<size_t>(columns) * ad.cap * sizeof(T));
    }

    const int ra = tile_rows[g], rb = tile_rows[g + 8], K = ad.k;
    const int k_lo = segment_at((K + 31) / 32, rank), k_hi = segment_at((K + 31) / 32, rank + 1);
    const uint4 zero = {0, 0, 0, 0};
    const T* xa = ra >= 0 ? x + ra * p.x_stride : nullptr;
    const T* xb = rb >= 0 ? x + rb * p.x_stride : nullptr;
    // G tiles a warp at once (t0, t0 + WARPS, ...), U blocks of k asked for at once
    const auto first_product = [&](auto G_, auto U_) {
        constexpr int G = G_, U = U_;
        for (int t0 = warp; t0 < ad.n_tiles; t0 += G * WARPS) {
            const T* from[G];
#pragma unroll
            for (int j = 0; j < G; ++j) from[j] = t0 + j * WARPS < ad.n_tiles ? ad.a_row(t0 + j * WARPS, g) : nullptr;
            float acc[G][4] = {};
            for (int k0 = k_lo; k0 < k_hi; k0 += U) {
                uint4 va[U], vb[U], w[U][G];
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int k = (k0 + i) * 32 + q * 8;
                    const bool in = k0 + i < k_hi && k < K;
                    va[i] = in && xa ? *reinterpret_cast<const uint4*>(xa + k) : zero;
                    vb[i] = in && xb ? *reinterpret_cast<const uint4*>(xb + k) : zero;
#pragma unroll
                    for (int j = 0; j < G; ++j)
                        w[i][j] = in && from[j] ? *reinterpret_cast<const uint4*>(from[j] + k) : zero;
                }
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const uint32_t a0[4] = {va[i].x, vb[i].x, va[i].y, vb[i].y};
                    const uint32_t a1[4] = {va[i].z, vb[i].z, va[i].w, vb[i].w};
                    if (k0 + i < k_hi)
#pragma unroll
                        for (int j = 0; j < G; ++j) {
                            mma<T>(acc[j], a0, w[i][j].x, w[i][j].y);
                            mma<T>(acc[j], a1, w[i][j].z, w[i][j].w);
                        }
                }
            }
#pragma unroll
            for (int j = 0; j < G; ++j)
                if (from[j])
#pragma unroll
                    for (int e = 0; e < 4; e += 2)
                        *reinterpret_cast<float2*>(
                            &u.sums[(g + e * 4) * u.cols + ad.template column<RP>(t0 + j * WARPS) + q * 2]) =
                            make_float2(acc[j][e], acc[j][e + 1]);
        }
    };
    if (ad.n_tiles <= WARPS) first_product(std::integral_constant<int, 1>(), std::integral_constant<int, 6>());
    else first_product(std::integral_constant<int, 3>(), std::integral_constant<int, 4>());
    cluster_sync_all();
    const float scale = p.ad.scales ? p.ad.scales[slot] : 1.0f;
    for (int r = rank * (M / FEW_CTAS) + warp; r < (rank + 1) * (M / FEW_CTAS); r += WARPS) {
        float2 v[RANK16];
        join_row<T, RANK16, FEW_CTAS>(u, r, ad.r8, v);
        store_row<T, RANK16, FEW_CTAS>(u, r, v, scale);
    }
    cluster_sync_all();     // (the last access to another CTA's memory was before it)

    for (int b = block_lo + warp; b < block_hi; b += WARPS) {
        const Block block = block_at(p, b);
        const int col = block.col + q * 8;
        const bool in = q * 8 < block.left, n_in = (g >> 1) * 8 < block.left;
        const uint4 ya = in && ra >= 0 ? *reinterpret_cast<const uint4*>(y + ra * p.y_stride + col) : zero;
        const uint4 yb = in && rb >= 0 ? *reinterpret_cast<const uint4*>(y + rb * p.y_stride + col) : zero;
        const T* w = ad.b + (static_cast<size_t>(block.col) + (g >> 1) * 8 + (g & 1)) * ad.cap;
        float acc[4][4] = {};
        second_product<T, RANK16>(acc, u, g * u.stride + block.m * RP, ad.r8, q, [&](int j, int s) {
            if constexpr (RANK16 == 1) {
                const uint2 v = n_in && q * 4 < ad.r8 ? *reinterpret_cast<const uint2*>(w + j * 2 * ad.cap + q * 4) : uint2{0, 0};
                return uint4{v.x, v.y, 0, 0};
            } else {
                return n_in && s * 16 + q * 8 < ad.r8 ? *reinterpret_cast<const uint4*>(w + j * 2 * ad.cap + s * 16 + q * 8)
                                                      : zero;
            }
        });
        const float fa = factor_of(u, g, block.m, scale), fb = factor_of(u, g + 8, block.m, scale);
        if (in && ra >= 0) *reinterpret_cast<uint4*>(out + ra * p.out_stride + col) = added<T>(ya, acc, 0, fa);
        if (in && rb >= 0) *reinterpret_cast<uint4*>(out + rb * p.out_stride + col) = added<T>(yb, acc, 2, fb);
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Many rows an adapter (prefill): tiles of 64 rows, CTAS a cluster; four shares of the columns by two groups of 32 rows
// (eight warps of two fragments, two CTAs an SM) or, from rank 33 on, where shared memory leaves one CTA an SM, by four
// groups of 16 (8192 x rank 16: 60 us against 72 with four groups, x rank 32 93 against 112; 3001 x rank 64: 80 against 83
// with two). One ring of shared memory carries both products: stages of 64 k of x and
// A, then stages of 128 columns of y and B, filled by 16-byte asynchronous copies, so that the second product's operands are
// on their way while the sums are joined. Rows of a stage are 128 bytes or more apart and their 16-byte pieces swapped by
// halves on odd rows (piece ^ 4), so that a quarter load (two rows, four pieces) meets every bank once.
// ---------------------------------------------------------------------------------------------------------------
constexpr int many_fragments(int rank16) { return rank16 >= 4 ? 1 : 2; }        // of 16 rows, a warp
constexpr int many_warps(int rank16) { return 16 / many_fragments(rank16); }
constexpr int MANY_ROWS = 64, MANY_TILES = 6, MANY_COLS = MANY_TILES * 8 * 4;      // inner columns it holds
constexpr int stage_bytes(int cols, int rank16) {
    const int first = (MANY_ROWS + cols) * 128, second = MANY_ROWS * 256 + 128 * rank16 * 32;
    return first > second ? first : second;
}
// From rank 33 on u's three parts of bf16 go over the sums and their levels, once every CTA has read them: beside them the
// ring would not have its three stages. That costs a cluster barrier, which fp16's two parts do not need (3001 x rank 64:
// 73 us without it, 74 with it).
constexpr bool parts_over(int rank16, int parts) { return rank16 >= 4 && parts > 2; }
constexpr int many_bytes(int cols, int rank16, int stages, int ctas, int parts) {
    const int sums = sums_bytes(MANY_ROWS, cols), levels = ctas >= 8 ? 0 : (ctas >= 4 ? 1 : 2) * sums;
    const int u = parts_bytes(MANY_ROWS, cols, parts);
    const int inner = parts_over(rank16, parts) ? (sums + levels > u ? sums + levels : u) : sums + (levels > u ? levels : u);
    return stages * stage_bytes(cols, rank16) + inner;
}

template <typename T, int RANK16, int CTAS>
__global__ void __launch_bounds__(many_warps(RANK16) * 32, RANK16 >= 4 ? 1 : 2) adapt_many(AdaptParams p, int stages) {
    constexpr int F = many_fragments(RANK16), GROUPS = 4 / F;
    constexpr int M = MANY_ROWS, WARPS = many_warps(RANK16), THREADS = WARPS * 32, RP = RANK16 * 16, OWN = SEGMENTS / CTAS;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int tile_rows[M];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    const int row_warp = warp % GROUPS, col_warp = warp / GROUPS;
    const int rank = blockIdx.x % CTAS, tile = blockIdx.x / CTAS;
    const int cols = p.ad.n_mats * RP, slot_bytes = stage_bytes(cols, RANK16);
    const Inner<T> u(smem + stages * slot_bytes, M, cols, parts_over(RANK16, PARTS<T>));
    pdl_launch_dependents();
    pdl_wait();
    const Tile mine = reinterpret_cast<const Tile*>(p.plan)[tile];
    if (mine.count == 0) return;        // (the whole cluster: one tile)
    if (tid < M) tile_rows[tid] = tid < mine.count ? p.plan[4 * p.max_tiles + mine.first + tid] : -1;
    __syncthreads();
    const Adapter<T> ad(p, mine.slot);
    if (ad.r8 == 0) return copy_rows<T>(p, tile_rows, mine.count, rank, CTAS, WARPS);
    const T* x = static_cast<const T*>(p.x);
    const T* y = static_cast<const T*>(p.y);
    const int K = ad.k, k_blocks = (K + 31) / 32, a_rows = ad.n_tiles * 8;
    const int blocks = block_count(p), block_lo = blocks * rank / CTAS, block_hi = blocks * (rank + 1) / CTAS;

    // Stages of the first product: each segment of k by itself, two blocks of 32 a stage; of the second: four blocks of
    // columns.
    int n_first = 0;
#pragma unroll
    for (int s = 0; s < OWN; ++s)
        n_first += (segment_at(k_blocks, rank * OWN + s + 1) - segment_at(k_blocks, rank * OWN + s) + 1) / 2;
    const int n_second = (block_hi - block_lo + 3) / 4, n_stages = n_first + n_second;

    // What this thread copies of a first stage: piece tid % 8 of rows tid / 8 + 32 i of x, then of A; of a second: piece tid
    // % 16 of rows tid / 16 + 16 i of y, then of B's. Rows of x and y that the tile lacks are left as they are (no other
    // row's result has anything of theirs).
    constexpr int TILES = RANK16 == 1 ? 2 : RANK16 == 2 ? 4 : MANY_TILES;       // n8 tiles of the first product a warp
    constexpr int STEP = THREADS / 8, X_PIECES = M / STEP, PIECES = X_PIECES + TILES * 8 * 4 / STEP;
    constexpr int Y_STEP = THREADS / 16, Y_PIECES = M / Y_STEP, ROW = RANK16 * 2;       // ROW: pieces of a row of B
    const int piece = tid & 7, piece_row = tid >> 3;
    const T* from_first[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int r = piece_row + i * STEP, a = r - M;
        if (i < X_PIECES) from_first[i] = tile_rows[r % M] >= 0 ? x + tile_rows[r % M] * p.x_stride + piece * 8 : nullptr;
        else from_first[i] = a < a_rows ? ad.a_row(a >> 3, a & 7) + piece * 8 : nullptr;
    }
    const T* from_y[Y_PIECES];
#pragma unroll
    for (int i = 0; i < Y_PIECES; ++i) {
        const int t = tile_rows[(tid >> 4) + i * Y_STEP];
        from_y[i] = t >= 0 ? y + t * p.y_stride + (tid & 3) * 8 : nullptr;
    }
    const uint32_t ring = smem_addr(smem), ring_end = ring + stages * slot_bytes;
    const uint32_t to_first = piece_row * 128 + (piece ^ (piece_row & 1) << 2) * 16;
    const uint32_t to_y = (tid >> 4) * 256 + ((tid & 15) ^ (tid >> 4 & 1) << 2) * 16;
    // The first block of a second stage, for the filling and for the use; `whole`: its four blocks are whole and of one
    // matrix, so that their columns follow from it.
    Block fill_at = block_lo < block_hi ? block_at(p, block_lo) : Block{0, 0, 0}, use_at = fill_at;
    const auto whole = [&](const Block& at, int b0) { return at.left >= 128 && b0 + 4 <= block_hi; };
    const auto advance = [&](Block& at, int b0) {       // on to block b0
        at.col += 128, at.left -= 128;
        if (at.left <= 0 && b0 < block_hi) at = block_at(p, b0);
    };
    int fill_stage = 0, fill_segment = rank * OWN, fill_block = segment_at(k_blocks, fill_segment);
    int fill_end = segment_at(k_blocks, fill_segment + 1);
    uint32_t fill_to = ring;
    const auto fill = [&] {         // the next stage
        if (fill_stage >= n_stages) return;
        if (fill_stage < n_first) {
            while (fill_block >= fill_end) fill_end = segment_at(k_blocks, ++fill_segment + 1);
            const int k = fill_block * 32;
            const uint32_t to = fill_to + to_first;
            if (k + piece * 8 < min(fill_end * 32, K)) {
#pragma unroll
                for (int i = 0; i < PIECES; ++i)
                    if (from_first[i]) cp_async16_sa(to + i * STEP * 128, from_first[i] + k);
            } else {
#pragma unroll
                for (int i = 0; i < PIECES; ++i)
                    if (i < X_PIECES || from_first[i]) st_shared_zero(to + i * STEP * 128);
            }
            fill_block = min(fill_block + 2, fill_end);
        } else {
            // y: [row][16 pieces], four blocks of four
            const int b0 = block_lo + (fill_stage - n_first) * 4;
            const bool all = whole(fill_at, b0);
            const int by = tid >> 2 & 3;
            Block block = {fill_at.m, fill_at.col + by * 32, fill_at.left - by * 32};
            if (!all) block = b0 + by < block_hi ? block_at(p, b0 + by) : Block{0, 0, 0};
            if ((tid & 3) * 8 < block.left)
#pragma unroll
                for (int i = 0; i < Y_PIECES; ++i)
                    if (from_y[i]) cp_async16_sa(fill_to + to_y + i * Y_STEP * 256, from_y[i] + block.col);
            // B: [block][j][g][RP]: row g of tile j is the block's column 8 (g / 2) + 2 j + g % 2
#pragma unroll
            for (int i = 0; i < (128 * ROW + THREADS - 1) / THREADS; ++i) {
                const int at = tid + i * THREADS, row = at / ROW, c = at % ROW, bb = row >> 5, j = row >> 3 & 3, gg = row & 7;
                if (row >= 128) break;
                const int n = (gg >> 1) * 8 + j * 2 + (gg & 1);
                const uint32_t to = fill_to + M * 256 + row * ROW * 16 + (ROW >= 8 ? c ^ (row & 1) << 2 : c) * 16;
                block = {fill_at.m, fill_at.col + bb * 32, fill_at.left - bb * 32};
                if (!all) block = b0 + bb < block_hi ? block_at(p, b0 + bb) : Block{0, 0, 0};
                if (n < block.left && c * 8 < ad.r8)
                    cp_async16_sa(to, ad.b + (static_cast<size_t>(block.col) + n) * ad.cap + c * 8);
                else
                    st_shared_zero(to);
            }
            advance(fill_at, b0 + 4);
        }
        ++fill_stage;
        if ((fill_to += slot_bytes) == ring_end) fill_to = ring;
    };
    for (int i = 0; i < stages - 1; ++i) fill(), cp_async_commit();
    uint32_t use = ring;
    const auto next = [&] {         // the next stage, whole and for all; the one behind it is filled again
        if (stages == 4) cp_async_wait<2>();
        else if (RANK16 != 2 || stages == 3) cp_async_wait<1>();
        else cp_async_wait<0>();
        __syncthreads();
        fill();
        cp_async_commit();
        const uint32_t at = use;
        if ((use += slot_bytes) == ring_end) use = ring;
        return at;
    };

    // u = x A^T, a segment at a time; sums of segments join as the tree's levels complete (level l of this thread's values
    // in shared memory).
    const int per = (ad.n_tiles + 3) / 4, t0 = col_warp * per, nt = min(per, ad.n_tiles - t0);
    const int la = row_warp * 16 * F + g;       // the first of this lane's rows: la + 16 f and la + 16 f + 8
    float* levels = u.sums + M * cols;      // (where u's parts will be)
    // lane (g, q)'s piece of half h of an even or odd row: q or q + 4
    const uint32_t x_at = la * 128 + q * 16, a_at = (M + t0 * 8 + g) * 128 + q * 16, odd = (g & 1) * 64;
#pragma unroll
    for (int s = 0; s < OWN; ++s) {
        float acc[F][TILES][4] = {};
        const int end = segment_at(k_blocks, rank * OWN + s + 1);
        for (int kb = segment_at(k_blocks, rank * OWN + s); kb < end; kb += 2) {
            const uint32_t from = next();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (kb + h >= end) break;
                const uint32_t half = h * 64 ^ odd;
                uint4 v[F][2], w[TILES];
#pragma unroll
                for (int f = 0; f < F; ++f)
#pragma unroll
                    for (int r = 0; r < 2; ++r) v[f][r] = ld_shared_v4(from + x_at + half + (f * 16 + r * 8) * 128);
#pragma unroll
                for (int j = 0; j < TILES; ++j)
                    if (j < nt) w[j] = ld_shared_v4(from + a_at + half + j * 8 * 128);
#pragma unroll
                for (int f = 0; f < F; ++f) {
                    const uint32_t a0[4] = {v[f][0].x, v[f][1].x, v[f][0].y, v[f][1].y};
                    const uint32_t a1[4] = {v[f][0].z, v[f][1].z, v[f][0].w, v[f][1].w};
#pragma unroll
                    for (int j = 0; j < TILES; ++j)
                        if (j < nt) mma<T>(acc[f][j], a0, w[j].x, w[j].y);
#pragma unroll
                    for (int j = 0; j < TILES; ++j)
                        if (j < nt) mma<T>(acc[f][j], a1, w[j].z, w[j].w);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
            if (j >= nt) break;
            const int col = ad.template column<RP>(t0 + j) + q * 2;
#pragma unroll
            for (int f = 0; f < F; ++f)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const int at = (la + f * 16 + e * 4) * cols + col;
                    float2 v = make_float2(acc[f][j][e], acc[f][j][e + 1]);
                    int level = 0;
#pragma unroll
                    for (int bit = s; bit & 1; bit >>= 1, ++level) {
                        const float2 o = *reinterpret_cast<const float2*>(&levels[level * M * cols + at]);
                        v.x = o.x + v.x, v.y = o.y + v.y;
                    }
                    *reinterpret_cast<float2*>(s == OWN - 1 ? &u.sums[at] : &levels[level * M * cols + at]) = v;
                }
        }
    }
    cluster_sync_all();
    const float scale = p.ad.scales ? p.ad.scales[mine.slot] : 1.0f;
    if constexpr (parts_over(RANK16, PARTS<T>)) {
        constexpr int ROWS = (M / CTAS + WARPS - 1) / WARPS;
        float2 v[ROWS][RANK16];
        const auto row = [&](int i) { return warp + i * WARPS < M / CTAS ? rank * (M / CTAS) + warp + i * WARPS : -1; };
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
            if (row(i) >= 0) join_row<T, RANK16, CTAS>(u, row(i), ad.r8, v[i]);
        cluster_sync_all();
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
            if (row(i) >= 0) store_row<T, RANK16, CTAS>(u, row(i), v[i], scale);
    } else {
        for (int r = rank * (M / CTAS) + warp; r < (rank + 1) * (M / CTAS); r += WARPS) {
            float2 v[RANK16];
            join_row<T, RANK16, CTAS>(u, r, ad.r8, v);
            store_row<T, RANK16, CTAS>(u, r, v, scale);
        }
    }
    cluster_sync_all();     // (the last access to another CTA's memory was before it)

    T* to[F][2];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = la + f * 16 + r * 8, at = tile_rows[row];
            to[f][r] = at >= 0 ? static_cast<T*>(p.out) + at * p.out_stride + q * 8 : nullptr;
        }
    const uint32_t y_at = la * 256 + (col_warp * 4 + q ^ (g & 1) << 2) * 16;
    const uint32_t b_at = M * 256 + (col_warp * 32 + g) * ROW * 16;
    const uint32_t row_bytes = u.stride * sizeof(T), u_at = smem_addr(u.part) + la * row_bytes, part_bytes = M * row_bytes;
    // steps s and s + 1 of row fragment f, for the matrix and part that start at `at`
    const auto fragment = [&](uint32_t at, int f, int s, uint32_t (&o)[2][4]) {
        const uint32_t a = at + f * 16 * row_bytes, b = a + 8 * row_bytes;
        if constexpr (RANK16 == 1) {
            const uint2 h0 = ld_shared_v2(a + q * 8), h1 = ld_shared_v2(b + q * 8);
            o[0][0] = h0.x, o[0][1] = h1.x, o[0][2] = h0.y, o[0][3] = h1.y;
        } else {
            const uint32_t off = s * 32 + q * 16;
            const uint4 h0 = ld_shared_v4(a + off), h1 = ld_shared_v4(b + off);
            o[0][0] = h0.x, o[0][1] = h1.x, o[0][2] = h0.y, o[0][3] = h1.y;
            o[1][0] = h0.z, o[1][1] = h1.z, o[1][2] = h0.w, o[1][3] = h1.w;
        }
    };
    for (int i = 0; i < n_second; ++i) {
        const uint32_t from = next();
        const int b0 = block_lo + i * 4;
        Block block = {use_at.m, use_at.col + col_warp * 32, use_at.left - col_warp * 32};
        if (!whole(use_at, b0)) block = b0 + col_warp < block_hi ? block_at(p, b0 + col_warp) : Block{0, 0, 0};
        advance(use_at, b0 + 4);
        if (block.left <= 0) continue;
        const uint32_t u_m = u_at + block.m * RP * sizeof(T);
        float acc[F][4][4] = {};
#pragma unroll
        for (int s = 0; s < RANK16; s += 2) {
            if (s * 16 >= ad.r8) break;
            uint4 w[4];
            const uint32_t c = RANK16 >= 4 ? (s * 2 + q ^ (g & 1) << 2) * 16 : q * 16;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (RANK16 == 1) {
                    const uint2 v = ld_shared_v2(from + b_at + j * 8 * ROW * 16 + q * 8);
                    w[j] = {v.x, v.y, 0, 0};
                } else {
                    w[j] = ld_shared_v4(from + b_at + j * 8 * ROW * 16 + c);
                }
            }
#pragma unroll
            for (int f = 0; f < F; ++f)
#pragma unroll
                for (int k = 0; k < PARTS<T>; ++k) {        // (in second_product's order)
                    uint32_t v[2][4];
                    fragment(u_m + k * part_bytes, f, s, v);
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma<T>(acc[f][j], v[0], w[j].x, w[j].y);
                    if constexpr (RANK16 > 1)
#pragma unroll
                        for (int j = 0; j < 4; ++j) mma<T>(acc[f][j], v[1], w[j].z, w[j].w);
                }
        }
        if (q * 8 >= block.left) continue;
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
            for (int r = 0; r < 2; ++r)
                if (to[f][r])
                    *reinterpret_cast<uint4*>(to[f][r] + block.col) =
                        added<T>(ld_shared_v4(from + y_at + (f * 16 + r * 8) * 256), acc[f], r * 2,
                                 factor_of(u, la + f * 16 + r * 8, block.m, scale));
    }
    cp_async_wait<0>();
}

template <typename T>
auto few_kernel(int rank16) -> void (*)(AdaptParams) {
    return rank16 == 1 ? adapt_few<T, 1> : rank16 == 2 ? adapt_few<T, 2> : rank16 == 4 ? adapt_few<T, 4> : adapt_few<T, 8>;
}
template <typename T, int CTAS>
auto many_kernel(int rank16) -> void (*)(AdaptParams, int) {
    return rank16 == 1   ? adapt_many<T, 1, CTAS>
           : rank16 == 2 ? adapt_many<T, 2, CTAS>
           : rank16 == 4 ? adapt_many<T, 4, CTAS>
                         : adapt_many<T, 8, CTAS>;
}
template <typename T>
auto many_kernel(int rank16, int ctas) {
    return ctas == 2 ? many_kernel<T, 2>(rank16) : ctas == 4 ? many_kernel<T, 4>(rank16) : many_kernel<T, 8>(rank16);
}

int rank_steps(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8; }

// Tiles a plan may need: every adapter's rows (and those without one) end with a tile that is not full.
long long max_tiles(int rows, int slots, int m) { return (rows + m - 1) / m + (rows < slots + 1 ? rows : slots + 1); }

constexpr int MAX_SMEM = 226 * 1024;    // a CTA's dynamic shared memory, beside its few static words
constexpr int HALF_SM = 112 * 1024 + 512;       // the same where two CTAs share an SM's 228 KB (1 KB of a CTA is the system's)
constexpr double CTA_COST = 0.06;       // of a tile's work, what a CTA spends on joining sums whatever its share is

}  // namespace
}  // namespace esp

extern "C" size_t esp_adapt_ws_bytes(int t_rows, int slots) {
    using namespace esp;
    if (t_rows <= NO_PLAN || slots < 1) return 0;
    return static_cast<size_t>(max_tiles(t_rows, slots, 16)) * sizeof(Tile) + static_cast<size_t>(t_rows) * sizeof(int);
}

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
    ESP_REQUIRE(ad->k >= 8 && ad->k % 8 == 0 && ad->k <= 1 << 30, ESP_ERR_INVALID,
                "esp_adapt: k %d is not a multiple of 8 up to 2^30", ad->k);
    long long n = 0;
    for (int m = 0; m < ad->n_mats; ++m) {
        ESP_REQUIRE(ad->widths[m] >= 8 && ad->widths[m] % 8 == 0, ESP_ERR_INVALID,
                    "esp_adapt: width %d is not a multiple of 8", ad->widths[m]);
        n += ad->widths[m];
    }
    ESP_REQUIRE(n <= 1 << 30, ESP_ERR_INVALID, "esp_adapt: %lld columns (up to 2^30)", n);
    ESP_REQUIRE(t_rows >= 0 && t_rows <= (1 << 26), ESP_ERR_INVALID, "esp_adapt: %d rows", t_rows);
    if (t_rows == 0) return ok();
    ESP_REQUIRE(ad->a && ad->b && x && y && ids && out, ESP_ERR_INVALID, "esp_adapt: null pointer");
    ESP_REQUIRE(aligned(ad->a, 16) && aligned(ad->b, 16) && aligned(x, 16) && aligned(y, 16) && aligned(out, 16) &&
                    x_stride % 8 == 0 && y_stride % 8 == 0 && out_stride % 8 == 0,
                ESP_ERR_INVALID, "esp_adapt: rows and weights must be 16-byte aligned");
    const size_t need = esp_adapt_ws_bytes(t_rows, ad->slots);
    ESP_REQUIRE(need == 0 || (ws && aligned(ws, 16) && ws_bytes >= need), ESP_ERR_SCRATCH,
                "esp_adapt: workspace of %zu bytes, %zu needed (16-byte aligned)", ws ? ws_bytes : 0, need);

    const int steps = rank_steps(ad->rank), cols = ad->n_mats * steps * 16;
    const bool half = ad->dtype == F16;
    const int parts = half ? PARTS<__half> : PARTS<__nv_bfloat16>;
    // Tiles of 64 rows where the inner columns fit a CTA, tiles of 16 need more than two rounds of the GPU's clusters, and
    // there are enough rows a slot that tiles of 64 are not mostly empty if every slot is in use (which ids occur is not known
    // here: with 12 of 512 slots in use, 8192 rows of rank 16 take 156 us for it, and 61 with 12 of 16). Measured, 16 / 64 rows
    // a tile, us, rank 16, 32 and 64, four prompts: 512 rows 15 / 19, 18 / 26, 23 / 27; 1024 rows 22 / 21, 27 / 29, 36 / 42;
    // 1536 rows 30 / 22, 39 / 29, 51 / 42. 64 adapters mixed row by row: 1536 rows 41 / 34, 53 / 48, 70 / 111; 3000 rows
    // 67 / 38, 82 / 53, 106 / 114.
    const int clusters = std::max(device_sms() / 18, 1) * (18 * 2 / FEW_CTAS);
    const bool many = t_rows > 2 * FEW_ROWS * clusters && t_rows / ad->slots >= (steps >= 4 ? 40 : 24) && cols <= MANY_COLS;
    const int m = many ? MANY_ROWS : FEW_ROWS;
    AdaptParams p{*ad, x, y, ids, out, nullptr, x_stride, y_stride, out_stride, t_rows, static_cast<int>(n), t_rows};
    if (t_rows > NO_PLAN) {
        p.max_tiles = static_cast<int>(max_tiles(t_rows, ad->slots, m));
        Tile* tiles = static_cast<Tile*>(ws);
        p.plan = static_cast<const int*>(ws);
        if (const int rc = launch(plan_kernel, dim3(1), dim3(1024), sizeof(int) * (ad->slots + 1), stream, true, p, tiles,
                                  reinterpret_cast<int*>(tiles + p.max_tiles), m))
            return rc;
    }
    if (!many) {
        const auto kernel = half ? few_kernel<__half>(steps) : few_kernel<__nv_bfloat16>(steps);
        const size_t smem = sums_bytes(m, cols) + parts_bytes(m, cols, parts);
        if (const int rc = allow_any_smem(kernel, smem)) return rc;
        if (const int rc = launch_cluster(kernel, dim3(static_cast<unsigned>(p.max_tiles) * FEW_CTAS), dim3(FEW_WARPS * 32),
                                          smem, stream, true, FEW_CTAS, p))
            return rc;
        return ok();
    }
    // CTAs a tile: what takes the least rounds x (a CTA's share of a tile + what it spends on joining sums). Places: two CTAs
    // an SM (one from rank 33 on, or where a ring of two stages does not fit twice), as many whole clusters as the 18 SMs of a
    // GPC hold. Measured: 8192 rows of rank 16 with 2 / 4 / 8 CTAs 60 / 65 / 83 us, of rank 32 124 / 93 / 111, 3001 of rank
    // 64 with 4 / 8 80 / 95 us.
    const int half_sm = HALF_SM, tiles = (t_rows + m - 1) / m + std::min(ad->slots, t_rows / m) / 2;
    int ctas = 8;       // (fits whatever fits at all)
    double best = 1e30;
    for (int c : {2, 4, 8}) {
        if (many_bytes(cols, steps, 3, c, parts) > MAX_SMEM) continue;
        const int an_sm = steps < 4 && many_bytes(cols, steps, steps == 2 ? 2 : 3, c, parts) <= half_sm ? 2 : 1;
        const int places = std::max(device_sms() / 18, 1) * (18 * an_sm / c) * c;
        const double work = ((tiles * c + places - 1) / places) * (1.0 / c + CTA_COST);
        if (work < best) best = work, ctas = c;
    }
    // Two stages where that leaves an SM to two CTAs: q | k | v at rank 32, 8192 rows 93 us against 127 with three and one CTA.
    const bool three = steps != 2 || many_bytes(cols, steps, 3, ctas, parts) <= half_sm;
    const int least = three || many_bytes(cols, steps, 2, ctas, parts) > half_sm ? 3 : 2;
    const int room = steps < 4 && many_bytes(cols, steps, least, ctas, parts) <= half_sm ? half_sm : MAX_SMEM;
    int stages = 4;
    while (stages > least && many_bytes(cols, steps, stages, ctas, parts) > room) --stages;
    const size_t smem = many_bytes(cols, steps, stages, ctas, parts);
    const auto kernel = half ? many_kernel<__half>(steps, ctas) : many_kernel<__nv_bfloat16>(steps, ctas);
    if (const int rc = allow_any_smem(kernel, smem)) return rc;
    if (const int rc = launch_cluster(kernel, dim3(static_cast<unsigned>(p.max_tiles) * ctas), dim3(many_warps(steps) * 32), smem,
                                      stream, true, ctas, p, stages))
        return rc;
    return ok();
}
