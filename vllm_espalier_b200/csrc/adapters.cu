// Low-rank adapters of many requests at once beside a shared projection.
//
// out[t] = y[t] + scale (x[t] A^T) B^T. Rows are grouped by adapter into tiles of M rows; a cluster of eight CTAs takes a
// tile. Each CTA multiplies its eighth of k (u = x A^T, partial), the partial sums meet in distributed shared memory (each
// CTA adds up an eighth of the tile's rows, in rank order, and stores them into all eight), and each CTA multiplies u by
// its eighth of the columns of B and adds y. Both products are m16n8k16 matrix instructions fed straight from global
// memory: the contraction index may be taken in any order as long as both operands agree, so a lane loads eight
// consecutive values (16 bytes) of a row and uses them as the fragments of two instructions, and no operand passes
// through shared memory but u.
//
// The sum over k has one order for every batch: a CTA's share of k in ascending order in one accumulator, then the eight
// CTAs' sums in rank order. So a row's bits do not depend on the tile's size or on the rows beside it.
#include <cuda_runtime.h>

#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "host.hpp"

namespace esp {
namespace {

constexpr int CTAS = 8, MAX_SLOTS = 4096;
constexpr int NO_PLAN = 64;             // up to this many rows every CTA finds its tile's rows itself

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
    for (int t0 = 0; t0 < p.rows; t0 += 1024) {
        const int t = t0 + tid, id = t < p.rows ? slot_of(p, t) : -2;
        const unsigned same = __match_any_sync(0xffffffffu, id);
        if (id >= -1 && lane == __ffs(same) - 1) atomicAdd(&count[id < 0 ? slots - 1 : id], __popc(same));
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
    for (int t0 = 0; t0 < p.rows; t0 += 1024) {
        const int t = t0 + tid, id = t < p.rows ? slot_of(p, t) : -2;
        const unsigned same = __match_any_sync(0xffffffffu, id);
        const int leader = __ffs(same) - 1;
        int at = 0;
        if (id >= -1 && lane == leader) at = atomicAdd(&count[id < 0 ? slots - 1 : id], __popc(same));
        at = __shfl_sync(0xffffffffu, at, leader);
        if (id >= -1) rows[at + __popc(same & ((1u << lane) - 1))] = t;
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
// The product: tiles of M = 16 ROW_WARPS rows, RANK16 = the capacity in steps of 16.
//   ROW_WARPS 1 (few rows an adapter): eight warps share the inner columns, operands straight from global memory, the
//   loads of many blocks of k asked for before the first product.
//   ROW_WARPS 4 (prefill): sixteen warps, four row groups by four shares of the columns, x and A through a ring of
//   shared memory (16-byte asynchronous copies, STAGE_K values of k a stage), so that a CTA's whole share is on its way
//   while the first stages are multiplied.
// ---------------------------------------------------------------------------------------------------------------
template <int ROW_WARPS>
struct Shape {
    static constexpr int M = 16 * ROW_WARPS;
    static constexpr int COL_WARPS = ROW_WARPS == 1 ? 8 : 4;    // warps that share a row group's columns of the output
    static constexpr int WARPS = ROW_WARPS * COL_WARPS, THREADS = 32 * WARPS;
    static constexpr int GROUP = ROW_WARPS == 1 ? 3 : 6;        // n8 tiles of the first product that a warp holds at once
};
constexpr int STAGE_K = 64, MAX_STAGES = 4, WIDE_COLS = Shape<4>::GROUP * 8 * Shape<4>::COL_WARPS;

// Shared memory: sums [M][cols] fp32, u_hi and u_lo [M][stride] 16-bit (stride: 64 bytes past a multiple of 128, so that
// the eight lanes of a quarter load meet every bank once), the rows' factors; with four row warps the same place holds the
// ring before.
__host__ __device__ constexpr int u_stride(int cols) { return cols + (192 - cols * 2 % 128) % 128 / 2; }
template <int ROW_WARPS>
__host__ __device__ constexpr int joined_bytes(int cols) {
    return Shape<ROW_WARPS>::M * (cols * 4 + 2 * u_stride(cols) * 2 + 8);
}
constexpr int stage_bytes(int cols) { return (Shape<4>::M + cols) * STAGE_K * 2; }

template <typename T, int ROW_WARPS, int RANK16>
__global__ void __launch_bounds__(Shape<ROW_WARPS>::THREADS, 2) adapt_kernel(AdaptParams p, int stages) {
    using S = Shape<ROW_WARPS>;
    constexpr int M = S::M, COL_WARPS = S::COL_WARPS, WARPS = S::WARPS, THREADS = S::THREADS, GROUP = S::GROUP;
    constexpr int RP = RANK16 * 16;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int tile_rows[M];
    __shared__ int tile_slot, tile_count, found[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    const int rank = blockIdx.x % CTAS, tile = blockIdx.x / CTAS;
    const int cap = p.ad.rank, K = p.ad.k, mats = p.ad.n_mats, cols = mats * RP, us = u_stride(cols);
    float* sums = reinterpret_cast<float*>(smem);
    T* u_hi = reinterpret_cast<T*>(sums + M * cols);
    T* u_lo = u_hi + M * us;
    float* factor = reinterpret_cast<float*>(u_lo + M * us);
    pdl_launch_dependents();
    pdl_wait();

    // The tile's adapter and rows.
    if (p.plan) {
        const Tile mine = reinterpret_cast<const Tile*>(p.plan)[tile];
        if (mine.count == 0) return;        // (the whole cluster: one tile)
        const int* rows = p.plan + 4 * p.max_tiles + mine.first;
        for (int i = tid; i < M; i += THREADS) tile_rows[i] = i < mine.count ? rows[i] : -1;
        if (tid == 0) tile_slot = mine.slot, tile_count = mine.count;
    } else {
        // Tile j is row j's if the rows of its adapter before it fill whole tiles; it takes the next M of them.
        const int slot = slot_of(p, tile);
        for (int i = tid; i < M; i += THREADS) tile_rows[i] = -1;
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
            if (lane == 0) tile_count = min(taken, M), found[0] = before % M == 0;
        }
        __syncthreads();
        if (!found[0]) return;
    }
    __syncthreads();
    const int slot = tile_slot, count = tile_count;
    int r8 = 0;             // the adapter's rank, in whole steps of 8
    if (slot >= 0) r8 = p.ad.ranks ? (min(max(p.ad.ranks[slot], 0), cap) + 7) / 8 * 8 : cap;
    const T* x = static_cast<const T*>(p.x);
    const T* y = static_cast<const T*>(p.y);
    T* out = static_cast<T*>(p.out);

    // this CTA's 32-column blocks of the output, matrix by matrix
    int blocks = 0;
    for (int m = 0; m < mats; ++m) blocks += (p.ad.widths[m] + 31) / 32;
    const int block_lo = blocks * rank / CTAS, block_hi = blocks * (rank + 1) / CTAS;

    if (r8 == 0) {          // nothing to add: y itself
        if (out == y && p.out_stride == p.y_stride) return;
        const int from = p.n / 8 * rank / CTAS, to = p.n / 8 * (rank + 1) / CTAS;
        for (int r = warp; r < count; r += WARPS)
            for (int c = from + lane; c < to; c += 32)
                reinterpret_cast<uint4*>(out + tile_rows[r] * p.out_stride)[c] =
                    reinterpret_cast<const uint4*>(y + tile_rows[r] * p.y_stride)[c];
        return;
    }

    const T* B = static_cast<const T*>(p.ad.b) + static_cast<size_t>(slot) * p.n * cap;
    {   // what the second product will read, into L2 meanwhile
        int col_lo = p.n, col_hi = 0, first = 0, col = 0;
        for (int m = 0; m < mats; ++m) {
            const int w = p.ad.widths[m], n = (w + 31) / 32, from = max(block_lo - first, 0), to = min(block_hi - first, n);
            if (from < to) col_lo = min(col_lo, col + from * 32), col_hi = max(col_hi, col + min(w, to * 32));
            first += n, col += w;
        }
        if (col_lo < col_hi) {
            if (tid < count) prefetch_l2(y + tile_rows[tid] * p.y_stride + col_lo, (col_hi - col_lo) * sizeof(T));
            if (tid == THREADS - 1)
                prefetch_l2(B + static_cast<size_t>(col_lo) * cap, static_cast<size_t>(col_hi - col_lo) * cap * sizeof(T));
        }
    }

    // u = x A^T over this CTA's blocks of k. n8 tile t of the inner columns is ranks 8 j .. 8 j + 7 of matrix m, t = m
    // (r8 / 8) + j.
    const int k_blocks = (K + 31) / 32, k_lo = k_blocks * rank / CTAS, k_hi = k_blocks * (rank + 1) / CTAS;
    const int tiles_a_mat = r8 / 8, n_tiles = mats * tiles_a_mat;
    const T* A = static_cast<const T*>(p.ad.a) + static_cast<size_t>(slot) * mats * cap * K;
    const int row_warp = ROW_WARPS == 1 ? 0 : warp % ROW_WARPS, col_warp = warp / ROW_WARPS;
    const int ra = tile_rows[row_warp * 16 + g], rb = tile_rows[row_warp * 16 + g + 8];
    const uint4 zero = {0, 0, 0, 0};
    const auto a_row = [&](int t, int r) {      // row r of tile t of A
        const int m = t / tiles_a_mat;
        return A + (static_cast<size_t>(m) * cap + (t - m * tiles_a_mat) * 8 + r) * K;
    };
    const auto column = [&](int t) {            // its first column in sums and u
        const int m = t / tiles_a_mat;
        return m * RP + (t - m * tiles_a_mat) * 8;
    };
    if constexpr (ROW_WARPS == 1) {
        const T* xa = ra >= 0 ? x + ra * p.x_stride : nullptr;
        const T* xb = rb >= 0 ? x + rb * p.x_stride : nullptr;
        // G tiles a warp at once (t0, t0 + WARPS, ...), U blocks of k asked for at once
        const auto product = [&](auto G_, auto U_) {
            constexpr int G = G_, U = U_;
            for (int t0 = warp; t0 < n_tiles; t0 += G * WARPS) {
                const T* from[G];
#pragma unroll
                for (int j = 0; j < G; ++j) from[j] = t0 + j * WARPS < n_tiles ? a_row(t0 + j * WARPS, g) : nullptr;
                float acc[G][4] = {};
                for (int k0 = k_lo; k0 < k_hi; k0 += U) {
                    uint4 va[U], vb[U], w[U][G];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int k = (k0 + u) * 32 + q * 8;
                        const bool in = k0 + u < k_hi && k < K;
                        va[u] = in && xa ? *reinterpret_cast<const uint4*>(xa + k) : zero;
                        vb[u] = in && xb ? *reinterpret_cast<const uint4*>(xb + k) : zero;
#pragma unroll
                        for (int j = 0; j < G; ++j)
                            w[u][j] = in && from[j] ? *reinterpret_cast<const uint4*>(from[j] + k) : zero;
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const uint32_t a0[4] = {va[u].x, vb[u].x, va[u].y, vb[u].y};
                        const uint32_t a1[4] = {va[u].z, vb[u].z, va[u].w, vb[u].w};
                        if (k0 + u < k_hi)
#pragma unroll
                            for (int j = 0; j < G; ++j) {
                                mma<T>(acc[j], a0, w[u][j].x, w[u][j].y);
                                mma<T>(acc[j], a1, w[u][j].z, w[u][j].w);
                            }
                    }
                }
#pragma unroll
                for (int j = 0; j < G; ++j)
                    if (from[j])
#pragma unroll
                        for (int e = 0; e < 4; e += 2)
                            *reinterpret_cast<float2*>(&sums[(g + e * 4) * cols + column(t0 + j * WARPS) + q * 2]) =
                                make_float2(acc[j][e], acc[j][e + 1]);
            }
        };
        if (n_tiles <= WARPS) product(std::integral_constant<int, 1>(), std::integral_constant<int, 6>());
        else product(std::integral_constant<int, GROUP>(), std::integral_constant<int, 4>());
    } else {
        // A stage: M rows of x, then the rows of A, 128 bytes each; 16-byte piece c of row r lies at c ^ 4 (r % 2), so that
        // the eight lanes of a quarter load (two rows, four pieces) meet every bank once.
        const int a_rows = n_tiles * 8, n_stages = ((k_hi - k_lo) * 32 + STAGE_K - 1) / STAGE_K;
        const auto fill = [&](int i) {
            unsigned char* to = smem + (i % stages) * stage_bytes(cols);
            const int k0 = k_lo * 32 + i * STAGE_K;
            for (int piece = tid; piece < (M + a_rows) * 8; piece += THREADS) {
                const int r = piece >> 3, c = piece & 7, k = k0 + c * 8;
                const T* from = nullptr;
                if (k < k_hi * 32 && k < K) {
                    if (r >= M) from = a_row((r - M) >> 3, (r - M) & 7) + k;
                    else if (tile_rows[r] >= 0) from = x + tile_rows[r] * p.x_stride + k;
                }
                uint4* at = reinterpret_cast<uint4*>(to + r * 128 + (c ^ (r & 1) << 2) * 16);
                if (from) cp_async16(at, from);
                else *at = zero;
            }
        };
        const int per = (n_tiles + COL_WARPS - 1) / COL_WARPS, t0 = col_warp * per, nt = min(per, n_tiles - t0);
        float acc[GROUP][4] = {};
        for (int i = 0; i < stages - 1; ++i) {
            if (i < n_stages) fill(i);
            cp_async_commit();
        }
        for (int i = 0; i < n_stages; ++i) {
            if (stages == 4) cp_async_wait<2>();        // the stage after this and the one behind it may be on their way
            else cp_async_wait<1>();
            __syncthreads();
            if (i + stages - 1 < n_stages) fill(i + stages - 1);
            cp_async_commit();
            const unsigned char* from = smem + (i % stages) * stage_bytes(cols);
#pragma unroll
            for (int h = 0; h < STAGE_K / 32; ++h) {
                const int kb = k_lo + i * (STAGE_K / 32) + h;
                if (kb >= k_hi) break;
                const auto piece = [&](int r) {
                    return *reinterpret_cast<const uint4*>(from + r * 128 + ((h * 4 + q) ^ (r & 1) << 2) * 16);
                };
                const uint4 va = piece(row_warp * 16 + g), vb = piece(row_warp * 16 + g + 8);
                const uint32_t a0[4] = {va.x, vb.x, va.y, vb.y}, a1[4] = {va.z, vb.z, va.w, vb.w};
#pragma unroll
                for (int j = 0; j < GROUP; ++j)
                    if (j < nt) {
                        const uint4 w = piece(M + (t0 + j) * 8 + g);
                        mma<T>(acc[j], a0, w.x, w.y);
                        mma<T>(acc[j], a1, w.z, w.w);
                    }
            }
        }
        cp_async_wait<0>();
        __syncthreads();        // the ring's place is free for the sums
#pragma unroll
        for (int j = 0; j < GROUP; ++j)
            if (j < nt)
#pragma unroll
                for (int e = 0; e < 4; e += 2)
                    *reinterpret_cast<float2*>(&sums[(row_warp * 16 + g + e * 4) * cols + column(t0 + j) + q * 2]) =
                        make_float2(acc[j][e], acc[j][e + 1]);
    }
    cluster_sync_all();

    // Add up the eight CTAs' sums of this CTA's eighth of the rows, in rank order, and store them into all eight as two
    // 16-bit halves (hi + lo is the sum to 2^-16 of it, so the second product rounds nothing that the output shows). For
    // fp16 a row is first scaled by a power of two that brings its largest value to [2^14, 2^15); the factor comes back
    // with the adapter's scale.
    const float scale = p.ad.scales ? p.ad.scales[slot] : 1.0f;
    for (int r = rank * (M / CTAS) + warp; r < (rank + 1) * (M / CTAS); r += WARPS) {
        float2 v[RANK16];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < RANK16; ++i) {
            const int c = lane * 2 + i * 64;
            v[i] = {0.0f, 0.0f};
            if (c < cols && c % RP < r8)
#pragma unroll
                for (int w = 0; w < CTAS; ++w) {
                    const float2 o = ld_cluster_f2(sums + r * cols + c, w);
                    v[i].x += o.x, v[i].y += o.y;
                }
            top = fmaxf(top, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
        }
        float up = 1.0f, down = scale;
        if constexpr (std::is_same_v<T, __half>) {
            top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
            if (top > 1e-30f && top < 1e30f) {
                const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14;
                up = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                down = scale * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            }
        }
#pragma unroll
        for (int i = 0; i < RANK16; ++i) {
            const int c = lane * 2 + i * 64;
            if (c >= cols) continue;
            const float a = v[i].x * up, b = v[i].y * up;
            const uint32_t hi = pack(a, b, T());
            const float2 back = unpack(hi, T());
            // (an infinite half leaves nothing to the other one)
            const uint32_t lo = pack(isinf(back.x) ? 0.0f : a - back.x, isinf(back.y) ? 0.0f : b - back.y, T());
#pragma unroll
            for (int w = 0; w < CTAS; ++w) {
                st_cluster_u32(u_hi + r * us + c, w, hi);
                st_cluster_u32(u_lo + r * us + c, w, lo);
            }
        }
        if (lane < CTAS) st_cluster_u32(factor + r, lane, __float_as_uint(down));
    }
    cluster_sync_all();     // (the last access to another CTA's memory was before it)

    // out = y + factor u B^T over this CTA's blocks of columns. The four n8 tiles of a block take columns so that a lane ends
    // up with eight consecutive ones: tile j's column c is 8 (c / 2) + 2 j + c % 2 of the block.
    const float fa = factor[row_warp * 16 + g], fb = factor[row_warp * 16 + g + 8];
    int m = -1, m_block = 0, m_col = 0, next_block = 0;       // the matrix of the block, its first block and column
    const T *h_at = nullptr, *l_at = nullptr;                 // this lane's halves of u for that matrix
    const auto halves = [&](const T* u, int s, uint32_t (&f)[2][4]) {       // the fragments of steps s and s + 1
        if constexpr (RANK16 == 1) {
            const uint2 va = *reinterpret_cast<const uint2*>(u + q * 4), vb = *reinterpret_cast<const uint2*>(u + 8 * us + q * 4);
            f[0][0] = va.x, f[0][1] = vb.x, f[0][2] = va.y, f[0][3] = vb.y;
        } else {
            const uint4 va = *reinterpret_cast<const uint4*>(u + s * 16 + q * 8);
            const uint4 vb = *reinterpret_cast<const uint4*>(u + 8 * us + s * 16 + q * 8);
            f[0][0] = va.x, f[0][1] = vb.x, f[0][2] = va.y, f[0][3] = vb.y;
            f[1][0] = va.z, f[1][1] = vb.z, f[1][2] = va.w, f[1][3] = vb.w;
        }
    };
    for (int b = block_lo + col_warp; b < block_hi; b += COL_WARPS) {
        if (b >= next_block) {
            while (b >= next_block) {
                if (m >= 0) m_col += p.ad.widths[m];
                m_block = next_block;
                next_block += (p.ad.widths[++m] + 31) / 32;
            }
            h_at = u_hi + (row_warp * 16 + g) * us + m * RP;
            l_at = u_lo + (row_warp * 16 + g) * us + m * RP;
        }
        const int width = p.ad.widths[m], base = (b - m_block) * 32;      // columns of matrix m
        const bool in = base + q * 8 < width;
        const int col = m_col + base + q * 8;
        const uint4 ya = in && ra >= 0 ? *reinterpret_cast<const uint4*>(y + ra * p.y_stride + col) : zero;
        const uint4 yb = in && rb >= 0 ? *reinterpret_cast<const uint4*>(y + rb * p.y_stride + col) : zero;
        const bool n_in = base + (g >> 1) * 8 < width;
        const T* w = B + (static_cast<size_t>(m_col) + base + (g >> 1) * 8 + (g & 1)) * cap;
        float acc[4][4] = {};
        uint32_t hi[2][4], lo[2][4];
        if constexpr (RANK16 == 1) {
            uint2 k[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                k[j] = n_in && q * 4 < r8 ? *reinterpret_cast<const uint2*>(w + j * 2 * cap + q * 4) : uint2{0, 0};
            halves(h_at, 0, hi);
            halves(l_at, 0, lo);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mma<T>(acc[j], hi[0], k[j].x, k[j].y);
                mma<T>(acc[j], lo[0], k[j].x, k[j].y);
            }
        } else {
#pragma unroll
            for (int s = 0; s < RANK16; s += 2) {
                if (s * 16 >= r8) break;
                uint4 k[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    k[j] = n_in && s * 16 + q * 8 < r8 ? *reinterpret_cast<const uint4*>(w + j * 2 * cap + s * 16 + q * 8)
                                                       : zero;
                halves(h_at, s, hi);
                halves(l_at, s, lo);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mma<T>(acc[j], hi[0], k[j].x, k[j].y);
                    mma<T>(acc[j], lo[0], k[j].x, k[j].y);
                    mma<T>(acc[j], hi[1], k[j].z, k[j].w);
                    mma<T>(acc[j], lo[1], k[j].z, k[j].w);
                }
            }
        }
        if (!in) continue;
        const auto add = [&](const uint4& v, int e, float f) {
            uint4 o;
            const uint32_t* from = &v.x;
            uint32_t* to = &o.x;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 b2 = unpack(from[j], T());
                to[j] = pack(fmaf(f, acc[j][e], b2.x), fmaf(f, acc[j][e + 1], b2.y), T());
            }
            return o;
        };
        if (ra >= 0) *reinterpret_cast<uint4*>(out + ra * p.out_stride + col) = add(ya, 0, fa);
        if (rb >= 0) *reinterpret_cast<uint4*>(out + rb * p.out_stride + col) = add(yb, 2, fb);
    }
}

using Kernel = void (*)(AdaptParams, int);

template <typename T, int ROW_WARPS>
Kernel kernel_of(int rank16) {
    return rank16 == 1   ? adapt_kernel<T, ROW_WARPS, 1>
           : rank16 == 2 ? adapt_kernel<T, ROW_WARPS, 2>
           : rank16 == 4 ? adapt_kernel<T, ROW_WARPS, 4>
                         : adapt_kernel<T, ROW_WARPS, 8>;
}

int rank_steps(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8; }

// Tiles a plan may need: every adapter's rows (and those without one) end with a tile that is not full.
long long max_tiles(int rows, int slots, int m) { return (rows + m - 1) / m + (rows < slots + 1 ? rows : slots + 1); }

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
    ESP_REQUIRE(ad->k >= 8 && ad->k % 8 == 0, ESP_ERR_INVALID, "esp_adapt: k %d is not a multiple of 8", ad->k);
    long long n = 0;
    for (int m = 0; m < ad->n_mats; ++m) {
        ESP_REQUIRE(ad->widths[m] >= 8 && ad->widths[m] % 8 == 0, ESP_ERR_INVALID,
                    "esp_adapt: width %d is not a multiple of 8", ad->widths[m]);
        n += ad->widths[m];
    }
    ESP_REQUIRE(n < INT_MAX - 128, ESP_ERR_INVALID, "esp_adapt: %lld columns", n);
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
    // Tiles of 64 rows where adapters have that many on average and their shared memory lets two CTAs on an SM.
    const bool wide = t_rows > NO_PLAN && t_rows / ad->slots >= 32 && cols <= WIDE_COLS;
    const int m = wide ? Shape<4>::M : Shape<1>::M, threads = wide ? Shape<4>::THREADS : Shape<1>::THREADS;
    const int stages = MAX_STAGES * stage_bytes(cols) <= 100 * 1024 ? MAX_STAGES : 3;
    const size_t smem = wide ? std::max(joined_bytes<4>(cols), stages * stage_bytes(cols))
                             : joined_bytes<1>(cols);
    const Kernel kernel = wide ? (half ? kernel_of<__half, 4>(steps) : kernel_of<__nv_bfloat16, 4>(steps))
                               : (half ? kernel_of<__half, 1>(steps) : kernel_of<__nv_bfloat16, 1>(steps));
    AdaptParams p{*ad, x, y, ids, out, nullptr, x_stride, y_stride, out_stride, t_rows, static_cast<int>(n), t_rows};
    if (t_rows > NO_PLAN) {
        p.max_tiles = static_cast<int>(max_tiles(t_rows, ad->slots, m));
        Tile* tiles = static_cast<Tile*>(ws);
        p.plan = static_cast<const int*>(ws);
        if (const int rc = launch(plan_kernel, dim3(1), dim3(1024), sizeof(int) * (ad->slots + 1), stream, true, p, tiles,
                                  reinterpret_cast<int*>(tiles + p.max_tiles), m))
            return rc;
    }
    if (const int rc = allow_smem(kernel, smem)) return rc;
    if (const int rc = launch_cluster(kernel, dim3(static_cast<unsigned>(p.max_tiles) * CTAS), dim3(threads), smem, stream,
                                      true, CTAS, p, stages))
        return rc;
    return ok();
}
