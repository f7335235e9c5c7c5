// Verification of drafted tokens against the target's probabilities: drafted token d_i of a request stands iff all before it
// do and u_i q_i(d_i) < p_i(d_i); the first that falls is replaced by a draw from max(p_i - q_i, 0), and after the last one a
// token is drawn from p. A draw is argmax_v w(v) / noise(v) with exponential noise: a race that needs no sum over w, no
// prefix sums and no second pass, and whose result does not depend on the order of anything.
//
// Bytes bound it where there are many requests (a row of 248320 bf16 logits is 0.5 MB, a request's noise 1 MB): rows past
// the first that falls are never read. With few, latency does: rows are taken one after another, about 2.5 us each (one
// pass over the row, one exchange in the cluster), then the race, 2.9 us. Measured: one request of 3 drafted tokens 11 us,
// 13 ragged ones (fp32, 150001 ids) 19 us, 96 requests 70 us for the 210 MB they cannot do without (47% of a plain copy;
// the exponentials alone take the special-function units about 30% of that time, the rest is waits at the rows' ends, which
// more and smaller CTAs only trade for more of them).
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

// 2^x to two units of fp32, 0 below 2^-126. Sums are fp32's own; a call's probabilities come out within 4e-7 of the 64-bit ones
// (relative, over the cases of the operators' benchmark; an fp32 softmax by exact exponentials and divisions: 2e-7).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// CTAs of 256 threads, four an SM. Measured, 1 / 13 ragged / 96 requests: 12 / 20 / 80 us so, 512 threads x 2 12 / 18 / 97,
// 1024 x 1 13 / 31 / 131, 128 x 8 15 / 22 / 73.
constexpr int THREADS = 256, WARPS = THREADS / 32, PACKS = 4, OCTETS = 1, SINGLES = 8, RESIDENT = 4;
// A request gets CTAs, up to one a segment of its vocabulary, until the batch has FILL an SM: with 1, 24 / 48 / 96 requests
// take 41 / 71 / 119 us, with 2 28 / 47 / 82, with 4 28 / 41 / 72, with 6 28 / 41 / 75.
constexpr int MAX_SEGMENTS = 16, SEGMENT = 16384, FILL = 4;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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

// What a CTA shares: its warps' values of a round, the cluster's of two rounds in turn, and what came of a round.
struct Shared {
    Part warps[MAX_SEGMENTS * WARPS];       // [own segment][warp]
    Part table[2][MAX_SEGMENTS];
    Part result;
    int gave_up;                            // a wait of the exchange did
    uint64_t full[2];                       // of the tables, armed for their next round
};

// What the CTAs of a cluster tell one another. In a round each warp puts a value into its CTA's `warps`; the CTA's first
// warp joins them, stores one value for each of the CTA's segments into every CTA's table (its place by segment, so what
// is made of the table does not depend on how many CTAs share the segments), counted there on the round's mbarrier, waits
// for its own table and joins that. Two tables in turn: a CTA gives to round r + 2 only after it has the whole of round
// r + 1, which every CTA gave to after it had read round r.
struct Exchange {
    Shared& sh;
    int ctas, segments, own;        // own: segments of this CTA
    int from;                       // the first of them
    int round = 0;

    __device__ __forceinline__ void arm(int r) {
        mbar_arrive_expect_tx(&sh.full[r], segments * static_cast<uint32_t>(sizeof(Part)));
    }

    // The first warp, all lanes: the round's table once it is whole (NULL after a wait that gave up).
    __device__ __forceinline__ const Part* whole(int r) {
        const bool there = mbar_wait(&sh.full[r & 1], (r >> 1) & 1);
        if (threadIdx.x == 0) arm(r & 1);
        if (__all_sync(0xffffffffu, there)) return sh.table[r & 1];
        if (threadIdx.x == 0) sh.gave_up = 1;
        return nullptr;
    }
    __device__ __forceinline__ void give(int r, int segment, int to, uint32_t a, uint32_t b, uint32_t c) {
        st_async_v4(&sh.table[r & 1][segment], &sh.full[r & 1], to, a, b, c, 0);
    }

    // The join of the parts that the cluster's warps put into `warps`, in every thread. After a wait that gave up: an
    // empty part.
    __device__ __forceinline__ Part part(float c) {
        const int lane = threadIdx.x & 31, r = round++;
        __syncthreads();
        if (threadIdx.x < 32) {
            for (int i = 0; i < own; i += 32 / WARPS) {     // four segments at once, eight lanes each
                const int s = i + lane / WARPS;
                Part t = {-INFINITY, 0.0f, INT_MAX, 0};
                if (s < own) t = sh.warps[i * WARPS + lane];
                t = lanes_part(t, c, WARPS / 2);
                if (s < own)
                    for (int to = lane % WARPS; to < ctas; to += WARPS)
                        give(r, from + s, to, __float_as_uint(t.m), __float_as_uint(t.z), t.at);
            }
            const Part* table = whole(r);
            Part t = {-INFINITY, 0.0f, INT_MAX, 0};
            if (table && lane < segments) t = table[lane];
            t = lanes_part(t, c, MAX_SEGMENTS / 2);
            if (lane == 0) sh.result = t;
        }
        __syncthreads();
        return sh.result;
    }

    // The largest of the keys that this CTA's and the others' warps put into `warps` (of the first own segment).
    __device__ __forceinline__ unsigned long long largest() {
        const int lane = threadIdx.x & 31, r = round++;
        __syncthreads();
        if (threadIdx.x < 32) {
            unsigned long long key = lane < WARPS ? as_key(sh.warps[lane]) : 0;
            key = lanes_max(key, 16);       // in every lane: each sends it to a CTA of its own
            if (lane < ctas)
                for (int s = 0; s < own; ++s)
                    give(r, from + s, lane, static_cast<uint32_t>(key >> 32), static_cast<uint32_t>(key), 0);
            const Part* table = whole(r);
            key = lanes_max(table && lane < segments ? as_key(table[lane]) : 0, MAX_SEGMENTS / 2);
            if (lane == 0) sh.result = {__uint_as_float(static_cast<uint32_t>(key >> 32)),
                                        __uint_as_float(static_cast<uint32_t>(key)), 0, 0};
        }
        __syncthreads();
        return as_key(sh.result);
    }

    static __device__ __forceinline__ unsigned long long as_key(const Part& t) {
        return static_cast<unsigned long long>(__float_as_uint(t.m)) << 32 | __float_as_uint(t.z);
    }
    // Over groups of 2 * half lanes from lane 0 on.
    static __device__ __forceinline__ Part lanes_part(Part t, float c, int half) {
#pragma unroll
        for (int k = half; k; k >>= 1)
            t = joined(t, {__shfl_xor_sync(0xffffffffu, t.m, k), __shfl_xor_sync(0xffffffffu, t.z, k),
                           __shfl_xor_sync(0xffffffffu, t.at, k), 0}, c);
        return t;
    }
    static __device__ __forceinline__ unsigned long long lanes_max(unsigned long long key, int half) {
#pragma unroll
        for (int k = half; k; k >>= 1) {
            const unsigned long long o = __shfl_xor_sync(0xffffffffu, key, k);
            key = o > key ? o : key;
        }
        return key;
    }
};

template <typename T>
struct alignas(16) Pack {
    T e[16 / sizeof(T)];
};

template <typename T>
struct alignas(16) Octet {
    T e[8];
};

// The largest of a thread's logits, NaN aside, two at an instruction where they are 16-bit.
__device__ __forceinline__ float largest_of(const Pack<float> (&k)[PACKS]) {
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < PACKS; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, k[u].e[e]);
    return top;
}
template <typename T>
__device__ __forceinline__ float largest_of(const Pack<T> (&k)[PACKS]) {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    T2 top = *reinterpret_cast<const T2*>(&k[0].e[0]);
#pragma unroll
    for (int u = 0; u < PACKS; ++u)
#pragma unroll
        for (int e = u ? 0 : 2; e < 8; e += 2) top = __hmax2(top, *reinterpret_cast<const T2*>(&k[u].e[e]));
    return fmaxf(f32(top.x), f32(top.y));
}

// This thread's share of the part [lo, hi) of a row, in one pass. The thread keeps the largest logit m that it has met
// and the sum of 2^(l c - mc) with mc = m c rounded; a larger m rescales the sum by 2^(mc - mc'). The rounding of mc is
// taken out once, at the end (2^(mc - m c)), so a logit costs one fma and one exponential. For c in [1e-6, 1e6], where a
// logit below FLOOR weighs nothing beside one above it. A row with NaN, +inf, an m c that overflows or nothing above
// FLOOR comes out with a sum that is NaN, infinite or 0, which the caller sees and takes careful_part instead.
constexpr float FLOOR = -1e30f;
template <typename T>
__device__ __forceinline__ Part fast_part(const T* row, int lo, int hi, float c) {
    constexpr int N = 16 / sizeof(T);
    float m = FLOOR, mc = 0.0f, z = 0.0f;
    int first = -1;         // where the batch starts among whose logits the largest was first met
    const auto raise = [&](float top, int v) {
        const float next = top * c;
        z = first < 0 ? 0.0f : z * ex2(mc - next);
        m = top, mc = next, first = v;
    };
    // 16-byte loads from the first boundary on, the ends one by one
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row + lo) % 16 / sizeof(T));
    const int head = min(hi, lo + (off ? N - off : 0)), packs = (hi - head) / N, tail = head + packs * N;
    const auto single = [&](int v) {
        const float l = f32(row[v]);
        if (l > m) raise(l, v);
        z += ex2(fmaf(l, c, -mc));
    };
    // PACKS packs, THREADS apart, from pack i on; those past the end read as the batch's first once more and weigh nothing.
    // The next batch is on its way while one is used.
    const auto load = [&](Pack<T> (&k)[PACKS], int i) {
#pragma unroll
        for (int u = 0; u < PACKS; ++u)
            k[u] = *reinterpret_cast<const Pack<T>*>(row + head + (u == 0 || i + u * THREADS < packs ? i + u * THREADS : i) * N);
    };
    const auto use = [&](const Pack<T> (&k)[PACKS], int i, auto whole) {
        const float top = largest_of(k);
        if (top > m) raise(top, head + i * N);
#pragma unroll
        for (int u = 0; u < PACKS; ++u)
            if (whole || u == 0 || i + u * THREADS < packs)
#pragma unroll
                for (int e = 0; e < N; ++e) z += ex2(fmaf(f32(k[u].e[e]), c, -mc));
    };
    // before the packs, so that a thread meets its places in order
    if (lo + static_cast<int>(threadIdx.x) < head) single(lo + threadIdx.x);
    int i = threadIdx.x;
    if (i < packs) {
        Pack<T> k[PACKS], then[PACKS];
        load(k, i);
        while (i + PACKS * THREADS < packs) {
            load(then, i + PACKS * THREADS);
            use(k, i, std::true_type());
#pragma unroll
            for (int u = 0; u < PACKS; ++u) k[u] = then[u];
            i += PACKS * THREADS;
        }
        use(k, i, std::false_type());
    }
    if (tail + static_cast<int>(threadIdx.x) < hi) single(tail + threadIdx.x);
    if (first >= 0) z *= ex2(-fmaf(m, c, -mc));
    return {m, z, first < 0 ? INT_MAX : first, 0};
}

// The lowest place of m among the logits of the batch that starts at v (a single one's place: that place), for a thread
// that met m there.
template <typename T>
__device__ __forceinline__ int place_of(const T* row, int v, int hi, float m) {
    constexpr int N = 16 / sizeof(T);
    for (int u = 0; u < PACKS; ++u)
        for (int e = 0; e < N; ++e) {
            const int at = v + u * THREADS * N + e;
            if (at < hi && f32(row[at]) == m) return at;
        }
    return v;
}

// The largest of a warp's values (no NaN), in every lane, by an integer whose order is the value's.
__device__ __forceinline__ float warp_max(float v) {
    const unsigned u = __float_as_uint(v);
    const unsigned r = __reduce_max_sync(0xffffffffu, u & 0x80000000u ? ~u : u | 0x80000000u);
    return __uint_as_float(r & 0x80000000u ? r & 0x7fffffffu : ~r);
}

// The join of a warp's threads into the CTA's table, for its i-th segment. `place`: a thread's lowest place of its
// largest, asked of the threads that have the warp's largest only.
template <typename Place>
__device__ __forceinline__ void put(Shared& sh, int i, Part t, float c, bool places, Place place) {
    const float m = warp_max(t.m);
    float z = t.m == m ? t.z : t.z * ex2((t.m - m) * c);
#pragma unroll
    for (int k = 16; k; k >>= 1) z += __shfl_xor_sync(0xffffffffu, z, k);
    int at = INT_MAX;
    if (places) at = __reduce_min_sync(0xffffffffu, t.m == m && t.at != INT_MAX ? place(t) : INT_MAX);
    if ((threadIdx.x & 31) == 0) sh.warps[i * WARPS + (threadIdx.x >> 5)] = {m, z, at, 0};
}

// The vocabulary in segments of `size` ids; this CTA's are [from, from + count).
struct Segments {
    int from, count, size, vocab;
    __device__ __forceinline__ int lo(int i) const { return min(vocab, (from + i) * size); }
    __device__ __forceinline__ int hi(int i) const { return min(vocab, (from + i + 1) * size); }
};

// The row's part for any row: NaN counts as -inf, weights as weight() has them. Takes CAREFUL_ROUNDS of the exchange,
// which the caller adds to its own count.
constexpr int CAREFUL_ROUNDS = 2;
template <typename T>
__device__ __noinline__ Part careful_part(const T* row, Segments own, float c, Exchange exchange) {
    const auto as_met = [](const Part& t) { return t.at; };
    for (int i = 0; i < own.count; ++i) {
        Part t = {-INFINITY, 0.0f, INT_MAX, 0};
        for (int v = own.lo(i) + threadIdx.x; v < own.hi(i); v += THREADS) {
            const float l = f32(row[v]);
            if (l > t.m) t = {l, 0.0f, v, 0};
        }
        put(exchange.sh, i, t, c, true, as_met);
    }
    Part all = exchange.part(c);
    for (int i = 0; i < own.count; ++i) {
        Part t = {0.0f, 0.0f, INT_MAX, 0};
        if (all.m > -INFINITY)
            for (int v = own.lo(i) + threadIdx.x; v < own.hi(i); v += THREADS) t.z += weight(f32(row[v]), all.m, c);
        put(exchange.sh, i, t, c, false, as_met);
    }
    all.z = exchange.part(c).z;
    return all;
}

struct NoProbs {};      // the drafter chose its token outright
template <typename Q>
__device__ __forceinline__ float draft_prob(const Q* q, long long i) {
    if constexpr (std::is_same_v<Q, NoProbs>) return 1.0f;
    else return f32(q[i]);
}

// A row's weights in the race: p(v) = e(l) scale with e(l) = 2^(l c - mc), mc = m c rounded and its rounding in `scale`;
// SAFE: weight() instead, for rows that careful_part summed.
struct Weights {
    float m, c, mc, scale;
    template <bool SAFE>
    __device__ __forceinline__ float e(float l) const {
        return SAFE ? weight(l, m, c) : ex2(fmaf(l, c, -mc));
    }
};

// A thread's best of the race so far: the largest max(p - q, 0) / noise and where it was met.
struct Best {
    float top = 0.0f;
    int at = -1;
};

// The race over [lo, hi) from w, by reciprocals of the noise (one unit of fp32 off, 0 past 2^126, infinite where it is
// subnormal: see race_exact): many loads are asked for before the first is used, a thread compares eight scores at
// once and `at` is where its eight consecutive ids start (or a single id). SUBTRACT: a drafted token was turned down and
// the drafter's probabilities are taken off.
template <bool SAFE, bool SUBTRACT, typename T, typename Q>
__device__ __forceinline__ void race(Best& best, const T* row, const Q* q, const float* noise, int out, int lo, int hi,
                                     const Weights& wt) {
    using O = std::conditional_t<SUBTRACT, Q, float>;
    const auto score = [&](T l, float e, float qv) { return fmaf(wt.e<SAFE>(f32(l)), wt.scale, SUBTRACT ? -qv : 0.0f) * rcp(e); };
    int v = lo;
    if ((reinterpret_cast<uintptr_t>(row + lo) | reinterpret_cast<uintptr_t>(noise + lo) |
         (SUBTRACT ? reinterpret_cast<uintptr_t>(q) + lo * sizeof(O) : 0)) % 16 == 0) {
        const int groups = (hi - lo) / 8;
        struct Octets {
            Octet<T> l[OCTETS];
            Octet<float> e[OCTETS];
            Octet<O> o[SUBTRACT ? OCTETS : 1];
        };
        const auto load = [&](Octets& k, int g) {
#pragma unroll
            for (int u = 0; u < OCTETS; ++u) {
                const int at = lo + (u == 0 || g + u * THREADS < groups ? g + u * THREADS : g) * 8;
                k.l[u] = *reinterpret_cast<const Octet<T>*>(row + at);
                k.e[u] = *reinterpret_cast<const Octet<float>*>(noise + at);
                if constexpr (SUBTRACT) k.o[u] = *reinterpret_cast<const Octet<O>*>(q + at);
            }
        };
        const auto use = [&](const Octets& k, int g) {
#pragma unroll
            for (int u = 0; u < OCTETS; ++u) {
                const int at = lo + (u == 0 || g + u * THREADS < groups ? g + u * THREADS : g) * 8;
                float s[8], top = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if constexpr (SUBTRACT) s[j] = score(k.l[u].e[j], k.e[u].e[j], f32(k.o[u].e[j]));
                    else s[j] = score(k.l[u].e[j], k.e[u].e[j], 0.0f);
                }
                if (!SUBTRACT && static_cast<unsigned>(out - at) < 8u) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (at + j == out) s[j] = 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, s[j]);
                if (top > best.top) best = {top, at};
            }
        };
        int g = threadIdx.x;
        if (g < groups) {
            Octets k, then;
            load(k, g);
            while (g + OCTETS * THREADS < groups) {
                load(then, g + OCTETS * THREADS);
                use(k, g);
                k = then;
                g += OCTETS * THREADS;
            }
            use(k, g);
        }
        v = lo + groups * 8;
    }
    for (v += threadIdx.x; v < hi; v += SINGLES * THREADS) {
        T l[SINGLES];
        float e[SINGLES];
        O o[SINGLES];
#pragma unroll
        for (int u = 0; u < SINGLES; ++u) {
            const int at = min(v + u * THREADS, hi - 1);        // past the end: an id that was met
            l[u] = row[at];
            e[u] = noise[at];
            if constexpr (SUBTRACT) o[u] = q[at];
        }
#pragma unroll
        for (int u = 0; u < SINGLES; ++u) {
            const int at = min(v + u * THREADS, hi - 1);
            float s;
            if constexpr (SUBTRACT) s = score(l[u], e[u], f32(o[u]));
            else s = at == out ? 0.0f : score(l[u], e[u], 0.0f);
            if (s > best.top) best = {s, at};
        }
    }
}

// The warp's best of the race over the CTA's segments, as a key in the CTA's table: the largest score, the lowest id among
// equals, 0 without a candidate. `out`: an id out of the race (-1: none).
template <bool SAFE, bool SUBTRACT, typename T, typename Q>
__device__ __forceinline__ void race_all(Shared& sh, const T* row, const Q* q, const float* noise, int out, const Segments& own,
                                         const Weights& wt) {
    Best best;
    for (int i = 0; i < own.count; ++i)
        race<SAFE, SUBTRACT>(best, row, q, noise, out, own.lo(i), own.hi(i), wt);
    const float top = warp_max(best.top);
    int id = INT_MAX;
    if (best.at >= 0 && best.top == top) {      // which of the eight (or of the one and those after it) it was
        id = best.at;
        for (int j = 0; j < 8 && best.at + j < own.vocab; ++j) {
            const int v = best.at + j;
            float qv = 0.0f;
            if constexpr (SUBTRACT) qv = f32(q[v]);
            const float s = fmaf(wt.e<SAFE>(f32(row[v])), wt.scale, SUBTRACT ? -qv : 0.0f) * rcp(noise[v]);
            if (v != out && s == top) {
                id = v;
                break;
            }
        }
    }
    id = __reduce_min_sync(0xffffffffu, id);
    if ((threadIdx.x & 31) == 0) {
        const unsigned long long key = id == INT_MAX ? 0 : score_key(top, id);
        sh.warps[threadIdx.x >> 5] = {__uint_as_float(static_cast<uint32_t>(key >> 32)),
                                      __uint_as_float(static_cast<uint32_t>(key)), 0, 0};
    }
}

// The race over row i of request b where its scores leave what rcp() and fp32 hold (noise that is subnormal or past 2^126):
// the same weights, the quotient in double, brought to where fp32 holds the largest, `top` by reciprocals. Pointers and ids
// are made anew, so that the kernel need not keep them for it.
constexpr float SCORE_LO = 0x1p-100f, SCORE_HI = 0x1p100f;
template <typename T, typename Q>
__device__ __noinline__ void race_exact(Shared& sh, const VerifyParams& p, int b, int i, Segments own, float m, float c,
                                        float inv_z, bool safe, float top) {
    constexpr bool GIVEN = !std::is_same_v<Q, NoProbs>;
    const long long at = static_cast<long long>(p.starts[b]) + i;
    const T* row = static_cast<const T*>(p.logits) + (at + b) * p.stride;
    const float* noise = p.noise + b * p.noise_stride;
    const bool fell = i < min(p.starts[b + 1] - p.starts[b], p.max_drafts);
    const int out = fell && !GIVEN ? p.drafts[at] : -1;
    const Weights wt{m, c, m * c, safe ? inv_z : inv_z * ex2(-fmaf(m, c, -(m * c)))};
    const double scale = top > 1.0f ? 0x1p-60 : 0x1p180;
    float best = 0.0f;
    int id = INT_MAX;
    for (int v = own.lo(0) + threadIdx.x; v < own.hi(own.count - 1); v += THREADS) {
        const float l = f32(row[v]), e = safe ? wt.e<true>(l) : wt.e<false>(l);
        float qv = 0.0f;
        if constexpr (GIVEN)
            if (fell) qv = f32(static_cast<const Q*>(p.draft_probs)[at * p.probs_stride + v]);
        const float s = static_cast<float>(static_cast<double>(fmaf(e, wt.scale, -qv)) / noise[v] * scale);
        if (v != out && s > best) best = s, id = v;
    }
    const float most = warp_max(best);
    id = __reduce_min_sync(0xffffffffu, best == most ? id : INT_MAX);
    if ((threadIdx.x & 31) == 0) {
        const unsigned long long key = id == INT_MAX ? 0 : score_key(most, id);
        sh.warps[threadIdx.x >> 5] = {__uint_as_float(static_cast<uint32_t>(key >> 32)),
                                      __uint_as_float(static_cast<uint32_t>(key)), 0, 0};
    }
}

struct Split {      // a request's vocabulary over segments and CTAs
    int ctas_log2, segments, own, size;
    bool ahead;
};

// A cluster of CTAs a request, each with its share of the vocabulary's segments: rows in order until a drafted token falls.
// Every CTA reads the same joined parts and so takes the same decisions.
template <typename T, typename Q>
__global__ void __launch_bounds__(THREADS, RESIDENT) verify_kernel(const __grid_constant__ VerifyParams p, Split split) {
    __shared__ Shared sh;
    constexpr bool GIVEN = !std::is_same_v<Q, NoProbs>;
    const int b = blockIdx.x >> split.ctas_log2, ctas = 1 << split.ctas_log2, rank = blockIdx.x & (ctas - 1);
    const int V = p.vocab, width = p.max_drafts + 1;
    const Segments own{rank * split.own, split.own, split.size, V};
    const int lo = own.lo(0), hi = own.hi(own.count - 1);
    const float* noise = p.noise + b * p.noise_stride;
    Exchange exchange{sh, ctas, split.segments, own.count, own.from};
    if (threadIdx.x == 0) {
        sh.gave_up = 0;
        for (int r = 0; r < 2; ++r) {
            mbar_init(&sh.full[r], 1);
            fence_mbar_init();
            exchange.arm(r);
        }
    }
    pdl_launch_dependents();
    pdl_wait();
    const long long at = p.starts[b], next = p.starts[b + 1];
    const float t = p.temperature ? p.temperature[b] : 1.0f;
    cluster_sync_all();     // every CTA of the cluster is there, its barriers armed, before the first store into it
    const long long first = at + b, k_all = next - at;
    const bool fits = at >= 0 && k_all >= 0 && at + k_all <= p.n_drafts && first + k_all < p.rows;
    const int k = static_cast<int>(min(k_all, static_cast<long long>(p.max_drafts)));
    const bool greedy = !(t > 0.0f);
    const float c = greedy ? LOG2E : LOG2E / fminf(fmaxf(t, 1e-30f), 1e30f);
    const bool fast = c >= 1e-6f && c <= 1e6f;
    // With a CTA an SM or less, all rows of the request at once: 2 / 4 / 9 requests 16.8 / 18.0 / 22.0 us, 18.1 / 19.3 / 22.6
    // without. With more CTAs the rows behind the first that falls cost more than the others gain: 24 / 32 requests 27.8 /
    // 29.8 us, 29.8 / 32.5 with all rows, 28.5 / 31.5 with one row more at a time.
    if (split.ahead && fits && threadIdx.x <= min(k, 31))
        prefetch_l2(static_cast<const T*>(p.logits) + (first + threadIdx.x) * p.stride + lo,
                    static_cast<size_t>(hi - lo) * sizeof(T));
    int* tokens = p.tokens + static_cast<size_t>(b) * width;
    float* probs = p.probs + static_cast<size_t>(b) * width;

    int n = 0, token = -1;
    float token_p = 0.0f;
    for (int i = 0; fits && i <= k; ++i) {
        const T* row = static_cast<const T*>(p.logits) + (first + i) * p.stride;
        const Q* q = static_cast<const Q*>(p.draft_probs) + (GIVEN ? (at + i) * p.probs_stride : 0);
        int d = i < k ? p.drafts[at + i] : -1;
        if (fast)
            for (int s = 0; s < own.count; ++s) {
                const int end = own.hi(s);
                put(sh, s, fast_part(row, own.lo(s), end, c), c, greedy,
                    [&](const Part& t) { return place_of(row, t.at, end, t.m); });
            }
        // asked for here, the drafted token's values arrive while the parts are joined
        float ld = 0.0f, qd = 0.0f, u = 0.0f;
        if (d < 0 || d >= V) d = -1;
        else ld = f32(row[d]), qd = draft_prob(q, d), u = p.uniform[at + i];
        n = i;
        Part all = {-INFINITY, 0.0f, INT_MAX, 0};
        if (fast) all = exchange.part(c);
        bool safe = false;
        if (!(all.z > 0.0f && all.z < INFINITY)) {
            safe = true;
            all = careful_part(row, own, c, exchange);
            exchange.round += CAREFUL_ROUNDS;
            if (all.m == -INFINITY) break;      // nothing left to choose from
        }
        const float m = all.m, inv_z = 1.0f / all.z;
        const float pd = d >= 0 ? weight(ld, m, c) * inv_z : 0.0f;
        if (d >= 0 && (greedy ? d == all.at : u * qd < pd)) {
            if (rank == 0 && threadIdx.x == 0) tokens[i] = d, probs[i] = pd;
            continue;
        }
        token = all.at;
        if (!greedy) {
            const float mc = m * c;
            const Weights wt{m, c, mc, safe ? inv_z : inv_z * ex2(-fmaf(m, c, -mc))};
            // On its way while the race's first loads are: 96 requests 70 us, 71 with no such order. Given at the start of
            // the kernel instead it takes 75: a fifth of these requests are greedy and never read their noise, and the
            // others' (a MB each) displaces rows that the race reads again.
            if (threadIdx.x == 0) prefetch_l2(noise + lo, static_cast<size_t>(hi - lo) * sizeof(float));
            const int out = GIVEN ? -1 : d;
            if (GIVEN && i < k) {
                if constexpr (GIVEN) {
                    if (safe) race_all<true, true>(sh, row, q, noise, out, own, wt);
                    else race_all<false, true>(sh, row, q, noise, out, own, wt);
                }
            } else {
                if (safe) race_all<true, false>(sh, row, q, noise, out, own, wt);
                else race_all<false, false>(sh, row, q, noise, out, own, wt);
            }
            unsigned long long key = exchange.largest();
            const float top = __uint_as_float(static_cast<uint32_t>(key >> 32));
            if (!(top >= SCORE_LO && top <= SCORE_HI)) {
                race_exact<T, Q>(sh, p, b, n, own, m, c, inv_z, safe, top);
                key = exchange.largest();
            }
            token = key_id(key);
            if (!key) {         // no weight left: the target's likeliest token
                token = careful_part(row, own, c, exchange).at;
                if (token == INT_MAX) token = -1;       // (a wait of the exchange gave up)
            }
        }
        if (token >= 0) token_p = weight(f32(row[token]), m, c) * inv_z;
        break;
    }
    if (rank == 0) {
        if (threadIdx.x == 0) p.accepted[b] = n;
        for (int i = n + threadIdx.x; i < width; i += THREADS) {
            tokens[i] = i == n ? token : -1;
            probs[i] = i == n ? token_p : 0.0f;
        }
    }
    cluster_sync_all();     // no CTA leaves while another may store into its shared memory,
    if (sh.gave_up) {       // nor, where it stopped waiting for a store, before that has had time to land
        const uint64_t from = global_ns();
        while (global_ns() - from < 20000) __nanosleep(1000);
    }
}

// Segments of a vocabulary: by its size alone, so that a row's sums do not depend on the batch.
int vocab_segments(int vocab) {
    int n = 1;
    while (n < MAX_SEGMENTS && vocab > n * SEGMENT) n *= 2;
    return n;
}

template <typename T>
auto kernel_of(bool given, int probs_dtype) {
    if (!given) return verify_kernel<T, NoProbs>;
    if (probs_dtype == F32) return verify_kernel<T, float>;
    return probs_dtype == BF16 ? verify_kernel<T, __nv_bfloat16> : verify_kernel<T, __half>;
}

constexpr int MAX_COUNT = 1 << 30;

bool known_dtype(int t) { return t == F16 || t == BF16 || t == F32; }

}  // namespace
}  // namespace esp

ESP_DEFINE_STATUS_READER(verify)

extern "C" int esp_verify(const void* logits, int dtype, long long stride, long long rows, int vocab, const int* starts,
                          int requests, const int* drafts, const float* uniform, long long n_drafts,
                          const void* draft_probs, int probs_dtype, long long probs_stride, const float* noise,
                          long long noise_stride, const float* temperature, int max_drafts, int* tokens, int* accepted,
                          float* probs, void* stream) {
    using namespace esp;
    ESP_REQUIRE(known_dtype(dtype), ESP_ERR_INVALID, "esp_verify: unknown logits dtype %d", dtype);
    ESP_REQUIRE(requests >= 0 && rows >= 0 && n_drafts >= 0 && max_drafts >= 0, ESP_ERR_INVALID,
                "esp_verify: negative size");
    // (ids and places are int, up to a batch of loads past the last)
    ESP_REQUIRE(vocab >= 1 && vocab <= MAX_COUNT && max_drafts <= MAX_COUNT, ESP_ERR_INVALID,
                "esp_verify: vocabulary of %d, %d drafted tokens (1..2^30, up to 2^30)", vocab, max_drafts);
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
    const int segments = vocab_segments(vocab), sms = device_sms();
    int log2 = 0;
    while (1 << log2 < segments && (static_cast<long long>(requests) << log2) < FILL * sms) ++log2;
    const int ctas = 1 << log2;
    ESP_REQUIRE(requests <= INT_MAX >> log2, ESP_ERR_INVALID, "esp_verify: %d requests", requests);
    if (ctas > 8)
        if (const int rc = allow_cluster16(kernel)) return rc;
    const Split split{log2, segments, segments >> log2, (vocab + 8 * segments - 1) / (8 * segments) * 8,
                      requests * ctas <= sms};
    if (const int rc = launch_cluster(kernel, dim3(static_cast<unsigned>(requests) << log2), dim3(THREADS), 0, stream, true,
                                      ctas, p, split))
        return rc;
    return ok();
}
