// Token log probabilities with entropy and top alternatives, forward and backward.
//
// For a row x of V logits, temperature T and z = x / T:
//   lse = log sum_v exp z_v,  log p_v = z_v - lse,  H = lse - sum_v p_v z_v,
//   top_j = log p of the j-th largest logit (equal logits: the lower index first)
//   dx_v = 1/T [ (g_lp [v = i] + sum_j g_top_j [v = top_j]) - p_v (g_lp + sum_j g_top_j)
//               - g_H p_v (log p_v + H) ]
// Bound by memory: the forward reads each live logit once, the backward reads it once more and writes the gradient
// once. Everything is kept in base 2 relative to the row's maximum: with k = log2(e) / T, d_v = (x_v - max) k,
// s = sum 2^d, t = sum 2^d d, so log p = ln2 (d - log2 s) and H = ln2 (log2 s - t / s). All sums are 32 bit.
//
// Four ways over the rows, every thread holding 32 logits in registers, so that logits are read once also where the
// largest are wanted. Times are of bf16 forward calls without the host's part, on both sides of each switch:
//   up to 512 entries (action sets): 16 lanes a row up to 64 entries, else 64, several rows a workgroup (131072 rows of
//   64: 11 us with 16 lanes, 42 us with 64; of 512: 73 us, 398 us as segments; 32 rows of 512: 3.9 and 4.6 us);
//   up to 256 longer rows (and more, where smaller segments offer too many largest entries): segments of up to 32768
//   logits, 1024 threads each. Of 32000 logits with entropy, 256 rows take 8 us and with the eight largest 15 us (10 and
//   20 us in segments of 8192), 257 rows 12 and 27 us (10 and 24 us), as a compute unit holds one such workgroup. Rows of
//   65536 entries on without largest ones would be better off in small segments (256 of 131072: 29 us, 24 us);
//   from 1024 rows on, where no largest are wanted: a workgroup walks a row of its own, see token_stream_fwd (1024 rows of
//   50001: 25 us, 32 us in segments). It is ahead from 257 rows on already (512 rows of 20000: 7.6 and 10 us);
//   else equal segments of up to 8192 logits, 256 threads each.
// The segments of a row are joined by a second, small kernel; a row of one segment needs none.
// 16384 rows of 131072 bf16 logits, three quarters of them live, take 0.55 to 0.6 ms forward (5.4 TB/s) and 1.33 ms
// backward (5.6 TB/s); a large copy reaches 4.9 TB/s here.
#include "common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 32;
constexpr int kSegment = kThreads * kPerThread;
constexpr int kMostTop = 32;
constexpr int64_t kManyRows = 1024;
constexpr int64_t kFewRows = 256;  // one for each compute unit
constexpr int kMostJoined = 4096;  // candidates that a row's segments may offer
constexpr int64_t kMostThreads = ((int64_t)1 << 32) - 1024;  // of a launch; more rows than that go in several
constexpr float kLn2 = 0.69314718055994531f;
// 2^-200 is zero in 32 bits: entries that far below the maximum count nothing, and 0 * -inf is kept out of the sums
constexpr float kFar = -200.f;

struct Rows {
    const void* base;
    int64_t inner;          // row r lies at (r / inner) * outer_stride + (r % inner) * inner_stride elements
    int64_t outer_stride;
    int64_t inner_stride;
};

template <typename T>
__device__ inline const T* row_of(const Rows& rows, int64_t r) {
    return (const T*)rows.base + (r / rows.inner) * rows.outer_stride + (r % rows.inner) * rows.inner_stride;
}

__device__ inline float to_f(float v) { return v; }
__device__ inline float to_f(__half v) { return __half2float(v); }
__device__ inline float to_f(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ inline T from_f(float v);
template <> __device__ inline float from_f<float>(float v) { return v; }
template <> __device__ inline __half from_f<__half>(float v) { return __float2half(v); }
template <> __device__ inline __hip_bfloat16 from_f<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

// 16 bytes of logits; rows of an odd length start anywhere, so the load assumes the element's alignment only
template <typename T>
struct Pack {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};
template <typename T>
__device__ inline Pack<T> load_pack(const T* p) {
    Pack<T> out;
    __builtin_memcpy(&out, p, 16);
    return out;
}
// a gradient is not read again soon: it goes past the caches (2% of a forward and backward pass over 4 GB)
typedef unsigned Quad __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
__device__ inline void store_pack(T* p, const Pack<T>& v) {
    Quad q;
    __builtin_memcpy(&q, &v, 16);
    __builtin_nontemporal_store(q, (Quad*)p);
}

// A value and its index as one integer: larger values first, among equal ones the lower index. -0 equals +0; NaN sorts
// above +inf. 0 is below every entry.
__device__ inline unsigned long long order_of(float x, int index) {
    int bits = __float_as_int(x + 0.f);
    unsigned ordered = (unsigned)(bits ^ ((bits >> 31) & 0x7fffffff)) ^ 0x80000000u;
    if (x != x) ordered = 0xffffffffu;
    return ((unsigned long long)ordered << 32) | (unsigned)(0x7fffffff - index);
}
__device__ inline int index_in(unsigned long long order) { return 0x7fffffff - (int)(unsigned)order; }
__device__ inline float value_in(unsigned long long order) {
    unsigned ordered = (unsigned)(order >> 32) ^ 0x80000000u;
    int bits = (int)ordered;
    return __int_as_float(bits ^ ((bits >> 31) & 0x7fffffff));
}

// (x - m) k in one operation where m k is small: its rounding, up to 2^-24 of it, is a factor of all sums that cancels in
// what comes out, but must not leave their range. Rows of huge logits take two operations.
struct Distance {
    float m, k, mk;
    bool far;
    __device__ inline Distance(float m_, float k_) : m(m_), k(k_), mk(m_ * k_), far(!(fabsf(mk) < 1e4f)) {}
    __device__ inline float operator()(float x) const { return far ? (x - m) * k : fmaf(x, k, -mk); }
    template <bool FAR> __device__ inline float at(float x) const { return FAR ? (x - m) * k : fmaf(x, k, -mk); }
    // from one reference to another, both as they are rounded
    __device__ inline float to_reference(float other) const {
#pragma clang fp contract(off)
        return far ? (other - m) * k : other * k - mk;
    }
};

struct Sums {
    float m, s, t;
};

// sums relative to `to` instead of their own maximum
__device__ inline void shift(Sums& a, float to, float k) {
    float d = fmaxf(Distance(to, k).to_reference(a.m), kFar);
    float f = __builtin_amdgcn_exp2f(d);
    a.t = f * (a.t + d * a.s);
    a.s = f * a.s;
    a.m = to;
}

__device__ inline Sums join(Sums a, Sums b, float k) {
    float m = fmaxf(a.m, b.m);
    shift(a, m, k);
    shift(b, m, k);
    return {m, a.s + b.s, a.t + b.t};
}

// Sums and maxima over W lanes. Within 16 lanes they go through the vector unit's own lane moves, not through LDS.
template <int CTRL>
__device__ inline float moved(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int W, typename F>
__device__ inline float group(float v, F&& f) {
    v = f(v, moved<0xb1>(v));   // lanes 1 0 3 2
    v = f(v, moved<0x4e>(v));   // lanes 2 3 0 1
    v = f(v, moved<0x141>(v));  // the half row turned round
    v = f(v, moved<0x140>(v));  // the row turned round
    if constexpr (W == 64) {
        auto row = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); };
        v = f(f(row(0), row(16)), f(row(32), row(48)));
    }
    return v;
}
template <int W>
__device__ inline float group_max(float v) {
    return group<W>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int W>
__device__ inline float group_sum(float v) {
    return group<W>(v, [](float a, float b) { return a + b; });
}
template <int W>
__device__ inline unsigned long long group_max(unsigned long long v) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
        unsigned long long u = __shfl_xor(v, o, W);
        v = u > v ? u : v;
    }
    return v;
}

struct Out {
    float* log_prob;      // [rows]
    float* entropy;       // [rows] or null
    float* stats;         // [rows, 2]: maximum, log2 s
    float* top_log_prob;  // [rows, top]
    int64_t* top_index;   // [rows, top]
};

__device__ inline float log2_of(float s) { return __builtin_amdgcn_logf(s); }

// What roundings put on the wrong side of zero is zero; NaN stays.
__device__ inline float at_most_zero(float v) { return v > 0.f ? 0.f : v; }
__device__ inline float at_least_zero(float v) { return v < 0.f ? 0.f : v; }

// what one lane writes for a row whose sums are known
template <typename T>
__device__ inline void write_row(const Out& out, int64_t r, Sums a, const T* x, int64_t token, int V, float k) {
    float log2s = log2_of(a.s);
    float lp = __builtin_nanf("");
    if (token >= 0 && token < V) lp = at_most_zero((Distance(a.m, k)(to_f(x[token])) - log2s) * kLn2);
    out.log_prob[r] = lp;
    if (out.entropy) out.entropy[r] = at_least_zero((log2s - a.t / a.s) * kLn2);
    out.stats[2 * r] = a.m;
    out.stats[2 * r + 1] = log2s;
}

__device__ inline void write_top(const Out& out, int64_t r, int top, int j, unsigned long long order, float m,
                                 float log2s, float k) {
    out.top_log_prob[r * top + j] = at_most_zero((Distance(m, k)(value_in(order)) - log2s) * kLn2);
    out.top_index[r * top + j] = index_in(order);
}

__device__ inline void write_nothing(const Out& out, int64_t r, int top, int lane, int lanes) {
    if (lane == 0) {
        out.log_prob[r] = 0.f;
        if (out.entropy) out.entropy[r] = 0.f;
        out.stats[2 * r] = 0.f;
        out.stats[2 * r + 1] = 0.f;
    }
    for (int j = lane; j < top; j += lanes) {
        out.top_log_prob[r * top + j] = 0.f;
        out.top_index[r * top + j] = -1;
    }
}

// ---------------------------------------------------------------------------------------------- short rows, forward
// LANES lanes hold a row in registers, PER entries each.
template <typename T, int LANES, int PER>
__global__ void __launch_bounds__(kThreads) token_short_fwd(
    Rows rows, const int64_t* __restrict__ index, Out out, int64_t first, int64_t end, int V, float k, int64_t ignore,
    int has_ignore, int top
) {
    int lane = threadIdx.x % LANES;
    int64_t r = first + (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    if (r >= end) return;
    int64_t token = index[r];
    if (has_ignore && token == ignore) {
        write_nothing(out, r, top, lane, LANES);
        return;
    }
    const T* x = row_of<T>(rows, r);
    float v[PER];
    Sums a{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        int c = j * LANES + lane;
        v[j] = c < V ? to_f(x[c]) : -INFINITY;
        a.m = fmaxf(a.m, v[j]);
    }
    a.m = group_max<LANES>(a.m);
    Distance distance(a.m == -INFINITY ? 0.f : a.m, k);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        float d = distance(v[j]);
        float e = __builtin_amdgcn_exp2f(d);
        a.s += e;
        a.t += e * fmaxf(d, kFar);
    }
    a.s = group_sum<LANES>(a.s);
    a.t = group_sum<LANES>(a.t);
    if (lane == 0) write_row(out, r, a, x, token, V, k);
    float log2s = log2_of(a.s);
    unsigned long long below = ~0ull;
    for (int j = 0; j < top; ++j) {
        unsigned long long best = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int c = i * LANES + lane;
            unsigned long long o = c < V ? order_of(v[i], c) : 0;
            if (o < below && o > best) best = o;
        }
        below = group_max<LANES>(best);
        if (lane == 0) write_top(out, r, top, j, below, a.m, log2s, k);
    }
}

// ----------------------------------------------------------------------------------------------- long rows, forward

// `top` largest of n orders in LDS, in descending order: each one's place is the number of larger ones
template <typename F>
__device__ inline void rank_orders(const unsigned long long* orders, int n, int top, F&& put) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        unsigned long long mine = orders[i];
        if (mine == 0) continue;
        int larger = 0;
        for (int j = 0; j < n && larger < top; ++j) larger += orders[j] > mine;
        if (larger < top) put(larger, mine);
    }
}

template <typename T, bool TOP, bool ENTROPY, int THREADS>
__global__ void __launch_bounds__(THREADS) token_segment_fwd(
    Rows rows, const int64_t* __restrict__ index, Out out, int64_t first, int V, int segments, int length, float k,
    int64_t ignore, int has_ignore, int top, float* __restrict__ partial, unsigned long long* __restrict__ offered
) {
    constexpr int N = Pack<T>::N;
    int64_t r = first + blockIdx.x / segments;
    int seg = blockIdx.x % segments;
    int tid = threadIdx.x;
    int64_t token = index[r];
    if (has_ignore && token == ignore) {
        if (seg == 0) write_nothing(out, r, top, tid, THREADS);
        return;
    }
    const T* x = row_of<T>(rows, r);
    int lo = seg * length, hi = min(V, lo + length);
    Pack<T> v[kPerThread / N];
#pragma unroll
    for (int j = 0; j < kPerThread / N; ++j) {
        int c = lo + (j * THREADS + tid) * N;
        if (c + N <= hi) {
            v[j] = load_pack(x + c);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[j].v[i] = c + i < hi ? x[c + i] : from_f<T>(-INFINITY);
        }
    }
    Sums a{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kPerThread / N; ++j)
#pragma unroll
        for (int i = 0; i < N; i += 2) a.m = fmaxf(a.m, fmaxf(to_f(v[j].v[i]), to_f(v[j].v[i + 1])));
    a.m = group_max<kWave>(a.m);
    Distance distance(a.m == -INFINITY ? 0.f : a.m, k);
    auto add = [&](auto far) {
#pragma unroll
        for (int j = 0; j < kPerThread / N; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float d = distance.template at<decltype(far)::value>(to_f(v[j].v[i]));
                float e = __builtin_amdgcn_exp2f(d);
                a.s += e;
                if (ENTROPY) a.t += e * fmaxf(d, kFar);
            }
    };
    if (distance.far)
        add(std::true_type{});
    else
        add(std::false_type{});
    a.s = group_sum<kWave>(a.s);
    if (ENTROPY) a.t = group_sum<kWave>(a.t);
    __shared__ Sums part[THREADS / kWave];
    if (tid % kWave == 0) part[tid / kWave] = a;

    // Largest entries. Of the largest of 64 groups of lanes, the top-th is a bound that all wanted entries reach, and only
    // `top` groups hold entries that reach it: at most top * GROUP * kPerThread candidates, and far fewer as a rule.
    constexpr int GROUP = THREADS / 64;
    __shared__ unsigned long long best[TOP ? 64 : 1];
    __shared__ unsigned long long bound_s;
    __shared__ unsigned long long candidates[TOP ? kMostTop * GROUP * kPerThread : 1];
    __shared__ int found;
    if constexpr (TOP) {
        unsigned long long mine = 0;
#pragma unroll
        for (int j = 0; j < kPerThread / N; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                int c = lo + (j * THREADS + tid) * N + i;
                unsigned long long o = c < hi ? order_of(to_f(v[j].v[i]), c) : 0;
                mine = o > mine ? o : mine;
            }
        mine = group_max<GROUP>(mine);
        if (tid % GROUP == 0) best[tid / GROUP] = mine;
        if (tid == 0) {
            bound_s = 1;  // fewer than `top` groups hold entries: all of theirs are candidates
            found = 0;
        }
        __syncthreads();
        if (tid < 64) {
            mine = best[tid];
            int larger = 0;
#pragma unroll 8
            for (int j = 0; j < 64; ++j) larger += best[j] > mine;
            if (mine != 0 && larger == top - 1) bound_s = mine;
        }
        __syncthreads();
        unsigned long long bound = bound_s;
#pragma unroll
        for (int j = 0; j < kPerThread / N; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                int c = lo + (j * THREADS + tid) * N + i;
                unsigned long long o = c < hi ? order_of(to_f(v[j].v[i]), c) : 0;
                if (o >= bound) candidates[atomicAdd(&found, 1)] = o;
            }
    }
    __syncthreads();
    Sums all = part[0];
#pragma unroll
    for (int w = 1; w < THREADS / kWave; ++w) all = join(all, part[w], k);
    if (segments == 1) {
        if (tid == 0) write_row(out, r, all, x, token, V, k);
        if constexpr (TOP) {
            float log2s = log2_of(all.s);
            rank_orders(candidates, found, top, [&](int j, unsigned long long o) {
                write_top(out, r, top, j, o, all.m, log2s, k);
            });
        }
    } else {
        if (tid == 0) {
            float* p = partial + 3 * (int64_t)blockIdx.x;
            p[0] = all.m;
            p[1] = all.s;
            p[2] = all.t;
        }
        if constexpr (TOP) {
            unsigned long long* mine = offered + (int64_t)blockIdx.x * top;
            for (int j = tid; j < top; j += THREADS)
                if (j >= found) mine[j] = 0;
            rank_orders(candidates, found, top, [&](int j, unsigned long long o) { mine[j] = o; });
        }
    }
}

// A workgroup walks a whole row, the next 8192 logits on their way while it sums the present ones; each thread keeps
// sums of its own and moves their reference when it meets a larger logit. For many rows: the chip is full then, and
// segments of their own would spend their time on starting (16384 rows of 131072 bf16 logits with entropy, of which three
// quarters are live: 0.57 ms, in segments 0.76 ms; 8184 rows of 50001, six tenths live: 125 us against 135).
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads) token_stream_fwd(
    Rows rows, const int64_t* __restrict__ index, Out out, int64_t first, int V, float k, int64_t ignore, int has_ignore
) {
    constexpr int N = Pack<T>::N, PACKS = kPerThread / N;
    int64_t r = first + blockIdx.x;
    int tid = threadIdx.x;
    int64_t token = index[r];
    if (has_ignore && token == ignore) {
        write_nothing(out, r, 0, tid, kThreads);
        return;
    }
    const T* x = row_of<T>(rows, r);
    Pack<T> now[PACKS], next[PACKS];
    auto load = [&](Pack<T>(&v)[PACKS], int lo) {
        if (lo + kSegment <= V) {
#pragma unroll
            for (int j = 0; j < PACKS; ++j) v[j] = load_pack(x + lo + (j * kThreads + tid) * N);
        } else {
#pragma unroll
            for (int j = 0; j < PACKS; ++j) {
                int c = lo + (j * kThreads + tid) * N;
                if (c + N <= V) {
                    v[j] = load_pack(x + c);
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) v[j].v[i] = c + i < V ? x[c + i] : from_f<T>(-INFINITY);
                }
            }
        }
    };
    Sums a{-INFINITY, 0.f, 0.f};
    load(now, 0);
    for (int lo = 0; lo < V; lo += kSegment) {
        if (lo + kSegment < V) load(next, lo + kSegment);
        float m = a.m;
#pragma unroll
        for (int j = 0; j < PACKS; ++j)
#pragma unroll
            for (int i = 0; i < N; i += 2) m = fmaxf(m, fmaxf(to_f(now[j].v[i]), to_f(now[j].v[i + 1])));
        if (m > a.m) shift(a, m, k);
        Distance distance(m == -INFINITY ? 0.f : m, k);
        auto add = [&](auto far) {
#pragma unroll
            for (int j = 0; j < PACKS; ++j)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    float d = distance.template at<decltype(far)::value>(to_f(now[j].v[i]));
                    float e = __builtin_amdgcn_exp2f(d);
                    a.s += e;
                    if (ENTROPY) a.t += e * fmaxf(d, kFar);
                }
        };
        if (distance.far)
            add(std::true_type{});
        else
            add(std::false_type{});
#pragma unroll
        for (int j = 0; j < PACKS; ++j) now[j] = next[j];
    }
    float m = group_max<kWave>(a.m);
    shift(a, m, k);
    a.s = group_sum<kWave>(a.s);
    if (ENTROPY) a.t = group_sum<kWave>(a.t);
    __shared__ Sums part[kThreads / kWave];
    if (tid % kWave == 0) part[tid / kWave] = a;
    __syncthreads();
    if (tid == 0) {
        Sums all = part[0];
#pragma unroll
        for (int w = 1; w < kThreads / kWave; ++w) all = join(all, part[w], k);
        write_row(out, r, all, x, token, V, k);
    }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) token_join(
    Rows rows, const int64_t* __restrict__ index, Out out, int64_t first, int64_t end, int V, int segments, float k,
    int64_t ignore, int has_ignore, int top, const float* __restrict__ partial,
    const unsigned long long* __restrict__ offered
) {
    // with largest entries a workgroup joins one row, else each of its waves does
    int lane = threadIdx.x % kWave;
    int64_t own = TOP ? blockIdx.x : (int64_t)blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave, r = first + own;
    if (r >= end) return;
    int64_t token = index[r];
    if (has_ignore && token == ignore) return;
    Sums a{-INFINITY, 0.f, 0.f};
    for (int g = lane; g < segments; g += kWave) {
        const float* p = partial + 3 * (own * segments + g);
        a = join(a, Sums{p[0], p[1], p[2]}, k);
    }
    float m = group_max<kWave>(a.m);
    shift(a, m, k);
    a.s = group_sum<kWave>(a.s);
    a.t = group_sum<kWave>(a.t);
    if (TOP ? threadIdx.x == 0 : lane == 0) write_row(out, r, a, row_of<T>(rows, r), token, V, k);
    if constexpr (TOP) {
        __shared__ unsigned long long orders[kMostJoined];
        int n = segments * top;
        for (int i = threadIdx.x; i < n; i += kThreads) orders[i] = offered[own * n + i];
        __syncthreads();
        float log2s = log2_of(a.s);
        rank_orders(orders, n, top, [&](int j, unsigned long long o) { write_top(out, r, top, j, o, a.m, log2s, k); });
    }
}

// --------------------------------------------------------------------------------------------------------- backward

struct Grads {
    const float* log_prob;  // [rows] or null
    const float* entropy;   // [rows] or null
    const float* top;       // [rows, top] or null
    const float* stats;
    const float* h;         // [rows]: the entropy itself, where its gradient is given
    const int64_t* top_index;
};

// what a row's gradient is made of: dx_v = p_v (c0 + c1 log2 p_v) + [v is one of the row's tokens] its own share
struct RowGrad {
    float m, log2s, c0, c1;
};

__device__ inline RowGrad row_grad(const Grads& g, int64_t r, int top, int64_t token, int V, float inv_t) {
    RowGrad a{g.stats[2 * r], g.stats[2 * r + 1], 0.f, 0.f};
    float sum = 0.f;
    if (g.log_prob) {
        sum = g.log_prob[r];
        if (token < 0 || token >= V) sum = __builtin_nanf("");
    }
    if (g.top)
        for (int j = 0; j < top; ++j) sum += g.top[r * top + j];
    a.c0 = -sum * inv_t;
    if (g.entropy) {
        float ge = g.entropy[r] * inv_t;
        a.c0 -= ge * g.h[r];
        a.c1 = -ge * kLn2;
    }
    return a;
}

template <bool FAR, bool ENTROPY>
__device__ inline float grad_at(const RowGrad& a, const Distance& distance, float x) {
    float d = distance.at<FAR>(x) - a.log2s, p = __builtin_amdgcn_exp2f(d);
    return ENTROPY ? p * fmaf(a.c1, fmaxf(d, kFar), a.c0) : p * a.c0;
}
__device__ inline float grad_at(const RowGrad& a, float x, float k) {
    Distance distance(a.m, k);
    return distance.far ? grad_at<true, true>(a, distance, x) : grad_at<false, true>(a, distance, x);
}

// the share of column c alone, and whether lane j is the one that adds it: lanes 0..top-1 stand for the largest
// entries, lane `top` for the token where it is none of them
__device__ inline bool own_share(const Grads& g, int64_t r, int top, int j, int64_t token, int V, float inv_t,
                                 int& column, float& share) {
    bool valid = g.log_prob && token >= 0 && token < V;
    float glp = valid ? g.log_prob[r] : 0.f;
    if (j < top && g.top) {
        column = (int)g.top_index[r * top + j];
        share = (g.top[r * top + j] + (valid && column == token ? glp : 0.f)) * inv_t;
        return true;
    }
    if (j == top && valid) {
        if (g.top)
            for (int i = 0; i < top; ++i)
                if (g.top_index[r * top + i] == token) return false;
        column = (int)token;
        share = glp * inv_t;
        return true;
    }
    return false;
}

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) token_short_bwd(
    Rows rows, const int64_t* __restrict__ index, Grads g, T* __restrict__ grad, int64_t first, int64_t end, int V,
    float k, float inv_t, int64_t ignore, int has_ignore, int top
) {
    int lane = threadIdx.x % LANES;
    int64_t r = first + (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    if (r >= end) return;
    int64_t token = index[r];
    T* out = grad + r * V;
    if (has_ignore && token == ignore) {
        for (int c = lane; c < V; c += LANES) out[c] = from_f<T>(0.f);
        return;
    }
    const T* x = row_of<T>(rows, r);
    RowGrad a = row_grad(g, r, top, token, V, inv_t);
    for (int c = lane; c < V; c += LANES) {
        float v = grad_at(a, to_f(x[c]), k);
        for (int j = 0; j <= top; ++j) {
            int column;
            float share;
            if (own_share(g, r, top, j, token, V, inv_t, column, share) && column == c) v += share;
        }
        out[c] = from_f<T>(v);
    }
}

template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads) token_segment_bwd(
    Rows rows, const int64_t* __restrict__ index, Grads g, T* __restrict__ grad, int64_t first, int V, int segments,
    int length, float k, float inv_t, int64_t ignore, int has_ignore, int top
) {
    constexpr int N = Pack<T>::N;
    int64_t r = first + blockIdx.x / segments;
    int lo = (blockIdx.x % segments) * length, hi = min(V, lo + length);
    int tid = threadIdx.x;
    int64_t token = index[r];
    T* out = grad + r * V;
    bool live = !(has_ignore && token == ignore);
    const T* x = row_of<T>(rows, r);
    RowGrad a{0.f, 0.f, 0.f, 0.f};
    if (live) a = row_grad(g, r, top, token, V, inv_t);
    Distance distance(a.m, k);
    auto write = [&](auto far) {
        constexpr bool FAR = decltype(far)::value;
#pragma unroll
        for (int j = 0; j < kPerThread / N; ++j) {
            int c = lo + (j * kThreads + tid) * N;
            if (c + N <= hi) {
                Pack<T> v, o;
                if (live) v = load_pack(x + c);
#pragma unroll
                for (int i = 0; i < N; ++i)
                    o.v[i] = from_f<T>(live ? grad_at<FAR, ENTROPY>(a, distance, to_f(v.v[i])) : 0.f);
                store_pack(out + c, o);
            } else {
                for (int i = 0; c + i < hi; ++i)
                    out[c + i] = from_f<T>(live ? grad_at<FAR, ENTROPY>(a, distance, to_f(x[c + i])) : 0.f);
            }
        }
    };
    if (distance.far)
        write(std::true_type{});
    else
        write(std::false_type{});
    if (!live) return;
    __syncthreads();  // the single columns are written again, whole, after the others
    int column;
    float share;
    if (tid <= top && own_share(g, r, top, tid, token, V, inv_t, column, share) && column >= lo &&
        column < hi)
        out[column] = from_f<T>(grad_at(a, to_f(x[column]), k) + share);
}

// ------------------------------------------------------------------------------------------------------------- host

// Leading dimensions fold into two where their strides allow it; `logits` is replaced by a dense copy where not.
Rows rows_of(torch::Tensor& logits) {
    for (;;) {
        int64_t size[2] = {1, 1}, stride[2] = {0, 0};
        int n = 0;  // folded dimensions so far, from the inner side
        bool fits = logits.stride(-1) == 1 || logits.size(-1) == 1;
        for (int64_t d = logits.dim() - 2; d >= 0 && fits; --d) {
            if (logits.size(d) == 1) continue;
            if (n > 0 && logits.stride(d) == stride[n - 1] * size[n - 1]) {
                size[n - 1] *= logits.size(d);
            } else if (n < 2) {
                size[n] = logits.size(d);
                stride[n++] = logits.stride(d);
            } else {
                fits = false;
            }
        }
        if (fits) return {logits.data_ptr(), size[0], stride[1], stride[0]};
        logits = logits.contiguous();
    }
}

void check_args(const torch::Tensor& logits, const torch::Tensor& index) {
    TORCH_CHECK(logits.is_cuda() && logits.dim() >= 1 && index.device() == logits.device() && index.is_contiguous() &&
                    index.scalar_type() == torch::kInt64 && index.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                "token_log_prob: logits [..., V] and index [...] must be on one HIP device");
    TORCH_CHECK(logits.size(-1) >= 1 && logits.size(-1) <= (1 << 30), "token_log_prob: V must be in [1, 2^30]");
}

// segments of a row are equally long, in whole packs
int length_of(int V, int segments) { return ((V + segments - 1) / segments + 7) / 8 * 8; }

// go(first, end) for as many rows at a time as a launch holds
template <typename F>
void in_launches(int64_t count, int64_t threads_a_row, F&& go) {
    int64_t most = std::max<int64_t>(1, kMostThreads / threads_a_row);
    for (int64_t first = 0; first < count; first += most) {
        go(first, std::min(count, first + most));
        HIP_CHECK_LAST();
    }
}

template <typename F>
void by_type(const torch::Tensor& x, F&& f) {
    switch (x.scalar_type()) {
        case torch::kFloat32: f((float*)nullptr); break;
        case torch::kFloat16: f((__half*)nullptr); break;
        case torch::kBFloat16: f((__hip_bfloat16*)nullptr); break;
        default: TORCH_CHECK(false, "expected float32, float16 or bfloat16");
    }
}

std::vector<torch::Tensor> token_log_prob_fwd(
    torch::Tensor logits, torch::Tensor index, double temperature, int64_t ignore, int64_t has_ignore,
    int64_t want_entropy, int64_t top
) {
    check_args(logits, index);
    c10::OptionalDeviceGuard guard(logits.device());
    Rows rows = rows_of(logits);
    int64_t count = index.numel();
    int V = (int)logits.size(-1);
    // few long rows: four times as many threads hold a segment, which saves the joining launch up to 32768 entries; else
    // where smaller segments would offer more candidates than the joining kernel holds
    bool large = V > kSegment && (count <= kFewRows || top * cdiv(V, kSegment) > kMostJoined);
    int segments = cdiv(V, large ? 4 * kSegment : kSegment);
    TORCH_CHECK(top >= 0 && top <= kMostTop && top <= V, "token_log_prob: top_k must be at most ", kMostTop, " and V");
    TORCH_CHECK(segments == 1 || top * segments <= kMostJoined, "token_log_prob: top_k times a row's segments of ",
                4 * kSegment, " entries must be at most ", kMostJoined, ", got ", top, " over ", V);
    auto opt = logits.options().dtype(torch::kFloat32);
    auto tops = index.sizes().vec();
    tops.push_back(top);
    auto log_prob = torch::empty(index.sizes(), opt);
    auto entropy = want_entropy ? torch::empty(index.sizes(), opt) : torch::empty({0}, opt);
    auto stats = torch::empty({count, 2}, opt);
    auto top_log_prob = top ? torch::empty(tops, opt) : torch::empty({0}, opt);
    auto top_index = top ? torch::empty(tops, opt.dtype(torch::kInt64)) : torch::empty({0}, opt.dtype(torch::kInt64));
    std::vector<torch::Tensor> result{log_prob, entropy, stats, top_log_prob, top_index};
    if (count == 0) return result;
    Out out{log_prob.data_ptr<float>(), want_entropy ? entropy.data_ptr<float>() : nullptr, stats.data_ptr<float>(),
            top_log_prob.data_ptr<float>(), top_index.data_ptr<int64_t>()};
    float k = (float)(1.4426950408889634 / temperature);
    hipStream_t stream = ding_current_stream();
    const int64_t* ix = index.data_ptr<int64_t>();
    by_type(logits, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        if (V <= 64) {
            in_launches(count, 16, [&](int64_t first, int64_t end) {
                token_short_fwd<T, 16, 4><<<cdiv(end - first, kThreads / 16), kThreads, 0, stream>>>(
                    rows, ix, out, first, end, V, k, ignore, has_ignore, top);
            });
        } else if (V <= 512) {
            in_launches(count, 64, [&](int64_t first, int64_t end) {
                token_short_fwd<T, 64, 8><<<cdiv(end - first, kThreads / 64), kThreads, 0, stream>>>(
                    rows, ix, out, first, end, V, k, ignore, has_ignore, top);
            });
        } else if (top == 0 && segments > 1 && count >= kManyRows) {
            in_launches(count, kThreads, [&](int64_t first, int64_t end) {
                auto go = [&](auto kernel) {
                    kernel<<<(unsigned)(end - first), kThreads, 0, stream>>>(rows, ix, out, first, V, k, ignore, has_ignore);
                };
                want_entropy ? go(token_stream_fwd<T, true>) : go(token_stream_fwd<T, false>);
            });
        } else {
            int threads = large ? 4 * kThreads : kThreads, length = length_of(V, segments);
            in_launches(count, (int64_t)segments * threads, [&](int64_t first, int64_t end) {
                int64_t groups = (end - first) * segments;
                torch::Tensor partial, offered;
                float* p = nullptr;
                unsigned long long* o = nullptr;
                if (segments > 1) {
                    partial = torch::empty({groups * 3}, opt);
                    p = partial.data_ptr<float>();
                    if (top > 0) {
                        offered = torch::empty({groups * top}, opt.dtype(torch::kInt64));
                        o = (unsigned long long*)offered.data_ptr<int64_t>();
                    }
                }
                auto go = [&](auto kernel) {
                    kernel<<<(unsigned)groups, threads, 0, stream>>>(rows, ix, out, first, V, segments, length, k, ignore,
                                                                     has_ignore, top, p, o);
                };
                if (top > 0)
                    large ? go(token_segment_fwd<T, true, true, 4 * kThreads>) : go(token_segment_fwd<T, true, true, kThreads>);
                else if (large)
                    go(token_segment_fwd<T, false, true, 4 * kThreads>);
                else if (want_entropy)
                    go(token_segment_fwd<T, false, true, kThreads>);
                else
                    go(token_segment_fwd<T, false, false, kThreads>);
                if (segments > 1) {
                    HIP_CHECK_LAST();
                    if (top > 0)
                        token_join<T, true><<<(unsigned)(end - first), kThreads, 0, stream>>>(
                            rows, ix, out, first, end, V, segments, k, ignore, has_ignore, top, p, o);
                    else
                        token_join<T, false><<<cdiv(end - first, kThreads / kWave), kThreads, 0, stream>>>(
                            rows, ix, out, first, end, V, segments, k, ignore, has_ignore, top, p, o);
                }
            });
        }
    });
    return result;
}

torch::Tensor token_log_prob_bwd(
    torch::Tensor logits, torch::Tensor index, torch::Tensor stats, torch::Tensor entropy, torch::Tensor top_index,
    torch::Tensor grad_log_prob, torch::Tensor grad_entropy, torch::Tensor grad_top, double temperature,
    int64_t ignore, int64_t has_ignore
) {
    check_args(logits, index);
    c10::OptionalDeviceGuard guard(logits.device());
    Rows rows = rows_of(logits);
    int64_t count = index.numel();
    int V = (int)logits.size(-1);
    int segments = cdiv(V, kSegment);
    int top = grad_top.defined() ? (int)top_index.size(-1) : 0;
    auto given = [&](const torch::Tensor& t, int64_t n) -> const float* {
        if (!t.defined() || t.numel() == 0) return nullptr;
        TORCH_CHECK(t.device() == logits.device() && t.is_contiguous() && t.scalar_type() == torch::kFloat32 &&
                        t.numel() == n, "token_log_prob: a gradient has another shape, type or device");
        return t.data_ptr<float>();
    };
    auto grad = torch::empty(logits.sizes(), logits.options());
    if (grad.numel() == 0) return grad;
    Grads g{given(grad_log_prob, count), given(grad_entropy, count), given(grad_top, count * top),
            given(stats, 2 * count), given(entropy, count), top ? top_index.data_ptr<int64_t>() : nullptr};
    TORCH_CHECK(g.stats && (g.h || !g.entropy), "token_log_prob: what the forward pass kept is missing");
    float k = (float)(1.4426950408889634 / temperature), inv_t = (float)(1.0 / temperature);
    hipStream_t stream = ding_current_stream();
    const int64_t* ix = index.data_ptr<int64_t>();
    by_type(logits, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        T* to = (T*)grad.data_ptr();
        if (V <= 64)
            in_launches(count, 16, [&](int64_t first, int64_t end) {
                token_short_bwd<T, 16><<<cdiv(end - first, kThreads / 16), kThreads, 0, stream>>>(
                    rows, ix, g, to, first, end, V, k, inv_t, ignore, has_ignore, top);
            });
        else if (V <= 512)
            in_launches(count, 64, [&](int64_t first, int64_t end) {
                token_short_bwd<T, 64><<<cdiv(end - first, kThreads / 64), kThreads, 0, stream>>>(
                    rows, ix, g, to, first, end, V, k, inv_t, ignore, has_ignore, top);
            });
        else
            in_launches(count, (int64_t)segments * kThreads, [&](int64_t first, int64_t end) {
                auto go = [&](auto kernel) {
                    kernel<<<(unsigned)((end - first) * segments), kThreads, 0, stream>>>(
                        rows, ix, g, to, first, V, segments, length_of(V, segments), k, inv_t, ignore, has_ignore, top);
                };
                g.entropy ? go(token_segment_bwd<T, true>) : go(token_segment_bwd<T, false>);
            });
    });
    return grad;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Rows keep their maximum and log-sum (8 bytes) for the backward pass, not their probabilities.
struct TokenLogProb : torch::autograd::Function<TokenLogProb> {
    static variable_list forward(AutogradContext* ctx, torch::Tensor logits, torch::Tensor index, double temperature,
                                 int64_t ignore, bool has_ignore, bool entropy, int64_t top) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto out = token_log_prob_fwd(logits, index, temperature, ignore, has_ignore, entropy, top);
        ctx->save_for_backward({logits, index, out[2], out[1], out[4]});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["ignore"] = ignore;
        ctx->saved_data["has_ignore"] = has_ignore;
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({out[4]});
        return {out[0], out[1], out[3], out[4]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        auto kept = ctx->get_saved_variables();
        torch::Tensor grad;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            auto dense = [](const torch::Tensor& t) { return t.defined() && t.numel() ? t.contiguous() : torch::Tensor(); };
            grad = token_log_prob_bwd(kept[0], kept[1], kept[2], kept[3], kept[4], dense(g[0]), dense(g[1]), dense(g[2]),
                                      ctx->saved_data["temperature"].toDouble(), ctx->saved_data["ignore"].toInt(),
                                      ctx->saved_data["has_ignore"].toBool());
        }
        torch::Tensor none;
        return ding_once_differentiable({grad, none, none, none, none, none, none}, "token_log_prob");
    }
};

}  // namespace

// log probabilities, entropy, top log probabilities and indexes of tokens; differentiable once
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> token_log_prob(
    torch::Tensor logits, torch::Tensor index, double temperature, c10::optional<int64_t> ignore_index, bool entropy,
    int64_t top_k
) {
    index = index.to(torch::kInt64).contiguous();
    if (logits.is_cuda() && logits.dim() > 0) rows_of(logits);  // what has to be copied is copied for both directions
    auto out = TokenLogProb::apply(logits, index, temperature, ignore_index.value_or(0), ignore_index.has_value(),
                                   entropy, top_k);
    return {out[0], out[1], out[2], out[3]};
}
