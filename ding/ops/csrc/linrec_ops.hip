// Gated linear recurrence over time, forward and backward.
//
//   a_t = sigmoid(f_t),  r_t = 0 where an episode starts at t, else 1
//   h_t = r_t a_t h_{t-1} + (1 - a_t) x_t
// Backward, with G_t the whole gradient of h_t:
//   G_t = g_t + r_{t+1} a_{t+1} G_{t+1}   (g_last joins at the last step)
//   dx_t = (1 - a_t) G_t,  df_t = G_t (r_t h_{t-1} - x_t) a_t (1 - a_t),  dh0 = r_0 a_0 G_0
// Bound by memory: two values read and one written a step forward, three read and two written backward. 32768 steps of
// 2 x 2048 in bfloat16 take 187 us forward (4.3 TB/s of what has to move; a large copy reaches 4.9) and 292 us backward
// (4.6 TB/s); waiting for earlier tiles is a tenth of that. Odd numbers of 16-bit channels cost a quarter more: every
// other row starts between two 4-byte words. The state is 32 bit throughout; the states that the backward pass needs are
// computed again from the states at the tiles' starts, not read from the rounded outputs.
//
// A tile is up to 128 steps of 64 lanes' columns (4 bytes of channels a lane: two of 16 bits, one of 32), held in
// registers: each of up to 8 waves takes kSteps steps, scans them from nothing, and gives the pair (A, B) that its steps
// make of a state s, A s + B. The waves' pairs are joined in LDS; the state that enters the tile comes from the tile
// before it. Inputs are so read once, at any length.
//
// Tiles of one column group follow each other by a chain in memory. A tile leaves two 64-bit words a column: its pair
// (A, B) as soon as it has it, and the state after the tile once it knows it. To know the state before it, a tile's
// waves look at the tiles before it, one each: the nearest known state is carried through the pairs of the tiles in
// between, one multiplication after the other, as if the state had been handed on from tile to tile; so results do not
// depend on who came first. The eighth wave waits for a state, the others for either word: states move eight tiles at a
// time. Tiles are handed out by a counter, in the order of time, so that what a tile waits for has been handed out
// before it, to a workgroup that runs already and that waits, if at all, for earlier ones only: every wait ends. The
// forward pass's words stay for the backward pass: they hold the states at the tiles' starts, and the states within a
// tile are computed again from them. The backward pass runs the same chain from the last tile to the first, with
// M_t = r_t a_t (g_t + M_{t+1}) in the place of the state.
//
// A reset makes A a negative zero: what comes before is then not multiplied but left out, also where it is not finite.
#include "common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

constexpr int kMostWaves = 8;
constexpr int kSteps = 16;  // of a wave, in a tile
constexpr int kTile = kMostWaves * kSteps;

template <typename T> __device__ inline T from_f(float v);
template <> __device__ inline float from_f<float>(float v) { return v; }

// 4 bytes of channels and what they stand for
template <typename T> struct Lane {
    static constexpr int N = 4 / sizeof(T);
};
__device__ inline float value_of(uint32_t raw, int j, const float*) { return __uint_as_float(raw); }
__device__ inline float value_of(uint32_t raw, int j, const __half*) {
    return __half2float(__ushort_as_half((unsigned short)(j ? raw >> 16 : raw)));
}
__device__ inline float value_of(uint32_t raw, int j, const __hip_bfloat16*) {
    return __uint_as_float(j ? raw & 0xffff0000u : raw << 16);
}
__device__ inline uint32_t bits_of(float v, const float*) { return __float_as_uint(v); }
__device__ inline uint32_t bits_of(float v, const __half*) { return __half_as_ushort(__float2half(v)); }
__device__ inline uint32_t bits_of(float v, const __hip_bfloat16*) {
    __hip_bfloat16 b = __float2bfloat16(v);
    unsigned short u;
    __builtin_memcpy(&u, &b, 2);
    return u;
}

// +inf as a gate keeps the state and takes nothing in: what stands for steps behind the last one
__device__ inline uint32_t open_gate(const float*) { return 0x7f800000u; }
__device__ inline uint32_t open_gate(const __half*) { return 0x7c007c00u; }
__device__ inline uint32_t open_gate(const __hip_bfloat16*) { return 0x7f807f80u; }

struct Seq {
    const void* base;
    int64_t t_stride, b_stride;  // elements; channels are dense
};

// The columns of a lane in an input. `dense`: every lane of the wave finds its channels side by side.
template <typename T>
struct Columns {
    int64_t at[2];
    bool dense;
    __device__ inline uint32_t load(const T* p) const {
        uint32_t raw;
        if constexpr (sizeof(T) == 4) {
            __builtin_memcpy(&raw, p + at[0], 4);
        } else if (dense) {
            __builtin_memcpy(&raw, p + at[0], 4);  // rows of an odd length start at any element
        } else {
            uint16_t lo, hi;
            __builtin_memcpy(&lo, p + at[0], 2);
            __builtin_memcpy(&hi, p + at[1], 2);
            raw = lo | (uint32_t)hi << 16;
        }
        return raw;
    }
};

// Lanes behind the last column read what the wave's first lane reads, and write nothing.
template <typename T>
__device__ inline Columns<T> columns_of(int64_t first, int count, int dim, int64_t b_stride) {
    Columns<T> c;
    int64_t base = first - (int64_t)(threadIdx.x % kWave) * Lane<T>::N;
    int64_t from = count > 0 ? first : base;
    c.at[0] = from / dim * b_stride + from % dim;
    int64_t next = count > 1 ? from + 1 : from;
    c.at[1] = next / dim * b_stride + next % dim;
    // a lane without columns reads both of the first lane's, which are side by side if the wave is dense
    c.dense = __all(count <= 0 || (count > 1 && c.at[1] == c.at[0] + 1));
    return c;
}

// results are not read again soon: they go past the caches (3 to 5% of the time)
typedef uint32_t Loose __attribute__((aligned(2)));
template <typename T>
__device__ inline void store(T* p, int64_t at, int count, const float* v) {
    if constexpr (sizeof(T) == 4) {
        if (count > 0) p[at] = from_f<T>(v[0]);
    } else {
        uint32_t lo = bits_of(v[0], (T*)nullptr), raw = lo | bits_of(v[1], (T*)nullptr) << 16;
        if (count > 1)
            __builtin_nontemporal_store(raw, (Loose*)(p + at));
        else if (count > 0)
            __builtin_memcpy(p + at, &lo, 2);
    }
}

// e = exp(-f) gives a = sigmoid(f) and b = 1 - a, both with a small relative error
__device__ inline float odds(float f) { return __builtin_amdgcn_exp2f(-1.44269504088896341f * f); }
__device__ inline void gate(float e, float& a, float& b) {
    a = __builtin_amdgcn_rcpf(1.f + e);
    b = e > 1e30f ? 1.f : e * a;
}

__device__ inline bool is_cut(float a) { return __float_as_uint(a) == 0x80000000u; }
// what a leaves of s
template <bool RESET>
__device__ inline float carry(float a, float s, float b) {
    if (RESET && is_cut(a)) return b;
    return fmaf(a, s, b);
}
template <bool RESET>
__device__ inline float chain(float a, float b) {
    if (RESET && (is_cut(a) || is_cut(b))) return -0.f;
    return a * b;
}

// bit i: an episode starts at the lane's step i
template <typename T, int STEPS>
__device__ inline void resets(const uint8_t* reset, int64_t t0, int64_t steps, int batch, int64_t first, int count,
                              int dim, uint32_t* mask) {
    int64_t b0 = (count > 0 ? first : 0) / dim, b1 = (count > 1 ? first + 1 : (count > 0 ? first : 0)) / dim;
    auto marks = [&](int64_t b) {
        uint8_t v[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) v[i] = reset[min(t0 + i, steps - 1) * batch + b];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) m |= (uint32_t)(v[i] != 0 && t0 + i < steps) << i;
        return m;
    };
    mask[0] = mask[1] = marks(b0);
    // a lane's two channels may belong to two batch entries
    if (Lane<T>::N == 2 && !__all(b0 == b1)) mask[1] = marks(b1);
}

// A state's word has a mark above the value. A pair's has A above B; A is at most 1, or a negative zero, or NaN, and
// never 2.0, whose bits are turned over in it: no pair is the zero that says that nothing is there.
typedef unsigned long long Word;
constexpr uint32_t kTurned = 0x40000000u;
__device__ inline void leave(Word* p, Word w) {
    __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline Word look(const Word* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline Word state_word(float s) { return (Word)1 << 32 | __float_as_uint(s); }
__device__ inline Word pair_word(float a, float b) {
    return (Word)(__float_as_uint(a) ^ kTurned) << 32 | __float_as_uint(b);
}

// The words of a chain: for each tile a row of states and a row of pairs.
struct Chain {
    Word* words;
    int64_t columns;
    __device__ inline Word* state(int64_t tile, int64_t c) const { return words + 2 * tile * columns + c; }
    __device__ inline Word* pair(int64_t tile, int64_t c) const { return words + (2 * tile + 1) * columns + c; }
};

template <int N>
struct Window {
    float a[kMostWaves][kWave * N], b[kMostWaves][kWave * N];
    int known[kMostWaves];
};

// The state that enters `tile`, from the tiles that lie `step` (-1 or 1) times 1 to 8 away, of which `first` is the end
// of the chain. Every wave of the workgroup calls it; all get the state.
template <int N, bool RESET>
__device__ inline void entering(const Chain& chain, Window<N>& window, int64_t tile, int step, int64_t end, int64_t c,
                                int count, int wave, int lane, float* s) {
    int64_t from = tile + (int64_t)step * (wave + 1);
    if (step < 0 ? from >= end : from <= end) {
        Word state[N], pair[N];
        bool known, there;
        for (;;) {
            known = there = true;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                state[j] = pair[j] = (Word)1 << 32;
                if (j < count) {
                    state[j] = look(chain.state(from, c + j));
                    if (wave + 1 < kMostWaves) pair[j] = look(chain.pair(from, c + j));
                }
                known = known && (state[j] >> 32);
                there = there && (pair[j] >> 32);
            }
            known = __all(known);
            there = __all(there) && wave + 1 < kMostWaves;
            if (known || there) break;
            __builtin_amdgcn_s_sleep(1);
        }
        if (lane == 0) window.known[wave] = known;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            window.a[wave][lane * N + j] = __uint_as_float((uint32_t)(pair[j] >> 32) ^ kTurned);
            window.b[wave][lane * N + j] = __uint_as_float((uint32_t)(known ? state[j] : pair[j]));
        }
    }
    __syncthreads();
    int at = 0;
    while (!window.known[at]) ++at;  // the end of the chain knows its state, as does what the eighth wave saw
#pragma unroll
    for (int j = 0; j < N; ++j) {
        s[j] = window.b[at][lane * N + j];
        for (int v = at - 1; v >= 0; --v)
            s[j] = carry<RESET>(window.a[v][lane * N + j], s[j], window.b[v][lane * N + j]);
    }
}

// the tile that this workgroup takes: column groups turn fastest, time follows
__device__ inline int64_t take_tile(unsigned* counter) {
    __shared__ unsigned taken;
    if (!counter) return blockIdx.x;
    if (threadIdx.x == 0) taken = atomicAdd(counter, 1u);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(taken);
}

template <typename T, int STEPS, bool RESET>
__global__ void __launch_bounds__(kMostWaves* kWave) linrec_fwd_kernel(
    Seq x, Seq f, const float* __restrict__ h0, const uint8_t* __restrict__ reset, T* __restrict__ h,
    float* __restrict__ last, Word* __restrict__ words, unsigned* __restrict__ counter, int64_t steps, int batch,
    int dim, int groups, int tiles
) {
    constexpr int N = Lane<T>::N;
    int64_t columns = (int64_t)batch * dim, taken = take_tile(counter), tile = taken / groups;
    int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    int waves = blockDim.x / kWave;
    int64_t c = taken % groups * (kWave * N) + lane * N;
    int count = (int)min((int64_t)N, max((int64_t)0, columns - c));
    int64_t t0 = tile * kTile + wave * STEPS;
    Columns<T> cx = columns_of<T>(c, count, dim, x.b_stride), cf = columns_of<T>(c, count, dim, f.b_stride);
    uint32_t rx[STEPS], rf[STEPS], mask[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        int64_t t = min(t0 + i, steps - 1);
        rx[i] = cx.load((const T*)x.base + t * x.t_stride);
        rf[i] = cf.load((const T*)f.base + t * f.t_stride);
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        rx[i] = t0 + i < steps ? rx[i] : 0;
        rf[i] = t0 + i < steps ? rf[i] : open_gate((T*)nullptr);
    }
    if (RESET) resets<T, STEPS>(reset, t0, steps, batch, c, count, dim, mask);
    // the wave's steps from nothing: h_t = add[t] + keep[t] s for a state s before them
    float add[STEPS][N], keep[STEPS][N], A[N], B[N];
#pragma unroll
    for (int j = 0; j < N; ++j) A[j] = 1.f, B[j] = 0.f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float a, b;
            gate(odds(value_of(rf[i], j, (T*)nullptr)), a, b);
            if (RESET && (mask[j] >> i & 1)) a = -0.f;
            B[j] = carry<RESET>(a, B[j], b * value_of(rx[i], j, (T*)nullptr));
            A[j] = chain<RESET>(A[j], a);
            add[i][j] = B[j];
            keep[i][j] = A[j];
        }
    __shared__ float la[kMostWaves][kWave * N], lb[kMostWaves][kWave * N];
    __shared__ Window<N> window;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        la[wave][lane * N + j] = A[j];
        lb[wave][lane * N + j] = B[j];
    }
    __syncthreads();
    Chain links{words, columns};
    float s[2], ta[N], tb[N];
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            ta[j] = A[j], tb[j] = B[j];
            for (int w = 1; w < waves; ++w) {
                float wa = la[w][lane * N + j];
                tb[j] = carry<RESET>(wa, tb[j], lb[w][lane * N + j]);
                ta[j] = chain<RESET>(ta[j], wa);
            }
            if (tile > 0 && tile + 1 < tiles && j < count) leave(links.pair(tile, c + j), pair_word(ta[j], tb[j]));
        }
    }
    if (tile == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) s[j] = h0 && j < count ? h0[c + j] : 0.f;
    } else {
        entering<N, RESET>(links, window, tile, -1, 0, c, count, wave, lane, s);
    }
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float after = carry<RESET>(ta[j], s[j], tb[j]);
            if (j < count) {
                if (tile + 1 < tiles) leave(links.state(tile, c + j), state_word(after));
                else last[c + j] = after;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
        for (int w = 0; w < wave; ++w) s[j] = carry<RESET>(la[w][lane * N + j], s[j], lb[w][lane * N + j]);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        float v[2];
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = carry<RESET>(keep[i][j], s[j], add[i][j]);
        store(h, (t0 + i) * columns + c, t0 + i < steps ? count : 0, v);
    }
}

template <typename T, int STEPS, bool RESET>
__global__ void __launch_bounds__(kMostWaves* kWave, 4) linrec_bwd_kernel(
    Seq x, Seq f, const float* __restrict__ h0, const uint8_t* __restrict__ reset, const Word* __restrict__ starts,
    const T* __restrict__ g, const float* __restrict__ g_last, T* __restrict__ dx, T* __restrict__ df,
    float* __restrict__ dh0, Word* __restrict__ words, unsigned* __restrict__ counter, int64_t steps, int batch,
    int dim, int groups, int tiles
) {
    constexpr int N = Lane<T>::N;
    int64_t columns = (int64_t)batch * dim, taken = take_tile(counter), tile = tiles - 1 - taken / groups;
    int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    int waves = blockDim.x / kWave;
    int64_t c = taken % groups * (kWave * N) + lane * N;
    int count = (int)min((int64_t)N, max((int64_t)0, columns - c));
    int64_t t0 = tile * kTile + wave * STEPS;
    Columns<T> cx = columns_of<T>(c, count, dim, x.b_stride), cf = columns_of<T>(c, count, dim, f.b_stride);
    Columns<T> cg = columns_of<T>(c, count, (int)min(columns, (int64_t)1 << 30), 0);
    if (columns > (int64_t)1 << 30) {
        cg.at[0] = count > 0 ? c : c - lane * N;
        cg.at[1] = cg.at[0] + (count > 1);
    }
    uint32_t rx[STEPS], rg[STEPS], mask[2] = {0, 0};
    float e[STEPS][N];
    {
        uint32_t rf[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            int64_t t = min(t0 + i, steps - 1);
            rf[i] = cf.load((const T*)f.base + t * f.t_stride);
            rx[i] = cx.load((const T*)x.base + t * x.t_stride);
            rg[i] = g ? cg.load(g + t * columns) : 0;
        }
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            bool in = t0 + i < steps;
            rf[i] = in ? rf[i] : open_gate((T*)nullptr);
            rx[i] = in ? rx[i] : 0;
            rg[i] = in ? rg[i] : 0;
#pragma unroll
            for (int j = 0; j < N; ++j) e[i][j] = odds(value_of(rf[i], j, (T*)nullptr));
        }
    }
    if (RESET) resets<T, STEPS>(reset, t0, steps, batch, c, count, dim, mask);
    // a state s before the wave's steps becomes A s + B after them; M after them becomes A M + Q before them
    float A[N], B[N], Q[N];
#pragma unroll
    for (int j = 0; j < N; ++j) A[j] = 1.f, B[j] = 0.f, Q[j] = 0.f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float a, b;
            gate(e[i][j], a, b);
            if (RESET && (mask[j] >> i & 1)) a = -0.f;
            B[j] = carry<RESET>(a, B[j], b * value_of(rx[i], j, (T*)nullptr));
            A[j] = chain<RESET>(A[j], a);
            Q[j] = carry<RESET>(A[j], value_of(rg[i], j, (T*)nullptr), Q[j]);
        }
    __shared__ float la[kMostWaves][kWave * N], lb[kMostWaves][kWave * N], lq[kMostWaves][kWave * N];
    __shared__ Window<N> window;
    // the gradients wait in LDS for the last pass: with them the registers of two workgroups a compute unit do not do
    __shared__ uint32_t waiting[STEPS][kMostWaves * kWave];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) waiting[i][threadIdx.x] = rg[i];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        la[wave][lane * N + j] = A[j];
        lb[wave][lane * N + j] = B[j];
        lq[wave][lane * N + j] = Q[j];
    }
    Chain kept{(Word*)starts, columns}, links{words, columns};
    float s[2], m[2], ta[N], tq[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        s[j] = 0.f;
        if (j < count) s[j] = tile > 0 ? __uint_as_float((uint32_t)*kept.state(tile - 1, c + j)) : h0 ? h0[c + j] : 0.f;
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            ta[j] = A[j], tq[j] = Q[j];
            for (int w = 1; w < waves; ++w) {
                tq[j] = carry<RESET>(ta[j], lq[w][lane * N + j], tq[j]);
                ta[j] = chain<RESET>(ta[j], la[w][lane * N + j]);
            }
            if (tile > 0 && tile + 1 < tiles && j < count) leave(links.pair(tile, c + j), pair_word(ta[j], tq[j]));
        }
    }
    if (tile == tiles - 1) {
#pragma unroll
        for (int j = 0; j < N; ++j) m[j] = g_last && j < count ? g_last[c + j] : 0.f;
    } else {
        entering<N, RESET>(links, window, tile, 1, tiles - 1, c, count, wave, lane, m);
    }
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float before = carry<RESET>(ta[j], m[j], tq[j]);
            if (j < count) {
                if (tile > 0) leave(links.state(tile, c + j), state_word(before));
                else if (dh0) dh0[c + j] = before;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        for (int w = 0; w < wave; ++w) s[j] = carry<RESET>(la[w][lane * N + j], s[j], lb[w][lane * N + j]);
        for (int w = waves - 1; w > wave; --w) m[j] = carry<RESET>(la[w][lane * N + j], m[j], lq[w][lane * N + j]);
    }
    float apart[STEPS][N];  // the state before a step less the step's input
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float a, b;
            // the compiler would keep the gates of the first pass, for which there are no registers
            asm volatile("" : "+v"(e[i][j]));
            gate(e[i][j], a, b);
            if (RESET && (mask[j] >> i & 1)) s[j] = 0.f;
            float in = value_of(rx[i], j, (T*)nullptr);
            apart[i][j] = s[j] - in;
            s[j] = fmaf(a, s[j], b * in);
        }
#pragma unroll
    for (int i = STEPS - 1; i >= 0; --i) {
        float vx[2], vf[2];
        uint32_t raw = waiting[i][threadIdx.x];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            asm volatile("" : "+v"(e[i][j]));
            float a, b, G = m[j] + value_of(raw, j, (T*)nullptr);
            gate(e[i][j], a, b);
            vx[j] = b * G;
            vf[j] = G * apart[i][j] * a * b;
            m[j] = RESET && (mask[j] >> i & 1) ? 0.f : a * G;
        }
        int here = t0 + i < steps ? count : 0;
        store(dx, (t0 + i) * columns + c, here, vx);
        store(df, (t0 + i) * columns + c, here, vf);
    }
}

Seq seq_of(const torch::Tensor& v) { return {v.data_ptr(), v.stride(0), v.stride(1)}; }

void check_seq(const torch::Tensor& v, const torch::Tensor& x) {
    TORCH_CHECK(v.is_cuda() && v.device() == x.device() && v.dim() == 3 && v.sizes() == x.sizes() &&
                    v.scalar_type() == x.scalar_type() && (v.stride(2) == 1 || v.size(2) == 1),
                "gated_linear_recurrence: x and gate must be [T, B, D] of one type and device with dense channels");
    TORCH_CHECK(v.size(0) >= 1 && v.size(1) * v.size(2) < (int64_t)1 << 31,
                "gated_linear_recurrence: T must be at least 1 and B * D below 2^31");
}

template <typename T>
const T* given(const torch::Tensor& v, const torch::Tensor& x, int64_t n, c10::ScalarType type) {
    if (!v.defined() || v.numel() == 0) return nullptr;
    TORCH_CHECK(v.device() == x.device() && v.is_contiguous() && v.numel() == n && v.scalar_type() == type,
                "gated_linear_recurrence: an argument has another size, type, layout or device");
    return (const T*)v.data_ptr();
}

template <typename F>
void by_type(const torch::Tensor& x, F&& f) {
    switch (x.scalar_type()) {
        case torch::kFloat32: f((float*)nullptr); break;
        case torch::kFloat16: f((__half*)nullptr); break;
        case torch::kBFloat16: f((__hip_bfloat16*)nullptr); break;
        default: TORCH_CHECK(false, "gated_linear_recurrence: expected float32, float16 or bfloat16");
    }
}

// How the work is cut: one step needs no more than a step of a lane; a sequence of one tile needs no chain.
struct Cut {
    int64_t columns;
    int groups, tiles, waves;
    bool single;
};

Cut cut_of(const torch::Tensor& x) {
    int64_t steps = x.size(0), columns = x.size(1) * x.size(2);
    int lanes = kWave * 4 / (int)x.element_size();
    Cut cut{columns, cdiv(columns, lanes), cdiv(steps, kTile), 0, steps == 1};
    cut.waves = cut.single ? 1 : (int)std::min<int64_t>(kMostWaves, (steps + kSteps - 1) / kSteps);
    TORCH_CHECK((int64_t)cut.groups * cut.tiles < (int64_t)1 << 31, "gated_linear_recurrence: too large");
    return cut;
}

// the chain's words, two a column for every tile, and the counter behind them, all zero
torch::Tensor words_of(const torch::Tensor& x, const Cut& cut) {
    auto opt = x.options().dtype(torch::kInt64);
    return cut.tiles > 1 ? torch::zeros({2 * cut.tiles * cut.columns + 1}, opt) : torch::empty({0}, opt);
}

template <typename F>
void by_case(const torch::Tensor& x, const Cut& cut, bool reset, F&& f) {
    by_type(x, [&](auto* null) {
        auto one = std::integral_constant<int, 1>{};
        auto many = std::integral_constant<int, kSteps>{};
        if (cut.single)
            reset ? f(null, one, std::true_type{}) : f(null, one, std::false_type{});
        else
            reset ? f(null, many, std::true_type{}) : f(null, many, std::false_type{});
    });
}

std::vector<torch::Tensor> linrec_fwd(torch::Tensor x, torch::Tensor gate, torch::Tensor h0, torch::Tensor reset) {
    check_seq(x, x);
    check_seq(gate, x);
    c10::OptionalDeviceGuard guard(x.device());
    auto h = torch::empty(x.sizes(), x.options());
    auto last = torch::empty({x.size(1), x.size(2)}, x.options().dtype(torch::kFloat32));
    if (h.numel() == 0) return {h, last, torch::empty({0}, x.options().dtype(torch::kInt64))};
    Cut cut = cut_of(x);
    auto words = words_of(x, cut);
    const float* h0p = given<float>(h0, x, cut.columns, torch::kFloat32);
    const uint8_t* rp = given<uint8_t>(reset, x, x.size(0) * x.size(1), torch::kBool);
    by_case(x, cut, rp, [&](auto* null, auto n, auto cuts) {
        using T = std::remove_pointer_t<decltype(null)>;
        Word* w = cut.tiles > 1 ? (Word*)words.data_ptr() : nullptr;
        linrec_fwd_kernel<T, decltype(n)::value, decltype(cuts)::value>
            <<<(unsigned)(cut.groups * cut.tiles), cut.waves * kWave, 0, ding_current_stream()>>>(
                seq_of(x), seq_of(gate), h0p, rp, (T*)h.data_ptr(), last.data_ptr<float>(), w,
                w ? (unsigned*)(w + 2 * cut.tiles * cut.columns) : nullptr, x.size(0), (int)x.size(1), (int)x.size(2),
                cut.groups, cut.tiles);
    });
    HIP_CHECK_LAST();
    return {h, last, words};
}

std::vector<torch::Tensor> linrec_bwd(
    torch::Tensor x, torch::Tensor gate, torch::Tensor h0, torch::Tensor reset, torch::Tensor starts,
    torch::Tensor grad_h, torch::Tensor grad_last, int64_t want_h0
) {
    check_seq(x, x);
    check_seq(gate, x);
    c10::OptionalDeviceGuard guard(x.device());
    auto opt = x.options().dtype(torch::kFloat32);
    auto dx = torch::empty(x.sizes(), x.options());
    auto df = torch::empty(x.sizes(), x.options());
    auto dh0 = want_h0 ? torch::empty({x.size(1), x.size(2)}, opt) : torch::empty({0}, opt);
    if (dx.numel() == 0) return {dx, df, dh0};
    Cut cut = cut_of(x);
    auto words = words_of(x, cut);
    int64_t steps = x.size(0);
    const float* h0p = given<float>(h0, x, cut.columns, torch::kFloat32);
    const uint8_t* rp = given<uint8_t>(reset, x, steps * x.size(1), torch::kBool);
    const void* gp = given<uint8_t>(grad_h, x, steps * cut.columns, x.scalar_type());
    const float* lp = given<float>(grad_last, x, cut.columns, torch::kFloat32);
    const Word* sp = given<Word>(starts, x, words.numel(), torch::kInt64);
    TORCH_CHECK(sp || cut.tiles == 1, "gated_linear_recurrence: the kept states are missing");
    by_case(x, cut, rp, [&](auto* null, auto n, auto cuts) {
        using T = std::remove_pointer_t<decltype(null)>;
        Word* w = cut.tiles > 1 ? (Word*)words.data_ptr() : nullptr;
        linrec_bwd_kernel<T, decltype(n)::value, decltype(cuts)::value>
            <<<(unsigned)(cut.groups * cut.tiles), cut.waves * kWave, 0, ding_current_stream()>>>(
                seq_of(x), seq_of(gate), h0p, rp, sp, (const T*)gp, lp, (T*)dx.data_ptr(), (T*)df.data_ptr(),
                want_h0 ? dh0.data_ptr<float>() : nullptr, w, w ? (unsigned*)(w + 2 * cut.tiles * cut.columns) : nullptr,
                steps, (int)x.size(1), (int)x.size(2), cut.groups, cut.tiles);
    });
    HIP_CHECK_LAST();
    return {dx, df, dh0};
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Recurrence : torch::autograd::Function<Recurrence> {
    static variable_list forward(AutogradContext* ctx, torch::Tensor x, torch::Tensor gate,
                                 c10::optional<torch::Tensor> h0, c10::optional<torch::Tensor> reset) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto start = h0 ? h0->to(torch::kFloat32).contiguous() : torch::Tensor();
        auto mask = reset ? reset->contiguous() : torch::Tensor();
        auto out = linrec_fwd(x, gate, start, mask);
        ctx->save_for_backward({x, gate, start, mask, out[2]});
        ctx->saved_data["h0"] = h0 ? (int64_t)h0->scalar_type() : (int64_t)-1;
        ctx->set_materialize_grads(false);
        return {out[0], out[1]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        auto kept = ctx->get_saved_variables();
        int64_t type = ctx->saved_data["h0"].toInt();
        bool want = type >= 0 && ctx->needs_input_grad(2);
        variable_list out;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            auto dense = [](const torch::Tensor& t) { return t.defined() ? t.contiguous() : t; };
            out = linrec_bwd(kept[0], kept[1], kept[2], kept[3], kept[4], dense(g[0]), dense(g[1]), want);
            if (want) out[2] = out[2].to((c10::ScalarType)type);
            else out[2] = torch::Tensor();
        }
        out.push_back(torch::Tensor());
        return ding_once_differentiable(std::move(out), "gated_linear_recurrence");
    }
};

}  // namespace

// x, gate [T, B, D], h0 [B, D], reset [T, B] -> h, the last state; differentiable once
std::tuple<torch::Tensor, torch::Tensor> gated_linear_recurrence(
    torch::Tensor x, torch::Tensor gate, c10::optional<torch::Tensor> h0, c10::optional<torch::Tensor> reset
) {
    auto dense = [](torch::Tensor v) { return v.stride(-1) == 1 || v.size(-1) == 1 ? v : v.contiguous(); };
    auto out = Recurrence::apply(dense(x), dense(gate), h0, reset);
    return {out[0], out[1]};
}
