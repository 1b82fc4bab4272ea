// Orthogonalisation of matrices by Newton-Schulz products.
//
//   X_0 = M / (|M|_F + eps), transposed where M is tall;  `steps` times:
//   G = X X^T,  X <- (a + b G + c G G) X
// Each step maps every singular value s to a s + b s^3 + c s^5 and leaves the singular vectors.
//
// Bound by the matrix units. The iteration multiplies early errors by a^steps (about 500), so 16-bit factors alone lose
// the small singular values, and 32-bit matrix instructions run at a tenth of the 16-bit rate. Every factor is therefore
// held as two half-precision numbers, v = (hi + lo) / scale with 22 significant bits, and a product is three matrix
// instructions,
//   hi hi + hi lo + lo hi   (lo lo is below 2^-22 of the result),
// summed in 32 bits. The scales are powers of two that the host derives from a bound of the singular values, so that
// nothing overflows and nothing but negligible entries becomes subnormal. A matrix given in 16 bits needs one number an
// entry until the first step has changed it: it is scaled by a power of two and the rest of its norm goes into the
// products' factors.
//
// Two ways through the same polynomial:
//   direct: G, G G and the product with X every step: m^2 n + m^3 + 2 m^2 n flops (symmetric results by half);
//   gram:   with Q = a + b G + c G G, P <- Q P and G <- Q G Q, all symmetric, and X <- P X once at the end of some steps.
// The second is cheaper, but errors of G grow by a^2 a step where those of X grow by a, and a matrix of one dominant
// direction has its others where such errors come to lie. It is taken for results that are rounded to 16 bits, over so
// few steps that it loses no more than a factor of four (two, with the usual coefficients).
//
// Large products run at 1.3 PFLOP/s of 16-bit instructions (4096 x 4096 over 8192: 623 us), as a library's product of
// plain half precision does here, and so at a third of that in results; 32-bit library products reach 0.15. It is the
// chip's power that bounds them: with zeros for factors the same instructions take a quarter to a third less. Smaller
// ones are held by LDS, which every tile's factors pass twice, and by 5 to 10 us a launch of filling, storing and
// starting.
//
// All products are "row times row" (C_ij = sum_k A_ik B_jk), which needs X and its transpose: both are kept. Columns are
// padded with zeros to a multiple of a stage's depth; rows of a tile that lie behind them are memory of ours that may
// hold anything, and reach nothing but such rows of the results.
#include "common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

constexpr int kThreads = 256;
constexpr int kNormBlocks = 1024;  // at most, for one matrix
constexpr int kStage = 32;       // depth of a stage
constexpr int kEdge = 64;        // tile side of the packing kernel

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef float float4v __attribute__((ext_vector_type(4)));

__device__ inline float to_f(float v) { return v; }
__device__ inline float to_f(__half v) { return __half2float(v); }
__device__ inline float to_f(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ inline T from_f(float v);
template <> __device__ inline float from_f<float>(float v) { return v; }
template <> __device__ inline __half from_f<__half>(float v) { return __float2half(v); }
template <> __device__ inline __hip_bfloat16 from_f<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

// a matrix of the batch, seen with its short side as rows
struct Matrix {
    const void* base;
    int64_t batch_stride, row_stride, col_stride;
    int rows, cols;
};

// Two planes of half precision. A plane lies in panels of kStage columns, [batch, panel, rows, kStage], so that what a
// tile needs of a stage is one dense piece of memory: rows at a stride of some KB would fall into few of the memory's
// channels (products of 2048 to 16384 columns took 1.05 to 1.35 times as long).
struct Split {
    _Float16 *hi, *lo;
    int64_t batch_stride;
    int rows;
    __device__ inline int64_t at(int64_t batch, int r, int k) const {
        return batch * batch_stride + ((int64_t)(k / kStage) * rows + r) * kStage + k % kStage;
    }
};

__device__ inline void split(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// Sums of squares in 64 bits, where no square of a 32-bit number overflows or vanishes. Lines of the dense direction are
// read 16 bytes a thread, four such on their way at a time; they may start at any element.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_kernel(Matrix m, double* __restrict__ partial) {
    constexpr int N = 16 / sizeof(T), AHEAD = 4;
    const T* p = (const T*)m.base + blockIdx.y * m.batch_stride;
    double sum = 0;
    bool flip = m.row_stride < m.col_stride;
    int lines = flip ? m.cols : m.rows, length = flip ? m.rows : m.cols;
    int64_t si = flip ? m.row_stride : m.col_stride, so = flip ? m.col_stride : m.row_stride;
    bool dense = si == 1;
    int groups = (length + N - 1) / N;
    int64_t n = (int64_t)lines * groups, stride = (int64_t)gridDim.x * kThreads;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += stride * AHEAD) {
        T v[AHEAD][N];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            int64_t g = i + k * stride;
            int64_t line = n < (int64_t)1 << 31 ? (unsigned)g / (unsigned)groups : g / groups;
            int at = (int)(g - line * groups) * N;
            const T* q = p + line * so + at * si;
            if (dense && g < n && at + N <= length) {
                __builtin_memcpy(v[k], q, 16);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) v[k][e] = g < n && at + e < length ? q[e * si] : from_f<T>(0.f);
            }
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
#pragma unroll
            for (int e = 0; e < N; ++e) sum += (double)to_f(v[k][e]) * to_f(v[k][e]);
    }
    __shared__ double part[kThreads / kWave];
    for (int o = kWave / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / kWave; ++w) sum += part[w];
        partial[blockIdx.y * gridDim.x + blockIdx.x] = sum;
    }
}

// No matrix but zero takes a larger factor: 2^-149 is the smallest number of 32 bits. With it zero stays zero whatever eps.
constexpr double kMostFactor = 0x1p200;
__device__ inline double at_most(double v, double most) { return v > most ? most : v; }  // NaN stays

// X and its transpose from M: a 64 x 64 tile a workgroup, turned in LDS. With `lo` planes X = M scale / (norm + eps);
// without, X = M times the next lower power of two, exactly, and `rest` takes what is left (in [1, 2)).
template <typename T>
__global__ void __launch_bounds__(kThreads) pack_kernel(
    Matrix m, const double* __restrict__ partial, int parts, double eps, float scale, Split x, Split xt,
    float* __restrict__ rest
) {
    __shared__ float tile[kEdge][kEdge + 1];
    __shared__ double sum_s[kThreads / kWave];
    int b = blockIdx.z;
    double sum = 0;
    for (int i = threadIdx.x; i < parts; i += kThreads) sum += partial[b * parts + i];
    for (int o = kWave / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    if (threadIdx.x % kWave == 0) sum_s[threadIdx.x / kWave] = sum;
    __syncthreads();
    sum = sum_s[0];
    for (int w = 1; w < kThreads / kWave; ++w) sum += sum_s[w];
    double whole = at_most(scale / (sqrt(sum) + eps), kMostFactor);
    float left = 1.f;
    if (!x.lo) {
        int e;
        frexp(whole, &e);
        double power = ldexp(1.0, min(max(e - 1, -300), 300));
        left = (float)(whole / power);
        whole = power;
    }
    // what 32 bits do not hold goes in two steps
    double near = whole < 0x1p-100 ? 0x1p-100 : at_most(whole, 0x1p100);
    float factor = (float)near, again = near == whole ? 1.f : (float)(whole / near);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) rest[b] = left;
    const T* p = (const T*)m.base + b * m.batch_stride;
    int i0 = blockIdx.y * kEdge, j0 = blockIdx.x * kEdge, lane = threadIdx.x % kEdge;
    bool flip = m.row_stride < m.col_stride;
#pragma unroll 4
    for (int r = threadIdx.x / kEdge; r < kEdge; r += kThreads / kEdge) {
        int i = flip ? lane : r, j = flip ? r : lane;
        bool in = i0 + i < m.rows && j0 + j < m.cols;
        tile[i][j] = in ? to_f(p[(i0 + i) * m.row_stride + (j0 + j) * m.col_stride]) * factor * again : 0.f;
    }
    __syncthreads();
    // 16 bytes a thread, 1 KB a wave
#pragma unroll
    for (int k = threadIdx.x; k < kEdge * kEdge / 8; k += kThreads) {
        int piece = k % 4, r = k / 4 % kEdge, c = k / (4 * kEdge) * 32 + piece * 8;
        half8 hi, lo;
        auto write = [&](const Split& to, int64_t at) {
            *(half8*)(to.hi + at) = hi;
            if (x.lo) *(half8*)(to.lo + at) = lo;
        };
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 h, l;
            split(tile[r][c + e], h, l);
            hi[e] = h, lo[e] = l;
        }
        write(x, x.at(b, i0 + r, j0 + c));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 h, l;
            split(tile[c + e][r], h, l);
            hi[e] = h, lo[e] = l;
        }
        write(xt, xt.at(b, j0 + r, i0 + c));
    }
}

struct Target {
    void* base;
    int64_t batch_stride, row_stride, col_stride;
    int rows, cols;
    int type;  // 0: float, 1: half, 2: bfloat16
};

// 16 bytes from global memory into LDS without a stop in registers; lane l of a wave writes to `to` + 16 l
__device__ inline void copy_to_lds(const void* from, void* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// Tile sides, the part of a tile that a wave computes, and the stages that are held in LDS.
template <int TILE_, int WM_, int WN_, int STAGES_>
struct Shape {
    static constexpr int TILE = TILE_, WM = WM_, WN = WN_, STAGES = STAGES_;
    static constexpr int WAVES = (TILE / WM) * (TILE / WN);
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int PLANE = TILE * kStage;              // halves of one plane of one factor's stage
    static constexpr int SIDE = WM % 32 || WN % 32 ? 16 : 32;  // of a matrix instruction
    // Where a row's four 16-byte pieces lie: the 16 lanes that LDS serves at once read as many different places.
    static __device__ inline int turn(int row) { return (row >> (SIDE == 32 ? 2 : 1)) & 3; }
};

// v_mfma of SIDE x SIDE results: lane l gives row l % SIDE of a factor, DEPTH / 8 pieces of 8 along the depth over the
// rest of l; it holds column l % SIDE of results, 4 rows at a time
template <int SIDE> struct Mfma;
template <> struct Mfma<32> {
    typedef float16v Acc;
    static constexpr int DEPTH = 16, QUADS = 4;
    static __device__ inline Acc run(half8 a, half8 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ inline int row(int q, int lane) { return q * 8 + lane / 32 * 4; }
};
template <> struct Mfma<16> {
    typedef float4v Acc;
    static constexpr int DEPTH = 32, QUADS = 1;
    static __device__ inline Acc run(half8 a, half8 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ inline int row(int q, int lane) { return lane / 16 * 4; }
};

enum Kind { SYMMETRIC, UPDATE, LAST };

// What a product is multiplied by and what is added: v = alpha rest^power C + beta E + diagonal [i = j]
struct Epilogue {
    float alpha, beta, diagonal;
    const float* rest;  // [batch] or null
    int power;          // alpha takes rest^power, beta takes rest^beta_power
    int beta_power;
    float inv_scale;
};

// The sums of a tile, as a wave's lanes hold them.
template <typename P>
struct Sums {
    typedef Mfma<P::SIDE> M;
    static constexpr int SI = P::WM / P::SIDE, SJ = P::WN / P::SIDE;
    typename M::Acc acc[SI][SJ];
};

// What becomes of the sums of tile (bi, bj).
template <typename P, Kind kind, int PA>
__device__ inline void finish(
    const Sums<P>& sums, int bi, int bj, int64_t batch, const Epilogue& ep, const Split& x, const Split& out,
    const Target& to
) {
    typedef Mfma<P::SIDE> M;
    constexpr int TILE = P::TILE, SIDE = P::SIDE, SI = Sums<P>::SI, SJ = Sums<P>::SJ;
    int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int wi = wave / (TILE / P::WN) * P::WM, wj = wave % (TILE / P::WN) * P::WN;
    const auto& acc = sums.acc;
    float alpha = ep.alpha, beta = ep.beta;
    if (ep.rest) {
        float r = ep.rest[batch];
        for (int p = 0; p < ep.power; ++p) alpha *= r;
        for (int p = 0; p < ep.beta_power; ++p) beta *= r;
    }
#pragma unroll
    for (int i = 0; i < SI; ++i)
#pragma unroll
        for (int j = 0; j < SJ; ++j)
#pragma unroll
            for (int q = 0; q < M::QUADS; ++q) {
                int r = bi * TILE + wi + i * SIDE + M::row(q, lane), c = bj * TILE + wj + j * SIDE + lane % SIDE;
                half4 hi, lo;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][q * 4 + e] * alpha;
                if (beta != 0.f) {
                    // the element itself: of a symmetric E, or of x, at (c, r)
                    int64_t at = x.at(batch, c, r);
                    half4 xh = *(const half4*)(x.hi + at);
                    if constexpr (kind == SYMMETRIC || PA == 2) {
                        half4 xl = *(const half4*)(x.lo + at);
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] += beta * ((float)xh[e] + (float)xl[e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] += beta * (float)xh[e];
                    }
                }
                if constexpr (kind == SYMMETRIC) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (r + e == c) v[e] += ep.diagonal;
                }
                if constexpr (kind == LAST) {
                    if (c < to.rows)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (r + e < to.cols) {
                                int64_t at = batch * to.batch_stride + c * to.row_stride + (r + e) * to.col_stride;
                                float w = v[e] * ep.inv_scale;
                                if (to.type == 0)
                                    ((float*)to.base)[at] = w;
                                else if (to.type == 1)
                                    ((__half*)to.base)[at] = from_f<__half>(w);
                                else
                                    ((__hip_bfloat16*)to.base)[at] = from_f<__hip_bfloat16>(w);
                            }
                    continue;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    _Float16 h, l;
                    split(v[e], h, l);
                    hi[e] = h;
                    lo[e] = l;
                }
                if constexpr (kind == UPDATE) {
                    int64_t at = x.at(batch, c, r);
                    *(half4*)(x.hi + at) = hi;
                    *(half4*)(x.lo + at) = lo;
                } else if (bi != bj) {
                    int64_t at = out.at(batch, c, r);
                    *(half4*)(out.hi + at) = hi;
                    *(half4*)(out.lo + at) = lo;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    int64_t at = out.at(batch, r + e, c);
                    out.hi[at] = hi[e];
                    out.lo[at] = lo[e];
                }
            }
}

// tile number t of the lower triangle
__device__ inline void triangle(int t, int& bi, int& bj) {
    bi = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while ((bi + 1) * (bi + 2) / 2 <= t) ++bi;
    while (bi * (bi + 1) / 2 > t) --bi;
    bj = t - bi * (bi + 1) / 2;
}

// C = A B^T over split factors of PA and PB planes, a TILE x TILE tile a workgroup.
//   SYMMETRIC: C is symmetric: tiles of the lower triangle, written twice. E = x where beta is not 0.
//   UPDATE:    A = X^T, B symmetric: C = (B X)^T; x <- beta x + C^T, its transpose to out. x may have one plane on the
//              way in (PA) and has two on the way out.
//   LAST:      the same, written to the caller's matrix in its type.
// Two symmetric products with the same A go in one launch: behind the first `matrices` of the grid's depth are those of
// the second B and out. A symmetric product may also be cut along its depth, gridDim.y parts of it: the parts' sums go to
// `partial` and join_kernel adds them up. That fills the chip where tiles are few, and keeps the sums of a long depth
// short: 130 x 8000 in single precision is 3.6e-6 off without.
// A stage of 32 columns is copied straight into LDS while the one before it is multiplied. Within a row of a stage the
// four 16-byte pieces change places with the row, so that eight rows read at once fall into different banks.
template <typename P, Kind kind, int PA, int PB>
__global__ void __launch_bounds__(P::THREADS) product_kernel(
    Split a, Split bm, int depth, Epilogue ep, Split x, Split out, Target to, int matrices, Split second_b,
    Split second_out, float* __restrict__ partial
) {
    typedef Mfma<P::SIDE> M;
    constexpr int TILE = P::TILE, SIDE = P::SIDE, SI = Sums<P>::SI, SJ = Sums<P>::SJ;
    __shared__ __attribute__((aligned(16))) _Float16 lds[P::STAGES][(PA + PB) * P::PLANE];
    int bi, bj, t = blockIdx.x;
    if constexpr (kind == SYMMETRIC) {
        // Workgroups go to the eight dies in turn: each die takes neighbouring tiles of the lower triangle, whose
        // factors meet in its cache (three of 1001: a tenth of the time; rectangles lost a third of theirs by it).
        int die = t % 8, each = gridDim.x / 8, over = gridDim.x % 8;
        t = die * each + min(die, over) + t / 8;
        triangle(t, bi, bj);
    } else {
        bi = blockIdx.x;
        bj = blockIdx.y;
    }
    int64_t batch = blockIdx.z;
    if (kind == SYMMETRIC && (int)blockIdx.z >= matrices) {
        batch -= matrices;
        bm = second_b;
        out = second_out;
    }
    int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    int wi = wave / (TILE / P::WN) * P::WM, wj = wave % (TILE / P::WN) * P::WN;
    Sums<P> sums;
    auto& acc = sums.acc;
#pragma unroll
    for (int i = 0; i < SI; ++i)
#pragma unroll
        for (int j = 0; j < SJ; ++j) acc[i][j] = (typename M::Acc)(0.f);

    // A wave copies 16 rows of a plane at a time: lane l takes piece l % 4 of row l / 4, from where it belongs. What
    // moves from copy to copy and from stage to stage is the same for all lanes and costs the vector unit nothing.
    constexpr int GROUPS = (PA + PB) * TILE / 16, COPIES = (GROUPS + P::WAVES - 1) / P::WAVES;
    constexpr int S = P::STAGES, STEPS = kStage / M::DEPTH;
    int stages = depth / kStage, now = 0, skip = 0;
    if (kind == SYMMETRIC && gridDim.y > 1) {
        int each = (stages + gridDim.y - 1) / gridDim.y;
        skip = min(each * (int)blockIdx.y, stages - 1);
        stages = max(0, min(each, stages - each * (int)blockIdx.y));
    }
    const unsigned own = lane / 4 * kStage + (lane % 4 ^ P::turn(lane / 4)) * 8;
    const _Float16* from[COPIES];
    int64_t step[COPIES];
    int place[COPIES];
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
        int group = min(c * P::WAVES + wave, GROUPS - 1);  // every wave issues as many: some copy the last group again
        int plane = group / (TILE / 16), first = group % (TILE / 16) * 16;
        const Split& f = plane < PA ? a : bm;
        step[c] = (int64_t)f.rows * kStage;
        from[c] = ((plane < PA ? plane : plane - PA) ? f.lo : f.hi) +
                  f.at(batch, (plane < PA ? bi : bj) * TILE + first, 0) + skip * step[c];
        place[c] = plane * P::PLANE + first * kStage;
    }
    // The stages in order; behind the last one it copies that again, which nobody reads, so that a wave always has as
    // many copies on their way.
    int fetched = 0;
    auto fetch = [&](_Float16* stage) {
        bool more = ++fetched < stages;
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
            copy_to_lds(from[c] + own, stage + place[c]);
            from[c] += more ? step[c] : 0;
        }
    };
    struct Factors {
        half8 a[PA][SI], b[PB][SJ];
    };
    auto read = [&](Factors& f, const _Float16* stage, int ks) {
        int piece = ks * (M::DEPTH / 8) + lane / SIDE;
        auto at = [&](int plane, int r) {
            return *(const half8*)(stage + plane * P::PLANE + r * kStage + (piece ^ P::turn(r)) * 8);
        };
#pragma unroll
        for (int p = 0; p < PA; ++p)
#pragma unroll
            for (int s = 0; s < SI; ++s) f.a[p][s] = at(p, wi + s * SIDE + lane % SIDE);
#pragma unroll
        for (int p = 0; p < PB; ++p)
#pragma unroll
            for (int s = 0; s < SJ; ++s) f.b[p][s] = at(PA + p, wj + s * SIDE + lane % SIDE);
    };
    auto multiply = [&](const Factors& f) {
        auto all = [&](const half8(&u)[SI], const half8(&v)[SJ]) {
#pragma unroll
            for (int i = 0; i < SI; ++i)
#pragma unroll
                for (int j = 0; j < SJ; ++j) acc[i][j] = M::run(u[i], v[j], acc[i][j]);
        };
        if constexpr (PA == 2) all(f.a[1], f.b[0]);
        if constexpr (PB == 2) all(f.a[0], f.b[1]);
        all(f.a[0], f.b[0]);
        // the next factors' reads are spread between these products
        constexpr int READS = PA * SI + PB * SJ, PRODUCTS = SI * SJ * (PA + PB - 1);
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS / READS > 0 ? PRODUCTS / READS : 1, 0);
        }
    };
    // The factors of the next product are read from LDS while the present ones are multiplied. Copies of a wave arrive
    // in the order of their issue: when only those of the S - 2 later stages are out, the next stage's are there; after
    // the barrier everyone's are, and everyone has read the present stage, which is overwritten then.
    Factors even, odd;
    auto turn_stage = [&](Factors& f) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * COPIES) : "memory");
        fetch(lds[now]);
        now = now + 1 == S ? 0 : now + 1;
        read(f, lds[now], 0);  // behind the last stage it reads what is there, and nobody uses it
    };
#pragma unroll
    for (int k = 0; k < S; ++k) fetch(lds[k]);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S - 1) * COPIES) : "memory");
    read(even, lds[0], 0);
    if constexpr (STEPS == 2) {
        for (int k = 0; k < stages; ++k) {
            read(odd, lds[now], 1);
            multiply(even);
            turn_stage(even);
            multiply(odd);
        }
    } else if constexpr (P::TILE == 192) {
        // two sets of factors do not fit in registers beside the sums
        for (int k = 0; k < stages; ++k) {
            multiply(even);
            turn_stage(even);
        }
    } else {
        // pairs of stages without a branch between them: the compiler would move reads behind it, next to their use
        int k = 0;
        if (stages % 2) {
            turn_stage(odd);
            multiply(even);
            even = odd;
            k = 1;
        }
        for (; k < stages; k += 2) {
            turn_stage(odd);
            multiply(even);
            turn_stage(even);
            multiply(odd);
        }
    }
    // nothing is on its way into LDS when the workgroup gives it back
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    if (kind == SYMMETRIC && gridDim.y > 1) {
        // a part of the depth: the sums themselves, a quad of a lane side by side with its neighbours'
        float4v* to_part = (float4v*)partial + (((int64_t)blockIdx.z * gridDim.x + t) * gridDim.y + blockIdx.y) *
                                                   (TILE * TILE / 4) + threadIdx.x;
#pragma unroll
        for (int i = 0; i < SI; ++i)
#pragma unroll
            for (int j = 0; j < SJ; ++j)
#pragma unroll
                for (int q = 0; q < M::QUADS; ++q) {
                    float4v v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[i][j][q * 4 + e];
                    to_part[((i * SJ + j) * M::QUADS + q) * P::THREADS] = v;
                }
        return;
    }
    finish<P, kind, PA>(sums, bi, bj, batch, ep, x, out, to);
}

// Adds the parts of a symmetric product's tiles up, in their order.
template <typename P>
__global__ void __launch_bounds__(P::THREADS) join_kernel(
    const float* __restrict__ partial, int parts, Epilogue ep, Split x, Split out, int matrices, Split second_out
) {
    typedef Mfma<P::SIDE> M;
    int64_t batch = blockIdx.z;
    if ((int)blockIdx.z >= matrices) {
        batch -= matrices;
        out = second_out;
    }
    int bi, bj;
    triangle(blockIdx.x, bi, bj);
    Sums<P> sums;
    const float4v* from = (const float4v*)partial +
                          ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * parts * (P::TILE * P::TILE / 4) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < Sums<P>::SI; ++i)
#pragma unroll
        for (int j = 0; j < Sums<P>::SJ; ++j)
#pragma unroll
            for (int q = 0; q < M::QUADS; ++q) {
                float4v v = (float4v)(0.f);
                for (int s = 0; s < parts; ++s)
                    v += from[(int64_t)s * (P::TILE * P::TILE / 4) + ((i * Sums<P>::SJ + j) * M::QUADS + q) * P::THREADS];
#pragma unroll
                for (int e = 0; e < 4; ++e) sums.acc[i][j][q * 4 + e] = v[e];
            }
    finish<P, SYMMETRIC, 2>(sums, bi, bj, batch, ep, x, out, Target{});
}

// ------------------------------------------------------------------------------------------------ small matrices
// A matrix of up to 128 x 256 has a workgroup of its own for the whole iteration: X stays in registers in 32 bits, its
// factors and G's lie in LDS, and nothing is launched or stored between the products, where a launch of its own takes
// about 5 us a product whatever its size. Up to 256 matrices of 64 x 64 take 14 us, of 128 x 128 55 us (six of them by
// launches: 95 us). Up to 256 of 128 x 256 take 92 to 110 us, by launches six take 104 us and 64 160 us. Products, LDS and the
// vector unit's splitting take about a third of the time each and hardly overlap: two waves a unit wait at the same
// barriers.
// X is held as the results of (B X)^T: rows r of X^T in parts of kPart, columns c; a wave has a half of a part's rows
// and a quarter of the columns. The same place in LDS holds X and X^T in turns, a part at a time.
struct Small {
    float gram, square, linear, update, keep;  // factors of C in G, of C and G in B, of C and x in x
    float scale, inv_scale;
    double eps;
    int steps;
};

template <int MP, int NP>
struct SmallShape {
    static constexpr int PART = NP < 128 ? NP : 128, PARTS = NP / PART;
    static constexpr int WAVES = 8, THREADS = WAVES * kWave;
    static constexpr int XI = PART / 2 / 16, GI = MP / 2 / 16, J = MP / 4 / 16;
    static constexpr int X_PLANE = MP * PART, G_PLANE = MP * MP;  // halves
};

// where element (row, k) of a plane of `rows` rows lies: panels of 32 columns, pieces changing places with the row
__device__ inline int small_at(int rows, int row, int k) {
    return (k / 32 * rows + row) * 32 + (((k / 8) & 3) ^ ((row >> 1) & 3)) * 8 + k % 8;
}

template <typename T, int MP, int NP>
__global__ void __launch_bounds__(512) small_kernel(Matrix m, Target to, Small p) {
    typedef SmallShape<MP, NP> S;
    typedef Mfma<16> M;
    __shared__ __attribute__((aligned(16))) _Float16 lx[2 * S::X_PLANE], lg[2 * S::G_PLANE];
    __shared__ double part[S::WAVES];
    int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int r_wave = wave / 4, c0 = wave % 4 * (MP / 4) + lane % 16, r_lane = lane / 16 * 4;
    auto row_x = [&](int q, int i) { return q * S::PART + r_wave * (S::PART / 2) + i * 16 + r_lane; };
    float x[S::PARTS][S::XI][S::J][4];
    double sum = 0;
#pragma unroll
    for (int q = 0; q < S::PARTS; ++q)
#pragma unroll
        for (int i = 0; i < S::XI; ++i)
#pragma unroll
            for (int j = 0; j < S::J; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // all loads go out before the first is waited for
                    int r = min(row_x(q, i) + e, m.cols - 1), c = min(c0 + j * 16, m.rows - 1);
                    x[q][i][j][e] =
                        to_f(((const T*)m.base)[blockIdx.x * m.batch_stride + c * m.row_stride + r * m.col_stride]);
                }
#pragma unroll
    for (int q = 0; q < S::PARTS; ++q)
#pragma unroll
        for (int i = 0; i < S::XI; ++i)
#pragma unroll
            for (int j = 0; j < S::J; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    bool in = row_x(q, i) + e < m.cols && c0 + j * 16 < m.rows;
                    float v = in ? x[q][i][j][e] : 0.f;
                    x[q][i][j][e] = v;
                    sum += (double)v * v;
                }
    for (int o = kWave / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    sum = part[0];
    for (int w = 1; w < S::WAVES; ++w) sum += part[w];
    double factor = at_most(p.scale / (sqrt(sum) + p.eps), kMostFactor);
    // a matrix of numbers below 2^-126 takes a factor that 32 bits do not hold: it goes in two steps
    float first = (float)fmin(factor, 0x1p100), second = (float)(factor / first);
#pragma unroll
    for (int q = 0; q < S::PARTS; ++q)
#pragma unroll
        for (int i = 0; i < S::XI; ++i)
#pragma unroll
            for (int j = 0; j < S::J; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[q][i][j][e] = x[q][i][j][e] * first * second;

    // acc[i][j] += rows `ra` of A times rows `rb` of B, over `depth` columns; planes lie behind each other
    auto multiply = [&](auto& acc, const _Float16* a, int a_rows, int ra, const _Float16* b, int b_rows, int depth) {
        constexpr int I = sizeof(acc) / sizeof(acc[0]);
        for (int k = 0; k < depth; k += 32) {
            half8 fa[2][I], fb[2][S::J];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < I; ++i)
                    fa[h][i] = *(const half8*)(a + h * a_rows * depth +
                                               small_at(a_rows, ra + i * 16 + lane % 16, k + lane / 16 * 8));
#pragma unroll
                for (int j = 0; j < S::J; ++j)
                    fb[h][j] = *(const half8*)(b + h * b_rows * depth +
                                               small_at(b_rows, c0 + j * 16, k + lane / 16 * 8));
            }
#pragma unroll
            for (int t = 0; t < 3; ++t)
#pragma unroll
                for (int i = 0; i < I; ++i)
#pragma unroll
                    for (int j = 0; j < S::J; ++j) acc[i][j] = M::run(fa[t == 0][i], fb[t == 1][j], acc[i][j]);
        }
    };

    for (int step = 0; step < p.steps; ++step) {
        // G, a part of X's columns at a time
        float4v acc[S::GI][S::J];
#pragma unroll
        for (int i = 0; i < S::GI; ++i)
#pragma unroll
            for (int j = 0; j < S::J; ++j) acc[i][j] = (float4v)(0.f);
#pragma unroll
        for (int q = 0; q < S::PARTS; ++q) {
            if (q > 0) __syncthreads();
#pragma unroll
            for (int i = 0; i < S::XI; ++i)
#pragma unroll
                for (int j = 0; j < S::J; ++j) {
                    half4 hi, lo;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        _Float16 h, l;
                        split(x[q][i][j][e], h, l);
                        hi[e] = h, lo[e] = l;
                    }
                    int at = small_at(MP, c0 + j * 16, row_x(0, i));
                    *(half4*)(lx + at) = hi;
                    *(half4*)(lx + S::X_PLANE + at) = lo;
                }
            __syncthreads();
            multiply(acc, lx, MP, r_wave * (MP / 2), lx, MP, S::PART);
        }
        // G is symmetric: its element (r, c) is written as (c, r)
        auto place = [&](int i, int j) { return small_at(MP, c0 + j * 16, r_wave * (MP / 2) + i * 16 + r_lane); };
        auto write_g = [&] {
#pragma unroll
            for (int i = 0; i < S::GI; ++i)
#pragma unroll
                for (int j = 0; j < S::J; ++j) {
                    half4 hi, lo;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        _Float16 h, l;
                        split(acc[i][j][e], h, l);
                        hi[e] = h, lo[e] = l;
                    }
                    *(half4*)(lg + place(i, j)) = hi;
                    *(half4*)(lg + S::G_PLANE + place(i, j)) = lo;
                }
        };
        float kept[S::GI][S::J][4];
#pragma unroll
        for (int i = 0; i < S::GI; ++i)
#pragma unroll
            for (int j = 0; j < S::J; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    acc[i][j][e] *= p.gram;
                    kept[i][j][e] = p.linear * acc[i][j][e];
                }
        write_g();
        __syncthreads();
        // B = b G + c G G in the place of G
#pragma unroll
        for (int i = 0; i < S::GI; ++i)
#pragma unroll
            for (int j = 0; j < S::J; ++j) acc[i][j] = (float4v)(0.f);
        multiply(acc, lg, MP, r_wave * (MP / 2), lg, MP, MP);
#pragma unroll
        for (int i = 0; i < S::GI; ++i)
#pragma unroll
            for (int j = 0; j < S::J; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = acc[i][j][e] * p.square + kept[i][j][e];
        __syncthreads();
        write_g();
        // x <- a x + (B X)^T, a part of X^T's rows at a time
#pragma unroll
        for (int q = 0; q < S::PARTS; ++q) {
            if (q > 0) __syncthreads();
#pragma unroll
            for (int i = 0; i < S::XI; ++i)
#pragma unroll
                for (int j = 0; j < S::J; ++j)
                {
                    // neighbouring lanes hold neighbouring columns: the even one writes both of rows 0 and 1, the odd one
                    // of rows 2 and 3
                    bool odd = lane & 1;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mine = odd ? x[q][i][j][2 + e] : x[q][i][j][e], given = odd ? x[q][i][j][e] : x[q][i][j][2 + e];
                        float other = __int_as_float(
                            __builtin_amdgcn_update_dpp(0, __float_as_int(given), 0xb1, 0xf, 0xf, true));
                        half2v hi, lo;
                        _Float16 h, l;
                        split(odd ? other : mine, h, l);
                        hi[0] = h, lo[0] = l;
                        split(odd ? mine : other, h, l);
                        hi[1] = h, lo[1] = l;
                        int at = small_at(S::PART, row_x(0, i) + e + (odd ? 2 : 0), (c0 & ~1) + j * 16);
                        *(half2v*)(lx + at) = hi;
                        *(half2v*)(lx + S::X_PLANE + at) = lo;
                    }
                }
            __syncthreads();
            float4v got[S::XI][S::J];
#pragma unroll
            for (int i = 0; i < S::XI; ++i)
#pragma unroll
                for (int j = 0; j < S::J; ++j) got[i][j] = (float4v)(0.f);
            multiply(got, lx, S::PART, r_wave * (S::PART / 2), lg, MP, MP);
#pragma unroll
            for (int i = 0; i < S::XI; ++i)
#pragma unroll
                for (int j = 0; j < S::J; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[q][i][j][e] = p.keep * x[q][i][j][e] + p.update * got[i][j][e];
        }
        __syncthreads();
    }
#pragma unroll
    for (int q = 0; q < S::PARTS; ++q)
#pragma unroll
        for (int i = 0; i < S::XI; ++i)
#pragma unroll
            for (int j = 0; j < S::J; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    int r = row_x(q, i) + e, c = c0 + j * 16;
                    if (c < to.rows && r < to.cols)
                        ((T*)to.base)[blockIdx.x * to.batch_stride + c * to.row_stride + r * to.col_stride] =
                            from_f<T>(x[q][i][j][e] * p.inv_scale);
                }
}

// whether one workgroup a matrix of m x n (m <= n) does all of it
bool small_takes(int64_t m, int64_t n, int64_t batch) {
    return m <= 128 && n <= 256 && (m <= 64 || n <= 128 || batch >= 16);
}

template <typename T>
void small_run(const Matrix& in, const Target& to, const Small& p, int64_t batch, hipStream_t stream) {
    auto go = [&](auto mp, auto np) {
        constexpr int MP = decltype(mp)::value, NP = decltype(np)::value;
        small_kernel<T, MP, NP><<<(unsigned)batch, 512, 0, stream>>>(in, to, p);
    };
    auto k64 = std::integral_constant<int, 64>{};
    auto k128 = std::integral_constant<int, 128>{};
    auto k256 = std::integral_constant<int, 256>{};
    if (in.rows <= 64)
        in.cols <= 64 ? go(k64, k64) : in.cols <= 128 ? go(k64, k128) : go(k64, k256);
    else
        in.cols <= 128 ? go(k128, k128) : go(k128, k256);
}

template <typename F>
void by_type(const torch::Tensor& x, F&& f) {
    switch (x.scalar_type()) {
        case torch::kFloat32: f((float*)nullptr); break;
        case torch::kFloat16: f((__half*)nullptr); break;
        case torch::kBFloat16: f((__hip_bfloat16*)nullptr); break;
        default: TORCH_CHECK(false, "orthogonalize: expected float32, float16 or bfloat16");
    }
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

int64_t tiles_of(int64_t m, int64_t n, int64_t batch, bool lower, int64_t side) {
    int64_t r = up(m, side) / side, c = up(n, side) / side;
    return (lower ? r * (r + 1) / 2 : r * c) * batch;
}

// How a product of m x n results (of which the lower triangle, or all) is cut: the tile side, and the parts of its depth.
// Taken is what has the busiest compute unit done first. Clocks of a stage of two planes, measured over a depth of 4096:
// of a tile that has its compute unit to itself, and of one among those that share it; a single plane takes 0.4 of them.
// Small tiles fill the chip where there are few; large ones need less from memory a product. Parts cost their sums' way
// through memory and another launch.
struct Plan {
    int side, parts;
};

Plan plan_of(int64_t m, int64_t n, int64_t depth, int64_t batch, bool lower, bool single = false) {
    static const struct { int side; double alone, shared; } costs[] = {
        {256, 5940, 5940}, {192, 3590, 3590}, {128, 1960, 1780}, {96, 1150, 1060}, {64, 680, 570}
    };
    Plan best{0, 1};
    double least = 0;
    int64_t stages = up(depth, kStage) / kStage;
    for (const auto& k : costs)
        for (int64_t parts = 1; parts <= (lower ? stages / 16 : 1) || parts == 1; ++parts) {
            if (parts > 64) break;
            int64_t tiles = tiles_of(m, n, batch, lower, k.side) * parts, each = (tiles + 255) / 256;
            double clocks = std::max(k.alone, each * k.shared) * ((stages + parts - 1) / parts) * (single ? 0.4 : 1.0);
            // 2300 clocks a microsecond; 4 us for the launch, and 4 bytes of a sum there and back at 4 TB/s
            if (parts > 1) clocks += 2300 * (4 + tiles * k.side * k.side * 8 / 4e6);
            if (!best.side || clocks < least) {
                least = clocks;
                best = {k.side, (int)parts};
            }
        }
    return best;
}

// The plans of all products of a call. The symmetric ones: G from X while that has one plane, G, products of m x m
// matrices, and two of those in one launch; then the product with X, whose depth is never cut.
struct Plans {
    Plan first, gram, one, two, update;
};

Plans plans_of(int64_t m, int64_t n, int64_t batch, bool single) {
    return {plan_of(m, m, n, batch, true, single), plan_of(m, m, n, batch, true), plan_of(m, m, m, batch, true),
            plan_of(m, m, m, 2 * batch, true), plan_of(m, n, m, batch, false)};
}

template <typename F>
void by_side(int side, int64_t tiles, F&& f) {
    switch (side) {
        case 256: f(Shape<256, 128, 64, 2>{}); break;
        case 192: f(Shape<192, 96, 48, 3>{}); break;
        case 128:
            // one tile a compute unit: eight waves hide each other's waiting; else two tiles do
            tiles <= 256 ? f(Shape<128, 64, 32, 4>{}) : f(Shape<128, 64, 64, 2>{});
            break;
        case 96: f(Shape<96, 48, 48, 3>{}); break;
        default: f(Shape<64, 32, 32, 3>{}); break;
    }
}

}  // namespace

// matrices [batch, rows, cols]. The scales are powers of two with |entry| * scale < 65504 for X, G, b G + c G G,
// Q = a + b G + c G G, and a product of `span` Qs; `span` 0 asks for the direct way, else P is applied every `span`
// steps.
torch::Tensor newton_schulz(
    torch::Tensor matrices, int64_t steps, double a, double b, double c, double eps, std::vector<double> scales,
    int64_t span
) {
    TORCH_CHECK(matrices.is_cuda() && matrices.dim() == 3, "orthogonalize: matrices must be [batch, m, n] on a HIP device");
    c10::OptionalDeviceGuard guard(matrices.device());
    auto result = torch::empty(matrices.sizes(), matrices.options());
    if (result.numel() == 0) return result;
    int64_t batch = matrices.size(0), rows = matrices.size(1), cols = matrices.size(2);
    bool tall = rows > cols;
    int64_t m = tall ? cols : rows, n = tall ? rows : cols;
    TORCH_CHECK(steps >= 1 && batch < 32768 && n <= (1 << 20) && scales.size() == 5,
                "orthogonalize: at least one step, fewer than 32768 matrices and sides of up to 2^20");
    double sx = scales[0], sg = scales[1], sb = scales[2], sq = scales[3], sp = scales[4];
    bool one = matrices.scalar_type() != torch::kFloat32;  // X has one plane until it is updated
    Plans plan = plans_of(m, n, batch, one);
    const std::pair<Plan, int64_t> plans[] = {
        {plan.first, batch}, {plan.gram, batch}, {plan.one, batch}, {plan.two, 2 * batch}
    };
    int rect = plan.update.side;
    // rows that tiles of either side reach, and whole tiles of the packing kernel
    int64_t mp = std::max(up(m, rect), up(m, kEdge)), np = std::max(up(n, rect), up(n, kEdge));
    for (const auto& [p, count] : plans) mp = std::max(mp, up(m, p.side));
    int depth_m = (int)up(m, kStage), depth_n = (int)up(n, kStage);
    Matrix in{matrices.data_ptr(), matrices.stride(0), matrices.stride(tall ? 2 : 1), matrices.stride(tall ? 1 : 2),
              (int)m, (int)n};
    int type = matrices.scalar_type() == torch::kFloat32 ? 0 : matrices.scalar_type() == torch::kFloat16 ? 1 : 2;
    Target to{result.data_ptr(), result.stride(0), result.stride(tall ? 2 : 1), result.stride(tall ? 1 : 2), (int)m,
              (int)n, type};
    hipStream_t stream = ding_current_stream();
    Small small{(float)(sg / (sx * sx)), (float)(c * sb / (sg * sg)), (float)(b * sb / sg), (float)(1.0 / sb), (float)a,
                (float)sx, (float)(1.0 / sx), eps, (int)steps};
    if (small_takes(m, n, batch)) {
        by_type(matrices, [&](auto* null) {
            using T = std::remove_pointer_t<decltype(null)>;
            small_run<T>(in, to, small, batch, stream);
        });
        HIP_CHECK_LAST();
        return result;
    }
    auto half = matrices.options().dtype(torch::kFloat16);
    int parts = (int)std::min<int64_t>(kNormBlocks, std::max<int64_t>(1, m * n / (kThreads * 32)));
    auto partial = torch::empty({batch * parts}, matrices.options().dtype(torch::kFloat64));
    auto rest = torch::empty({batch}, matrices.options().dtype(torch::kFloat32));
    std::vector<torch::Tensor> kept;
    auto planes = [&](int64_t r, int64_t q) {
        kept.push_back(torch::empty({2, batch, r, q}, half));
        _Float16* p = (_Float16*)kept.back().data_ptr();
        return Split{p, p + batch * r * q, r * q, (int)r};
    };
    Split x = planes(mp, np), xt = planes(np, mp), g = planes(mp, mp), q = planes(mp, mp);
    by_type(matrices, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        norm_kernel<T><<<dim3(parts, (unsigned)batch), kThreads, 0, stream>>>(in, partial.data_ptr<double>());
        HIP_CHECK_LAST();
        Split px = x, pt = xt;
        if (one) px.lo = pt.lo = nullptr;
        dim3 grid((unsigned)(up(n, kEdge) / kEdge), (unsigned)(up(m, kEdge) / kEdge), (unsigned)batch);
        pack_kernel<T><<<grid, kThreads, 0, stream>>>(in, partial.data_ptr<double>(), parts, eps, (float)sx, px, pt,
                                                      rest.data_ptr<float>());
        HIP_CHECK_LAST();
    });
    int64_t most = 0;
    for (const auto& [p, count] : plans)
        if (p.parts > 1) most = std::max(most, tiles_of(m, m, count, true, p.side) * p.parts * p.side * p.side);
    auto sums = torch::empty({most}, matrices.options().dtype(torch::kFloat32));
    float* partial_sums = sums.data_ptr<float>();
    // out = (alpha A B^T + beta E) scaled, for symmetric results; with a second B and out if given
    auto symmetric = [&](Split u, Split v, int depth, Epilogue ep, Split e, Split out, bool single,
                         const Split* v2 = nullptr, const Split* out2 = nullptr) {
        int64_t count = v2 ? 2 * batch : batch;
        Plan cut = v2 ? plan.two : single ? plan.first : depth == depth_m ? plan.one : plan.gram;
        by_side(cut.side, tiles_of(m, m, count, true, cut.side) * cut.parts, [&](auto shape) {
            using P = decltype(shape);
            unsigned r = (unsigned)up(m, P::TILE) / P::TILE, tiles = r * (r + 1) / 2;
            dim3 grid(tiles, (unsigned)cut.parts, (unsigned)count);
            auto go = [&](auto kernel) {
                kernel<<<grid, P::THREADS, 0, stream>>>(u, v, depth, ep, e, out, to, (int)batch, v2 ? *v2 : v,
                                                        out2 ? *out2 : out, partial_sums);
            };
            if (single)
                go(product_kernel<P, SYMMETRIC, 1, 1>);
            else
                go(product_kernel<P, SYMMETRIC, 2, 2>);
            if (cut.parts > 1) {
                HIP_CHECK_LAST();
                join_kernel<P><<<dim3(tiles, 1, (unsigned)count), P::THREADS, 0, stream>>>(
                    partial_sums, cut.parts, ep, e, out, (int)batch, out2 ? *out2 : out);
            }
        });
        HIP_CHECK_LAST();
    };
    // x <- beta x + p x
    auto update = [&](Split p, double scale, double beta, bool last, Split& next) {
        Epilogue ep{(float)(1.0 / scale), (float)beta, 0.f, one ? rest.data_ptr<float>() : nullptr, 1, 1,
                    (float)(1.0 / sx)};
        by_side(rect, tiles_of(m, n, batch, false, rect), [&](auto shape) {
            using P = decltype(shape);
            dim3 grid((unsigned)up(n, P::TILE) / P::TILE, (unsigned)up(m, P::TILE) / P::TILE, (unsigned)batch);
            auto go = [&](auto kernel) {
                kernel<<<grid, P::THREADS, 0, stream>>>(xt, p, depth_m, ep, x, next, to, (int)batch, p, next, nullptr);
            };
            if (last)
                one ? go(product_kernel<P, LAST, 1, 2>) : go(product_kernel<P, LAST, 2, 2>);
            else
                one ? go(product_kernel<P, UPDATE, 1, 2>) : go(product_kernel<P, UPDATE, 2, 2>);
        });
        HIP_CHECK_LAST();
        if (!last) std::swap(xt, next);
        one = false;
    };
    auto gram = [&] {
        symmetric(x, x, depth_n, {(float)(sg / (sx * sx)), 0.f, 0.f, one ? rest.data_ptr<float>() : nullptr, 2, 0, 0.f},
                  x, g, one);
    };
    if (span == 0) {
        Split next = steps > 1 ? planes(np, mp) : xt;
        for (int64_t s = 0; s < steps; ++s) {
            gram();
            symmetric(g, g, depth_m, {(float)(c * sb / (sg * sg)), (float)(b * sb / sg), 0.f, nullptr, 0, 0, 0.f}, g, q,
                      false);
            update(q, sb, a, s + 1 == steps, next);
        }
        return result;
    }
    Split next = steps > span ? planes(np, mp) : xt;
    Split p[2] = {planes(mp, mp), planes(mp, mp)}, y = planes(mp, mp);
    for (int64_t s = 0; s < steps; s += span) {
        int64_t count = std::min(span, steps - s);
        gram();
        for (int64_t i = 0; i < count; ++i) {
            // P is Q of the first step; it is written in P's scale then
            Split into = i == 0 ? p[0] : q;
            double s_into = i == 0 ? sp : sq;
            symmetric(g, g, depth_m,
                      {(float)(c * s_into / (sg * sg)), (float)(b * s_into / sg), (float)(a * s_into), nullptr, 0, 0, 0.f},
                      g, into, false);
            Epilogue plain{(float)(1.0 / s_into), 0.f, 0.f, nullptr, 0, 0, 0.f};
            bool more = i + 1 < count;
            // P <- Q P and Y = Q G, together where both are wanted; then G <- Y Q
            if (i > 0 && more)
                symmetric(q, g, depth_m, plain, g, y, false, &p[(i + 1) % 2], &p[i % 2]);
            else if (i > 0)
                symmetric(q, p[(i + 1) % 2], depth_m, plain, g, p[i % 2], false);
            else if (more)
                symmetric(into, g, depth_m, plain, g, y, false);
            if (more) symmetric(y, into, depth_m, plain, g, g, false);
        }
        update(p[(count + 1) % 2], sp, 0.0, s + count == steps, next);
    }
    return result;
}

// How newton_schulz cuts the products of a batch: for G of one plane (or as the next where the type has two), G, one and
// two m x m products and the product with X the tile's side, the parts of the depth and the workgroups. Nothing where a
// workgroup takes a whole matrix. It needs no device.
std::vector<std::vector<int64_t>> newton_schulz_plan(int64_t batch, int64_t rows, int64_t cols, bool single) {
    int64_t m = std::min(rows, cols), n = std::max(rows, cols);
    if (small_takes(m, n, batch)) return {};
    Plans p = plans_of(m, n, batch, single);
    auto row = [&](Plan k, int64_t width, int64_t count, bool lower) -> std::vector<int64_t> {
        return {k.side, k.parts, tiles_of(m, width, count, lower, k.side) * k.parts};
    };
    return {row(p.first, m, batch, true), row(p.gram, m, batch, true), row(p.one, m, batch, true),
            row(p.two, m, 2 * batch, true), row(p.update, n, batch, false)};
}
