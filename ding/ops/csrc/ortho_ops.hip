// Orthogonalisation of matrices by Newton-Schulz products.
//
//   X_0 = M / (|M|_F + eps), transposed where M is tall;  five times or so:
//   G = X X^T,  B = b G + c G G,  X <- a X + B X
// Each step maps every singular value s to a s + b s^3 + c s^5 and leaves the singular vectors.
//
// Bound by the matrix units. There is no wide 32-bit matrix instruction here, and the iteration multiplies early errors by
// a^steps (about 500), so 16-bit factors alone lose the small singular values. Every factor is therefore held as two
// half-precision numbers, v = (hi + lo) / scale with 22 significant bits, and a product is three matrix instructions,
//   hi hi + hi lo + lo hi   (lo lo is below 2^-22 of the result),
// summed in 32 bits. The scales are powers of two that the host derives from a bound of the singular values, so that
// nothing overflows and nothing but negligible entries becomes subnormal. G and G G are symmetric: half their tiles are
// computed and written twice.
//
// All three products are "row times row" (C_ij = sum_k A_ik B_jk), which needs X and its transpose: both are kept.
// Sides are padded with zeros to a multiple of kPad, so that the product kernels have no edges.
#include "common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace {

constexpr int kPad = 128;
constexpr int kThreads = 256;
constexpr int kNormBlocks = 64;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

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

// two planes [batch, rows, cols] of half precision
struct Split {
    _Float16 *hi, *lo;
    int64_t batch_stride;
    int cols;
};

__device__ inline void split(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// sums of squares in 64 bits, where no square of a 32-bit number overflows or vanishes
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_kernel(Matrix m, double* __restrict__ partial) {
    const T* p = (const T*)m.base + blockIdx.y * m.batch_stride;
    double sum = 0;
    bool flip = m.row_stride < m.col_stride;  // walk the dense direction
    int64_t inner = flip ? m.rows : m.cols, n = (int64_t)m.rows * m.cols;
    int64_t si = flip ? m.row_stride : m.col_stride, so = flip ? m.col_stride : m.row_stride;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)kNormBlocks * kThreads) {
        double v = to_f(p[i / inner * so + i % inner * si]);
        sum += v * v;
    }
    __shared__ double part[kThreads / kWave];
    for (int o = kWave / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / kWave; ++w) sum += part[w];
        partial[blockIdx.y * kNormBlocks + blockIdx.x] = sum;
    }
}

// X and its transpose from M: a 64 x 64 tile a workgroup, turned in LDS
template <typename T>
__global__ void __launch_bounds__(kThreads) pack_kernel(
    Matrix m, const double* __restrict__ partial, double eps, float scale, Split x, Split xt
) {
    __shared__ float tile[64][65];
    __shared__ float factor_s;
    int b = blockIdx.z;
    if (threadIdx.x < kWave) {
        double sum = threadIdx.x < kNormBlocks ? partial[b * kNormBlocks + threadIdx.x] : 0;
        for (int o = kWave / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
        if (threadIdx.x == 0) factor_s = (float)(scale / (sqrt(sum) + eps));
    }
    __syncthreads();
    float factor = factor_s;
    const T* p = (const T*)m.base + b * m.batch_stride;
    int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64, lane = threadIdx.x % 64;
    bool flip = m.row_stride < m.col_stride;
    for (int r = threadIdx.x / 64; r < 64; r += kThreads / 64) {
        int i = flip ? lane : r, j = flip ? r : lane;
        bool in = i0 + i < m.rows && j0 + j < m.cols;
        tile[i][j] = in ? to_f(p[(i0 + i) * m.row_stride + (j0 + j) * m.col_stride]) * factor : 0.f;
    }
    __syncthreads();
    for (int r = threadIdx.x / 64; r < 64; r += kThreads / 64) {
        _Float16 hi, lo;
        split(tile[r][lane], hi, lo);
        int64_t at = b * x.batch_stride + (int64_t)(i0 + r) * x.cols + j0 + lane;
        x.hi[at] = hi;
        x.lo[at] = lo;
        split(tile[lane][r], hi, lo);
        at = b * xt.batch_stride + (int64_t)(j0 + r) * xt.cols + i0 + lane;
        xt.hi[at] = hi;
        xt.lo[at] = lo;
    }
}

enum Kind { GRAM, SQUARE, UPDATE, LAST };

struct Target {
    void* base;
    int64_t batch_stride, row_stride, col_stride;
    int rows, cols;
};

// C = A B^T over split factors, a TILE x TILE tile a workgroup, a quarter of it a wave.
//   GRAM:   A = B = X;      out = G, both triangles
//   SQUARE: A = B = G;      out = b G + c C, both triangles
//   UPDATE: A = X^T, B = b G + c G G (symmetric): C = (B X)^T; x <- a x + C^T and its transpose to out
//   LAST:   the same, written to the caller's matrix in its type
template <int TILE, Kind kind, typename T>
__global__ void __launch_bounds__(kThreads) product_kernel(
    Split a, Split bm, int depth, float alpha, float beta, float inv_scale, Split x, Split out, Target to
) {
    constexpr int K = 32;               // depth of a stage
    constexpr int W = TILE / 2;         // a wave's side
    constexpr int S = W / 32;           // matrix instructions along it
    constexpr int CHUNKS = TILE * K / 8;  // 16-byte pieces of a plane of a stage
    __shared__ half8 sa[2][CHUNKS], sb[2][CHUNKS];
    int bi, bj;
    if constexpr (kind == GRAM || kind == SQUARE) {
        // tile number t of the lower triangle
        int t = blockIdx.x;
        bi = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
        while ((bi + 1) * (bi + 2) / 2 <= t) ++bi;
        while (bi * (bi + 1) / 2 > t) --bi;
        bj = t - bi * (bi + 1) / 2;
    } else {
        bi = blockIdx.x;
        bj = blockIdx.y;
    }
    int64_t batch = blockIdx.z;
    int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int wi = wave / 2 * W, wj = wave % 2 * W;
    float16v acc[S][S];
    for (int i = 0; i < S; ++i)
        for (int j = 0; j < S; ++j) acc[i][j] = (float16v)(0.f);
    const _Float16* pa[2] = {a.hi + batch * a.batch_stride, a.lo + batch * a.batch_stride};
    const _Float16* pb[2] = {bm.hi + batch * bm.batch_stride, bm.lo + batch * bm.batch_stride};
    for (int k0 = 0; k0 < depth; k0 += K) {
        __syncthreads();
#pragma unroll
        for (int c = threadIdx.x; c < CHUNKS; c += kThreads) {
            int row = c / 4, piece = c % 4;
            int at = row * 4 + (piece ^ ((row >> 1) & 3));  // eight rows' pieces fall into different banks
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                sa[p][at] = *(const half8*)(pa[p] + (int64_t)(bi * TILE + row) * a.cols + k0 + piece * 8);
                sb[p][at] = *(const half8*)(pb[p] + (int64_t)(bj * TILE + row) * bm.cols + k0 + piece * 8);
            }
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < K / 16; ++ks) {
            half8 fa[2][S], fb[2][S];
#pragma unroll
            for (int s = 0; s < S; ++s) {
                int ra = wi + s * 32 + lane % 32, rb = wj + s * 32 + lane % 32, piece = ks * 2 + lane / 32;
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    fa[p][s] = sa[p][ra * 4 + (piece ^ ((ra >> 1) & 3))];
                    fb[p][s] = sb[p][rb * 4 + (piece ^ ((rb >> 1) & 3))];
                }
            }
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[1][i], fb[0][j], acc[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0][i], fb[1][j], acc[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0][i], fb[0][j], acc[i][j], 0, 0, 0);
                }
        }
    }
    // a lane holds column lane % 32 of rows 8 q + 4 (lane / 32) + 0..3
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = 0; j < S; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                int r = bi * TILE + wi + i * 32 + q * 8 + lane / 32 * 4, c = bj * TILE + wj + j * 32 + lane % 32;
                half4 hi, lo;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][q * 4 + e] * alpha;
                if constexpr (kind != GRAM) {
                    // the element itself: of G at (c, r), of x at (c, r)
                    int64_t at = batch * x.batch_stride + (int64_t)c * x.cols + r;
                    half4 xh = *(const half4*)(x.hi + at), xl = *(const half4*)(x.lo + at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += beta * ((float)xh[e] + (float)xl[e]);
                }
                if constexpr (kind == LAST) {
                    if (c < to.rows)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (r + e < to.cols)
                                ((T*)to.base)[batch * to.batch_stride + c * to.row_stride + (r + e) * to.col_stride] =
                                    from_f<T>(v[e] * inv_scale);
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
                    int64_t at = batch * x.batch_stride + (int64_t)c * x.cols + r;
                    *(half4*)(x.hi + at) = hi;
                    *(half4*)(x.lo + at) = lo;
                } else if (bi != bj) {
                    int64_t at = batch * out.batch_stride + (int64_t)c * out.cols + r;
                    *(half4*)(out.hi + at) = hi;
                    *(half4*)(out.lo + at) = lo;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    int64_t at = batch * out.batch_stride + (int64_t)(r + e) * out.cols + c;
                    out.hi[at] = hi[e];
                    out.lo[at] = lo[e];
                }
            }
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

}  // namespace

// matrices [batch, rows, cols]; the scales are powers of two with |entry| * scale < 65504
torch::Tensor newton_schulz(
    torch::Tensor matrices, int64_t steps, double a, double b, double c, double eps, double scale_x, double scale_g,
    double scale_b
) {
    TORCH_CHECK(matrices.is_cuda() && matrices.dim() == 3, "orthogonalize: matrices must be [batch, m, n] on a HIP device");
    c10::OptionalDeviceGuard guard(matrices.device());
    auto result = torch::empty(matrices.sizes(), matrices.options());
    if (result.numel() == 0) return result;
    int64_t batch = matrices.size(0), rows = matrices.size(1), cols = matrices.size(2);
    bool tall = rows > cols;
    int64_t m = tall ? cols : rows, n = tall ? rows : cols;
    TORCH_CHECK(steps >= 1 && batch < 65536 && n <= (1 << 20), "orthogonalize: at least one step, fewer than 65536 "
                "matrices and sides of up to 2^20");
    int64_t mp = (m + kPad - 1) / kPad * kPad, np = (n + kPad - 1) / kPad * kPad;
    Matrix in{matrices.data_ptr(), matrices.stride(0), matrices.stride(tall ? 2 : 1), matrices.stride(tall ? 1 : 2),
              (int)m, (int)n};
    Target to{result.data_ptr(), result.stride(0), result.stride(tall ? 2 : 1), result.stride(tall ? 1 : 2), (int)m,
              (int)n};
    auto half = matrices.options().dtype(torch::kFloat16);
    auto partial = torch::empty({batch * kNormBlocks}, matrices.options().dtype(torch::kFloat64));
    std::vector<torch::Tensor> kept;
    auto planes = [&](int64_t r, int64_t q) {
        kept.push_back(torch::empty({2, batch, r, q}, half));
        _Float16* p = (_Float16*)kept.back().data_ptr();
        return Split{p, p + batch * r * q, r * q, (int)q};
    };
    Split x = planes(mp, np), xt[2] = {planes(np, mp), planes(np, mp)}, g = planes(mp, mp), bg = planes(mp, mp);
    hipStream_t stream = ding_current_stream();
    by_type(matrices, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        norm_kernel<T><<<dim3(kNormBlocks, (unsigned)batch), kThreads, 0, stream>>>(in, partial.data_ptr<double>());
        HIP_CHECK_LAST();
        pack_kernel<T><<<dim3((unsigned)(np / 64), (unsigned)(mp / 64), (unsigned)batch), kThreads, 0, stream>>>(
            in, partial.data_ptr<double>(), eps, (float)scale_x, x, xt[0]);
        HIP_CHECK_LAST();
        constexpr int TILE = 128;
        unsigned tiles = (unsigned)(mp / TILE), wide = (unsigned)(np / TILE);
        dim3 half_grid(tiles * (tiles + 1) / 2, 1, (unsigned)batch), grid(wide, tiles, (unsigned)batch);
        for (int64_t s = 0; s < steps; ++s) {
            Split from = xt[s % 2], next = xt[(s + 1) % 2];
            product_kernel<TILE, GRAM, T><<<half_grid, kThreads, 0, stream>>>(
                x, x, (int)np, (float)(scale_g / (scale_x * scale_x)), 0.f, 0.f, x, g, to);
            product_kernel<TILE, SQUARE, T><<<half_grid, kThreads, 0, stream>>>(
                g, g, (int)mp, (float)(c * scale_b / (scale_g * scale_g)), (float)(b * scale_b / scale_g), 0.f, g, bg,
                to);
            float alpha = (float)(1.0 / scale_b);
            if (s + 1 < steps)
                product_kernel<TILE, UPDATE, T><<<grid, kThreads, 0, stream>>>(
                    from, bg, (int)mp, alpha, (float)a, 0.f, x, next, to);
            else
                product_kernel<TILE, LAST, T><<<grid, kThreads, 0, stream>>>(
                    from, bg, (int)mp, alpha, (float)a, (float)(1.0 / scale_x), x, next, to);
            HIP_CHECK_LAST();
        }
    });
    return result;
}
