// orthogonalize.hip — updates of matrices made nearly orthogonal by Newton-Schulz products, many
// matrices in the same launches.
//
//     X = G / (|G| + eps)   (G or its transpose: the one with m <= n),   then `steps` times
//     A = X X^T,   P = b A + c A^2,   X <- a X + P X
//
// Three products a step, of the form L R^T with both operands' rows along the contracted axis: A and P
// are symmetric (tiles on and above the diagonal are computed, and stored twice), and X is kept in
// both orders. Products run on the matrix cores in float16: of one plane for results of 16 bits of
// 8-bit precision, of two (hi and what it leaves, 22 bits; the product of the two small ones, 2^-24, is
// left out) for float32 and float16 results. Numbers are scaled by powers of two so that neither plane
// leaves float16's range: X (|X| about 1) by 64 sqrt(n), its entries then are about 1 to 64, A and P by
// 2^10. Sums are float32's; what X keeps of itself (a X, and P's diagonal times X) never goes through
// one plane: X is held in two, the diagonal apart in float32. With one plane, what is left of the
// rounding of A and P to 11 bits is 2 to 5 parts in 10^4 of the result (bfloat16's own: 16).
#include <algorithm>
#include <climits>
#include <cmath>
#include <memory>
#include <new>

#include "policy_common.hpp"

namespace navi_policy {
namespace {

using h8 = _Float16 __attribute__((ext_vector_type(8)));
using h4 = _Float16 __attribute__((ext_vector_type(4)));
using f16x16 = float __attribute__((ext_vector_type(16)));

constexpr int kMatrices = 28;       // of a launch: its arguments stay under 4 KiB
constexpr int kNormBlocks = 64;     // workgroups that sum a matrix's squares
constexpr int kDepth = 64;          // of a product's step
constexpr float kScaleA = 1024.0f;  // of A and P
constexpr int64_t kGroupBytes = int64_t{1} << 30;  // of workspace that matrices in one launch share

struct Matrix {
    const void* from;
    void* to;
    int64_t from_stride[2], to_stride[2];  // of X's rows and columns
    _Float16* rows;     // [planes][M][N] X
    _Float16* turned;   // [2][2][N][M] X^T, this step's and the next's, each hi and what it leaves
    _Float16* gram;     // [planes][M][M]
    _Float16* poly;     // [planes][M][M] P without its diagonal
    float* diagonal;    // [M] a + P's diagonal
    double* squares;    // [kNormBlocks]
    int32_t m, n, M, N;  // and rounded up to whole tiles
    int32_t from_dtype, to_dtype;
    int32_t first_tile, first_piece;  // of those of all matrices
    float scale;        // of X
};

struct Params {
    Matrix matrix[kMatrices];
    int32_t count, tiles;
    int32_t current;   // which of the two X^T is this step's
    float a, b, c, eps;
};
static_assert(sizeof(Params) <= 4096, "a launch's arguments");

__device__ inline float load_any(const void* from, int32_t dtype, int64_t at) {
    if (dtype == NAVI_POLICY_F32) return static_cast<const float*>(from)[at];
    if (dtype == NAVI_POLICY_BF16) return to_float(static_cast<const bf16*>(from)[at]);
    return to_float(static_cast<const f16*>(from)[at]);
}

__device__ inline void store_any(void* to, int32_t dtype, int64_t at, float x) {
    if (dtype == NAVI_POLICY_F32)
        static_cast<float*>(to)[at] = x;
    else if (dtype == NAVI_POLICY_BF16)
        static_cast<bf16*>(to)[at] = from_float<bf16>(x);
    else
        static_cast<f16*>(to)[at] = from_float<f16>(x);
}

// Squares of a matrix: workgroups take lines along its contiguous axis in turn.
__global__ __launch_bounds__(256) void newton_squares_kernel(Params P) {
    __shared__ double part[4];
    const Matrix& x = P.matrix[blockIdx.y];
    const bool along = x.from_stride[1] == 1;
    const int64_t lines = along ? x.m : x.n, length = along ? x.n : x.m, stride = along ? x.from_stride[0] : x.from_stride[1];
    double sum = 0.0;
    for (int64_t line = blockIdx.x; line < lines; line += kNormBlocks)
        for (int64_t i = threadIdx.x; i < length; i += 256) {
            const double v = load_any(x.from, x.from_dtype, line * stride + i);
            sum += v * v;
        }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) x.squares[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// The last matrix whose first tile (or piece) is not after `at`.
template <class F>
__device__ inline int matrix_of(const Params& P, int at, F first) {
    int lo = 0, hi = P.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (first(P.matrix[mid]) <= at)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

__device__ inline void split(float x, _Float16& hi, _Float16& lo) {
    hi = static_cast<_Float16>(x);
    lo = static_cast<_Float16>(x - static_cast<float>(hi));
}

// X from G: 64 x 64 numbers a workgroup, in both orders, zeros past the matrix.
template <int kPlanes16>
__global__ __launch_bounds__(256) void newton_begin_kernel(Params P) {
    __shared__ float tile[64][65];
    const int at = blockIdx.x, index = matrix_of(P, at, [](const Matrix& x) { return x.first_piece; });
    const Matrix& x = P.matrix[index];
    const int piece = at - x.first_piece, across = x.N / 64, row0 = piece / across * 64, col0 = piece % across * 64;
    const int lane = threadIdx.x & 63, wave = wave_of_workgroup();
    double sum = x.squares[lane];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    const double factor = x.scale / (sqrt(sum) + static_cast<double>(P.eps));
    const bool along = x.from_stride[1] == 1;
    for (int i = wave; i < 64; i += 4) {
        const int row = row0 + (along ? i : lane), col = col0 + (along ? lane : i);
        float v = 0.0f;
        if (row < x.m && col < x.n)
            v = static_cast<float>(load_any(x.from, x.from_dtype, row * x.from_stride[0] + col * x.from_stride[1]) * factor);
        tile[along ? i : lane][along ? lane : i] = v;
    }
    __syncthreads();
    const int64_t size = static_cast<int64_t>(x.M) * x.N;
    _Float16* turned = x.turned + P.current * 2 * size;
    for (int i = wave; i < 64; i += 4) {
        _Float16 hi, lo;
        split(tile[i][lane], hi, lo);
        const int64_t to = static_cast<int64_t>(row0 + i) * x.N + col0 + lane;
        x.rows[to] = hi;
        if (kPlanes16 == 2) x.rows[size + to] = lo;
        split(tile[lane][i], hi, lo);
        const int64_t back = static_cast<int64_t>(col0 + i) * x.M + row0 + lane;
        turned[back] = hi;
        turned[size + back] = lo;
    }
}

enum { kGram, kPoly, kApply, kLast };

// A product's operands from memory to LDS, 16 bytes a lane, without registers between: a row of 64
// numbers is eight pieces, piece p of row r in place p ^ (r % 8), so that the eight lanes that read
// one piece of eight rows at once find them in all banks.
template <int kRows, int kThreads>
__device__ inline void stage(const _Float16* from, int64_t stride, _Float16* lds) {
    constexpr int kAtOnce = kThreads / 8;  // rows
    const int row = threadIdx.x >> 3, piece = (threadIdx.x & 7) ^ (row & 7);
    const _Float16* lane = from + row * stride + piece * 8;
    _Float16* to = lds + wave_of_workgroup() * 512;  // (the wave's; its lanes follow each other)
#pragma unroll
    for (int i = 0; i < kRows / kAtOnce; ++i)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(lane + i * kAtOnce * stride),
                                         (__attribute__((address_space(3))) void*)(to + i * kAtOnce * kDepth), 16, 0, 0);
}

// Tiles of one of the three products, kTile x kTile a workgroup, kTile / 2 x 64 a wave.
template <int kTile, int kPlanes16, int kMode>
__global__ __launch_bounds__(kTile * 2) void newton_product_kernel(Params P) {
    constexpr int kThreads = kTile * 2, kAcross = kTile / 64;  // waves side by side (two down)
    constexpr int kDown = kTile / 64;                          // results of 32 x 32 of a wave: down, and two across
    constexpr bool kSymmetric = kMode == kGram || kMode == kPoly;
    __shared__ __attribute__((aligned(16))) _Float16 lds[2][2][kTile * kDepth];
    const int wave = wave_of_workgroup(), lane = threadIdx.x & 63;
    // Workgroups go round the 8 XCDs in turn: each XCD takes a run of tiles.
    const int each = (P.tiles + 7) / 8, at = static_cast<int>(blockIdx.x % 8) * each + static_cast<int>(blockIdx.x / 8);
    if (static_cast<int>(blockIdx.x / 8) >= each || at >= P.tiles) return;
    const Matrix& x = P.matrix[matrix_of(P, at, [](const Matrix& y) { return y.first_tile; })];
    int tile_row, tile_col;
    {
        const int n = at - x.first_tile;
        if (kSymmetric) {  // tiles (i, j) with i <= j, a column of tiles after the other
            int j = static_cast<int>((sqrtf(8.0f * n + 1.0f) - 1.0f) * 0.5f);
            while ((j + 1) * (j + 2) / 2 <= n) ++j;
            while (j * (j + 1) / 2 > n) --j;
            tile_col = j;
            tile_row = n - j * (j + 1) / 2;
        } else {  // all rows of tiles of a column after the other: P is read again, X once
            const int down = x.M / kTile;
            tile_col = n / down;
            tile_row = n % down;
        }
    }
    const int64_t size = static_cast<int64_t>(x.M) * x.N, square = static_cast<int64_t>(x.M) * x.M;
    const _Float16* turned = x.turned + P.current * 2 * size;
    const int depth = kMode == kGram ? x.N : x.M;
    const _Float16* left = kMode == kGram ? x.rows : kMode == kPoly ? x.gram : x.poly;
    const _Float16* right = kMode == kGram ? x.rows : kMode == kPoly ? x.gram : turned;
    const int64_t left_plane = kMode == kGram ? size : square, right_plane = kMode == kPoly ? square : size;
    left += static_cast<int64_t>(tile_row) * kTile * depth;
    right += static_cast<int64_t>(tile_col) * kTile * depth;
    const int steps = depth / kDepth, all = (kPlanes16 == 2 ? 3 : 1) * steps;
    const auto load = [&](int step, int buffer) {  // the smallest products first
        const int term = kPlanes16 == 2 ? step / steps : 2, k = kPlanes16 == 2 ? step % steps : step;
        stage<kTile, kThreads>(left + (term == 0 ? left_plane : 0) + k * kDepth, depth, lds[buffer][0]);
        stage<kTile, kThreads>(right + (term == 1 ? right_plane : 0) + k * kDepth, depth, lds[buffer][1]);
    };
    const int row0 = wave / kAcross * (kTile / 2), col0 = wave % kAcross * 64;  // the wave's in the tile
    f16x16 sum[kDown][2];
#pragma unroll
    for (int i = 0; i < kDown; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int s = 0; s < 16; ++s) sum[i][j][s] = 0.0f;
    load(0, 0);
    for (int step = 0; step < all; ++step) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (step + 1 < all) load(step + 1, (step + 1) & 1);
        const _Float16* l = lds[step & 1][0];
        const _Float16* r = lds[step & 1][1];
#pragma unroll
        for (int k = 0; k < kDepth / 16; ++k) {
            const int piece = ((2 * k + (lane >> 5)) ^ (lane & 7)) * 8;
            h8 a[kDown], b[2];
#pragma unroll
            for (int i = 0; i < kDown; ++i) a[i] = *reinterpret_cast<const h8*>(&l[(row0 + 32 * i + (lane & 31)) * kDepth + piece]);
#pragma unroll
            for (int j = 0; j < 2; ++j) b[j] = *reinterpret_cast<const h8*>(&r[(col0 + 32 * j + (lane & 31)) * kDepth + piece]);
#pragma unroll
            for (int i = 0; i < kDown; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) sum[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i], b[j], sum[i][j], 0, 0, 0);
        }
    }
    // A lane has column l % 32 of each 32 x 32, rows 8 q + 4 (l / 32) to + 3.
    _Float16* next = x.turned + (1 - P.current) * 2 * size;
#pragma unroll
    for (int i = 0; i < kDown; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = tile_row * kTile + row0 + 32 * i + 8 * q + 4 * (lane >> 5), col = tile_col * kTile + col0 + 32 * j + (lane & 31);
                f4 v = {sum[i][j][4 * q], sum[i][j][4 * q + 1], sum[i][j][4 * q + 2], sum[i][j][4 * q + 3]};
                if constexpr (kSymmetric) {
                    _Float16* to = kMode == kGram ? x.gram : x.poly;
                    if constexpr (kMode == kGram) {
                        v = v * (kScaleA / (x.scale * x.scale));
                    } else {
                        const h4 hi = *reinterpret_cast<const h4*>(x.gram + static_cast<int64_t>(col) * x.M + row);
                        f4 g = __builtin_convertvector(hi, f4);
                        if constexpr (kPlanes16 == 2)
                            g += __builtin_convertvector(*reinterpret_cast<const h4*>(x.gram + square + static_cast<int64_t>(col) * x.M + row), f4);
                        v = P.b * g + v * (P.c / kScaleA);
#pragma unroll
                        for (int s = 0; s < 4; ++s)
                            if (row + s == col) {
                                x.diagonal[col] = P.a + v[s] * (1.0f / kScaleA);
                                v[s] = 0.0f;
                            }
                    }
                    h4 hi, lo;
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        _Float16 h, r;
                        split(v[s], h, r);
                        hi[s] = h;
                        lo[s] = r;
                    }
                    *reinterpret_cast<h4*>(to + static_cast<int64_t>(col) * x.M + row) = hi;
                    if constexpr (kPlanes16 == 2) *reinterpret_cast<h4*>(to + square + static_cast<int64_t>(col) * x.M + row) = lo;
                    if (tile_row != tile_col) {
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            to[static_cast<int64_t>(row + s) * x.M + col] = hi[s];
                            if constexpr (kPlanes16 == 2) to[square + static_cast<int64_t>(row + s) * x.M + col] = lo[s];
                        }
                    }
                } else {
                    const int64_t back = static_cast<int64_t>(col) * x.M + row;
                    const f4 own = __builtin_convertvector(*reinterpret_cast<const h4*>(turned + back), f4) +
                                   __builtin_convertvector(*reinterpret_cast<const h4*>(turned + size + back), f4);
                    v = *reinterpret_cast<const f4*>(x.diagonal + row) * own + v * (1.0f / kScaleA);
                    if constexpr (kMode == kApply) {
                        h4 hi, lo;
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            _Float16 h, r;
                            split(v[s], h, r);
                            hi[s] = h;
                            lo[s] = r;
                            const int64_t to = static_cast<int64_t>(row + s) * x.N + col;
                            x.rows[to] = h;
                            if constexpr (kPlanes16 == 2) x.rows[size + to] = r;
                        }
                        *reinterpret_cast<h4*>(next + back) = hi;
                        *reinterpret_cast<h4*>(next + size + back) = lo;
                    } else {
#pragma unroll
                        for (int s = 0; s < 4; ++s)
                            if (row + s < x.m && col < x.n)
                                store_any(x.to, x.to_dtype, (row + s) * x.to_stride[0] + col * x.to_stride[1], v[s] / x.scale);
                    }
                }
            }
}

int launched() {
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess)
        return set_error(NAVI_POLICY_E_LAUNCH, "navi_orthogonalize: kernel launch failed: %s", hipGetErrorString(err));
    return NAVI_POLICY_OK;
}

int64_t rounded(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Matrices of few tiles take smaller ones: with 256 x 256 a CU holds one workgroup, whose waves have
// twice the products for what they read.
int tile_of(const navi_orthogonalize_matrix* x, int count) {
    int64_t tiles = 0;
    for (int i = 0; i < count; ++i) tiles += ((x[i].rows + 255) / 256) * ((x[i].cols + 255) / 256);
    return tiles >= 256 ? 256 : 128;
}

int planes_of(const navi_orthogonalize_matrix& x) { return x.to_dtype == NAVI_POLICY_BF16 ? 1 : 2; }

int64_t bytes_of(const navi_orthogonalize_matrix& x, int tile, int planes) {
    const int64_t M = rounded(std::min(x.rows, x.cols), tile), N = rounded(std::max(x.rows, x.cols), tile);
    return 2 * (planes * M * N + 4 * M * N + 2 * planes * M * M) + rounded(4 * M, 256) + 8 * kNormBlocks;
}

// Matrices from `at` on that go together: of one number of planes, as many as a launch names and the
// workspace holds.
int group_end(const navi_orthogonalize_matrix* x, int count, int at, int tile, int64_t* bytes) {
    const int planes = planes_of(x[at]);
    int64_t total = 0;
    int end = at, named = 0;
    for (; end < count && named < kMatrices; ++end) {
        if (x[end].rows == 0 || x[end].cols == 0) continue;
        if (planes_of(x[end]) != planes) break;
        const int64_t own = bytes_of(x[end], tile, planes);
        if (named > 0 && total + own > kGroupBytes) break;
        total += own;
        ++named;
    }
    *bytes = total;
    return end;
}

int check(const navi_orthogonalize_matrix* x, int32_t count) {
    if (count < 0 || (count > 0 && !x)) return set_error(NAVI_POLICY_E_ARG, "matrices must be non-null");
    for (int i = 0; i < count; ++i) {
        if (x[i].rows < 0 || x[i].cols < 0 || x[i].rows > (1 << 20) || x[i].cols > (1 << 20) || x[i].rows * x[i].cols > INT32_MAX)
            return set_error(NAVI_POLICY_E_ARG, "matrix %d must have at most 2^20 rows and columns, and 2^31 numbers", i);
        for (int32_t t : {x[i].from_dtype, x[i].to_dtype})
            if (t < NAVI_POLICY_F32 || t > NAVI_POLICY_F16)
                return set_error(NAVI_POLICY_E_ARG, "matrix %d must be float32, bfloat16 or float16", i);
        if (x[i].rows == 0 || x[i].cols == 0) continue;
        if (!x[i].from || !x[i].to) return set_error(NAVI_POLICY_E_ARG, "matrix %d is null", i);
        if (!aligned(x[i].from_dtype == NAVI_POLICY_F32 ? 4 : 2, x[i].from) || !aligned(x[i].to_dtype == NAVI_POLICY_F32 ? 4 : 2, x[i].to))
            return set_error(NAVI_POLICY_E_ARG, "matrix %d must be aligned to its elements", i);
        if (x[i].from_stride[0] != 1 && x[i].from_stride[1] != 1)
            return set_error(NAVI_POLICY_E_ARG, "matrix %d must be contiguous along its rows or its columns", i);
    }
    return NAVI_POLICY_OK;
}

struct Span {  // a matrix's bytes, from its first number to its last
    uintptr_t first, end;
    int32_t matrix;
};

Span span_of(const navi_orthogonalize_matrix& x, const void* p, const int64_t (&stride)[2], int32_t dtype, int32_t index) {
    const Extent e = extent_of(p, {x.rows, x.cols, 1, 1}, {stride[0], stride[1], 0, 0}, dtype == NAVI_POLICY_F32 ? 4 : 2);
    return Span{e.first, e.end, index};
}

// Results are written while other matrices are read or written: they lie apart, but for one in its own place.
int check_apart(const navi_orthogonalize_matrix* x, int count) {
    const std::unique_ptr<Span[]> spans(new (std::nothrow) Span[std::max(count, 1)]);
    if (!spans) return set_error(NAVI_POLICY_E_ARG, "out of host memory for %d matrices", count);
    int written = 0;
    for (int i = 0; i < count; ++i)
        if (x[i].rows > 0 && x[i].cols > 0) spans[written++] = span_of(x[i], x[i].to, x[i].to_stride, x[i].to_dtype, i);
    std::sort(&spans[0], &spans[0] + written, [](const Span& a, const Span& b) { return a.first < b.first; });
    for (int i = 1; i < written; ++i)
        if (spans[i - 1].end > spans[i].first)
            return set_error(NAVI_POLICY_E_ARG, "matrices %d and %d that are written share memory",
                             std::min(spans[i - 1].matrix, spans[i].matrix), std::max(spans[i - 1].matrix, spans[i].matrix));
    for (int i = 0; i < count; ++i) {
        if (x[i].rows == 0 || x[i].cols == 0) continue;
        const Span read = span_of(x[i], x[i].from, x[i].from_stride, x[i].from_dtype, i);
        // (the squares and X are taken of a matrix before its result is written: its own memory it may share in any way)
        for (const Span* next = std::partition_point(&spans[0], &spans[0] + written, [&](const Span& s) { return s.end <= read.first; });
             next != &spans[0] + written && next->first < read.end; ++next)
            if (next->matrix != i)
                return set_error(NAVI_POLICY_E_ARG, "matrix %d that is read and matrix %d that is written share memory", i, next->matrix);
    }
    return NAVI_POLICY_OK;
}

template <int kTile, int kPlanes16>
int run_group(Params& P, int squares_rows, int pieces, int steps, hipStream_t stream) {
    hipLaunchKernelGGL(newton_squares_kernel, dim3(kNormBlocks, squares_rows), dim3(256), 0, stream, P);
    hipLaunchKernelGGL(newton_begin_kernel<kPlanes16>, dim3(pieces), dim3(256), 0, stream, P);
    Params S = P, X = P;  // tiles of the symmetric products, and of the other
    S.tiles = X.tiles = 0;
    for (int i = 0; i < P.count; ++i) {
        const int down = P.matrix[i].M / kTile, across = P.matrix[i].N / kTile;
        S.matrix[i].first_tile = S.tiles;
        X.matrix[i].first_tile = X.tiles;
        S.tiles += down * (down + 1) / 2;
        X.tiles += down * across;
    }
    const dim3 symmetric((S.tiles + 7) / 8 * 8), whole((X.tiles + 7) / 8 * 8), threads(kTile * 2);
    for (int step = 0; step < steps; ++step) {
        S.current = X.current = step & 1;
        hipLaunchKernelGGL((newton_product_kernel<kTile, kPlanes16, kGram>), symmetric, threads, 0, stream, S);
        hipLaunchKernelGGL((newton_product_kernel<kTile, kPlanes16, kPoly>), symmetric, threads, 0, stream, S);
        if (step + 1 < steps)
            hipLaunchKernelGGL((newton_product_kernel<kTile, kPlanes16, kApply>), whole, threads, 0, stream, X);
        else
            hipLaunchKernelGGL((newton_product_kernel<kTile, kPlanes16, kLast>), whole, threads, 0, stream, X);
    }
    return launched();
}

}  // namespace
}  // namespace navi_policy

extern "C" int64_t navi_orthogonalize_workspace(int32_t count, const navi_orthogonalize_matrix* matrices) {
    using namespace navi_policy;
    const int code = check(matrices, count);
    if (code != NAVI_POLICY_OK) return code;
    const int tile = tile_of(matrices, count);
    int64_t most = 0;
    for (int at = 0; at < count;) {
        int64_t bytes;
        at = group_end(matrices, count, at, tile, &bytes);
        most = std::max(most, bytes);
    }
    return most;
}

extern "C" int navi_orthogonalize(int32_t count, const navi_orthogonalize_matrix* matrices, int32_t steps, float a, float b, float c,
                                  float eps, void* workspace, void* stream) {
    using namespace navi_policy;
    const int code = check(matrices, count);
    if (code != NAVI_POLICY_OK) return code;
    if (steps < 1 || steps > 100) return set_error(NAVI_POLICY_E_ARG, "steps must be in [1, 100]");
    if (!(eps >= 0.0f)) return set_error(NAVI_POLICY_E_ARG, "eps must not be negative");
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return set_error(NAVI_POLICY_E_ARG, "the factors must be finite");
    const int shared = check_apart(matrices, count);
    if (shared != NAVI_POLICY_OK) return shared;
    const int tile = tile_of(matrices, count);
    for (int at = 0; at < count;) {
        int64_t bytes;
        const int end = group_end(matrices, count, at, tile, &bytes);
        if (bytes > 0 && (!workspace || !aligned(256, workspace)))
            return set_error(NAVI_POLICY_E_ARG, "workspace must be non-null and 256-byte aligned");
        Params P{};
        P.a = a;
        P.b = b;
        P.c = c;
        P.eps = eps;
        int planes = 1, pieces = 0;
        char* place = static_cast<char*>(workspace);
        for (; at < end; ++at) {
            const navi_orthogonalize_matrix& given = matrices[at];
            if (given.rows == 0 || given.cols == 0) continue;
            planes = planes_of(given);
            Matrix& x = P.matrix[P.count++];
            const int turn = given.rows > given.cols;  // X is the transpose
            x.from = given.from;
            x.to = given.to;
            for (int k = 0; k < 2; ++k) {
                x.from_stride[k] = given.from_stride[k ^ turn];
                x.to_stride[k] = given.to_stride[k ^ turn];
            }
            x.m = static_cast<int32_t>(turn ? given.cols : given.rows);
            x.n = static_cast<int32_t>(turn ? given.rows : given.cols);
            x.M = static_cast<int32_t>(rounded(x.m, tile));
            x.N = static_cast<int32_t>(rounded(x.n, tile));
            x.from_dtype = given.from_dtype;
            x.to_dtype = given.to_dtype;
            x.scale = std::exp2(std::round(std::log2(std::sqrt(static_cast<float>(x.n)))) + 6.0f);
            x.first_piece = pieces;
            pieces += x.M / 64 * (x.N / 64);
            const int64_t size = static_cast<int64_t>(x.M) * x.N, square = static_cast<int64_t>(x.M) * x.M;
            x.rows = reinterpret_cast<_Float16*>(place);
            x.turned = x.rows + planes * size;
            x.gram = x.turned + 4 * size;
            x.poly = x.gram + planes * square;
            x.diagonal = reinterpret_cast<float*>(x.poly + planes * square);
            x.squares = reinterpret_cast<double*>(reinterpret_cast<char*>(x.diagonal) + rounded(4 * static_cast<int64_t>(x.M), 256));
            place = reinterpret_cast<char*>(x.squares + kNormBlocks);
        }
        if (P.count == 0) continue;
        hipStream_t on = as_stream(stream);
        int result;
        if (tile == 256)
            result = planes == 1 ? run_group<256, 1>(P, P.count, pieces, steps, on) : run_group<256, 2>(P, P.count, pieces, steps, on);
        else
            result = planes == 1 ? run_group<128, 1>(P, P.count, pieces, steps, on) : run_group<128, 2>(P, P.count, pieces, steps, on);
        if (result != NAVI_POLICY_OK) return result;
    }
    return NAVI_POLICY_OK;
}
