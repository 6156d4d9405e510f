// orthogonalize.hip — updates of matrices made nearly orthogonal by Newton-Schulz products, many
// matrices in the same launches.
//
//     X = G / (|G| + eps)   (G or its transpose: the one with m <= n),   then `steps` times
//     A = X X^T,   P = b A + c A^2,   X <- a X + P X
//
// Three products a step, of the form L R^T with both operands' rows along the contracted axis: A and P
// are symmetric (tiles on and above the diagonal are computed, and stored twice), and X is kept in
// both orders. Products run on the matrix cores in float16: of one plane for bfloat16 results of matrices with more
// than 256 rows and columns, of two (hi and what it leaves, 22 bits; the product of the two small ones, 2^-24, is
// left out) for all others. Numbers are scaled by powers of two so that neither plane
// leaves float16's range: A and P by 2^10, X (|X| about 1) by 64 sqrt(n), which brings the entries of an X
// whose size is spread out to about 1 to 64, but by no more than leaves an entry of X's largest singular value
// (all of it in one place) below 65504: 2^15 with the default factors, whose steps take singular values
// to 1.2025. An X of a million columns spread out then has entries of 32. Factors that take singular values
// past 7.9 between steps, or P past 62, are refused: their planes would not hold A or P. Sums are float32's;
// what X keeps of itself (a X, and P's diagonal times X) never goes through one plane: X is held in two, the
// diagonal apart in float32. With one plane, what is left of the
// rounding of A, P and the X in products to 11 bits is 3 to 7 parts in 10^4 of the result before its own rounding
// (bfloat16's: 16; 6 at widths of 300, 3.3 at 2000); X in one plane too would leave 10^-2 where singular values lie
// far apart. With two, 1 to 3 parts in 10^6.
//
// 8 blocks of width 2000 (32 squares, 16 of twice the length; 9.6e12 operations, of which symmetry spares a third)
// take 15 ms: A 0.72 ms and P 0.58 at 840 and 800 TFLOP/s of what is computed, X 1.7 ms at 640: a workgroup's 256 x 256
// tile reads 256 KB of X and writes 384 (both orders, what is left of the rounding) after its products, 4.3 GB in all,
// and all workgroups do so at about the same time. Half as wide tiles, two workgroups a CU: 1.68 ms, for registers
// spilled. 26 matrices of width 256: 174 us in 17 launches of 8 to 16 us each, the trips to memory of one tile.
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

constexpr int kMatrices = 62;       // of a launch: its arguments stay under 4 KiB
constexpr int kNormBlocks = 64;     // workgroups that sum a matrix's squares
constexpr int kDepth = 32;          // of a product's stage
constexpr float kScaleA = 1024.0f;  // of A and P
constexpr int64_t kGroupBytes = int64_t{4} << 30;  // of workspace that matrices in one launch share

struct Matrix {
    const void* from;
    void* to;
    int64_t from_line;      // elements between X's rows, or (`turned`) its columns; those along them lie side by side
    int64_t to_stride[2];   // of X's rows and columns
    int32_t m, n;           // X
    uint32_t place;         // in the workspace, 256 bytes
    int8_t from_dtype, to_dtype, turned;
    int8_t scale;           // X times two to this
};
struct Params {
    Matrix matrix[kMatrices];
    int32_t first[kMatrices];  // of a launch's tiles (or pieces) of all matrices
    char* workspace;
    int32_t count, tiles;
    int32_t tile;      // M and N are m and n rounded up to it
    int32_t current;   // which of the two X^T is this step's
    float a, b, c, eps;
};
static_assert(sizeof(Params) <= 4096, "a launch's arguments");

// Where a matrix's part of the workspace holds what.
template <int kPlanes16>
struct Parts {
    int32_t M, N;
    int64_t size, square;
    _Float16* rows;     // [planes][M][N] X
    _Float16* turned;   // [2][2][N][M] X^T, this step's and the next's, each hi and what it leaves
    _Float16* gram;     // [planes][M][M]
    _Float16* poly;     // [planes][M][M] P without its diagonal
    float* diagonal;    // [M] a + P's diagonal
    double* squares;    // [kNormBlocks]
    float scale;

    __device__ Parts(const Params& P, const Matrix& x, int tile) {
        M = (x.m + tile - 1) / tile * tile;
        N = (x.n + tile - 1) / tile * tile;
        size = static_cast<int64_t>(M) * N;
        square = static_cast<int64_t>(M) * M;
        squares = reinterpret_cast<double*>(P.workspace + 256 * static_cast<uint64_t>(x.place));
        diagonal = reinterpret_cast<float*>(squares + kNormBlocks);
        rows = reinterpret_cast<_Float16*>(diagonal + M);
        turned = rows + kPlanes16 * size;
        gram = turned + 4 * size;
        poly = gram + kPlanes16 * square;
        scale = __builtin_ldexpf(1.0f, x.scale);
    }
};

// Sixteen bytes at any element's address (vector accesses of global memory need no more).
template <class E>
struct __attribute__((packed, aligned(sizeof(E)))) Vector {
    u4 words;
};

// The squares of `count` numbers, by 256 threads. In float64: those of any float32 are in range.
template <class E>
__device__ inline double sum_of_squares(const E* from, int64_t count) {
    constexpr int kEach = 16 / sizeof(E);
    const int64_t whole = count / kEach;
    double sum = 0.0;
    const auto add = [&](u4 words) {
        union {
            u4 words;
            E elements[kEach];
        } got{words};
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const double v = to_float(got.elements[n]);
            sum += v * v;
        }
    };
    int64_t i = threadIdx.x;
    for (; i + 768 < whole; i += 1024) {
        u4 words[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) words[n] = reinterpret_cast<const Vector<E>*>(from)[i + 256 * n].words;
#pragma unroll
        for (int n = 0; n < 4; ++n) add(words[n]);
    }
    for (; i < whole; i += 256) add(reinterpret_cast<const Vector<E>*>(from)[i].words);
    const int64_t left = whole * kEach + threadIdx.x;
    if (left < count) {
        const double v = to_float(from[left]);
        sum += v * v;
    }
    return sum;
}

// Squares of a matrix: workgroups take lines along its contiguous axis in turn, or parts of all of them
// where those lie one after the other.
__global__ __launch_bounds__(256) void newton_squares_kernel(Params P) {
    __shared__ double part[4];
    const Matrix& x = P.matrix[blockIdx.y];
    int64_t lines = x.turned ? x.n : x.m, length = x.turned ? x.m : x.n, stride = x.from_line;
    if (stride == length) {  // (parts begin at multiples of 16 bytes from the first number)
        const int64_t all = lines * length;
        length = ((all + kNormBlocks - 1) / kNormBlocks + 7) / 8 * 8;
        lines = (all + length - 1) / length;
        stride = length;
        if (static_cast<int64_t>(blockIdx.x) + 1 == lines) length = all - blockIdx.x * length;
    }
    double sum = 0.0;
    for (int64_t line = blockIdx.x; line < lines; line += kNormBlocks) {
        if (x.from_dtype == NAVI_POLICY_F32)
            sum += sum_of_squares(static_cast<const float*>(x.from) + line * stride, length);
        else if (x.from_dtype == NAVI_POLICY_BF16)
            sum += sum_of_squares(static_cast<const bf16*>(x.from) + line * stride, length);
        else
            sum += sum_of_squares(static_cast<const f16*>(x.from) + line * stride, length);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) Parts<1>(P, x, P.tile).squares[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// The matrix that tile (or piece) `at` of a launch is of: the last whose first is not after it, each lane
// looking at one (arguments come from the host's memory: a search would wait for them several times).
__device__ inline int matrix_of(const Params& P, int at) {
    const int lane = threadIdx.x & 63;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < P.count && P.first[lane < kMatrices ? lane : 0] <= at)) - 1);
}

__device__ inline void split(float x, _Float16& hi, _Float16& lo) {
    hi = static_cast<_Float16>(x);
    lo = static_cast<_Float16>(x - static_cast<float>(hi));
}

// X from G: 64 x 64 numbers a workgroup, in both orders, zeros past the matrix.
template <int kPlanes16>
__global__ __launch_bounds__(256) void newton_begin_kernel(Params P) {
    __shared__ float tile[64][65];
    const int at = blockIdx.x, index = matrix_of(P, at);
    const Matrix& x = P.matrix[index];
    const Parts<kPlanes16> w(P, x, P.tile);
    const int piece = at - P.first[index], across = w.N / 64, row0 = piece / across * 64, col0 = piece % across * 64;
    const int lane = threadIdx.x & 63, wave = wave_of_workgroup();
    double sum = w.squares[lane];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    const double factor = w.scale / (sqrt(sum) + static_cast<double>(P.eps));
    const bool along = !x.turned;
    // Sixteen numbers a lane, all on their way at once; eight at a time leave.
    float v[16];
    const auto fetch = [&](const auto* from) {
#pragma unroll
        for (int n = 0; n < 16; ++n) {
            const int i = wave + 4 * n, row = row0 + (along ? i : lane), col = col0 + (along ? lane : i);
            v[n] = 0.0f;
            if (row < x.m && col < x.n) v[n] = to_float(from[along ? row * x.from_line + col : col * x.from_line + row]);
        }
    };
    if (x.from_dtype == NAVI_POLICY_F32)
        fetch(static_cast<const float*>(x.from));
    else if (x.from_dtype == NAVI_POLICY_BF16)
        fetch(static_cast<const bf16*>(x.from));
    else
        fetch(static_cast<const f16*>(x.from));
#pragma unroll
    for (int n = 0; n < 16; ++n) {
        const int i = wave + 4 * n;
        tile[along ? i : lane][along ? lane : i] = static_cast<float>(v[n] * factor);
    }
    __syncthreads();
    const int64_t size = w.size;
    _Float16* turned = w.turned + P.current * 2 * size;
    const int c = threadIdx.x % 8 * 8;
#pragma unroll
    for (int r = threadIdx.x / 8; r < 64; r += 32) {
        h8 hi, lo;
        const auto part = [&](auto number) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                _Float16 high, low;
                split(number(k), high, low);
                hi[k] = high;
                lo[k] = low;
            }
        };
        part([&](int k) { return tile[r][c + k]; });
        const int64_t to = static_cast<int64_t>(row0 + r) * w.N + col0 + c;
        *reinterpret_cast<h8*>(w.rows + to) = hi;
        if (kPlanes16 == 2) *reinterpret_cast<h8*>(w.rows + size + to) = lo;
        part([&](int k) { return tile[c + k][r]; });
        const int64_t back = static_cast<int64_t>(col0 + r) * w.M + row0 + c;
        *reinterpret_cast<h8*>(turned + back) = hi;
        *reinterpret_cast<h8*>(turned + size + back) = lo;
    }
}

enum { kGram, kPoly, kApply, kLast };

// A product's operands lie in LDS in rows of 32 numbers, four pieces of 16 bytes; piece p of row r in place
// p ^ place_of_row(r), so that the lanes that read one piece of 8 or 16 rows at once find them in all banks.
__device__ inline int place_of_row(int row) { return ((row >> 1) ^ (row >> 3)) & 3; }

// From memory to LDS, 16 bytes a lane, without registers between.
template <int kRows>
__device__ inline void stage(const _Float16* from, int64_t stride, _Float16* lds) {
    const int row = threadIdx.x >> 2, piece = (threadIdx.x & 3) ^ place_of_row(row);
    const _Float16* lane = from + row * stride + piece * 8;
    _Float16* to = lds + wave_of_workgroup() * 512;  // (the wave's; its lanes follow each other)
#pragma unroll
    for (int i = 0; i < kRows / 64; ++i)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(lane + i * 64 * stride),
                                         (__attribute__((address_space(3))) void*)(to + i * 64 * kDepth), 16, 0, 0);
}

// A tile of results on its way to memory: its columns one after the other, apart by rows that begin in
// other banks.
template <int kTile>
using Tile = _Float16[kTile][kTile + 8];

// From an array whose rows are the tile's columns.
template <int kTile>
__device__ inline void get_tile(Tile<kTile>& tile, const _Float16* from, int64_t stride) {
    constexpr int kAcross = kTile / 8, kAtOnce = 256 / kAcross, kBatch = kTile / kAtOnce < 8 ? kTile / kAtOnce : 8;
    const int row = threadIdx.x / kAcross, column = threadIdx.x % kAcross * 8;
    for (int i = row; i < kTile; i += kAtOnce * kBatch) {
        h8 x[kBatch];
#pragma unroll
        for (int n = 0; n < kBatch; ++n) x[n] = *reinterpret_cast<const h8*>(from + (i + n * kAtOnce) * stride + column);
#pragma unroll
        for (int n = 0; n < kBatch; ++n) *reinterpret_cast<h8*>(&tile[i + n * kAtOnce][column]) = x[n];
    }
}

// And back.
template <int kTile>
__device__ inline void put_straight(const Tile<kTile>& tile, _Float16* to, int64_t stride) {
    constexpr int kAcross = kTile / 8, kAtOnce = 256 / kAcross;
    const int row = threadIdx.x / kAcross, column = threadIdx.x % kAcross * 8;
#pragma unroll 4
    for (int k = 0; k < kTile / kAtOnce; ++k)
        *reinterpret_cast<h8*>(to + (row + k * kAtOnce) * stride + column) = *reinterpret_cast<const h8*>(&tile[row + k * kAtOnce][column]);
}

// Sixteen rows of the tile (numbers 16 r to 16 r + 15 of its columns), 32 columns from 32 c on: a lane has
// row 16 r + l % 16, columns 32 c + 8 (l / 16) to + 7.
template <int kTile>
__device__ inline h8 turned_eight(const Tile<kTile>& tile, int r, int c) {
    const int lane = threadIdx.x & 63, i = lane & 15;
    const _Float16* from = &tile[32 * c + 8 * (lane >> 4) + (i >> 2)][16 * r + 4 * (i & 3)];
    const u2 a = read_transposed(reinterpret_cast<const uint16_t*>(from)), b = read_transposed(reinterpret_cast<const uint16_t*>(from + 4 * (kTile + 8)));
    return __builtin_bit_cast(h8, u4{a.x, a.y, b.x, b.y});
}

// To an array whose rows are the tile's rows.
template <int kTile>
__device__ inline void put_turned(const Tile<kTile>& tile, _Float16* to, int64_t stride) {
    const int wave = wave_of_workgroup(), lane = threadIdx.x & 63;
#pragma unroll 4
    for (int k = 0; k < kTile / 16 * (kTile / 32) / 4; ++k) {
        const int n = 4 * k + wave, r = n / (kTile / 32), c = n % (kTile / 32);
        *reinterpret_cast<h8*>(to + (16 * r + (lane & 15)) * stride + 32 * c + 8 * (lane >> 4)) = turned_eight<kTile>(tile, r, c);
    }
}

// Eight numbers `step` apart, those of `count` that there are.
__device__ inline void put_eight(_Float16* to, int64_t step, h8 x, int count) {
    if (step == 1 && count >= 8 && reinterpret_cast<uintptr_t>(to) % 16 == 0) {
        *reinterpret_cast<h8*>(to) = x;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < count) to[i * step] = x[i];
    }
}

// Both for results of 16 bits at any address, the first `rows` of the array's rows, `columns` of its columns.
template <int kTile>
__device__ inline void put_straight_to(const Tile<kTile>& tile, _Float16* to, int64_t stride, int rows, int columns) {
    constexpr int kAcross = kTile / 8, kAtOnce = 256 / kAcross;
    const int column = threadIdx.x % kAcross * 8;
    for (int i = threadIdx.x / kAcross; i < rows; i += kAtOnce)
        put_eight(to + i * stride + column, 1, *reinterpret_cast<const h8*>(&tile[i][column]), columns - column);
}

template <int kTile>
__device__ inline void put_turned_to(const Tile<kTile>& tile, _Float16* to, int64_t stride, int64_t step, int rows, int columns) {
    const int wave = wave_of_workgroup(), lane = threadIdx.x & 63;
    for (int n = wave; n < kTile / 16 * (kTile / 32); n += 4) {
        const int row = n / (kTile / 32) * 16 + (lane & 15), column = n % (kTile / 32) * 32 + 8 * (lane >> 4);
        const h8 x = turned_eight<kTile>(tile, n / (kTile / 32), n % (kTile / 32));  // (by all lanes)
        if (row < rows) put_eight(to + row * stride + column * step, step, x, columns - column);
    }
}

// Stages in LDS at once: as many as 128 KB hold, four at most. X's products of tiles of 64 take 32 KB, so that four
// workgroups share a CU and one reads and writes X while others multiply (26 matrices of width 256, two planes: 15.7
// us, with 64 KB 18.0; the symmetric ones, whose tiles the card holds at once, 9.6 with 64 KB, 10.7 with 32).
template <int kTile, int kPlanes16, int kMode>
inline constexpr int kStages = kTile == 64 && (kMode == kApply || kMode == kLast) ? 4 / kPlanes16 : kTile * kPlanes16 <= 256 ? 4 : 2;

// Tiles of one of the three products, kTile x kTile a workgroup, a quarter a wave. Two or four stages of 32
// numbers along the contracted axis, of all planes, are on their way or in LDS; a wave reads the operands of
// the next 16 while it multiplies those it has.
template <int kTile, int kPlanes16, int kMode>
__global__ __launch_bounds__(256, kTile == 256 ? 1 : kTile == 128 && kPlanes16 == 2 ? 1 : 2) void newton_product_kernel(Params P) {
    constexpr int kEach = kTile / 64;          // results of 32 x 32 of a wave, down and across
    constexpr int kLoads = 2 * kPlanes16 * kTile / 64;  // of a lane for a stage
    constexpr int kBuffers = kStages<kTile, kPlanes16, kMode>;
    constexpr bool kSymmetric = kMode == kGram || kMode == kPoly;
    extern __shared__ __attribute__((aligned(16))) char lds_bytes[];
    auto& lds = *reinterpret_cast<_Float16 (*)[kBuffers][2][kPlanes16][kTile * kDepth]>(lds_bytes);
    const int wave = wave_of_workgroup(), lane = threadIdx.x & 63;
    // Workgroups go round the 8 XCDs in turn: each XCD takes a run of tiles.
    const int each = (P.tiles + 7) / 8, at = static_cast<int>(blockIdx.x % 8) * each + static_cast<int>(blockIdx.x / 8);
    if (static_cast<int>(blockIdx.x / 8) >= each || at >= P.tiles) return;
    const int index = matrix_of(P, at);
    const Matrix& x = P.matrix[index];
    const Parts<kPlanes16> w(P, x, kTile);
    int tile_row, tile_col;
    {
        const int n = at - P.first[index];
        if (kSymmetric) {  // tiles (i, j) with i <= j, a column of tiles after the other
            int j = static_cast<int>((sqrtf(8.0f * n + 1.0f) - 1.0f) * 0.5f);
            while ((j + 1) * (j + 2) / 2 <= n) ++j;
            while (j * (j + 1) / 2 > n) --j;
            tile_col = j;
            tile_row = n - j * (j + 1) / 2;
        } else {  // all rows of tiles of a column after the other: P is read again, X once
            const int down = w.M / kTile;
            tile_col = n / down;
            tile_row = n % down;
        }
    }
    const int64_t size = w.size, square = w.square;
    const _Float16* turned = w.turned + P.current * 2 * size;
    const int depth = kMode == kGram ? w.N : w.M;
    const _Float16* left = kMode == kGram ? w.rows : kMode == kPoly ? w.gram : w.poly;
    const _Float16* right = kMode == kGram ? w.rows : kMode == kPoly ? w.gram : turned;
    const int64_t left_plane = kMode == kGram ? size : square, right_plane = kMode == kPoly ? square : size;
    left += static_cast<int64_t>(tile_row) * kTile * depth;
    right += static_cast<int64_t>(tile_col) * kTile * depth;
    const int steps = depth / kDepth;  // (at least two)
    const auto load = [&](int step, int buffer) {
#pragma unroll
        for (int n = 0; n < kPlanes16; ++n) {
            stage<kTile>(left + n * left_plane + step * kDepth, depth, lds[buffer][0][n]);
            stage<kTile>(right + n * right_plane + step * kDepth, depth, lds[buffer][1][n]);
        }
    };
    const int row0 = (wave >> 1) * (kTile / 2), col0 = (wave & 1) * (kTile / 2);  // the wave's in the tile
    using Operand = h8[kPlanes16][kEach];
    const auto read = [&](int buffer, int k, Operand& a, Operand& b) {
        const int piece = ((2 * k + (lane >> 5)) ^ place_of_row(lane & 31)) * 8;
#pragma unroll
        for (int n = 0; n < kPlanes16; ++n)
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                a[n][i] = *reinterpret_cast<const h8*>(&lds[buffer][0][n][(row0 + 32 * i + (lane & 31)) * kDepth + piece]);
                b[n][i] = *reinterpret_cast<const h8*>(&lds[buffer][1][n][(col0 + 32 * i + (lane & 31)) * kDepth + piece]);
            }
    };
    f16x16 sum[kEach][kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
#pragma unroll
        for (int j = 0; j < kEach; ++j)
#pragma unroll
            for (int s = 0; s < 16; ++s) sum[i][j][s] = 0.0f;
    // Rows of results from `from` to `to`, the smallest products first.
    const auto multiply = [&](const Operand& a, const Operand& b, int from, int to) {
#pragma unroll
        for (int term = 2 * (kPlanes16 - 1); term >= 0; --term)
#pragma unroll
            for (int i = from; i < to; ++i)
#pragma unroll
                for (int j = 0; j < kEach; ++j)
                    sum[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[term == 2][i], b[term == 1][j], sum[i][j], 0, 0, 0);
    };
    Operand a[2], b[2];
#pragma unroll
    for (int s = 0; s < kBuffers; ++s) load(s < steps ? s : steps - 1, s);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((kBuffers - 1) * kLoads) : "memory");
    read(0, 0, a[0], b[0]);
    for (int step = 0; step < steps; ++step) {
        multiply(a[0], b[0], 0, 1);  // (these operands have come: nothing else is waited for)
        __builtin_amdgcn_sched_barrier(0);
        read(step % kBuffers, 1, a[1], b[1]);
        __builtin_amdgcn_sched_barrier(0);
        multiply(a[0], b[0], 1, kEach);
        __builtin_amdgcn_sched_barrier(0);
        // This stage has been read by all waves (each waits for what it read), the next has come for all;
        // those after it may be on their way. (Past the end the last stage comes again, unused.)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kBuffers - 2) * kLoads) : "memory");
        load(step + kBuffers < steps ? step + kBuffers : steps - 1, step % kBuffers);
        read((step + 1) % kBuffers, 0, a[0], b[0]);
        __builtin_amdgcn_sched_barrier(0);
        multiply(a[1], b[1], 0, kEach);
        __builtin_amdgcn_sched_barrier(0);
    }
    // (nothing comes into LDS any more)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    auto& tile = *reinterpret_cast<Tile<kTile>*>(lds_bytes);
    const int64_t first_row = static_cast<int64_t>(tile_row) * kTile, first_col = static_cast<int64_t>(tile_col) * kTile;
    // A lane has column l % 32 of each 32 x 32, rows 8 q + 4 (l / 32) to + 3: f(their place in the tile, their sums).
    const auto each_four = [&](auto f) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
#pragma unroll
            for (int j = 0; j < kEach; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    f4 v = {sum[i][j][4 * q], sum[i][j][4 * q + 1], sum[i][j][4 * q + 2], sum[i][j][4 * q + 3]};
                    f(row0 + 32 * i + 8 * q + 4 * (lane >> 5), col0 + 32 * j + (lane & 31), v);
#pragma unroll
                    for (int s = 0; s < 4; ++s) sum[i][j][4 * q + s] = v[s];
                }
    };
    // Adds a factor (of each row) times a tile of an array whose rows are the tile's columns.
    const auto add_tile = [&](const _Float16* from, int64_t stride, auto factor) {
        get_tile<kTile>(tile, from + first_col * stride + first_row, stride);
        __syncthreads();
        each_four([&](int row, int col, f4& v) { v += factor(row) * __builtin_convertvector(*reinterpret_cast<const h4*>(&tile[col][row]), f4); });
        __syncthreads();
    };
    // What the sums round to, into the tile; they keep the rest.
    const auto put_rounded = [&] {
        each_four([&](int row, int col, f4& v) {
            const h4 hi = __builtin_convertvector(v, h4);
            *reinterpret_cast<h4*>(&tile[col][row]) = hi;
            v -= __builtin_convertvector(hi, f4);
        });
        __syncthreads();
    };
    if constexpr (kSymmetric) {
        _Float16* to = kMode == kGram ? w.gram : w.poly;
        const float scale = kMode == kGram ? kScaleA / (w.scale * w.scale) : P.c / kScaleA;
        each_four([&](int, int, f4& v) { v *= scale; });
        if constexpr (kMode == kPoly) {
#pragma unroll
            for (int plane = kPlanes16 - 1; plane >= 0; --plane) add_tile(w.gram + plane * square, w.M, [&](int) { return P.b; });
            if (tile_row == tile_col)
                each_four([&](int row, int col, f4& v) {
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        if (row + s == col) {
                            w.diagonal[first_col + col] = P.a + v[s] * (1.0f / kScaleA);
                            v[s] = 0.0f;
                        }
                });
        }
#pragma unroll
        for (int plane = 0; plane < kPlanes16; ++plane) {
            put_rounded();
            put_straight<kTile>(tile, to + plane * square + first_col * w.M + first_row, w.M);
            if (tile_row != tile_col) put_turned<kTile>(tile, to + plane * square + first_row * w.M + first_col, w.M);
            if (plane + 1 < kPlanes16) __syncthreads();
        }
    } else {
        each_four([&](int, int, f4& v) { v *= 1.0f / kScaleA; });
#pragma unroll
        for (int plane = 1; plane >= 0; --plane)
            add_tile(turned + plane * size, w.M, [&](int row) { return *reinterpret_cast<const f4*>(w.diagonal + first_row + row); });
        if constexpr (kMode == kApply) {
            _Float16* next = w.turned + (1 - P.current) * 2 * size;
#pragma unroll
            for (int plane = 0; plane < 2; ++plane) {
                put_rounded();
                put_straight<kTile>(tile, next + plane * size + first_col * w.M + first_row, w.M);
                if (plane < kPlanes16) put_turned<kTile>(tile, w.rows + plane * size + first_row * w.N + first_col, w.N);
                if (plane == 0) __syncthreads();
            }
        } else {
            const float scale = 1.0f / w.scale;
            const int rows = static_cast<int>(x.m - first_row < kTile ? x.m - first_row : kTile);
            const int cols = static_cast<int>(x.n - first_col < kTile ? x.n - first_col : kTile);
            const int64_t down = x.to_stride[0], across = x.to_stride[1], base = first_row * down + first_col * across;
            if (x.to_dtype == NAVI_POLICY_F32) {
                float* to = static_cast<float*>(x.to) + base;
                each_four([&](int row, int col, f4& v) {
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        if (row + s < rows && col < cols) to[(row + s) * down + col * across] = v[s] * scale;
                });
            } else {
                each_four([&](int row, int col, f4& v) {
                    h4 y;
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        y[s] = x.to_dtype == NAVI_POLICY_F16 ? static_cast<_Float16>(v[s] * scale)
                                                              : __builtin_bit_cast(_Float16, static_cast<__bf16>(v[s] * scale));
                    *reinterpret_cast<h4*>(&tile[col][row]) = y;
                });
                __syncthreads();
                _Float16* to = static_cast<_Float16*>(x.to) + base;
                if (down == 1)
                    put_straight_to<kTile>(tile, to, across, cols, rows);
                else
                    put_turned_to<kTile>(tile, to, down, across, rows, cols);
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

// The largest that X's singular values s come to before a step, and b A + c A A in one, whatever X is: at the
// ends of [0, s] and where the polynomials' slopes are zero. No entry is larger. (X's last values are no plane's.)
struct Largest {
    double x, gram, poly;
};

Largest largest_of(double a, double b, double c, int steps) {
    Largest most{1.0, 1.0, 0.0};
    double s = 1.0;  // (|X| <= 1)
    for (int step = 0; step < steps; ++step) {
        const double t = s * s;  // of A
        double poly = std::fabs(b * t + c * t * t), next = std::fabs(s * (a + b * t + c * t * t));
        const double top = -b / (2.0 * c);
        if (top > 0.0 && top < t) poly = std::max(poly, std::fabs(top * (b + c * top)));
        // a + 3 b t + 5 c t^2 = 0 (no difference of numbers that are nearly the same, and c may be 0)
        const double root = 9.0 * b * b - 20.0 * a * c, q = -0.5 * (3.0 * b + std::copysign(std::sqrt(std::max(root, 0.0)), b));
        for (const double at : {q / (5.0 * c), a / q})
            if (root >= 0.0 && at > 0.0 && at < t) next = std::max(next, std::fabs(std::sqrt(at) * (a + b * at + c * at * at)));
        most = {std::max(most.x, s), std::max(most.gram, t), std::max(most.poly, poly)};
        if (!(most.gram < 1e30 && most.poly < 1e30)) break;  // (out of any range, and before it is out of double's)
        s = next;
    }
    return most;
}

constexpr double kLargest = 65504.0 / 1.02;  // of float16; the planes' roundings change singular values by less

// One plane for bfloat16 results, but for matrices with a short side of up to 256: few products, whose errors do
// not average out (6 to 16 parts in 10^4 of the result with one plane, as much as its own rounding), and times that
// the launches are most of (26 matrices of 4 blocks of width 64: 170 us either way; width 256: 204 and 255 with two;
// 98 of 16 blocks: 621 and 880). From 8 blocks of width 512 on two take 1.8 to 2.4 times as long: 976 us and 1734, of 2000
// 15.8 ms and 37.1.
constexpr int64_t kShort = 256;

int planes_of(const navi_orthogonalize_matrix& x) {
    return x.to_dtype == NAVI_POLICY_BF16 && std::min(x.rows, x.cols) > kShort ? 1 : 2;
}

bool takes_part(const navi_orthogonalize_matrix& x, int planes) { return x.rows > 0 && x.cols > 0 && planes_of(x) == planes; }

// The largest tiles that leave every CU one (256 x 256: a CU holds one workgroup, whose waves have twice the
// products for what they read of 128's; 64 for matrices of a small policy), by the matrices of `planes` planes.
int tile_of(const navi_orthogonalize_matrix* x, int count, int planes) {
    for (const int tile : {256, 128}) {
        int64_t tiles = 0;
        for (int i = 0; i < count; ++i)
            if (takes_part(x[i], planes)) tiles += ((x[i].rows + tile - 1) / tile) * ((x[i].cols + tile - 1) / tile);
        if (tiles >= 256) return tile;
    }
    return 64;
}

int64_t bytes_of(const navi_orthogonalize_matrix& x, int tile, int planes) {
    const int64_t M = rounded(std::min(x.rows, x.cols), tile), N = rounded(std::max(x.rows, x.cols), tile);
    return 8 * kNormBlocks + 4 * M + 2 * (planes * M * N + 4 * M * N + 2 * planes * M * M);  // (a multiple of 256: M is one of 64)
}

// Matrices of `planes` planes from `at` on that go together: as many as a launch names and the workspace holds.
int group_end(const navi_orthogonalize_matrix* x, int count, int at, int planes, int tile, int64_t* bytes) {
    int64_t total = 0;
    int end = at, named = 0;
    for (; end < count && named < kMatrices; ++end) {
        if (!takes_part(x[end], planes)) continue;
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

template <int kTile, int kPlanes16, int kMode>
int launch(const Params& P, hipStream_t stream) {
    constexpr int staged = kStages<kTile, kPlanes16, kMode> * 2 * kPlanes16 * kTile * kDepth * sizeof(_Float16), tile = sizeof(Tile<kTile>), lds = staged > tile ? staged : tile;
    const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(newton_product_kernel<kTile, kPlanes16, kMode>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (err != hipSuccess) return set_error(NAVI_POLICY_E_LAUNCH, "navi_orthogonalize: %s", hipGetErrorString(err));
    hipLaunchKernelGGL((newton_product_kernel<kTile, kPlanes16, kMode>), dim3((P.tiles + 7) / 8 * 8), dim3(256), lds, stream, P);
    return launched();
}

template <int kTile, int kPlanes16>
int run_group(Params& P, int pieces, int steps, hipStream_t stream) {
    hipLaunchKernelGGL(newton_squares_kernel, dim3(kNormBlocks, P.count), dim3(256), 0, stream, P);
    hipLaunchKernelGGL(newton_begin_kernel<kPlanes16>, dim3(pieces), dim3(256), 0, stream, P);
    Params S = P, X = P;  // tiles of the symmetric products, and of the other
    S.tiles = X.tiles = 0;
    for (int i = 0; i < P.count; ++i) {
        const int down = (P.matrix[i].m + kTile - 1) / kTile, across = (P.matrix[i].n + kTile - 1) / kTile;
        S.first[i] = S.tiles;
        X.first[i] = X.tiles;
        S.tiles += down * (down + 1) / 2;
        X.tiles += down * across;
    }
    for (int step = 0; step < steps; ++step) {
        S.current = X.current = step & 1;
        int code = launch<kTile, kPlanes16, kGram>(S, stream);
        if (code == NAVI_POLICY_OK) code = launch<kTile, kPlanes16, kPoly>(S, stream);
        if (code == NAVI_POLICY_OK)
            code = step + 1 < steps ? launch<kTile, kPlanes16, kApply>(X, stream) : launch<kTile, kPlanes16, kLast>(X, stream);
        if (code != NAVI_POLICY_OK) return code;
    }
    return launched();
}

// A call whose arguments have been looked over.
struct Matrices {
    const navi_orthogonalize_matrix* given;
    int count, steps;
    float a, b, c, eps;
    int most_scale;
    char* workspace;
    hipStream_t stream;

    // The matrices of `planes` planes, group after group.
    int run(int planes) const {
        const int tile = tile_of(given, count, planes);
        for (int at = 0; at < count;) {
            int64_t bytes;
            const int end = group_end(given, count, at, planes, tile, &bytes);
            if (bytes > 0 && (!workspace || !aligned(256, workspace)))
                return set_error(NAVI_POLICY_E_ARG, "workspace must be non-null and 256-byte aligned");
            Params P{};
            P.a = a;
            P.b = b;
            P.c = c;
            P.eps = eps;
            P.workspace = workspace;
            P.tile = tile;
            int pieces = 0;
            int64_t place = 0;
            for (; at < end; ++at) {
                if (!takes_part(given[at], planes)) continue;
                P.first[P.count] = pieces;
                P.matrix[P.count] = matrix_at(given[at], place);
                const Matrix& x = P.matrix[P.count++];
                pieces += static_cast<int>(rounded(x.m, tile) / 64 * (rounded(x.n, tile) / 64));
                place += bytes_of(given[at], tile, planes);
            }
            if (P.count == 0) continue;
            int code;
            if (tile == 256)
                code = planes == 1 ? run_group<256, 1>(P, pieces, steps, stream) : run_group<256, 2>(P, pieces, steps, stream);
            else if (tile == 128)
                code = planes == 1 ? run_group<128, 1>(P, pieces, steps, stream) : run_group<128, 2>(P, pieces, steps, stream);
            else
                code = planes == 1 ? run_group<64, 1>(P, pieces, steps, stream) : run_group<64, 2>(P, pieces, steps, stream);
            if (code != NAVI_POLICY_OK) return code;
        }
        return NAVI_POLICY_OK;
    }

    Matrix matrix_at(const navi_orthogonalize_matrix& from, int64_t place) const {
        Matrix x{};
        const int turn = from.rows > from.cols;  // X is the transpose
        x.from = from.from;
        x.to = from.to;
        x.turned = from.from_stride[1 ^ turn] != 1;
        x.from_line = from.from_stride[x.turned ? 1 ^ turn : turn];
        for (int k = 0; k < 2; ++k) x.to_stride[k] = from.to_stride[k ^ turn];
        x.m = static_cast<int32_t>(turn ? from.cols : from.rows);
        x.n = static_cast<int32_t>(turn ? from.rows : from.cols);
        x.place = static_cast<uint32_t>(place / 256);
        x.from_dtype = static_cast<int8_t>(from.from_dtype);
        x.to_dtype = static_cast<int8_t>(from.to_dtype);
        x.scale = static_cast<int8_t>(std::min(static_cast<int>(std::lround(0.5 * std::log2(static_cast<double>(x.n)))) + 6, most_scale));
        return x;
    }
};

}  // namespace
}  // namespace navi_policy

extern "C" int64_t navi_orthogonalize_workspace(int32_t count, const navi_orthogonalize_matrix* matrices) {
    using namespace navi_policy;
    const int code = check(matrices, count);
    if (code != NAVI_POLICY_OK) return code;
    int64_t most = 0;
    for (const int planes : {1, 2}) {
        const int tile = tile_of(matrices, count, planes);
        for (int at = 0; at < count;) {
            int64_t bytes;
            at = group_end(matrices, count, at, planes, tile, &bytes);
            most = std::max(most, bytes);
        }
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
    const Largest most = largest_of(a, b, c, steps);
    if (!(kScaleA * most.gram <= kLargest && kScaleA * most.poly <= kLargest))
        return set_error(NAVI_POLICY_E_ARG, "the factors take singular values s past 7.9 between steps, or b s^2 + c s^4 past 62");
    const int most_scale = static_cast<int>(std::floor(std::log2(kLargest / most.x)));
    const int shared = check_apart(matrices, count);
    if (shared != NAVI_POLICY_OK) return shared;
    Matrices call{matrices, count, steps, a, b, c, eps, most_scale, static_cast<char*>(workspace), as_stream(stream)};
    for (const int planes : {1, 2}) {
        const int code = call.run(planes);
        if (code != NAVI_POLICY_OK) return code;
    }
    return NAVI_POLICY_OK;
}
