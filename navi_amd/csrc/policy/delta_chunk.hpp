// delta_chunk.hpp — what the chunked kernels of the gated delta rule share: a chunk's gates,
// its rows in LDS and its two triangles.
//
// Mathematics. Inside a chunk of 64 tokens with the state S before it, G_i the sum of g up to
// token i (from the chunk's first on), D_ij = exp(G_i - G_j) for i >= j of one episode and 0
// for two, E_i = exp(G_i) as long as no episode has started, F_i = exp(G_last - G_i) where
// none starts after i, the updates u of all tokens solve one unit lower triangular system:
//
//     (I + A) u = r,  A_ij = D_ij (k_i . k_j) beta_j  (i > j),   r_i = v_i - E_i S^T k_i
//     o_i = scale E_i S^T q_i + sum_j P_ij u_j,  P_ij = scale D_ij (q_i . k_j) beta_j  (i >= j)
//     S  <- E_last S + sum_i k_i (F_i beta_i u_i)^T
//
// and with X = (I + A)^-1, u = X r. X and P are the chunk's two triangles; they do not depend
// on S or v. (k_i . k_j is close to 1 between frames that look alike, so X comes from
// substitution in 16 x 16 blocks, whose entries stay bounded, not from powers of A.)
//
// G is summed in float64 and kept as a float and its rest: D needs differences of sums that
// may be large, to float32's precision.
#pragma once

#include <cstddef>

#include "policy_common.hpp"

namespace navi_policy {

constexpr int kChunk = NAVI_POLICY_CHUNK;
constexpr int kTiles = 10;         // 16 x 16 tiles of a lower triangle of 64
constexpr float kStart = -1e5f;    // a decay below exp(kStart) is the start of an episode
constexpr float kLog2E = 1.44269504088896340736f;

struct RuleParams {
    navi_delta_rule r;
    navi_delta_gradients d;
    int32_t group;        // value heads of a key head
    int32_t n_chunks;
    int32_t wide_qk, wide_v, wide_do;  // rows that 16-byte loads can read
    int32_t wide_out;     // rows of four-number stores
    int32_t wide_state;   // rows of states and updates that 16-byte accesses can
    float* dstates;       // [env, head][chunks - 1][K][V] gradient of the state after each chunk but the last
    float* rgrads;        // [env, head][steps][V] gradient of r
    // Long sequences of few heads are walked in segments of chunks (delta_join_kernel)
    int32_t n_segments;
    int32_t blocks, summary_blocks;  // of 64 columns: of V, and of V and the unit matrix
    float* segment_states;    // [env, head][n_segments - 1][K][V]
    float* segment_matrices;  // [env, head][n_segments - 1][K][K]
    float* dq_heads;      // [env][step][value head][K] where heads are shared
    float* dk_heads;
};

// Tile (i, j), j <= i, of a triangle; a tile is 64 lanes of four numbers as products leave
// them: slot l has column l % 16, rows 4 (l / 16) to 4 (l / 16) + 3.
__device__ constexpr int tile_of(int i, int j) { return i * (i + 1) / 2 + j; }

template <int N>
using Triangle = uint16_t[kTiles][N][64][4];  // its planes

// What delta_triangles_kernel leaves of a chunk for the kernels that walk the chunks.
struct ChunkMatrices {
    f4 x[kTiles][64], p[kTiles][64];
    float e[kChunk], fb[kChunk];  // E, and F beta
};
static_assert(sizeof(ChunkMatrices) == 4 * NAVI_POLICY_CHUNK_MATRICES, "the header's size");

struct ChunkGates {
    float hi[kChunk], lo[kChunk];  // G
    float e[kChunk], f[kChunk], beta[kChunk];
    int32_t episode[kChunk];       // episodes started in the chunk so far
};

// Rows in LDS hold every 32 columns in the order in which two tiles of a product's result hold a
// column: 4 g to 4 g + 3 of the first tile, then of the second, for g = 0 to 3. A lane's part
// (g) of an operand is then 16 adjacent bytes, whether the other operand is such a result or
// rows like these.
__device__ inline int place_of(int column) {
    return (column & ~31) + ((column & 12) << 1) + ((column & 16) >> 2) + (column & 3);
}

// Eight columns from a multiple of eight on, to their places.
template <int kPitch>
__device__ inline void put_columns(uint16_t (&row)[kPitch], int column, u4 x) {
    uint16_t* to = &row[place_of(column)];
    *reinterpret_cast<u2*>(to) = u2{x[0], x[1]};
    *reinterpret_cast<u2*>(to + 8) = u2{x[2], x[3]};
}

template <class E, int KP>
struct ChunkRows {
    static constexpr int kPitch = KP + 8;
    uint16_t q[kPlanes<E>][kChunk][kPitch];
    uint16_t k[kPlanes<E>][kChunk][kPitch];
};

template <class E>
__device__ inline const E* at(const void* base, const int64_t (&stride)[3], int64_t env, int64_t step, int64_t head) {
    return static_cast<const E*>(base) + env * stride[0] + step * stride[1] + head * stride[2];
}

// Eight elements of a row as floats, those from `valid` on as zeros.
template <class E>
__device__ inline void load8(const E* row, int valid, bool wide, float (&x)[8]) {
    if (wide && valid >= 8) {
        union {
            u4 words[sizeof(E) == 4 ? 2 : 1];
            E elements[8];
        } got;
        got.words[0] = *reinterpret_cast<const u4*>(row);
        if constexpr (sizeof(E) == 4) got.words[1] = *reinterpret_cast<const u4*>(row + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_float(got.elements[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < valid ? to_float(row[i]) : 0.0f;
    }
}

// The chunk's queries and keys into LDS, zeros past the last token and the key dimension.
template <class E, int KP>
__device__ inline void load_rows(const RuleParams& P, ChunkRows<E, KP>& rows, int64_t env, int head, int64_t t0,
                                 int tokens) {
    constexpr int kPieces = KP / 8;
    const int key_head = head / P.group;
#pragma unroll 1
    for (int piece = threadIdx.x; piece < kChunk * kPieces; piece += blockDim.x) {
        const int t = piece / kPieces, c = piece % kPieces * 8;
        const int valid = t < tokens ? P.r.key_dim - c : 0;
        float x[8];
        u4 plane[kPlanes<E>];
        load8(at<E>(P.r.q, P.r.q_stride, env, t0 + (t < tokens ? t : 0), key_head) + c, valid, P.wide_qk, x);
        split8(x, plane);
#pragma unroll
        for (int n = 0; n < kPlanes<E>; ++n) put_columns(rows.q[n][t], c, plane[n]);
        load8(at<E>(P.r.k, P.r.k_stride, env, t0 + (t < tokens ? t : 0), key_head) + c, valid, P.wide_qk, x);
        split8(x, plane);
#pragma unroll
        for (int n = 0; n < kPlanes<E>; ++n) put_columns(rows.k[n][t], c, plane[n]);
    }
}

// A chunk's gates, a token a lane of one wave: read, and summed into LDS.
struct GatesFetch {
    float g, beta;
    int start;

    __device__ void fetch(const RuleParams& P, int64_t env, int head, int64_t t0, int tokens) {
        const int lane = threadIdx.x & 63;
        g = beta = 0.0f;
        start = 0;
        if (lane < tokens) {
            g = *at<float>(P.r.g, P.r.g_stride, env, t0 + lane, head);
            beta = *at<float>(P.r.beta, P.r.beta_stride, env, t0 + lane, head);
            if (P.r.starts) start = P.r.starts[env * P.r.starts_stride[0] + (t0 + lane) * P.r.starts_stride[1]];
        }
    }

    __device__ void put(ChunkGates& gates) const {
        const int lane = threadIdx.x & 63;
        const bool starts = start != 0 || g < kStart;
        double sum = starts ? 0.0 : static_cast<double>(g);
        const uint64_t all = __ballot(starts);
        const int episode = __popcll(all << (63 - lane)), last_episode = __popcll(all);
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double s = __shfl_up(sum, d);
            sum += lane >= d ? s : 0.0;
        }
        const float hi = static_cast<float>(sum), lo = static_cast<float>(sum - hi);
        const double last = __shfl(sum, 63);
        gates.hi[lane] = hi;
        gates.lo[lane] = lo;
        gates.e[lane] = episode == 0 ? expf(hi) * (1.0f + lo) : 0.0f;
        gates.f[lane] = episode == last_episode ? expf(static_cast<float>(last - sum)) : 0.0f;
        gates.beta[lane] = beta;
        gates.episode[lane] = episode;
    }
};

__device__ inline float decay(const ChunkGates& gates, int i, float hi_j, float lo_j, int episode_j) {
    const float d = (gates.hi[i] - hi_j) + (gates.lo[i] - lo_j);
    return gates.episode[i] == episode_j ? __builtin_amdgcn_exp2f(d * kLog2E) : 0.0f;
}

// Operands of products from rows in LDS: rows row0 to row0 + 15, the lane's part of columns 32 m
// to 32 m + 31 (the other operand: a result's two tiles 2 m, or rows read in the same way);
template <int N, int kPitch>
__device__ inline void operand_rows(int lane, const uint16_t (&rows)[N][kChunk][kPitch], int row0, int m, u4 (&x)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n)
        x[n] = *reinterpret_cast<const u4*>(&rows[n][row0 + (lane & 15)][32 * m + 8 * (lane >> 4)]);
}

// and columns 16 c to 16 c + 15 as the operand's rows, tokens 32 m to 32 m + 31 contracted in
// the order of results.
template <int N, int kPitch>
__device__ inline void operand_columns(int lane, const uint16_t (&rows)[N][kChunk][kPitch], int c, int m, u4 (&x)[N]) {
    const int i = lane & 15;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const uint16_t* from = &rows[n][32 * m + 4 * (lane >> 4) + (i >> 2)][32 * (c >> 1) + 4 * (c & 1) + 8 * (i & 3)];
        const u2 a = read_transposed(from), b = read_transposed(from + 16 * kPitch);
        x[n] = u4{a.x, a.y, b.x, b.y};
    }
}

// A triangle's rows 16 i to 16 i + 15, columns 32 m to 32 m + 31 (32 m <= 16 i) as an operand
// whose contracted axis is in the order of results;
template <int N>
__device__ inline void operand_triangle(int lane, const Triangle<N>& t, int i, int m, u4 (&x)[N]) {
    const int l = lane & 15;
    const int slot = (l & 3) * 16 + 4 * (lane >> 4) + (l >> 2);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const u2 a = read_transposed(t[tile_of(i, 2 * m)][n][slot]);
        const u2 b = 2 * m + 1 <= i ? read_transposed(t[tile_of(i, 2 * m + 1)][n][slot]) : u2{0, 0};
        x[n] = u4{a.x, a.y, b.x, b.y};
    }
}

// and of its transpose, rows 16 j on, columns 32 m on (16 j < 32 m + 32).
template <int N>
__device__ inline void operand_transpose(int lane, const Triangle<N>& t, int j, int m, u4 (&x)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const u2 a = 2 * m >= j ? *reinterpret_cast<const u2*>(t[tile_of(2 * m, j)][n][lane]) : u2{0, 0};
        const u2 b = *reinterpret_cast<const u2*>(t[tile_of(2 * m + 1, j)][n][lane]);
        x[n] = u4{a.x, a.y, b.x, b.y};
    }
}

template <int N>
__device__ inline void store_slot(Triangle<N>& t, int tile, int slot, f4 x) {
    uint32_t a[N], b[N];
    split_pair<N>(x[0], x[1], a);
    split_pair<N>(x[2], x[3], b);
#pragma unroll
    for (int n = 0; n < N; ++n) *reinterpret_cast<u2*>(t[tile][n][slot]) = u2{a[n], b[n]};
}

__device__ constexpr int tile_row(int tile) { return tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3; }

// The inverse of I + the strictly lower triangle in `a`, in its place (unit diagonal and zeros
// above it within diagonal tiles; tiles above are not touched). All threads of the workgroup.
__device__ inline void invert_triangle(float (&a)[kChunk][kChunk + 4], int wave, int waves) {
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    // Diagonal tiles by forward substitution, a column a lane, four tiles in a wave.
    if (wave == 0) {
        const int at = 16 * g;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = i == col ? 1.0f : 0.0f;
#pragma unroll
            for (int m = 0; m < i; m += 4) {
                const f4 row = *reinterpret_cast<const f4*>(&a[at + i][at + m]);
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    if (m + n < i) s -= row[n] * x[m + n];
            }
            x[i] = s;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) a[at + i][at + col] = x[i];
    }
    __syncthreads();
    // The tile below two diagonal ones: -X22 A21 X11.
    for (int pair = wave; pair < 2; pair += waves) {
        const int lo = 32 * pair, hi = lo + 16;
        const f4 below = *reinterpret_cast<const f4*>(&a[hi + col][lo + 4 * g]);
        const f4 left = *reinterpret_cast<const f4*>(&a[hi + col][hi + 4 * g]);
        f4 t = {0, 0, 0, 0}, x = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < 4; ++s) t = mfma_f32(below[s], a[lo + 4 * g + s][lo + col], t);
#pragma unroll
        for (int s = 0; s < 4; ++s) x = mfma_f32(left[s], t[s], x);
#pragma unroll
        for (int s = 0; s < 4; ++s) a[hi + 4 * g + s][lo + col] = -x[s];
    }
    __syncthreads();
    // The four tiles below those pairs, by columns of tiles.
    f4 x[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        if (j % waves != wave) continue;
        f4 t[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            t[i] = f4{0, 0, 0, 0};
#pragma unroll
            for (int m = j; m < 2; ++m) {
                const f4 below = *reinterpret_cast<const f4*>(&a[32 + 16 * i + col][16 * m + 4 * g]);
#pragma unroll
                for (int s = 0; s < 4; ++s) t[i] = mfma_f32(below[s], a[16 * m + 4 * g + s][16 * j + col], t[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[j][i] = f4{0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m <= i; ++m) {
                const f4 left = *reinterpret_cast<const f4*>(&a[32 + 16 * i + col][32 + 16 * m + 4 * g]);
#pragma unroll
                for (int s = 0; s < 4; ++s) x[j][i] = mfma_f32(left[s], t[m][s], x[j][i]);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (j % waves == wave)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int s = 0; s < 4; ++s) a[32 + 16 * i + 4 * g + s][16 * j + col] = -x[j][i][s];
    __syncthreads();
}

// A chunk's rows, then (when no wave needs them) its triangle, in the same memory: more
// workgroups of a CU hide each other's waits.
template <class E, int KP>
struct TriangleLds {
    union {
        ChunkRows<E, KP> rows;
        float work[kChunk][kChunk + 4];  // A, then X
    };
    ChunkGates gates;
};

// X and P of the chunk whose rows and gates are in LDS, by the four waves of a workgroup, three
// tiles each (the last of the ten thrice, with the same numbers: no branch stands between tiles).
template <class E, int KP>
__device__ inline void make_triangles(TriangleLds<E, KP>& lds, ChunkMatrices& to, float scale, int wave) {
    constexpr int N = kPlanes<E>, kEach = (kTiles + 3) / 4;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    f4 a[kEach];
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
        const int tile = wave + 4 * n < kTiles ? wave + 4 * n : kTiles - 1;
        const int i = tile_row(tile), j = tile - tile_of(i, 0);
        f4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < KP / 32; ++m) {
            u4 ki[N], qi[N], kj[N];
            operand_rows(lane, lds.rows.k, 16 * j, m, kj);
            operand_rows(lane, lds.rows.k, 16 * i, m, ki);
            kk = mma(ki, kj, kk);
            operand_rows(lane, lds.rows.q, 16 * i, m, qi);
            qk = mma(qi, kj, qk);
        }
        const int column = 16 * j + col;
        const float hi = lds.gates.hi[column], lo = lds.gates.lo[column], beta = lds.gates.beta[column];
        const int episode = lds.gates.episode[column];
        f4 p;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int row = 16 * i + 4 * g + s;
            const float d = row >= column ? decay(lds.gates, row, hi, lo, episode) * beta : 0.0f;
            a[n][s] = row > column ? d * kk[s] : 0.0f;
            p[s] = scale * d * qk[s];
        }
        to.p[tile][lane] = p;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
        const int tile = wave + 4 * n < kTiles ? wave + 4 * n : kTiles - 1;
        const int i = tile_row(tile), j = tile - tile_of(i, 0);
#pragma unroll
        for (int s = 0; s < 4; ++s) lds.work[16 * i + 4 * g + s][16 * j + col] = a[n][s];
    }
    __syncthreads();
    invert_triangle(lds.work, wave, 4);
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
        const int tile = wave + 4 * n < kTiles ? wave + 4 * n : kTiles - 1;
        const int i = tile_row(tile), j = tile - tile_of(i, 0);
        f4 x;
#pragma unroll
        for (int s = 0; s < 4; ++s) x[s] = lds.work[16 * i + 4 * g + s][16 * j + col];
        to.x[tile][lane] = x;
    }
}

// A chunk's inputs on their way: read into registers while the chunk before it is computed,
// put into LDS once that is done with it. (Rows that 16-byte loads cannot read come then.)
// Without kAll, keys and X alone: what the state needs of a chunk whose outputs nobody asks for.
template <class E, int KP, int kThreads, bool kAll>
struct ChunkFetch {
    static constexpr int kPieces = kChunk * KP / 8 / kThreads;                  // of rows of q, and of k
    static constexpr int kSlots = ((kAll ? 2 : 1) * kTiles * 64 + kThreads - 1) / kThreads;  // of X and P
    static constexpr int kWords = sizeof(E) == 4 ? 2 : 1;
    u4 q[kAll ? kPieces : 1][kWords], k[kPieces][kWords];
    f4 slot[kSlots];
    float gate;

    __device__ void fetch(const RuleParams& P, const ChunkMatrices& from, int64_t env, int head, int64_t t0, int tokens) {
        if (P.wide_qk) {
            const int key_head = head / P.group;
            if constexpr (kAll)
                fetch_rows(at<E>(P.r.q, P.r.q_stride, env, t0, key_head), static_cast<uint32_t>(P.r.q_stride[1]) * sizeof(E),
                           P.r.key_dim, tokens, q);
            fetch_rows(at<E>(P.r.k, P.r.k_stride, env, t0, key_head), static_cast<uint32_t>(P.r.k_stride[1]) * sizeof(E),
                       P.r.key_dim, tokens, k);
        }
        const Buffer matrices = buffer_of(&from, sizeof from);
#pragma unroll
        for (int i = 0; i < kSlots; ++i)  // (P follows X, the gates P)
            slot[i] = __builtin_bit_cast(f4, buffer_load16(matrices, 16 * (threadIdx.x + i * kThreads)));
        gate = buffer_load<float>(matrices, threadIdx.x < 2 * kChunk ? offsetof(ChunkMatrices, e) + 4 * threadIdx.x : kOutside);
    }

    __device__ static void fetch_rows(const E* base, uint32_t row_bytes, int dim, int tokens, u4 (&to)[kPieces][kWords]) {
        const Buffer rows = buffer_of(base, tokens > 0 ? (tokens - 1) * row_bytes + dim * sizeof(E) : 0);
        constexpr int kAcross = KP / 8, kDown = kThreads / kAcross;  // pieces of a row; rows at once
        const int t = threadIdx.x / kAcross, c = threadIdx.x % kAcross * 8;
        const uint32_t lane = c < dim ? t * row_bytes + c * sizeof(E) : kOutside;
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
            for (int w = 0; w < kWords; ++w) to[i][w] = buffer_load16(rows, lane + i * kDown * row_bytes + 16 * w);
    }

    __device__ static void put_piece(uint16_t (&rows)[kPlanes<E>][kChunk][KP + 8], int t, int c, const u4 (&from)[kWords]) {
        if constexpr (kPlanes<E> == 1) {
            put_columns(rows[0][t], c, from[0]);
        } else {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (kWords == 2)
                    x[i] = float_of(from[i / 4][i % 4]);
                else
                    x[i] = to_float(__builtin_bit_cast(f16, static_cast<uint16_t>(from[0][i / 2] >> (16 * (i % 2)))));
            }
            u4 plane[kPlanes<E>];
            split8(x, plane);
#pragma unroll
            for (int n = 0; n < kPlanes<E>; ++n) put_columns(rows[n][t], c, plane[n]);
        }
    }

    // The rows alone, at once.
    __device__ static void load(const RuleParams& P, ChunkRows<E, KP>& rows, int64_t env, int head, int64_t t0, int tokens) {
        if (!P.wide_qk) {
            load_rows<E, KP>(P, rows, env, head, t0, tokens);
            return;
        }
        u4 q[kPieces][kWords], k[kPieces][kWords];
        const int key_head = head / P.group;
        fetch_rows(at<E>(P.r.q, P.r.q_stride, env, t0, key_head), static_cast<uint32_t>(P.r.q_stride[1]) * sizeof(E),
                   P.r.key_dim, tokens, q);
        fetch_rows(at<E>(P.r.k, P.r.k_stride, env, t0, key_head), static_cast<uint32_t>(P.r.k_stride[1]) * sizeof(E),
                   P.r.key_dim, tokens, k);
        put_rows(rows, q, k);
    }

    __device__ static void put_rows(ChunkRows<E, KP>& rows, const u4 (&q)[kAll ? kPieces : 1][kWords], const u4 (&k)[kPieces][kWords]) {
        constexpr int kAcross = KP / 8, kDown = kThreads / kAcross;
        const int t = threadIdx.x / kAcross, c = threadIdx.x % kAcross * 8;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if constexpr (kAll) put_piece(rows.q, t + i * kDown, c, q[i]);
            put_piece(rows.k, t + i * kDown, c, k[i]);
        }
    }

    __device__ void put(const RuleParams& P, ChunkRows<E, KP>& rows, Triangle<3>& x, Triangle<3>& p, float (&gates)[2][kChunk],
                        int64_t env, int head, int64_t t0, int tokens) const {
        if (P.wide_qk) {
            put_rows(rows, q, k);
        } else {
            load_rows<E, KP>(P, rows, env, head, t0, tokens);
        }
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            const int n = threadIdx.x + i * kThreads;
            if (n < kTiles * 64)
                store_slot<3>(x, n >> 6, n & 63, slot[i]);
            else if (kAll && n < 2 * kTiles * 64)
                store_slot<3>(p, (n >> 6) - kTiles, n & 63, slot[i]);
        }
        if (threadIdx.x < 2 * kChunk) (&gates[0][0])[threadIdx.x] = gate;
    }
};

}  // namespace navi_policy
