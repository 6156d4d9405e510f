// selective_scan.hip — a selective state space scan over chunks of 64 tokens, and its gradients.
//
// Per env and head, with beta_t = softplus(dt_t + dt_bias), g_t = beta_t a (no decay but a cleared
// state at a token that begins an episode), the state S a state_dim x head_dim matrix:
//
//     S <- exp(g_t) S + beta_t b_t x_t^T,    y_t = S^T c_t + d x_t
//
// Inside a chunk with the state S before it, G_i the sum of g up to token i, D_ij = exp(G_i - G_j)
// for j < i of one episode and 0 for two, E_i = exp(G_i) as long as no episode has begun, F_i =
// exp(G_last - G_i) where none begins after i:
//
//     y_i = E_i S^T c_i + sum over j < i of D_ij (c_i . b_j) beta_j x_j + (beta_i (c_i . b_i) + d) x_i
//     S  <- E_last S + sum_i b_i (F_i beta_i x_i)^T
//
// The gradients are three scans of the same form, with the queries, keys and values (c, b, x) in other
// roles and the last two in the opposite order (the decay then is that of the token after, and beta
// multiplies the results instead of the values):
//
//     dc: queries dy, keys x, values b, forwards, the same state transposed
//     dx: queries b, keys c, values dy, backwards from the gradient of the last state
//     db: queries x, keys dy, values c, backwards, that state transposed
//
// The gradient of g_t collects what passes from before t to t and after, W_ij = D_ij beta_j (c_i . b_j)
// (dy_i . x_j) from token j to token i of a chunk and what the states carry:
//
//     dg_t = sum over j < t <= i of W_ij + sum over i >= t of rho_i + sum over j < t of kappa_j + E_last <S, dS>
//     rho_i = E_i c_i . (S^T's dy_i),   kappa_j = F_j beta_j x_j . (dS^T b_j)
//
// with the state S before the chunk and the gradient dS of that after it. (dg is also a sum to the
// sequence's end of c . dc - beta b . db, which needs no state; but the two differ by less than float32
// leaves of them after some hundred tokens: 3e-4 of da at 4096.) The dc scan leaves S for the
// db scan, which holds dS in the same layout, where a chunk has both.
//
// The matrix cores' float32 sums of 16-bit products lie below the exact ones by about a hundredth of
// their rounding, whatever their sign (measured: -0.004 to -0.009 of 2^-24 of the sum's size where
// small products join a large sum, against a spread of 0.85; none for products of float32). That is
// nothing in one number, but gradients of a and dt_bias add up a hundred thousand such numbers of both
// signs: 1e-4 of da for 1024 x 128 steps. So keys are negated in every other chunk and environment,
// and all that follows from them until it is used: the errors cancel.
//
// A workgroup walks the chunks of 64 columns of a head's state: long walks of few heads are cut into segments
// (what each makes of zeros, then their join, then all at once), whose chain is what bounds them (1 x 16384 tokens
// of 16 heads of 128 x 64: 35 + 8 + 77 us, 16 times the floor of memory). With many walks no single unit is full:
// 1024 x 128 steps of 4 heads of 64 x 64 in bfloat16 take 95 us forward for 168 MB, the vector units 46% busy with
// splits, factors and conversions, the matrix cores 13%, LDS 31%; the three scans back 340 us (three times 95 and
// the float32 gradients of b and c that each head leaves: 268 MB), the gates' gradients 66. More or fewer workgroups
// a CU than the registers allow without spills change nothing (forward 93 with two) or cost (130 with four).
//
// G is summed in float64 and kept as a float and its rest (delta_chunk.hpp has the layouts of rows
// and triangles in LDS, policy_common.hpp the planes that products run on).
#include <algorithm>
#include <climits>

#include "delta_chunk.hpp"

namespace navi_policy {
namespace {

constexpr int kColumns = 64;  // of the state that a workgroup holds, 16 a wave

struct Operand {
    const void* p;
    int64_t stride[3];  // env, step, head
    int32_t share;      // heads of the scan that read one of its heads
    int32_t wide;       // rows that 16-byte loads can read
};

// What a scan takes and leaves.
struct Role {
    Operand q, k, v, z;
    int32_t K, V;          // numbers of a query or key, of a value
    int32_t blocks;        // of kColumns columns
    int32_t reverse;       // from the last token to the first, beta on the results
    int32_t skip;          // d times the values is added
    int32_t wide_out;
    int32_t state_row, state_column;  // strides of the states outside
    void* out;             // [env][step][head][V], of the inputs' type
    float* out_heads;      // instead, in float32
    const float* from;     // the state before the first token, or NULL for zeros
    float* to;             // the state after the last, or NULL
    float* state_dots;     // [env, head][blocks][steps] z . (what the state adds to a result), or NULL
    float* dots;           // likewise, of what all other tokens do, or NULL
    float* keep_states;    // [env, head][chunks][blocks][4][KP / 16][64][4] the state before a chunk, written,
    const float* other_states;  // read, and multiplied with this scan's into
    float* through;        // [env, head][chunks][blocks][4] (chunks in the order of tokens)
    int32_t keep_from, keep_to;  // chunks that need it
    float* segment_states; // [env, head][n_segments - 1][K][V]
    float* segment_keeps;  // [env, head][n_segments]
};

struct ScanParams {
    int64_t envs, steps;
    int32_t heads, group;  // heads of a group
    int32_t n_chunks, n_segments;
    const float* dt;
    int64_t dt_stride[3];
    const float* a;
    const float* d;
    const float* dt_bias;
    const uint8_t* starts;
    int64_t starts_stride[2];
    Role role[3];
};

// A lane's neighbours by moves within the vector unit: lane l - n of its row of 16, or (143 and 142) the
// last lane of the row or the half before it; 0 where there is none.
template <int kControl, int kRows = 15>
__device__ inline double lane_before(double x) {
    const u2 w = __builtin_bit_cast(u2, x);
    return __builtin_bit_cast(double, u2{static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(w.x), kControl, kRows, 15, false)),
                                         static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(w.y), kControl, kRows, 15, false))});
}

// Sums over the lanes up to each.
__device__ inline double sum_up(double x) {
    x += lane_before<0x111>(x);
    x += lane_before<0x112>(x);
    x += lane_before<0x114>(x);
    x += lane_before<0x118>(x);
    x += lane_before<0x142, 10>(x);
    x += lane_before<0x143, 12>(x);
    return x;
}

__device__ inline double of_lane(double x, int lane) {
    const u2 w = __builtin_bit_cast(u2, x);
    return __builtin_bit_cast(double, u2{static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(w.x), lane)),
                                         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(w.y), lane))});
}

__device__ inline float softplus(float z) { return fmaxf(z, 0.0f) + log1pf(expf(-fabsf(z))); }

// A chunk's gates in LDS.
struct ScanGates {
    float hi[kChunk], lo[kChunk];  // G
    float e[kChunk], f[kChunk];    // E; F, times beta where that is on the values
    float beta[kChunk], diagonal[kChunk];  // (diagonal: q . k of each token)
    int32_t episode[kChunk];       // episodes begun in the chunk so far
    // D_ij (beta_j) of tiles below the diagonal as down_i across_j, from and to the first token of i's tile
    float down[kChunk], across[3][kChunk];
};

struct ScanGatesFetch {
    float dt, after;
    int start;

    // A chunk of tokens from `low` on, in the walk's order.
    __device__ void fetch(const ScanParams& P, bool reverse, int64_t env, int head, int64_t low, int tokens) {
        const int lane = threadIdx.x & 63;
        const int64_t t = low + (reverse ? tokens - 1 - lane : lane), u = reverse ? t + 1 : t;  // whose decay comes before
        const float* from = P.dt + env * P.dt_stride[0] + head * P.dt_stride[2];
        dt = after = 0.0f;
        start = 0;
        if (lane >= tokens) return;
        dt = from[t * P.dt_stride[1]];
        if (reverse && u < P.steps) after = from[u * P.dt_stride[1]];
        if (P.starts && u < P.steps) start = P.starts[env * P.starts_stride[0] + u * P.starts_stride[1]];
    }

    __device__ void put(const ScanParams& P, ScanGates& gates, bool reverse, int head, int64_t low, int tokens) const {
        const int lane = threadIdx.x & 63;
        const float bias = P.dt_bias ? P.dt_bias[head] : 0.0f, a = P.a[head];
        const bool inside = lane < tokens;
        const float beta = inside ? softplus(dt + bias) : 0.0f;
        // (backwards nothing decays before the last token)
        const bool decays = inside && !(reverse && lane == 0 && low + tokens == P.steps);
        const double g = decays ? static_cast<double>(reverse ? softplus(after + bias) : beta) * a : 0.0;
        const bool starts = start != 0 || g < kStart;
        const double sum = sum_up(starts ? 0.0 : g);
        const uint64_t all = __ballot(starts);
        const int episode = __popcll(all << (63 - lane)), last_episode = __popcll(all);
        const float hi = static_cast<float>(sum), lo = static_cast<float>(sum - hi);
        const double last = of_lane(sum, 63);
        const float f = episode == last_episode ? expf(static_cast<float>(last - sum)) : 0.0f;
        double own = of_lane(sum, 0);  // of the first token of the lane's tile
        int own_episode = __builtin_amdgcn_readlane(episode, 0);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const double first = of_lane(sum, 16 * i + 16);
            const int first_episode = __builtin_amdgcn_readlane(episode, 16 * i + 16);
            const float x = episode == first_episode ? expf(static_cast<float>(first - sum)) : 0.0f;
            gates.across[i][lane] = reverse ? x : x * beta;
            own = lane >= 16 * i + 16 ? first : own;
            own_episode = lane >= 16 * i + 16 ? first_episode : own_episode;
        }
        gates.down[lane] = episode == own_episode ? expf(static_cast<float>(sum - own)) : 0.0f;
        gates.hi[lane] = hi;
        gates.lo[lane] = lo;
        gates.e[lane] = episode == 0 ? expf(hi) * (1.0f + lo) : 0.0f;
        gates.f[lane] = reverse ? f : f * beta;
        gates.beta[lane] = beta;
        gates.episode[lane] = episode;
    }
};

// Values of a chunk: planes, or float32 as it is, which takes less of the LDS than three of them: two workgroups of
// 64 rows fit a CU (float32, 1024 x 128 steps of 4 heads of 64 x 64: forward 169 us, 261 with planes; with gradients
// 924 and 1371).
template <class E>
using Values = std::conditional_t<sizeof(E) == 4, float[kChunk][kColumns + 4], uint16_t[kPlanes<E>][kChunk][kColumns + 8]>;

template <class E, int KP>
struct ScanLds {
    union {
        uint16_t q[kPlanes<E>][kChunk][KP + 8];
        Triangle<3> p;  // once the queries have been used
    };
    uint16_t k[kPlanes<E>][kChunk][KP + 8];
    __attribute__((aligned(16))) Values<E> v;
    ScanGates gates;
};

template <class E, int KP>
struct ScanGradientsLds : ScanLds<E, KP> {
    float dots[2][4][2][kChunk];
};

// Rows of a chunk on their way to LDS: kCols columns from `column` on, 256 threads.
template <class E, int kCols>
struct RowsFetch {
    static constexpr int kAcross = kCols / 8, kDown = 256 / kAcross, kPieces = kChunk / kDown;
    Part<E, 8> part[kPieces];

    __device__ void fetch(const Operand& from, int64_t env, int head, int64_t low, int tokens, bool reverse, int column, int width) {
        const uint32_t row_bytes = static_cast<uint32_t>(from.stride[1]) * sizeof(E);
        const E* base = static_cast<const E*>(from.p) + env * from.stride[0] + low * from.stride[1] + head / from.share * from.stride[2];
        const Buffer rows = buffer_of(base, (tokens - 1) * row_bytes + width * sizeof(E));
        const int c = column + threadIdx.x % kAcross * 8;
        if (from.wide) {
            // Rows past the last are beyond the buffer's end in either order (backwards their offsets wrap
            // around to 2^31 and more).
            const int t = threadIdx.x / kAcross;
            const uint32_t lane = (c < width ? c * static_cast<uint32_t>(sizeof(E)) : kOutside) + (reverse ? tokens - 1 - t : t) * row_bytes;
            const uint32_t step = (reverse ? -kDown : kDown) * row_bytes;
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
#pragma unroll
                for (int w = 0; w < Part<E, 8>::kWords; ++w) part[i].words[w] = buffer_load16(rows, lane + i * step + 16 * w);
        } else {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int t = threadIdx.x / kAcross + i * kDown, row = reverse ? tokens - 1 - t : t;
                part[i].load(rows, row * row_bytes + c * sizeof(E), t < tokens ? width - c : 0, false);
            }
        }
    }

    // `signs`: 0x80008000 to negate them, or 0.
    template <int kPitch>
    __device__ void put(uint16_t (&rows)[kPlanes<E>][kChunk][kPitch], uint32_t signs = 0) const {
        const int c = threadIdx.x % kAcross * 8;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int t = threadIdx.x / kAcross + i * kDown;
            if constexpr (kPlanes<E> == 1) {
                put_columns(rows[0][t], c, part[i].words[0] ^ signs);
            } else {
                float x[8];
                u4 plane[kPlanes<E>];
                part[i].floats(x);
                split8(x, plane);
#pragma unroll
                for (int n = 0; n < kPlanes<E>; ++n) put_columns(rows[n][t], c, plane[n] ^ signs);
            }
        }
    }
};

// As they are, where they are float32.
template <int kPieces, int kPitch>
__device__ inline void put_floats(const Part<float, 8> (&part)[kPieces], float (&rows)[kChunk][kPitch]) {
    const int c = threadIdx.x % (kColumns / 8) * 8;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int t = threadIdx.x / (kColumns / 8) + i * (256 / (kColumns / 8));
#pragma unroll
        for (int w = 0; w < 2; ++w) *reinterpret_cast<u4*>(&rows[t][c + 4 * w]) = part[i].words[w];
    }
}

// Eight numbers of operands as floats: their planes' sum.
template <int N>
__device__ inline void join8(const u4 (&plane)[N], float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = 0.0f;
#pragma unroll
        for (int n = N - 1; n >= 0; --n) {
            const uint32_t word = plane[n][i / 2];
            x[i] += float_of(i % 2 ? word & 0xffff0000u : word << 16);
        }
    }
}

// Four numbers of a row in LDS, columns 4 g of the 16 from 16 c on.
template <int N, int kPitch>
__device__ inline f4 four_of(const uint16_t (&rows)[N][kChunk][kPitch], int row, int c, int g) {
    f4 x = {0, 0, 0, 0};
#pragma unroll
    for (int n = N - 1; n >= 0; --n) {
        const u2 w = *reinterpret_cast<const u2*>(&rows[n][row][32 * (c >> 1) + 8 * g + 4 * (c & 1)]);
        x += f4{float_of(w.x << 16), float_of(w.x & 0xffff0000u), float_of(w.y << 16), float_of(w.y & 0xffff0000u)};
    }
    return x;
}

// The same of values that are float32.
template <int kPitch>
__device__ inline f4 four_of(const float (&rows)[kChunk][kPitch], int row, int c, int g) {
    return *reinterpret_cast<const f4*>(&rows[row][16 * c + 4 * g]);
}

// The wave's 16 columns of 32 tokens of values that are float32, as operand_columns orders them.
template <int kPitch>
__device__ inline void column_values(int lane, const float (&v)[kChunk][kPitch], int wave, int m, float (&x)[8]) {
#pragma unroll
    for (int s = 0; s < 8; ++s) x[s] = v[32 * m + 16 * (s >> 2) + 4 * (lane >> 4) + (s & 3)][16 * wave + (lane & 15)];
}

// The tiles of a triangle that a wave computes: its own on the diagonal, and of those below one or two
// (i and j, two bits each, for n = 1 and 2; 3 for none).
__device__ inline int tile_of_wave(int wave, int n) {
    constexpr uint32_t kBelow = 0x84u | 0xc9u << 8 | 0x3du << 16 | 0x3eu << 24;
    return n == 0 ? 5 * wave : kBelow >> (8 * wave + 4 * (n - 1)) & 15;
}

// D of a tile (beta_j D_ij forwards), for the lane's column and four rows; zeros on the diagonal and above.
__device__ inline f4 decays(const ScanGates& gates, int i, int j, bool reverse) {
    const int lane = threadIdx.x & 63, g = lane >> 4, column = 16 * j + (lane & 15), row = 16 * i + 4 * g;
    if (i != j) return *reinterpret_cast<const f4*>(&gates.down[row]) * gates.across[i - 1][column];
    const float hi = gates.hi[column], lo = gates.lo[column], beta = reverse ? 1.0f : gates.beta[column];
    const int episode = gates.episode[column];
    const f4 row_hi = *reinterpret_cast<const f4*>(&gates.hi[row]), row_lo = *reinterpret_cast<const f4*>(&gates.lo[row]);
    using i4 = int32_t __attribute__((ext_vector_type(4)));
    const i4 row_episode = *reinterpret_cast<const i4*>(&gates.episode[row]);
    f4 x;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const float d = (row_hi[s] - hi) + (row_lo[s] - lo);
        x[s] = row + s > column && row_episode[s] == episode ? __builtin_amdgcn_exp2f(d * kLog2E) * beta : 0.0f;
    }
    return x;
}

// Rows i of q times rows j of k.
template <int N, int kPitch>
__device__ inline f4 tile_product(const uint16_t (&q)[N][kChunk][kPitch], const uint16_t (&k)[N][kChunk][kPitch], int i, int j) {
    const int lane = threadIdx.x & 63;
    f4 x = {0, 0, 0, 0};
#pragma unroll
    for (int m = 0; m < kPitch / 32; ++m) {
        u4 qi[N], kj[N];
        operand_rows(lane, q, 16 * i, m, qi);
        operand_rows(lane, k, 16 * j, m, kj);
        x = mma(qi, kj, x);
    }
    return x;
}

// The lane's number of a tile's diagonal, if it has one.
template <class F>
__device__ inline void diagonal_of(f4 x, F to) {
    const int lane = threadIdx.x & 63, s = (lane & 15) - 4 * (lane >> 4);
    if (s >= 0 && s < 4) to(lane & 15, s == 0 ? x[0] : s == 1 ? x[1] : s == 2 ? x[2] : x[3]);
}

template <int KP>
__device__ inline void add_state(const Role& R, const float* from, int64_t row, int64_t column, int first, f4 (&state)[KP / 16]) {
    const int lane = threadIdx.x & 63, c = first + (lane & 15);
#pragma unroll
    for (int i = 0; i < KP / 16; ++i)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int k = 16 * i + 4 * (lane >> 4) + s;
            if (k < R.K && c < R.V) state[i][s] = from[k * row + c * column];
        }
}

template <int KP>
__device__ inline void store_state(const Role& R, float* to, int64_t row, int64_t column, int first, float factor, const f4 (&state)[KP / 16]) {
    const int lane = threadIdx.x & 63, c = first + (lane & 15);
#pragma unroll
    for (int i = 0; i < KP / 16; ++i)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int k = 16 * i + 4 * (lane >> 4) + s;
            if (k < R.K && c < R.V) to[k * row + c * column] = factor == 0.0f ? 0.0f : state[i][s] * factor;
        }
}

// Results alone; with what the gradients of the gates need; what a segment makes of zeros, and what it
// multiplies a state before it with.
enum { kResults, kGradients, kSegments };

// Four numbers of a row each of the lane's tokens (l % 16 of each tile), its columns of the wave's 16.
template <class E>
struct FourFetch {
    using Words = std::conditional_t<sizeof(E) == 4, u4, u2>;
    Words words[4];

    __device__ void fetch(const Operand& from, int64_t env, int head, int64_t low, int tokens, bool reverse, int first, int width) {
        const int lane = threadIdx.x & 63, t = lane & 15, c = first + 4 * (lane >> 4);
        const uint32_t row_bytes = static_cast<uint32_t>(from.stride[1]) * sizeof(E);
        const E* base = static_cast<const E*>(from.p) + env * from.stride[0] + low * from.stride[1] + head / from.share * from.stride[2];
        const Buffer rows = buffer_of(base, (tokens - 1) * row_bytes + width * sizeof(E));
        const uint32_t at = (c < width ? c * static_cast<uint32_t>(sizeof(E)) : kOutside) + (reverse ? tokens - 1 - t : t) * row_bytes;
        const uint32_t step = (reverse ? -16 : 16) * row_bytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (from.wide) {
                if constexpr (sizeof(E) == 4)
                    words[i] = buffer_load16(rows, at + i * step);
                else
                    words[i] = __builtin_bit_cast(u2, __builtin_amdgcn_raw_buffer_load_b64(rows, at + i * step, 0, 0));
            } else {
                E x[4];
#pragma unroll
                for (int s = 0; s < 4; ++s) x[s] = buffer_load<E>(rows, c + s < width ? at + i * step + s * static_cast<uint32_t>(sizeof(E)) : kOutside);
                words[i] = __builtin_bit_cast(Words, x);
            }
        }
    }

    __device__ f4 floats(int i) const {
        if constexpr (sizeof(E) == 4) {
            return __builtin_bit_cast(f4, words[i]);
        } else {
            f4 x;
#pragma unroll
            for (int s = 0; s < 4; ++s) x[s] = to_float(__builtin_bit_cast(E, static_cast<uint16_t>(words[i][s / 2] >> (16 * (s % 2)))));
            return x;
        }
    }
};

// Workgroups that a CU's LDS holds and its registers allow: 36 KiB each for bfloat16 and 64 (40 with gradients), up to
// 122 (126) for float32 and 128.
template <class E, int KP>
inline constexpr int kWorkgroups = kPlanes<E> == 1 ? (KP == 64 ? 3 : 2) : KP == 64 ? 2 : 1;

// A workgroup walks the chunks of a segment with 64 columns of a head's state in registers, 16 a wave.
template <class E, int KP, int kMode>
__global__ __launch_bounds__(256, (kWorkgroups<E, KP>)) void selective_scan_kernel(ScanParams P) {
    constexpr bool kSummary = kMode == kSegments, kGates = kMode == kGradients;
    constexpr int N = kPlanes<E>;
    extern __shared__ char lds_bytes[];
    auto& lds = *reinterpret_cast<std::conditional_t<kGates, ScanGradientsLds<E, KP>, ScanLds<E, KP>>*>(lds_bytes);
    const Role& R = P.role[blockIdx.y];
    const int wave = wave_of_workgroup(), lane = threadIdx.x & 63, g = lane >> 4;
    // Workgroups go round the 8 XCDs in turn: those of one env, group and segment, which read the same
    // rows, are 8 apart (or one after the other where there are fewer than 8 such).
    const uint32_t inner = P.group * R.blocks, segments = kSummary ? P.n_segments - 1 : P.n_segments;
    const int64_t groups = P.heads / P.group, units = P.envs * groups * segments;
    const uint32_t round = units < 8 ? blockIdx.x : blockIdx.x / 8;
    const int64_t unit = units < 8 ? round / inner : static_cast<int64_t>(round / inner) * 8 + blockIdx.x % 8;
    if (unit >= units) return;
    const int segment = static_cast<int>(unit % segments);
    const int64_t outer = unit / segments, env = outer / groups;
    const int head = static_cast<int>(outer % groups) * P.group + static_cast<int>(round % inner) / R.blocks;
    const int block = static_cast<int>(round % inner) % R.blocks, first = block * kColumns + 16 * wave;
    const int64_t sequence = env * P.heads + head, kv = static_cast<int64_t>(R.K) * R.V;
    const bool reverse = kMode != kResults && R.reverse, working = first < R.V;
    const int begin = static_cast<int>(static_cast<int64_t>(segment) * P.n_chunks / P.n_segments);
    const int end = static_cast<int>((segment + 1ll) * P.n_chunks / P.n_segments);

    f4 state[KP / 16];
#pragma unroll
    for (int i = 0; i < KP / 16; ++i) state[i] = f4{0, 0, 0, 0};
    bool empty = true;
    if constexpr (!kSummary) {
        if (segment > 0) {
            empty = false;
            add_state<KP>(R, R.segment_states + (sequence * (P.n_segments - 1) + segment - 1) * kv, R.V, 1, first, state);
        } else if (R.from) {
            empty = false;
            add_state<KP>(R, R.from + sequence * kv, R.state_row, R.state_column, first, state);
        }
    }
    RowsFetch<E, KP> q_next, k_next;
    RowsFetch<E, kColumns> v_next;
    ScanGatesFetch gates_next;
    // Chunks of both directions are the same tokens; backwards they are counted from the last.
    const auto place_of = [&](int chunk) { return reverse ? P.n_chunks - 1 - chunk : chunk; };
    const auto tokens_of = [&](int64_t low) { return static_cast<int>(P.steps - low < kChunk ? P.steps - low : kChunk); };
    const auto fetch = [&](int chunk) {
        const int64_t low = static_cast<int64_t>(place_of(chunk)) * kChunk;
        const int tokens = tokens_of(low);
        if (!kSummary) q_next.fetch(R.q, env, head, low, tokens, reverse, 0, R.K);
        k_next.fetch(R.k, env, head, low, tokens, reverse, 0, R.K);
        v_next.fetch(R.v, env, head, low, tokens, reverse, block * kColumns, R.V);
        if (wave == 0) gates_next.fetch(P, reverse, env, head, low, tokens);
    };
    const auto sign_of = [&](int chunk) { return (env + place_of(chunk)) & 1 ? -1.0f : 1.0f; };  // of keys, states and results
    float total = 1.0f, sign = begin < end ? sign_of(begin) : 1.0f;
#pragma unroll
    for (int i = 0; i < KP / 16; ++i) state[i] = sign * state[i];
    if (begin < end) fetch(begin);
    for (int chunk = begin; chunk < end; ++chunk) {
        const int place = place_of(chunk);
        const int64_t low = static_cast<int64_t>(place) * kChunk;
        const int tokens = tokens_of(low);
        if (chunk > begin) {
            sign = -sign;
#pragma unroll
            for (int i = 0; i < KP / 16; ++i) state[i] = -state[i];
            __syncthreads();
        }
        if (!kSummary) q_next.put(lds.q);
        k_next.put(lds.k, sign < 0.0f ? 0x80008000u : 0u);
        if constexpr (sizeof(E) == 4)
            put_floats(v_next.part, lds.v);
        else
            v_next.put(lds.v);
        if (wave == 0) gates_next.put(P, lds.gates, reverse, head, low, tokens);
        __syncthreads();
        if (chunk + 1 < end) fetch(chunk + 1);
        const float keep = lds.gates.e[kChunk - 1];
        total = keep == 0.0f ? 0.0f : total * keep;
        FourFetch<E> z;
        if (kGates && R.state_dots) z.fetch(R.z, env, head, low, tokens, reverse, first, working ? R.V : 0);
        // z . o of the lane's tokens and columns
        const auto dots = [&](const f4 (&o)[4], float (&to)[2][kChunk]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f4 x = z.floats(i) * o[i];
                float sum = sign * ((x[0] + x[1]) + (x[2] + x[3]));
                sum += __shfl_xor(sum, 32);
                if (g < 2) to[g][16 * i + (lane & 15)] = sum;
            }
        };
        f4 o[4], p[3];
        const int64_t slot = ((sequence * P.n_chunks + place) * R.blocks + block) * 4 + wave;
        if (kGates && R.through && !working && lane == 0) R.through[slot] = 0.0f;
        if constexpr (kGates) {
            if (working && R.keep_states && place >= R.keep_from && place < R.keep_to) {
                f4* to = reinterpret_cast<f4*>(R.keep_states) + slot * (KP / 16) * 64 + lane;
#pragma unroll
                for (int i = 0; i < KP / 16; ++i) to[i * 64] = state[i];
            }
            if (working && R.through) {
                float dot = 0.0f;
                if (place >= R.keep_from && place < R.keep_to) {
                    const f4* from = reinterpret_cast<const f4*>(R.other_states) + slot * (KP / 16) * 64 + lane;
#pragma unroll
                    for (int i = 0; i < KP / 16; ++i) {
                        const f4 x = state[i] * from[i * 64];
                        dot += (x[0] + x[1]) + (x[2] + x[3]);
                    }
#pragma unroll
                    for (int d = 1; d < 64; d *= 2) dot += __shfl_xor(dot, d);
                }
                // (what is held backwards has not passed the decay before the chunk's first place)
                if (lane == 0) R.through[slot] = lds.gates.e[0] == 0.0f ? 0.0f : lds.gates.e[0] * dot;
            }
        }
        if constexpr (!kSummary) {
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                const int tile = tile_of_wave(wave, n), i = tile >> 2, j = tile & 3;
                if (tile == 3) continue;
                p[n] = tile_product(lds.q, lds.k, i, j);
                if (n == 0) diagonal_of(p[0], [&](int t, float x) { lds.gates.diagonal[16 * i + t] = sign * x; });
                p[n] *= decays(lds.gates, i, j, reverse);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = f4{0, 0, 0, 0};
            // (a state that the chunk's first token forgets may hold anything)
            if (lds.gates.e[0] == 0.0f)
#pragma unroll
                for (int i = 0; i < KP / 16; ++i) state[i] = f4{0, 0, 0, 0};
            if (working && !empty && lds.gates.e[0] != 0.0f) {
#pragma unroll
                for (int m = 0; m < KP / 32; ++m) {
                    u4 b[3];
                    split8(state[2 * m], state[2 * m + 1], b);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        u4 a[N];
                        operand_rows(lane, lds.q, 16 * i, m, a);
                        o[i] = mma(b, a, o[i]);  // (transposed: the operands hold rows and columns alike)
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = lds.gates.e[16 * i + (lane & 15)] * o[i];
            }
            if constexpr (kGates) {
                if (R.state_dots && working) dots(o, lds.dots[0][wave]);
            }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                const int tile = tile_of_wave(wave, n);
                if (tile != 3) store_slot<3>(lds.p, tile_of(tile >> 2, tile & 3), lane, p[n]);
            }
        }
        u4 value[2][N];
        float values[sizeof(E) == 4 ? 2 : 1][8];
        if (working) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if constexpr (sizeof(E) == 4) {
                    column_values(lane, lds.v, wave, m, values[m]);
                    split8(values[m], value[m]);
                } else {
                    operand_columns(lane, lds.v, wave, m, value[m]);
                }
            }
#pragma unroll
            for (int i = 0; i < KP / 16; ++i)
#pragma unroll
                for (int s = 0; s < 4; ++s) state[i][s] = keep == 0.0f ? 0.0f : keep * state[i][s];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                u4 r[3];
                float(&x)[8] = values[sizeof(E) == 4 ? m : 0];
                if constexpr (sizeof(E) != 4) join8(value[m], x);
                const f4 f0 = *reinterpret_cast<const f4*>(&lds.gates.f[32 * m + 4 * g]);
                const f4 f1 = *reinterpret_cast<const f4*>(&lds.gates.f[32 * m + 16 + 4 * g]);
                split8(f0 * f4{x[0], x[1], x[2], x[3]}, f1 * f4{x[4], x[5], x[6], x[7]}, r);
#pragma unroll
                for (int i = 0; i < KP / 16; ++i) {
                    u4 a[N];
                    operand_columns(lane, lds.k, i, m, a);
                    state[i] = mma(a, r, state[i]);
                }
            }
            empty = false;
        }
        if constexpr (!kSummary) {
            __syncthreads();
            if (working) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    u4 a[3];
                    operand_triangle<3>(lane, lds.p, i, 0, a);
                    o[i] = mma(value[0], a, o[i]);
                    if (i >= 2) {
                        operand_triangle<3>(lane, lds.p, i, 1, a);
                        o[i] = mma(value[1], a, o[i]);
                    }
                }
            }
        }
        if constexpr (kSummary) continue;
        if constexpr (kGates) if (R.state_dots) {
            if (working) {
                if (R.dots) dots(o, lds.dots[1][wave]);
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) lds.dots[0][wave][i][lane] = lds.dots[1][wave][i][lane] = 0.0f;
            }
            __syncthreads();
            float* to = wave == 0 ? R.state_dots : R.dots;
            if (wave < 2 && lane < tokens && to) {
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const auto& from = lds.dots[wave][w];
                    sum += from[0][lane] + from[1][lane];
                }
                to[(sequence * R.blocks + block) * P.steps + low + (reverse ? tokens - 1 - lane : lane)] = sum;
            }
        }
        if (!working) continue;
        // A lane has token l % 16 of each tile, four columns of it.
        const float skip = R.skip && P.d ? P.d[head] : 0.0f;
        const int column = 4 * g, width = R.V - first < 16 ? R.V - first : 16;
        const int64_t row0 = (env * P.steps + low) * P.heads + head;
        const auto store = [&](auto* base) {
            using T = std::remove_reference_t<decltype(*base)>;
            const uint32_t row_bytes = static_cast<uint32_t>(P.heads) * R.V * sizeof(T);
            const Buffer to = buffer_of(base + row0 * R.V + first, (tokens - 1) * row_bytes + width * sizeof(T));
            // (rows past the last: as in RowsFetch)
            const uint32_t own = (column < width ? column * static_cast<uint32_t>(sizeof(T)) : kOutside) +
                                 (reverse ? tokens - 1 - (lane & 15) : lane & 15) * row_bytes;
            const uint32_t step = (reverse ? -16 : 16) * row_bytes;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 16 * i + (lane & 15);
                const float beta = lds.gates.beta[t];
                const f4 x = (reverse ? sign * beta : sign) * o[i] + (beta * lds.gates.diagonal[t] + skip) * four_of(lds.v, t, wave, g);
                const uint32_t offset = own + i * step;
                const T y[4] = {from_float<T>(x[0]), from_float<T>(x[1]), from_float<T>(x[2]), from_float<T>(x[3])};
                if (R.wide_out) {
                    buffer_store_four(to, offset, y);
                } else {
#pragma unroll
                    for (int s = 0; s < 4; ++s) buffer_store<T>(to, column + s < width ? offset + s * sizeof(T) : kOutside, y[s]);
                }
            }
        };
        if (kGates && R.out_heads)
            store(R.out_heads);
        else
            store(static_cast<E*>(R.out));
    }
    if constexpr (kSummary) {
        if (working) store_state<KP>(R, R.segment_states + (sequence * (P.n_segments - 1) + segment) * kv, R.V, 1, first, sign, state);
        if (block == 0 && threadIdx.x == 0) R.segment_keeps[sequence * P.n_segments + segment] = total;
    } else if (R.to && segment + 1 == P.n_segments && working) {
        float factor = sign;
        if (reverse) {  // what the first token's decay leaves of it
            const float beta = softplus(P.dt[env * P.dt_stride[0] + head * P.dt_stride[2]] + (P.dt_bias ? P.dt_bias[head] : 0.0f));
            factor *= expf(beta * P.a[head]);
            if (P.starts && P.starts[env * P.starts_stride[0]]) factor = 0.0f;
        }
        store_state<KP>(R, R.to + sequence * kv, R.state_row, R.state_column, first, factor, state);
    }
}

// The states before segments from what each makes of zeros, in their place: four numbers a lane,
// from segment to segment.
__global__ __launch_bounds__(256) void selective_join_kernel(ScanParams P) {
    const Role& R = P.role[blockIdx.y];
    const int64_t kv = static_cast<int64_t>(R.K) * R.V, i = blockIdx.x * 256ll + threadIdx.x;
    const int64_t sequence = i / kv, n = i % kv;
    if (sequence >= P.envs * P.heads) return;
    float* at = R.segment_states + sequence * (P.n_segments - 1) * kv + n;
    const float* keep = R.segment_keeps + sequence * P.n_segments;
    float state = 0.0f;
    if (R.from) state = R.from[sequence * kv + n / R.V * R.state_row + n % R.V * R.state_column];
    for (int s = 0; s + 1 < P.n_segments; s += 8) {
        float made[8], factor[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            made[j] = factor[j] = 0.0f;
            if (s + j + 1 < P.n_segments) made[j] = at[(s + j) * kv], factor[j] = keep[s + j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            state = made[j] + (factor[j] == 0.0f ? 0.0f : factor[j] * state);
            if (s + j + 1 < P.n_segments) at[(s + j) * kv] = state;
        }
    }
}

struct GateParams {
    ScanParams scan;
    Operand x, b, c, dy;
    int32_t state_dim, head_dim;
    const float* rho;      // [env, head][rho_blocks][steps]
    const float* kappa;    // [env, head][delta_blocks][steps] without beta
    const float* delta;    // likewise: x . dx / beta, but for the token's own term
    const float* through;  // [env, head][chunks][through_waves], or NULL
    int32_t rho_blocks, delta_blocks, through_waves;
    float* d_dt;      // [env][step][head]
    double* partial;  // [env, head][chunks][3]: d_a, d_d, d_dt_bias
};

template <class E, int KP>
struct GateLds {
    uint16_t q[kPlanes<E>][kChunk][KP + 8];
    uint16_t k[kPlanes<E>][kChunk][KP + 8];
    Triangle<3> w;
    ScanGates gates;
    float bc[kChunk], dyx[kChunk], pairs[kChunk];
};

// dg of a chunk's tokens and what follows from it, a workgroup a chunk of a head: both triangles of
// products, W, its sums (a product with the triangle of ones: sum over j < t, then over rows i >= t),
// and a token a lane.
template <class E, int KP>
__global__ __launch_bounds__(256, 2) void selective_gates_kernel(GateParams P) {
    extern __shared__ char lds_bytes[];
    auto& lds = *reinterpret_cast<GateLds<E, KP>*>(lds_bytes);
    const ScanParams& S = P.scan;
    const int wave = wave_of_workgroup(), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int64_t sequence = blockIdx.x / static_cast<uint32_t>(S.n_chunks), env = sequence / S.heads;
    const int chunk = static_cast<int>(blockIdx.x % static_cast<uint32_t>(S.n_chunks)), head = static_cast<int>(sequence % S.heads);
    const int64_t t0 = static_cast<int64_t>(chunk) * kChunk;
    const int tokens = static_cast<int>(S.steps - t0 < kChunk ? S.steps - t0 : kChunk);
    const float sign = (env + chunk) & 1 ? -1.0f : 1.0f;  // of b, x and W
    RowsFetch<E, KP> c, b, dy, x;
    c.fetch(P.c, env, head, t0, tokens, false, 0, P.state_dim);
    b.fetch(P.b, env, head, t0, tokens, false, 0, P.state_dim);
    dy.fetch(P.dy, env, head, t0, tokens, false, 0, P.head_dim);
    x.fetch(P.x, env, head, t0, tokens, false, 0, P.head_dim);
    const bool inside = lane < tokens;
    const int64_t t = t0 + lane;
    // What the last wave needs at the end it reads now (1024 x 128 steps of 4 heads: 66 us, 77 with loads there and
    // sums by shuffles). Both dimensions have two blocks of columns at most.
    static_assert(NAVI_POLICY_MAX_STATE_DIM <= 2 * kColumns, "partial sums of rho, kappa and delta");
    float rho = 0.0f, kappa = 0.0f, delta = 0.0f, through = 0.0f, z = 0.0f, more[3] = {};
    if (wave == 3) {
        if (inside) {
            rho = P.rho[sequence * P.rho_blocks * S.steps + t];
            kappa = P.kappa[sequence * P.delta_blocks * S.steps + t];
            delta = P.delta[sequence * P.delta_blocks * S.steps + t];
            if (P.rho_blocks > 1) more[0] = P.rho[(sequence * P.rho_blocks + 1) * S.steps + t];
            if (P.delta_blocks > 1) {
                more[1] = P.kappa[(sequence * P.delta_blocks + 1) * S.steps + t];
                more[2] = P.delta[(sequence * P.delta_blocks + 1) * S.steps + t];
            }
            z = S.dt[env * S.dt_stride[0] + t * S.dt_stride[1] + head * S.dt_stride[2]];
        }
        if (P.through && lane < P.through_waves) through = P.through[(sequence * S.n_chunks + chunk) * P.through_waves + lane];
    }
    if (wave == 0) {
        ScanGatesFetch gates;
        gates.fetch(S, false, env, head, t0, tokens);
        gates.put(S, lds.gates, false, head, t0, tokens);
    }
    c.put(lds.q);
    b.put(lds.k, sign < 0.0f ? 0x80008000u : 0u);
    __syncthreads();
    f4 bc[3];
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        const int tile = tile_of_wave(wave, n);
        if (tile != 3) bc[n] = tile_product(lds.q, lds.k, tile >> 2, tile & 3);
    }
    __syncthreads();
    dy.put(lds.q);
    x.put(lds.k, sign < 0.0f ? 0x80008000u : 0u);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        const int tile = tile_of_wave(wave, n), i = tile >> 2, j = tile & 3;
        if (tile == 3) continue;
        const f4 dyx = sign * tile_product(lds.q, lds.k, i, j);
        if (n == 0) {
            diagonal_of(bc[0], [&](int t, float y) { lds.bc[16 * i + t] = sign * y; });
            diagonal_of(dyx, [&](int t, float y) { lds.dyx[16 * i + t] = y; });
        }
        store_slot<3>(lds.w, tile_of(i, j), lane, decays(lds.gates, i, j, false) * bc[n] * dyx);  // (of either sign as well)
    }
    __syncthreads();
    {
        const int t = 16 * wave + col;
        f4 sums[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[i] = f4{0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            u4 before[1];  // ones for tokens before t
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int j = 32 * m + 16 * (n >> 1) + 4 * g + 2 * (n & 1);
                before[0][n] = (j < t ? 0x3f80u : 0u) | (j + 1 < t ? 0x3f800000u : 0u);
            }
#pragma unroll
            for (int i = 2 * m; i < 4; ++i) {
                u4 w[3];
                operand_triangle<3>(lane, lds.w, i, m, w);
                sums[i] = mma(w, before, sums[i]);
            }
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s) sum += 16 * i + 4 * g + s >= t ? sums[i][s] : 0.0f;
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (g == 0) lds.pairs[t] = sign * sum;
    }
    __syncthreads();
    if (wave != 3) return;
    const float beta = lds.gates.beta[lane], a = S.a[head], keep = lds.gates.e[kChunk - 1];
    z += S.dt_bias ? S.dt_bias[head] : 0.0f;
    const double carried = of_lane(sum_up(through), 63);
    // sums from each token on, and up to the token before each
    const double from = rho + more[0], to = static_cast<double>(beta) * (kappa + more[1]);
    const double from_up = sum_up(from), to_up = sum_up(to);
    const double dg = lds.pairs[lane] + (of_lane(from_up, 63) - (from_up - from)) + (to_up - to) + (keep == 0.0f ? 0.0 : keep * carried);
    double sums[3] = {};
    if (inside) {
        const double dbeta = (delta + more[2]) + static_cast<double>(lds.bc[lane]) * lds.dyx[lane] + a * dg;
        const float d_dt = static_cast<float>(dbeta) / (1.0f + expf(-z));
        P.d_dt[(env * S.steps + t) * S.heads + head] = d_dt;
        sums[0] = beta * dg;
        sums[1] = lds.dyx[lane];
        sums[2] = d_dt;
    }
    if (!P.partial) return;
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        const double sum = of_lane(sum_up(sums[n]), 63);
        if (lane == 0) P.partial[3 * static_cast<int64_t>(blockIdx.x) + n] = sum;
    }
}

// Sums over environments and chunks: a workgroup a head.
__global__ __launch_bounds__(256) void selective_sums_kernel(const double* partial, int64_t envs, int32_t heads, int32_t chunks, float* d_a,
                                                             float* d_d, float* d_bias) {
    __shared__ double lds[3][4];
    const int head = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double sum[3] = {};
    for (int64_t i = threadIdx.x; i < envs * chunks; i += 256) {
        const double* from = partial + 3 * ((i / chunks * heads + head) * chunks + i % chunks);
#pragma unroll
        for (int n = 0; n < 3; ++n) sum[n] += from[n];
    }
#pragma unroll
    for (int n = 0; n < 3; ++n) {
#pragma unroll
        for (int d = 1; d < 64; d *= 2) sum[n] += __shfl_xor(sum[n], d);
        if (lane == 0) lds[n][wave] = sum[n];
    }
    __syncthreads();
    if (threadIdx.x >= 3) return;
    float* to[3] = {d_a, d_d, d_bias};
    const double* part = lds[threadIdx.x];
    if (to[threadIdx.x]) to[threadIdx.x][head] = static_cast<float>((part[0] + part[1]) + (part[2] + part[3]));
}

// Gradients of b and c from those of the heads that share them, eight numbers a thread.
template <class E>
__global__ __launch_bounds__(256) void selective_groups_kernel(const float* from0, const float* from1, E* to0, E* to1, int64_t rows, int32_t group, int32_t dim) {
    const float* from = blockIdx.y ? from1 : from0;
    E* to = blockIdx.y ? to1 : to0;
    const int32_t pieces = (dim + 7) / 8;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * pieces; i += gridDim.x * 256ll) {
        const int64_t row = i / pieces;
        const int32_t c = static_cast<int32_t>(i % pieces) * 8;
        float sum[8] = {};
        const float* at = from + row * group * dim + c;
        if (dim % 8 == 0) {
            int32_t h = 0;
            for (; h + 4 <= group; h += 4) {  // (on their way at once: 1024 x 128 rows of 4 heads of 64 take 60 us, 5 TB/s)
                float x[4][8];
#pragma unroll
                for (int m = 0; m < 4; ++m) load_eight(at + static_cast<int64_t>(h + m) * dim, x[m]);
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int n = 0; n < 8; ++n) sum[n] += x[m][n];
            }
            for (; h < group; ++h) {
                float x[8];
                load_eight(at + static_cast<int64_t>(h) * dim, x);
#pragma unroll
                for (int n = 0; n < 8; ++n) sum[n] += x[n];
            }
        } else {
            for (int32_t h = 0; h < group; ++h)
#pragma unroll
                for (int n = 0; n < 8; ++n) sum[n] += c + n < dim ? at[static_cast<int64_t>(h) * dim + n] : 0.0f;
        }
#pragma unroll
        for (int n = 0; n < 8; ++n)
            if (c + n < dim) to[row * dim + c + n] = from_float<E>(sum[n]);
    }
}

int64_t chunks_of(int64_t steps) { return (steps + kChunk - 1) / kChunk; }
int32_t blocks_of(int32_t columns) { return (columns + kColumns - 1) / kColumns; }
int64_t rounded(int64_t floats) { return (floats + 3) / 4 * 4; }

// Walks that leave the card's 256 CUs without two workgroups each are cut, into segments of at
// least two chunks.
int32_t segments_of(const navi_selective_scan_args& a, int32_t blocks) {
    const int64_t walks = a.envs * a.heads * blocks, chunks = chunks_of(a.steps);
    if (walks <= 0 || walks >= 256 || chunks < 8) return 1;
    return static_cast<int32_t>(std::max<int64_t>(1, std::min({(512 + walks - 1) / walks, chunks / 2, int64_t{64}})));
}

int32_t segments_of(const navi_selective_scan_args& a, bool back) {
    return segments_of(a, back ? blocks_of(a.head_dim) + 2 * blocks_of(a.state_dim) : blocks_of(a.head_dim));
}

// What a role's segments need.
int64_t segment_floats(const navi_selective_scan_args& a, int32_t segments) {
    if (segments <= 1) return 0;
    const int64_t sequences = a.envs * a.heads;
    return rounded(sequences * (segments - 1) * a.state_dim * a.head_dim) + rounded(sequences * segments);
}

int check(const navi_selective_scan_args* a) {
    if (!a) return set_error(NAVI_POLICY_E_ARG, "args must be non-null");
    if (a->dtype < NAVI_POLICY_F32 || a->dtype > NAVI_POLICY_F16)
        return set_error(NAVI_POLICY_E_ARG, "dtype must be float32, bfloat16 or float16");
    if (a->groups <= 0 || a->heads <= 0 || a->heads % a->groups != 0)
        return set_error(NAVI_POLICY_E_ARG, "heads must be a positive multiple of groups");
    if (a->state_dim <= 0 || a->state_dim > NAVI_POLICY_MAX_STATE_DIM || a->head_dim <= 0 || a->head_dim > NAVI_POLICY_MAX_STATE_DIM)
        return set_error(NAVI_POLICY_E_ARG, "state_dim and head_dim must be in [1, %d]", NAVI_POLICY_MAX_STATE_DIM);
    if (a->heads > NAVI_POLICY_MAX_HEADS) return set_error(NAVI_POLICY_E_ARG, "heads must be at most %d", NAVI_POLICY_MAX_HEADS);
    if (a->envs < 0 || a->steps < 0) return set_error(NAVI_POLICY_E_ARG, "envs and steps must not be negative");
    if (a->steps > INT32_MAX || a->envs > INT32_MAX / 4 / a->heads)
        return set_error(NAVI_POLICY_E_ARG, "steps and 4 * envs * heads must be below 2^31");
    if (a->envs == 0) return 1;
    if (!a->a || (a->steps > 0 && (!a->x || !a->dt || !a->b || !a->c)))
        return set_error(NAVI_POLICY_E_ARG, "x, dt, a, b and c must be non-null");
    const int64_t bytes = a->dtype == NAVI_POLICY_F32 ? 4 : 2;
    if (!aligned(bytes, a->x, a->b, a->c, a->out, a->grad_out, a->d_x, a->d_b, a->d_c) ||
        !aligned(4, a->dt, a->a, a->d, a->dt_bias, a->initial_state, a->final_state, a->grad_final_state, a->d_dt, a->d_a, a->d_d,
                 a->d_dt_bias, a->d_initial_state))
        return set_error(NAVI_POLICY_E_ARG, "arrays must be aligned to their elements");
    return NAVI_POLICY_OK;
}

constexpr int64_t kFarthest = INT32_MAX / kChunk - (1 << 18);  // bytes between steps

bool rows_apart(const int64_t (&stride)[3], int64_t bytes, int64_t row) {
    return stride[1] >= row && stride[1] * bytes <= kFarthest;
}

Operand operand_of(const void* p, const int64_t (&stride)[3], int64_t bytes, int32_t dim, int32_t share) {
    Operand o{p, {stride[0], stride[1], stride[2]}, share, 0};
    o.wide = dim % 8 == 0 && aligned16(p) && stride[0] * bytes % 16 == 0 && stride[1] * bytes % 16 == 0 && stride[2] * bytes % 16 == 0;
    return o;
}

// An output's rows of `heads` heads: stores reach them by 32-bit offsets.
bool wide_out(const void* p, int32_t dim) { return aligned16(p) && dim % 4 == 0; }

// Workgroups of a launch of scans whose states have up to `blocks` blocks of columns.
int64_t scan_grid(const ScanParams& P, int64_t segments, int blocks) {
    const int64_t units = P.envs * (P.heads / P.group) * segments;
    return (units < 8 ? units : (units + 7) / 8 * 8) * P.group * blocks;
}

struct Setup {
    ScanParams P{};
    Operand x, b, c, dy;
};

int setup(const navi_selective_scan_args* args, bool back, Setup& s) {
    const int code = check(args);
    if (code != NAVI_POLICY_OK) return code;
    navi_selective_scan_args a = *args;
    const int64_t bytes = a.dtype == NAVI_POLICY_F32 ? 4 : 2;
    const int32_t group = a.heads / a.groups;
    if (a.envs * a.heads * chunks_of(a.steps) > INT32_MAX)
        return set_error(NAVI_POLICY_E_ARG, "envs * heads * chunks must be below 2^31");
    if (a.steps == 1) {  // (the stride of an axis of one may be anything)
        a.x_stride[1] = a.grad_out_stride[1] = a.head_dim;
        a.b_stride[1] = a.c_stride[1] = a.state_dim;
    }
    if (a.envs == 1) a.x_stride[0] = a.b_stride[0] = a.c_stride[0] = a.grad_out_stride[0] = 0;
    if (a.heads == 1) a.x_stride[2] = a.grad_out_stride[2] = 0;
    if (a.groups == 1) a.b_stride[2] = a.c_stride[2] = 0;
    if (a.steps > 0 && !(rows_apart(a.x_stride, bytes, a.head_dim) && rows_apart(a.b_stride, bytes, a.state_dim) &&
                         rows_apart(a.c_stride, bytes, a.state_dim) && (!back || rows_apart(a.grad_out_stride, bytes, a.head_dim))))
        return set_error(NAVI_POLICY_E_ARG, "the steps of x, b, c or grad_out overlap or lie too far apart");
    if (static_cast<int64_t>(a.heads) * std::max(a.head_dim, a.state_dim) * 4 > kFarthest)
        return set_error(NAVI_POLICY_E_ARG, "heads * head_dim or heads * state_dim is too large");
    ScanParams& P = s.P;
    P.envs = a.envs;
    P.steps = a.steps;
    P.heads = a.heads;
    P.group = group;
    P.n_chunks = static_cast<int32_t>(chunks_of(a.steps));
    P.n_segments = segments_of(a, back);
    if (!launchable(scan_grid(P, P.n_segments, blocks_of(back ? std::max(a.head_dim, a.state_dim) : a.head_dim)), 256) ||
        (back && !launchable(a.envs * a.heads * P.n_chunks, 256)))
        return set_error(NAVI_POLICY_E_ARG, "too many envs and heads (in the backward pass: and chunks): a launch has fewer than 2^32 threads");
    P.dt = a.dt;
    std::copy(a.dt_stride, a.dt_stride + 3, P.dt_stride);
    P.a = a.a;
    P.d = a.d;
    P.dt_bias = a.dt_bias;
    P.starts = a.starts;
    std::copy(a.starts_stride, a.starts_stride + 2, P.starts_stride);
    s.x = operand_of(a.x, a.x_stride, bytes, a.head_dim, 1);
    s.b = operand_of(a.b, a.b_stride, bytes, a.state_dim, group);
    s.c = operand_of(a.c, a.c_stride, bytes, a.state_dim, group);
    s.dy = operand_of(a.grad_out, a.grad_out_stride, bytes, a.head_dim, 1);
    return NAVI_POLICY_OK;
}

Role role_of(const navi_selective_scan_args& a, const Operand& q, const Operand& k, const Operand& v, bool transposed, bool reverse) {
    Role r{};
    r.q = q;
    r.k = k;
    r.v = v;
    r.K = transposed ? a.head_dim : a.state_dim;
    r.V = transposed ? a.state_dim : a.head_dim;
    r.state_row = transposed ? 1 : a.head_dim;
    r.state_column = transposed ? a.head_dim : 1;
    r.blocks = blocks_of(r.V);
    r.reverse = reverse;
    return r;
}

int launched(const char* name) {
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return set_error(NAVI_POLICY_E_LAUNCH, "%s: kernel launch failed: %s", name, hipGetErrorString(err));
    return NAVI_POLICY_OK;
}

template <class E, int KP, int kMode>
int launch_scan(const ScanParams& P, int roles, int segments, hipStream_t stream) {
    constexpr int lds = kMode == kGradients ? sizeof(ScanGradientsLds<E, KP>) : sizeof(ScanLds<E, KP>);
    static_assert(lds * kWorkgroups<E, KP> <= 160 * 1024, "a CU's LDS");
    const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(selective_scan_kernel<E, KP, kMode>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (err != hipSuccess) return set_error(NAVI_POLICY_E_LAUNCH, "navi_selective_scan: %s", hipGetErrorString(err));
    int blocks = 0;
    for (int i = 0; i < roles; ++i) blocks = std::max(blocks, P.role[i].blocks);
    const dim3 grid(static_cast<unsigned>(scan_grid(P, segments, blocks)), roles);  // (setup has looked at it)
    hipLaunchKernelGGL((selective_scan_kernel<E, KP, kMode>), grid, dim3(256), lds, stream, P);
    return launched("navi_selective_scan");
}

// All roles of P (of one KP) over all segments.
template <class E, int KP>
int scan(const ScanParams& P, int roles, bool back, hipStream_t stream) {
    if (P.n_segments > 1) {
        const int code = launch_scan<E, KP, kSegments>(P, roles, P.n_segments - 1, stream);
        if (code != NAVI_POLICY_OK) return code;
        const int64_t numbers = P.envs * P.heads * P.role[0].K * P.role[0].V;
        hipLaunchKernelGGL(selective_join_kernel, dim3(static_cast<unsigned>((numbers + 255) / 256), roles), dim3(256), 0, stream, P);
    }
    return back ? launch_scan<E, KP, kGradients>(P, roles, P.n_segments, stream) : launch_scan<E, KP, kResults>(P, roles, P.n_segments, stream);
}

template <class E>
int scans(const ScanParams& P, int roles, bool back, bool wide, hipStream_t stream) {
    // those of one KP together
    ScanParams few = P, many = P;
    int n_few = 0, n_many = 0;
    for (int i = 0; i < roles; ++i) {
        if (P.role[i].K <= 64 && !wide)
            few.role[n_few++] = P.role[i];
        else
            many.role[n_many++] = P.role[i];
    }
    if (n_few > 0) {
        const int code = scan<E, 64>(few, n_few, back, stream);
        if (code != NAVI_POLICY_OK) return code;
    }
    return n_many > 0 ? scan<E, 128>(many, n_many, back, stream) : NAVI_POLICY_OK;
}

template <class E, int KP>
int launch_gates(const GateParams& P, hipStream_t stream) {
    constexpr int lds = sizeof(GateLds<E, KP>);
    static_assert(lds <= 160 * 1024, "a CU's LDS");
    const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(selective_gates_kernel<E, KP>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (err != hipSuccess) return set_error(NAVI_POLICY_E_LAUNCH, "navi_selective_scan_backward: %s", hipGetErrorString(err));
    const int64_t blocks = P.scan.envs * P.scan.heads * P.scan.n_chunks;
    hipLaunchKernelGGL((selective_gates_kernel<E, KP>), dim3(static_cast<unsigned>(blocks)), dim3(256), lds, stream, P);
    return launched("navi_selective_scan_backward");
}

template <class E>
int gates(const GateParams& P, hipStream_t stream) {
    return std::max(P.state_dim, P.head_dim) <= 64 ? launch_gates<E, 64>(P, stream) : launch_gates<E, 128>(P, stream);
}

int scans_typed(const ScanParams& P, int32_t dtype, int roles, bool back, bool wide, hipStream_t stream) {
    if (dtype == NAVI_POLICY_F32) return scans<float>(P, roles, back, wide, stream);
    if (dtype == NAVI_POLICY_BF16) return scans<bf16>(P, roles, back, wide, stream);
    return scans<f16>(P, roles, back, wide, stream);
}

float* place_segments(Role& r, const navi_selective_scan_args& a, int32_t segments, float* at) {
    if (segments <= 1) return at;
    r.segment_states = at;
    r.segment_keeps = at + rounded(a.envs * a.heads * (segments - 1) * a.state_dim * a.head_dim);
    return r.segment_keeps + rounded(a.envs * a.heads * segments);
}

// The chunks that have a state before them and a gradient of the one after them.
int32_t keep_from(const navi_selective_scan_args& a) { return a.initial_state ? 0 : 1; }
int32_t keep_to(const navi_selective_scan_args& a) { return static_cast<int32_t>(chunks_of(a.steps)) - (a.grad_final_state ? 0 : 1); }
bool states_needed(const navi_selective_scan_args& a) { return keep_from(a) < keep_to(a); }

// The gradients' scans have keys of state_dim and head_dim numbers, and kernels of 64 and 128 rows run one after the
// other. Where both are needed and the card holds all workgroups of 128 at once, all scans take those: dc and dx then
// run together (bfloat16 with gradients: 9 x 77 steps of 6 heads of 48 x 80, 51 us on the device and 65 apart; 20 x 40
// of 4 heads of 128 x 64, 37 and 46).
bool widened(const navi_selective_scan_args& a, int32_t segments) {
    const int64_t resident = 256 * (a.dtype == NAVI_POLICY_F32 ? kWorkgroups<float, 128> : a.dtype == NAVI_POLICY_BF16 ? kWorkgroups<bf16, 128> : kWorkgroups<f16, 128>);
    const int32_t blocks = blocks_of(a.head_dim) + (states_needed(a) ? 1 : 2) * blocks_of(a.state_dim);
    return (a.state_dim <= 64) != (a.head_dim <= 64) && a.envs * a.heads * segments * blocks <= resident;
}

// What the backward pass keeps for itself.
struct Workspace {
    int64_t partial, rho, kappa, delta, through, states, db, dc, segments, floats;
};

Workspace workspace_of(const navi_selective_scan_args& a) {
    const int64_t sequences = a.envs * a.heads, tokens = sequences * a.steps, chunks = chunks_of(a.steps);
    Workspace w{};
    int64_t at = 0;
    const auto take = [&](int64_t floats) {
        const int64_t here = at;
        at += rounded(floats);
        return here;
    };
    w.partial = take(6 * sequences * chunks);  // (float64)
    w.rho = take(tokens * blocks_of(a.state_dim));
    w.kappa = take(tokens * blocks_of(a.head_dim));
    w.delta = take(tokens * blocks_of(a.head_dim));
    const bool needed = states_needed(a);
    w.through = take(needed ? sequences * chunks * blocks_of(a.state_dim) * 4 : 0);
    w.states = take(needed ? sequences * chunks * blocks_of(a.state_dim) * kColumns * (a.head_dim <= 64 && !widened(a, segments_of(a, true)) ? 64 : 128) : 0);
    const int64_t heads = a.heads > a.groups ? tokens * a.state_dim : 0;
    w.db = take(heads);
    w.dc = take(heads);
    w.segments = take(3 * segment_floats(a, segments_of(a, true)));
    w.floats = at;
    return w;
}

Extent rows_extent(const void* p, const navi_selective_scan_args& a, int64_t heads, int64_t dim, const int64_t (&s)[3], int64_t each) {
    return p && a.steps > 0 ? extent_of(p, {a.envs, a.steps, heads, dim}, {s[0], s[1], s[2], 1}, each) : Extent{0, 0};
}

}  // namespace

int check_selective(const navi_selective_scan_args* a) { return check(a); }

// Workgroups read the inputs in any order, so what is written shares no memory with them: but the
// state after may be the state before in the form for single tokens, and out x there.
int check_selective_apart(const navi_selective_scan_args& a, bool in_place) {
    const int64_t bytes = a.dtype == NAVI_POLICY_F32 ? 4 : 2, H = a.heads, G = a.groups, N = a.state_dim, V = a.head_dim;
    const auto vector = [&](const float* p, int64_t n) { return p ? extent_of(p, {n, 1, 1, 1}, {1, 0, 0, 0}, 4) : Extent{0, 0}; };
    const Extent out = rows_extent(a.out, a, H, V, {a.steps * H * V, H * V, V}, bytes), last = vector(a.final_state, a.envs * H * N * V);
    const Extent x = rows_extent(a.x, a, H, V, a.x_stride, bytes), first = vector(a.initial_state, a.envs * H * N * V);
    const Extent inputs[] = {rows_extent(a.b, a, G, N, a.b_stride, bytes), rows_extent(a.c, a, G, N, a.c_stride, bytes),
                             rows_extent(a.dt, a, H, 1, a.dt_stride, 4), vector(a.a, H), vector(a.d, H), vector(a.dt_bias, H),
                             rows_extent(a.starts, a, 1, 1, {a.starts_stride[0], a.starts_stride[1], 0}, 1)};
    bool fine = apart(out, last) && apart(out, first) && apart(last, x);
    for (const Extent& r : inputs) fine = fine && apart(out, r) && apart(last, r);
    const bool own = in_place && a.out == a.x && a.steps == 1 && (H == 1 || a.x_stride[2] == V) && (a.envs == 1 || a.x_stride[0] == H * V);
    fine = fine && (own || apart(out, x)) && ((in_place && a.final_state == a.initial_state) || apart(last, first));
    return fine ? NAVI_POLICY_OK : set_error(NAVI_POLICY_E_ARG, "out or the state after shares memory with what is read");
}

}  // namespace navi_policy

using namespace navi_policy;

extern "C" int navi_selective_scan(const navi_selective_scan_args* args, void* stream) {
    Setup s;
    const int code = setup(args, false, s);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : NAVI_POLICY_OK;
    if (args->steps > 0 && !args->out) return set_error(NAVI_POLICY_E_ARG, "out must be non-null");
    if (args->steps == 0 && !args->final_state) return NAVI_POLICY_OK;
    if (s.P.n_segments > 1 && (!args->scratch || !aligned16(args->scratch)))
        return set_error(NAVI_POLICY_E_ARG, "scratch must be non-null and 16-byte aligned");
    const int shared = check_selective_apart(*args, false);
    if (shared != NAVI_POLICY_OK) return shared;
    Role& r = s.P.role[0] = role_of(*args, s.c, s.b, s.x, false, false);
    r.skip = 1;
    r.out = args->out;
    r.wide_out = wide_out(args->out, args->head_dim);
    r.from = args->initial_state;
    r.to = args->final_state;
    place_segments(r, *args, s.P.n_segments, static_cast<float*>(args->scratch));
    return scans_typed(s.P, args->dtype, 1, false, false, as_stream(stream));
}

extern "C" int64_t navi_selective_scan_scratch(const navi_selective_scan_args* args) {
    const int code = check(args);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : 0;
    return 4 * segment_floats(*args, segments_of(*args, false));
}

extern "C" int64_t navi_selective_scan_workspace(const navi_selective_scan_args* args) {
    const int code = check(args);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : 0;
    return 4 * workspace_of(*args).floats;
}

extern "C" int navi_selective_scan_backward(const navi_selective_scan_args* args, void* stream) {
    Setup s;
    const int code = setup(args, true, s);
    if (code < 0) return code;
    if (code != NAVI_POLICY_OK || args->steps == 0) return set_error(NAVI_POLICY_E_ARG, "the backward pass needs at least one token");
    const navi_selective_scan_args& a = *args;
    if (!a.grad_out || !a.d_x || !a.d_b || !a.d_c || !a.d_dt || !a.workspace)
        return set_error(NAVI_POLICY_E_ARG, "grad_out, d_x, d_b, d_c, d_dt and workspace must be non-null");
    if (!aligned16(a.workspace)) return set_error(NAVI_POLICY_E_ARG, "workspace must be 16-byte aligned");
    const Workspace w = workspace_of(a);
    float* base = static_cast<float*>(a.workspace);
    const bool shared = a.heads > a.groups;
    ScanParams& P = s.P;
    Role& dc = P.role[0] = role_of(a, s.dy, s.x, s.b, true, false);
    dc.z = s.c;
    dc.out = a.d_c;
    dc.out_heads = shared ? base + w.dc : nullptr;
    dc.wide_out = wide_out(shared ? static_cast<void*>(dc.out_heads) : a.d_c, a.state_dim);
    dc.from = a.initial_state;
    dc.state_dots = base + w.rho;
    Role& dx = P.role[1] = role_of(a, s.b, s.c, s.dy, false, true);
    dx.z = s.x;
    dx.skip = 1;
    dx.out = a.d_x;
    dx.wide_out = wide_out(a.d_x, a.head_dim);
    dx.from = a.grad_final_state;
    dx.to = a.d_initial_state;
    dx.state_dots = base + w.kappa;
    dx.dots = base + w.delta;
    Role& db = P.role[2] = role_of(a, s.x, s.dy, s.c, true, true);
    db.out = a.d_b;
    db.out_heads = shared ? base + w.db : nullptr;
    db.wide_out = wide_out(shared ? static_cast<void*>(db.out_heads) : a.d_b, a.state_dim);
    db.from = a.grad_final_state;
    const bool needed = states_needed(a);
    if (needed) {
        dc.keep_states = base + w.states;
        db.other_states = base + w.states;
        db.through = base + w.through;
        for (Role* r : {&dc, &db}) r->keep_from = keep_from(a), r->keep_to = keep_to(a);
    }
    float* at = base + w.segments;
    for (Role& r : P.role) at = place_segments(r, a, P.n_segments, at);
    GateParams G{};
    G.scan = P;
    // (the db scan reads what the dc scan leaves)
    const bool wide = widened(a, P.n_segments);
    int result = scans_typed(P, a.dtype, needed ? 2 : 3, true, wide, as_stream(stream));
    if (result != NAVI_POLICY_OK) return result;
    if (needed) {
        P.role[0] = db;
        result = scans_typed(P, a.dtype, 1, true, wide, as_stream(stream));
        if (result != NAVI_POLICY_OK) return result;
    }
    G.x = s.x;
    G.b = s.b;
    G.c = s.c;
    G.dy = s.dy;
    G.state_dim = a.state_dim;
    G.head_dim = a.head_dim;
    G.rho = base + w.rho;
    G.kappa = base + w.kappa;
    G.delta = base + w.delta;
    G.through = needed ? base + w.through : nullptr;
    G.rho_blocks = blocks_of(a.state_dim);
    G.delta_blocks = blocks_of(a.head_dim);
    G.through_waves = 4 * blocks_of(a.state_dim);
    G.d_dt = a.d_dt;
    const bool sums = a.d_a || a.d_d || a.d_dt_bias;
    G.partial = sums ? reinterpret_cast<double*>(base + w.partial) : nullptr;
    result = a.dtype == NAVI_POLICY_F32 ? gates<float>(G, as_stream(stream))
             : a.dtype == NAVI_POLICY_BF16 ? gates<bf16>(G, as_stream(stream)) : gates<f16>(G, as_stream(stream));
    if (result != NAVI_POLICY_OK) return result;
    if (sums)
        hipLaunchKernelGGL(selective_sums_kernel, dim3(a.heads), dim3(256), 0, as_stream(stream), G.partial, a.envs, a.heads, P.n_chunks, a.d_a,
                           a.d_d, a.d_dt_bias);
    if (shared) {
        const int64_t rows = a.envs * a.steps * a.groups, pieces = rows * ((a.state_dim + 7) / 8);
        const dim3 grid(static_cast<unsigned>(std::min<int64_t>((pieces + 255) / 256, 4096)), 2);
        const auto join = [&](auto* to_b, auto* to_c) {
            using E = std::remove_reference_t<decltype(*to_b)>;
            hipLaunchKernelGGL(selective_groups_kernel<E>, grid, dim3(256), 0, as_stream(stream), base + w.db, base + w.dc, to_b, to_c,
                               rows, a.heads / a.groups, a.state_dim);
        };
        if (a.dtype == NAVI_POLICY_F32)
            join(static_cast<float*>(a.d_b), static_cast<float*>(a.d_c));
        else if (a.dtype == NAVI_POLICY_BF16)
            join(static_cast<bf16*>(a.d_b), static_cast<bf16*>(a.d_c));
        else
            join(static_cast<f16*>(a.d_b), static_cast<f16*>(a.d_c));
    }
    return launched("navi_selective_scan_backward");
}
