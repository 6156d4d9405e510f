// delta_rule.hip — the gated delta rule over chunks of 64 tokens: forward, and the two
// kernels of its backward pass (mathematics in delta_chunk.hpp).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "delta_chunk.hpp"

namespace navi_policy {
namespace {

// A wave's 16 columns of an array of T in the layout of products: lane l has column l % 16 and
// rows 4 (l / 16) + s of each tile of 16. A row's address is a scalar, the lane's part of it
// one register for all rows and chunks.
template <class T>
struct Columns {
    uint32_t row_bytes, lane, width;

    // `stride` elements from row to row; `columns` from the wave's first to the array's last
    __device__ Columns(int64_t stride, int columns) {
        const int l = threadIdx.x & 63;
        row_bytes = static_cast<uint32_t>(stride) * sizeof(T);
        width = (columns < 0 ? 0 : columns < 16 ? columns : 16) * static_cast<uint32_t>(sizeof(T));
        lane = (l & 15) < columns ? 4 * (l >> 4) * row_bytes + (l & 15) * sizeof(T) : kOutside;
    }

    __device__ Buffer rows(const T* base, int rows) const {
        return buffer_of(base, rows > 0 ? (rows - 1) * row_bytes + width : 0);
    }

    // The lane's part, where the compiler does not see that it is the same for every chunk: it
    // would keep the offset of every row in a register.
    __device__ uint32_t fresh() const {
        uint32_t x = lane;
        asm volatile("" : "+v"(x));
        return x;
    }

    template <int kTilesOfRows, class F>
    __device__ void load(Buffer from, F to) const {
        const uint32_t own = fresh();
#pragma unroll
        for (int i = 0; i < kTilesOfRows; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s) to(i, s, buffer_load<T>(from, own + (16 * i + s) * row_bytes));
    }

    template <int kTilesOfRows, class F>
    __device__ void store(Buffer to, F from) const {
        const uint32_t own = fresh();
#pragma unroll
        for (int i = 0; i < kTilesOfRows; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s) buffer_store<T>(to, own + (16 * i + s) * row_bytes, from(i, s));
    }
};

__device__ inline f4 four(const float (&x)[kChunk], int row) { return *reinterpret_cast<const f4*>(&x[row]); }

// A wave's 16 columns of 64 rows on their way to the layout of products: two loads of a lane hold
// 8 columns of a row each, of tile 2 m (lanes 0 to 31) and 2 m + 1; a product with the unit matrix
// (exact: each sum has one term) puts them where results stand.
template <class E>
struct ColumnFetch {
    Part<E, 8> part[2];

    __device__ void fetch(const E* base, int64_t stride, int columns, int tokens, bool wide) {
        const int l = threadIdx.x & 63, g = l >> 4;
        const uint32_t row_bytes = static_cast<uint32_t>(stride) * sizeof(E);
        const int width = columns < 0 ? 0 : columns < 16 ? columns : 16;
        const Buffer from = buffer_of(base, (tokens - 1) * row_bytes + width * sizeof(E));
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int token = 32 * m + 16 * (g >> 1) + (l & 15), column = 8 * (g & 1);
            part[m].load(from, token * row_bytes + column * sizeof(E), token < tokens ? width - column : 0, wide);
        }
    }

    // x of the 64 rows added to `to`.
    __device__ void add(f4 (&to)[4]) const {
        const int l = threadIdx.x & 63, at = (l & 15) - 8 * ((l >> 4) & 1);  // the one of the lane's eight, if any
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            u4 x[kPlanes<E>];
            if constexpr (kPlanes<E> == 1) {
                x[0] = part[m].words[0];
            } else {
                float y[8];
                part[m].floats(y);
                split8(y, x);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                u4 unit;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    unit[i] = l >> 5 == n && at >> 1 == i ? (at & 1 ? 0x3f800000u : 0x3f80u) : 0u;
#pragma unroll
                for (int p = kPlanes<E> - 1; p >= 0; --p) to[2 * m + n] = mfma(x[p], unit, to[2 * m + n]);
            }
        }
    }
};

// Sixteen columns of 64 rows from transposed results: a lane has row l % 16 of each tile, four
// columns of it.
template <class E>
__device__ inline void store_transposed(E* base, int64_t stride, int columns, int tokens, bool wide, const f4 (&x)[4]) {
    const int l = threadIdx.x & 63, column = 4 * (l >> 4);
    const uint32_t row_bytes = static_cast<uint32_t>(stride) * sizeof(E);
    const int width = columns < 16 ? columns : 16;
    const Buffer to = buffer_of(base, (tokens - 1) * row_bytes + width * sizeof(E));
    const uint32_t lane = (l & 15) * row_bytes + column * sizeof(E);
    if (wide) {
        const uint32_t own = column < width ? lane : kOutside;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const E y[4] = {from_float<E>(x[i][0]), from_float<E>(x[i][1]), from_float<E>(x[i][2]), from_float<E>(x[i][3])};
            buffer_store_four(to, own + 16 * i * row_bytes, y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s)
                buffer_store<E>(to, column + s < width ? lane + 16 * i * row_bytes + s * sizeof(E) : kOutside, from_float<E>(x[i][s]));
    }
}

// x * factor, 0 where the factor is 0 whatever x is: a state that an episode's start clears.
__device__ inline f4 gated(f4 x, f4 factor) {
    f4 y;
#pragma unroll
    for (int s = 0; s < 4; ++s) y[s] = factor[s] == 0.0f ? 0.0f : x[s] * factor[s];
    return y;
}

// The lane, where the compiler does not see that it has been asked for before: it would hold
// every address that comes from it in a register of its own from the first step on.
__device__ inline int fresh_lane() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

// Keeps the compiler from reading what later steps need from LDS early, into more registers
// than there are.
__device__ inline void settle() { __builtin_amdgcn_sched_barrier(0); }

__device__ inline int tokens_of(const RuleParams& P, int chunk) {
    const int64_t left = P.r.steps - static_cast<int64_t>(chunk) * kChunk;
    return static_cast<int>(left < kChunk ? left : kChunk);
}

// The triangles and gates of every chunk, which need no state: a workgroup each, so that the
// walks, which go from chunk to chunk, do not wait for a substitution. Bound by memory where there are
// many chunks: 1024 x 128 steps, 4 heads of 64, bfloat16, 70 us for 134 MB of rows and 172 MB of
// triangles (4.4 TB/s, a large copy reaches 4.8).
template <class E, int KP>
__global__ __launch_bounds__(256) void delta_triangles_kernel(RuleParams P) {
    extern __shared__ char lds_bytes[];
    auto& lds = *reinterpret_cast<TriangleLds<E, KP>*>(lds_bytes);
    const int wave = wave_of_workgroup();
    const int64_t sequence = blockIdx.x / static_cast<uint32_t>(P.n_chunks);
    const int chunk = static_cast<int>(blockIdx.x % static_cast<uint32_t>(P.n_chunks));
    const int64_t env = sequence / P.r.value_heads, t0 = static_cast<int64_t>(chunk) * kChunk;
    const int head = static_cast<int>(sequence % P.r.value_heads), tokens = tokens_of(P, chunk);
    ChunkMatrices& to = reinterpret_cast<ChunkMatrices*>(P.r.matrices)[blockIdx.x];
    GatesFetch gates;
    if (wave == 0) gates.fetch(P, env, head, t0, tokens);
    ChunkFetch<E, KP, 256, true>::load(P, lds.rows, env, head, t0, tokens);
    if (wave == 0) gates.put(lds.gates);
    __syncthreads();
    if (threadIdx.x < kChunk) {
        to.e[threadIdx.x] = lds.gates.e[threadIdx.x];
        to.fb[threadIdx.x] = lds.gates.f[threadIdx.x] * lds.gates.beta[threadIdx.x];
    }
    make_triangles<E, KP>(lds, to, P.r.scale, wave);
}

template <class E, int KP>
struct ScanLds {
    ChunkRows<E, KP> rows;
    Triangle<3> x, p;
    float gates[2][kChunk];  // E, F beta
};

template <int KP>
__device__ inline void load_state(const Columns<float>& at, const float* from, int K, f4 (&state)[KP / 16]) {
    at.load<KP / 16>(at.rows(from, from ? K : 0), [&](int c, int s, float x) { state[c][s] = x; });
}

template <int KP>
__device__ inline void store_state(const Columns<float>& at, float* to, int K, const f4 (&state)[KP / 16]) {
    at.store<KP / 16>(at.rows(to, K), [&](int c, int s) { return state[c][s]; });
}

// Columns of the state that a workgroup holds, 16 a wave. Two workgroups of 64 fit a CU and wait
// apart: 2 x 4001 steps, 8 heads of 128, 413 us forward and back against 435 with one of 128; 256 x
// 128 steps, 4 heads of 128, forward, 93 and 99. Rows of 128 float32 leave a CU's LDS to one
// workgroup, which then has eight waves: the same, 208 us against 313.
template <class E, int KP>
inline constexpr int kWalkColumns = sizeof(E) == 4 && KP == 128 ? 128 : 64;
template <class E, int KP>
inline constexpr int kWalkThreads = 4 * kWalkColumns<E, KP>;

// The chunks of a segment in the order that a kernel walks them, and the state before the
// first: segment 0 begins with `given` (or zeros), the others with what delta_join_kernel
// found. In summary, the columns past V (rounded up to 16) are those of the unit matrix, and
// there are no inputs for them: the state after the segment is then the matrix that it
// multiplies the state before it with.
struct Walk {
    int32_t begin, end;  // chunks, counted in the walk's order
    const float* from;   // state before, or NULL for zeros
    float* to;           // state after, or NULL
    int32_t first;       // column of the wave's first
    int32_t columns;     // that the array behind `from` and `to` has
    bool working, unit;

    // The sequence and columns of a workgroup. Workgroups go round the 8 XCDs in turn: those of
    // one sequence are 8 apart, so that what they all read is in one XCD's L2.
    template <int kColumns>
    __device__ static bool place(const RuleParams& P, int blocks, int64_t& sequence, int& first) {
        const uint32_t id = blockIdx.x, round = id / 8;
        sequence = static_cast<int64_t>(round / blocks) * 8 + id % 8;
        first = static_cast<int>(round % blocks) * kColumns;
        return sequence < P.r.envs * P.r.value_heads;
    }

    template <bool kSummary>
    __device__ static Walk of(const RuleParams& P, int64_t sequence, int first, const float* given, float* result) {
        const int segment = blockIdx.z, V = P.r.value_dim, K = P.r.key_dim;
        const int64_t slots = sequence * (P.n_segments - 1);
        Walk w;
        w.begin = static_cast<int>(static_cast<int64_t>(segment) * P.n_chunks / P.n_segments);
        w.end = static_cast<int>((segment + 1ll) * P.n_chunks / P.n_segments);
        w.first = first;
        w.columns = V;
        w.working = first < V;
        w.unit = false;
        const int64_t kv = static_cast<int64_t>(K) * V;
        w.from = segment == 0 ? (given ? given + sequence * kv : nullptr)
                              : kSummary ? nullptr : P.segment_states + (slots + segment - 1) * kv;
        w.to = kSummary ? P.segment_states + (slots + segment) * kv
                        : result && segment + 1 == P.n_segments ? result + sequence * kv : nullptr;
        const int rounded = (V + 15) / 16 * 16;
        if (kSummary && first >= rounded) {
            w.unit = true;
            w.first = first - rounded;
            w.columns = K;
            w.working = segment > 0 && w.first < K;
            w.from = nullptr;
            w.to = P.segment_matrices + (slots + segment) * K * K;
        }
        return w;
    }

    template <int KP>
    __device__ void begin_state(const Columns<float>& at, int K, f4 (&state)[KP / 16]) const {
        load_state<KP>(at, from ? from + first : nullptr, K, state);
        if (unit) {
            const int l = threadIdx.x & 63;
#pragma unroll
            for (int c = 0; c < KP / 16; ++c)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    state[c][s] = 16 * c + 4 * (l >> 4) + s == first + (l & 15) ? 1.0f : 0.0f;
        }
    }
};

// u or its gradient from the rows of X, all tiles of a stage side by side.
template <int N, int NB>
__device__ inline void times_triangle(int lane, const Triangle<N>& t, const u4 (&b)[2][NB], f4 (&x)[4]) {
    u4 a[4][N];
#pragma unroll
    for (int i = 0; i < 4; ++i) operand_triangle<N>(lane, t, i, 0, a[i]);
    mma_each<4>(a, b[0], x);
    u4 below[2][N];
    f4 y[2] = {x[2], x[3]};
#pragma unroll
    for (int i = 0; i < 2; ++i) operand_triangle<N>(lane, t, 2 + i, 1, below[i]);
    mma_each<2>(below, b[1], y);
    x[2] = y[0];
    x[3] = y[1];
}

// The same with the result transposed.
template <int N, int NB>
__device__ inline void times_triangle_transposed(int lane, const Triangle<N>& t, const u4 (&b)[2][NB], f4 (&x)[4]) {
    u4 a[4][N];
#pragma unroll
    for (int i = 0; i < 4; ++i) operand_triangle<N>(lane, t, i, 0, a[i]);
    mma_each_transposed<4>(a, b[0], x);
    u4 below[2][N];
    f4 y[2] = {x[2], x[3]};
#pragma unroll
    for (int i = 0; i < 2; ++i) operand_triangle<N>(lane, t, 2 + i, 1, below[i]);
    mma_each_transposed<2>(below, b[1], y);
    x[2] = y[0];
    x[3] = y[1];
}

template <int N, int NB>
__device__ inline void times_transpose(int lane, const Triangle<N>& t, const u4 (&b)[2][NB], f4 (&x)[4]) {
    u4 a[4][N];
#pragma unroll
    for (int j = 0; j < 4; ++j) operand_transpose<N>(lane, t, j, 1, a[j]);
    mma_each<4>(a, b[1], x);
    u4 left[2][N];
    f4 y[2] = {x[0], x[1]};
#pragma unroll
    for (int j = 0; j < 2; ++j) operand_transpose<N>(lane, t, j, 0, left[j]);
    mma_each<2>(left, b[0], y);
    x[0] = y[0];
    x[1] = y[1];
}

// Columns of rows in LDS times b, added to four tiles of a state from tile c on.
template <int N, int kPitch, int NB, int kCount>
__device__ inline void add_columns(int lane, const uint16_t (&rows)[N][kChunk][kPitch], int c, const u4 (&b)[2][NB], f4 (&state)[kCount]) {
    f4 x[4] = {state[c], state[c + 1], state[c + 2], state[c + 3]};
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        u4 a[4][N];
#pragma unroll
        for (int n = 0; n < 4; ++n) operand_columns(lane, rows, c + n, m, a[n]);
        mma_each<4>(a, b[m], x);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) state[c + n] = x[n];
}

// A wave holds 16 columns of the state as results of products (KP / 16 tiles), a workgroup of
// four waves 64 of one head; it walks the chunks with the state in registers.
// The state is the second operand of S^T k without a move: its tiles hold the contracted axis
// in the order of results, which the rows in LDS are kept in as well.
//
// With many sequences memory bounds it: 1024 x 128 steps, 4 heads of 64, bfloat16, with what the
// gradients need, 152 us for 374 MB read and 269 MB written (4.2 TB/s). With few, the chain from
// chunk to chunk does: 16384 steps, 16 heads of 128 in 16 segments, 145 us, 9.1 us a chunk of which
// the products' own time is 3.3 (what lies between: reads of LDS for the operands, with bank
// conflicts in a fifth of the cycles, splits of the state into planes, two barriers).
template <class E, int KP, bool kSummary>
__global__ __launch_bounds__((kWalkThreads<E, KP>), 2) void delta_forward_kernel(RuleParams P) {
    constexpr int N = kPlanes<E>;
    extern __shared__ char lds_bytes[];
    auto& lds = *reinterpret_cast<ScanLds<E, KP>*>(lds_bytes);
    const int wave = wave_of_workgroup(), lane = threadIdx.x & 63, g = lane >> 4;
    int64_t sequence;
    int block;
    if (!Walk::place<kWalkColumns<E, KP>>(P, kSummary ? P.summary_blocks : P.blocks, sequence, block)) return;
    const int64_t env = sequence / P.r.value_heads;
    const int head = static_cast<int>(sequence % P.r.value_heads);
    const int K = P.r.key_dim, V = P.r.value_dim;
    const Walk walk = Walk::of<kSummary>(P, sequence, block + 16 * wave, P.r.initial_state,
                                         P.r.final_state);
    const int first = walk.first;
    const ChunkMatrices* matrices = reinterpret_cast<const ChunkMatrices*>(P.r.matrices) + sequence * P.n_chunks;
    const E* v = at<E>(P.r.v, P.r.v_stride, env, 0, head) + first;
    const Columns<float> rows_state(walk.columns, walk.columns - first);

    f4 state[KP / 16];
    walk.begin_state<KP>(rows_state, K, state);

    ChunkFetch<E, KP, kWalkThreads<E, KP>, !kSummary> next;
    ColumnFetch<E> v_next;
    const auto fetch = [&](int chunk) {
        const int64_t t0 = static_cast<int64_t>(chunk) * kChunk;
        next.fetch(P, matrices[chunk], env, head, t0, tokens_of(P, chunk));
        v_next.fetch(v + t0 * P.r.v_stride[1], P.r.v_stride[1], walk.unit ? 0 : V - first, tokens_of(P, chunk), P.wide_v);
    };
    if (walk.begin < walk.end) fetch(walk.begin);
    for (int chunk = walk.begin; chunk < walk.end; ++chunk) {
        const int64_t t0 = static_cast<int64_t>(chunk) * kChunk;
        const int tokens = tokens_of(P, chunk);
        if (chunk > walk.begin) __syncthreads();
        next.put(P, lds.rows, lds.x, lds.p, lds.gates, env, head, t0, tokens);
        const ColumnFetch<E> values = v_next;
        __syncthreads();
        if (chunk + 1 < walk.end) fetch(chunk + 1);
        if (!walk.working) continue;

        if (!kSummary && P.r.states && chunk > 0)
            store_state<KP>(rows_state, P.r.states + (sequence * (P.n_chunks - 1) + chunk - 1) * K * V + first, K, state);
        f4 u[4], o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = o[i] = f4{0, 0, 0, 0};
        // (a state that the chunk's first token forgets may hold anything)
        const bool forgotten = lds.gates[0][0] == 0.0f;
        if (forgotten)
#pragma unroll
            for (int c = 0; c < KP / 16; ++c) state[c] = f4{0, 0, 0, 0};
        if (!forgotten && (chunk > walk.begin || walk.from || walk.unit)) {
#pragma unroll
            for (int m = 0; m < KP / 32; ++m) {
                u4 b[3], a[4][N];
                split8(state[2 * m], state[2 * m + 1], b);
#pragma unroll
                for (int i = 0; i < 4; ++i) operand_rows(lane, lds.rows.k, 16 * i, m, a[i]);
                mma_each<4>(a, b, u);
                if constexpr (!kSummary) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) operand_rows(lane, lds.rows.q, 16 * i, m, a[i]);
                    mma_each_transposed<4>(a, b, o);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = -four(lds.gates[0], 16 * i + 4 * g) * u[i];
            o[i] = P.r.scale * lds.gates[0][16 * i + (lane & 15)] * o[i];
        }
        values.add(u);
        u4 r[2][3];
#pragma unroll
        for (int m = 0; m < 2; ++m) split8(u[2 * m], u[2 * m + 1], r[m]);
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = f4{0, 0, 0, 0};
        times_triangle<3>(lane, lds.x, r, u);
        if (!kSummary && P.r.updates)
            rows_state.store<4>(rows_state.rows(P.r.updates + (sequence * P.r.steps + t0) * V + first, tokens),
                                [&](int i, int s) { return u[i][s]; });
        // The state first: the next chunk waits for it.
        const float keep = lds.gates[0][kChunk - 1];
#pragma unroll
        for (int m = 0; m < 2; ++m)
            split8(u[2 * m] * four(lds.gates[1], 32 * m + 4 * g), u[2 * m + 1] * four(lds.gates[1], 32 * m + 16 + 4 * g), r[m]);
#pragma unroll
        for (int c = 0; c < KP / 16; ++c) state[c] = keep * state[c];
#pragma unroll
        for (int c = 0; c < KP / 16; c += 4) add_columns(lane, lds.rows.k, c, r, state);
        if constexpr (!kSummary) {
#pragma unroll
            for (int m = 0; m < 2; ++m) split8(u[2 * m], u[2 * m + 1], r[m]);
            times_triangle_transposed<3>(lane, lds.p, r, o);
            store_transposed(static_cast<E*>(P.r.out) + ((env * P.r.steps + t0) * P.r.value_heads + head) * V + first,
                             static_cast<int64_t>(P.r.value_heads) * V, V - first, tokens, P.wide_out, o);
        }
    }
    if (walk.to && walk.working) store_state<KP>(rows_state, walk.to + first, K, state);
}

// Backward through the chunks from the last to the first, the gradient dS of the state after
// a chunk in registers as the state is in the forward pass:
//
//     du = P^T do + beta F (k dS),   dr = X^T du  (= dv),
//     dS <- E_last dS + q^T (scale E do) - k^T (E dr)
//
// dS and dr go to memory for delta_gradients_kernel. Bound as the forward pass is: 146 us for the
// same traffic at 1024 x 128 steps, 4 heads of 64 (4.4 TB/s).
template <class E, int KP, bool kSummary>
__global__ __launch_bounds__((kWalkThreads<E, KP>), 2) void delta_reverse_kernel(RuleParams P) {
    constexpr int N = kPlanes<E>;
    extern __shared__ char lds_bytes[];
    auto& lds = *reinterpret_cast<ScanLds<E, KP>*>(lds_bytes);
    const int wave = wave_of_workgroup(), lane = threadIdx.x & 63, g = lane >> 4;
    int64_t sequence;
    int block;
    if (!Walk::place<kWalkColumns<E, KP>>(P, kSummary ? P.summary_blocks : P.blocks, sequence, block)) return;
    const int64_t env = sequence / P.r.value_heads;
    const int head = static_cast<int>(sequence % P.r.value_heads);
    const int K = P.r.key_dim, V = P.r.value_dim;
    const Walk walk = Walk::of<kSummary>(P, sequence, block + 16 * wave, P.d.grad_final_state,
                                         P.d.d_initial_state);
    const int first = walk.first;
    const ChunkMatrices* matrices = reinterpret_cast<const ChunkMatrices*>(P.r.matrices) + sequence * P.n_chunks;
    const E* grad = at<E>(P.d.grad_out, P.d.grad_out_stride, env, 0, head) + first;
    const Columns<E> rows_v(static_cast<int64_t>(P.r.value_heads) * V, V - first);
    const Columns<float> rows_state(walk.columns, walk.columns - first);

    f4 dstate[KP / 16];
    walk.begin_state<KP>(rows_state, K, dstate);

    ChunkFetch<E, KP, kWalkThreads<E, KP>, true> next;
    ColumnFetch<E> grad_next;
    const auto fetch = [&](int chunk) {
        const int64_t t0 = static_cast<int64_t>(chunk) * kChunk;
        next.fetch(P, matrices[chunk], env, head, t0, tokens_of(P, chunk));
        grad_next.fetch(grad + t0 * P.d.grad_out_stride[1], P.d.grad_out_stride[1], walk.unit ? 0 : V - first,
                        tokens_of(P, chunk), P.wide_do);
    };
    const int last = P.n_chunks - 1;
    if (walk.begin < walk.end) fetch(last - walk.begin);
    for (int step = walk.begin; step < walk.end; ++step) {
        const int chunk = last - step;
        const int64_t t0 = static_cast<int64_t>(chunk) * kChunk;
        const int tokens = tokens_of(P, chunk);
        if (step > walk.begin) __syncthreads();
        next.put(P, lds.rows, lds.x, lds.p, lds.gates, env, head, t0, tokens);
        const ColumnFetch<E> grads = grad_next;
        __syncthreads();
        if (step + 1 < walk.end) fetch(chunk - 1);
        if (!walk.working) continue;

        if (!kSummary && step > 0)
            store_state<KP>(rows_state, P.dstates + (sequence * (P.n_chunks - 1) + chunk) * K * V + first, K, dstate);
        f4 du[4], dO[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) du[i] = dO[i] = f4{0, 0, 0, 0};
        grads.add(dO);
        if (step > walk.begin || walk.from || walk.unit) {
#pragma unroll
            for (int m = 0; m < KP / 32; ++m) {
                u4 b[3], a[4][N];
                split8(dstate[2 * m], dstate[2 * m + 1], b);
#pragma unroll
                for (int i = 0; i < 4; ++i) operand_rows(lane, lds.rows.k, 16 * i, m, a[i]);
                mma_each<4>(a, b, du);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) du[i] = du[i] * four(lds.gates[1], 16 * i + 4 * g);
        }
        {
            u4 raw[2][N];
#pragma unroll
            for (int m = 0; m < 2; ++m) split8(dO[2 * m], dO[2 * m + 1], raw[m]);
            times_transpose<3>(lane, lds.p, raw, du);
        }
        u4 b[2][3];
#pragma unroll
        for (int m = 0; m < 2; ++m) split8(du[2 * m], du[2 * m + 1], b[m]);
#pragma unroll
        for (int j = 0; j < 4; ++j) du[j] = f4{0, 0, 0, 0};
        times_transpose<3>(lane, lds.x, b, du);  // dr
        if constexpr (!kSummary) {
            rows_v.template store<4>(
                rows_v.rows(static_cast<E*>(P.d.d_v) + ((env * P.r.steps + t0) * P.r.value_heads + head) * V + first, tokens),
                [&](int j, int s) { return from_float<E>(du[j][s]); });
            rows_state.store<4>(rows_state.rows(P.rgrads + (sequence * P.r.steps + t0) * V + first, tokens),
                                [&](int j, int s) { return du[j][s]; });
        }
        if (chunk > 0 || kSummary || P.d.d_initial_state) {
            const float keep = lds.gates[0][kChunk - 1];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f4 e = four(lds.gates[0], 16 * j + 4 * g);
                du[j] = -e * du[j];
                dO[j] = P.r.scale * e * dO[j];
            }
#pragma unroll
            for (int c = 0; c < KP / 16; ++c) dstate[c] = keep * dstate[c];
#pragma unroll
            for (int m = 0; m < 2; ++m) split8(du[2 * m], du[2 * m + 1], b[m]);
#pragma unroll
            for (int c = 0; c < KP / 16; c += 4) add_columns(lane, lds.rows.k, c, b, dstate);
#pragma unroll
            for (int m = 0; m < 2; ++m) split8(dO[2 * m], dO[2 * m + 1], b[m]);
#pragma unroll
            for (int c = 0; c < KP / 16; c += 4) add_columns(lane, lds.rows.q, c, b, dstate);
        }
    }
    if (walk.to && walk.working) store_state<KP>(rows_state, walk.to + first, K, dstate);
}

// Sixteen rows of results, KP / 16 tiles across, into `rows` rows of `columns` numbers.
template <class T, int KP>
__device__ inline void store_tiles(T* base, int64_t stride, int rows, int columns, const f4 (&x)[KP / 16]) {
#pragma unroll
    for (int c = 0; c < KP / 16; ++c) {
        const Columns<T> at(stride, columns - 16 * c);
        at.template store<1>(at.rows(base + 16 * c, rows < 16 ? rows : 16), [&](int, int s) { return from_float<T>(x[c][s]); });
    }
}

// The gradients of one chunk of one head, all chunks at once, from the states S before and
// the state gradients dS after each, u and dr. With H = do u^T, R = dr u^T (lower triangles),
// Y = do S^T, Z = dr S^T, W = u dS^T:
//
//     N_ij = scale D_ij H_ij beta_j (i >= j),  M_ij = -R_ij D_ij beta_j (i > j)
//     dq_i = scale E_i Y_i + sum_j N_ij k_j
//     dk_i = beta_i F_i W_i - E_i Z_i + sum_j M_ij k_j + sum_j (N_ji q_j + M_ji k_j)
//     dbeta_j = F_j k_j . W_j + sum_i (scale D_ij H_ij q_i . k_j - R_ij D_ij k_i . k_j)
//     dG_i = sum_j B_ij - sum_j B_ji + scale E_i q_i . Y_i - E_i k_i . Z_i - beta_i F_i k_i . W_i,
//     B_ij = N_ij q_i . k_j + M_ij k_i . k_j (i > j),
//     dG_last += sum_j beta_j F_j k_j . W_j + E_last <S, dS>,  dg_t = sum_{i >= t} dG_i
//
// The same number stands at +i and -j of dG, so what cancels in dg cancels to its rounding.
//
// Eight waves: four of 16 tokens each take the terms of do (Y, H, W, N, dq, their part of dk), four
// those of dr (Z, R, M, the rest of dk). V is taken 32 columns at a time. Two workgroups fit a CU
// with 64 keys of bfloat16, one with more. Rows of 64 float16 (two planes) leave room for one, but
// for two of four waves with both kinds of terms, whose rows come after V into the stage's place:
// 1024 x 128 steps, 4 heads of 64, forward and back, float16 733 us with four waves, 835 with
// eight; bfloat16 626 and 609; 2 x 4001 steps, 8 heads of 128, bfloat16 531 and 413. The
// kernel alone takes 271 to 289 us of the 609, for 622 MB read and 151 MB written (2.7 to 2.8 TB/s):
// VALU and LDS are each busy half of that time, and waves wait for their chunk's rows.
template <class E, int KP>
inline constexpr int kGradientWaves = KP == 64 && kPlanes<E> == 2 ? 4 : 8;

template <int KP>
struct GradientStage {
    uint16_t s[KP / 16][3][64][8], ds[KP / 16][3][64][8];  // 32 columns of S and dS as operands
    uint16_t u[4][3][64][8];                                // and of u
};

template <class E, int KP>
struct GradientTriangles {
    Triangle<3> n, m;
    float beta_part[kGradientWaves<E, KP>][kChunk], g_part[kGradientWaves<E, KP>][kChunk];
};

struct GradientRest {
    ChunkGates gates;
    float beta_row[kChunk], g_row[2][kChunk], dot_part[8];
};

template <class E, int KP>
union GradientRows {
    ChunkRows<E, KP> rows;
    f4 exchange[4][KP / 16][64];
};

// The rows of q and k stay in LDS where a workgroup has the room; else they come after V.
template <class E, int KP>
inline constexpr bool kRowsStay = kGradientWaves<E, KP> == 8 && (sizeof(E) == 2 || KP == 64);

template <class E, int KP, bool kStay = kRowsStay<E, KP>>
struct GradientLds {
    union {
        GradientStage<KP> stage;
        GradientTriangles<E, KP> tri;
    };
    GradientRows<E, KP> of;
    GradientRest rest;
};

template <class E, int KP>
struct GradientLds<E, KP, false> {
    union {
        GradientStage<KP> stage;
        struct {
            GradientTriangles<E, KP> tri;
            GradientRows<E, KP> of;
        };
    };
    GradientRest rest;
};

__device__ inline float sum16(float x) {  // over 16 lanes in a row
    const auto moved = [](float y, auto control) {
        return float_of(__builtin_amdgcn_mov_dpp(bits_of(y), decltype(control)::value, 0xf, 0xf, true));
    };
    x += moved(x, std::integral_constant<int, 0xb1>{});   // lanes 1, 0, 3, 2 of four
    x += moved(x, std::integral_constant<int, 0x4e>{});   // 2, 3, 0, 1
    x += moved(x, std::integral_constant<int, 0x141>{});  // the other four of eight
    x += moved(x, std::integral_constant<int, 0x140>{});  // the other eight
    return x;
}

// Over the four lanes that have a column's tokens in a tile of results
__device__ inline float sum_tokens(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// Four floats into the planes of an operand's lane, its first or second half.
__device__ inline void stage_part(uint16_t (&tile)[3][64][8], int slot, int half, const float (&x)[4]) {
    uint32_t a[3], b[3];
    split_pair<3>(x[0], x[1], a);
    split_pair<3>(x[2], x[3], b);
#pragma unroll
    for (int n = 0; n < 3; ++n) *reinterpret_cast<u2*>(&tile[n][slot][4 * half]) = u2{a[n], b[n]};
}

__device__ inline void staged_operand(int lane, const uint16_t (&tile)[3][64][8], u4 (&x)[3]) {
#pragma unroll
    for (int n = 0; n < 3; ++n) x[n] = *reinterpret_cast<const u4*>(tile[n][lane]);
}

// The states before the segments but the first, one after another, from what the summary left
// of each: S <- M S + N with N the state that it makes of zeros (of the given state, for
// segment 0) and M its matrix. Takes N's place. A workgroup holds 16 columns, its four waves a
// quarter of the rows each: M's rows come straight into the wave that multiplies with them, S's
// planes go through LDS. A chain of products, each after the one before it: 3 us for one of
// 128 x 128 (64 columns a workgroup, M's planes in LDS: 4.7 us; products of float32 in place of
// planes: 3 us as well).
template <int KP>
__global__ __launch_bounds__(256) void delta_join_kernel(RuleParams P) {
    constexpr int kOwn = KP / 64;  // tiles of a wave's rows
    __shared__ alignas(16) uint16_t planes[2][KP / 32][3][64][8];
    const int wave = wave_of_workgroup(), lane = threadIdx.x & 63;
    const int64_t sequence = blockIdx.x;
    const int first = blockIdx.y * 16, top = 16 * kOwn * wave;
    const int K = P.r.key_dim, V = P.r.value_dim;
    const int64_t kv = static_cast<int64_t>(K) * V, slots = sequence * (P.n_segments - 1);
    const Columns<float> columns(V, V - first);
    const auto rows_of = [&](int segment) {
        return columns.rows(P.segment_states + (slots + segment) * kv + static_cast<int64_t>(top) * V + first, K - top);
    };
    f4 state[kOwn], next[kOwn], part[kOwn][KP / 32][2];
    const bool wide = K % 4 == 0;
    // Of a segment while the one before it is computed: its N, and the wave's rows of its M as
    // operands (a lane holds columns 4 g and 16 + 4 g on of 32, in the order of results)
    const auto fetch = [&](int segment) {
        const Buffer matrix = buffer_of(P.segment_matrices + (slots + segment) * K * K, 4 * K * K);
#pragma unroll
        for (int c = 0; c < kOwn; ++c)
#pragma unroll
            for (int m = 0; m < KP / 32; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = top + 16 * c + (lane & 15), column = 32 * m + 4 * (lane >> 4) + 16 * h;
                    const uint32_t offset = 4 * (row * K + column);
                    if (wide) {
                        part[c][m][h] = __builtin_bit_cast(f4, buffer_load16(matrix, row < K && column < K ? offset : kOutside));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            part[c][m][h][i] = buffer_load<float>(matrix, row < K && column + i < K ? offset + 4 * i : kOutside);
                    }
                }
        columns.load<kOwn>(rows_of(segment), [&](int c, int s, float x) { next[c][s] = x; });
    };
    columns.load<kOwn>(rows_of(0), [&](int c, int s, float x) { state[c][s] = x; });
    fetch(1);
    for (int segment = 1; segment + 1 < P.n_segments; ++segment) {
        auto& shared = planes[segment & 1];  // (who still reads the other has passed the last barrier but one)
#pragma unroll
        for (int c = 0; c < kOwn; ++c) {
            const int tile = kOwn * wave + c;
            const float x[4] = {state[c][0], state[c][1], state[c][2], state[c][3]};
            stage_part(shared[tile / 2], lane, tile % 2, x);
        }
        u4 a[KP / 32][kOwn][3];
#pragma unroll
        for (int c = 0; c < kOwn; ++c) {
            state[c] = next[c];
#pragma unroll
            for (int m = 0; m < KP / 32; ++m) split8(part[c][m][0], part[c][m][1], a[m][c]);
        }
        __syncthreads();
        if (segment + 2 < P.n_segments) fetch(segment + 1);
#pragma unroll
        for (int m = 0; m < KP / 32; ++m) {
            u4 b[3];
            staged_operand(lane, shared[m], b);
            mma_each<kOwn>(a[m], b, state);
        }
        columns.store<kOwn>(rows_of(segment), [&](int c, int s) { return state[c][s]; });
    }
}

// A triangle's rows times 32 rows in LDS.
template <int N, int kPitch, int kCount>
__device__ inline void add_products(int lane, const u4 (&a)[3], const uint16_t (&rows)[N][kChunk][kPitch], int m, f4 (&x)[kCount]) {
#pragma unroll
    for (int c = 0; c < kCount; ++c) {
        u4 b[N];
        operand_columns(lane, rows, c, m, b);
        x[c] = mma(a, b, x[c]);
        if (c % 2) settle();
    }
}

// What a wave computes of do's terms (kDo: x is do, y is Y, h is H) or of dr's (dr, Z, R), for
// the tokens 16 wave on.
template <class E, int KP>
struct GradientTerms {
    static constexpr int N = kPlanes<E>;
    f4 y[KP / 16], h[4], row_sum;

    __device__ void clear() {
#pragma unroll
        for (int c = 0; c < KP / 16; ++c) y[c] = f4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = f4{0, 0, 0, 0};
    }

    template <int kOwn>
    __device__ void products(int lane, int wave, const GradientStage<KP>& stage, bool with_state, const u4 (&x)[kOwn]) {
        u4 b[3];
        if (with_state)
#pragma unroll
            for (int c = 0; c < KP / 16; ++c) {
                staged_operand(lane, stage.s[c], b);
                y[c] = mma(x, b, y[c]);
                settle();
            }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > wave) continue;
            staged_operand(lane, stage.u[j], b);
            h[j] = mma(x, b, h[j]);
            settle();
        }
    }

    template <bool kDo>
    __device__ static const auto& left_rows(const ChunkRows<E, KP>& rows) {
        if constexpr (kDo)
            return rows.q;
        else
            return rows.k;
    }

    template <bool kDo>
    __device__ static auto& triangle(GradientTriangles<E, KP>& tri) {
        if constexpr (kDo)
            return tri.n;
        else
            return tri.m;
    }

    // N or M, and the sums over its rows (kept) and columns (parts of the workgroup's sums: with
    // eight waves M's own, with four N's, which it adds to).
    template <bool kDo>
    __device__ void make_triangle(int lane, int wave, const ChunkRows<E, KP>& rows, const ChunkGates& gates,
                                  GradientTriangles<E, KP>& tri, float scale) {
        constexpr bool kAdd = !kDo && kGradientWaves<E, KP> == 4;
        const int col = lane & 15, g = lane >> 4, row = 16 * wave + 4 * g;
        const int part = wave + (kDo || kAdd ? 0 : 4);
        row_sum = f4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float beta_sum = 0.0f, g_sum = 0.0f;
            if (j <= wave) {
                f4 xk = {0, 0, 0, 0};  // q . k or k . k
#pragma unroll
                for (int m = 0; m < KP / 32; ++m) {
                    u4 a[N], b[N];
                    operand_rows(lane, rows.k, 16 * j, m, b);
                    operand_rows(lane, left_rows<kDo>(rows), 16 * wave, m, a);
                    xk = mma(a, b, xk);
                }
                const int column = 16 * j + col;
                const float hi = gates.hi[column], lo = gates.lo[column], beta = gates.beta[column];
                const int episode = gates.episode[column];
                const float factor = kDo ? scale : -1.0f;
                f4 n;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const bool below = row + s > column, on = kDo ? row + s >= column : below;
                    const float d = on ? decay(gates, row + s, hi, lo, episode) : 0.0f;
                    const float x = on ? factor * d * h[j][s] : 0.0f, xb = x * beta;
                    n[s] = xb;
                    const float pair = below ? xb * xk[s] : 0.0f;
                    beta_sum += on ? x * xk[s] : 0.0f;
                    g_sum += pair;
                    row_sum[s] += pair;
                }
                store_slot<3>(triangle<kDo>(tri), tile_of(wave, j), lane, n);
                settle();
            }
            beta_sum = sum_tokens(beta_sum);
            g_sum = sum_tokens(g_sum);
            if (g == 0) {
                tri.beta_part[part][16 * j + col] = (kAdd ? tri.beta_part[part][16 * j + col] : 0.0f) + beta_sum;
                tri.g_part[part][16 * j + col] = (kAdd ? tri.g_part[part][16 * j + col] : 0.0f) + g_sum;
            }
        }
    }

    // y becomes scale E Y or -E Z; its product with q or k is added to the sums of rows.
    template <bool kDo>
    __device__ void close_rows(int lane, int wave, const ChunkRows<E, KP>& rows, const ChunkGates& gates, float scale) {
        const int row = 16 * wave + 4 * (lane >> 4);
        const f4 e = four(gates.e, row);
        const float factor = kDo ? scale : -1.0f;
#pragma unroll
        for (int c = 0; c < KP / 16; ++c) {
            y[c] = factor * gated(y[c], e);
            row_sum = row_sum + row_products(lane, row, left_rows<kDo>(rows), c, y[c]);
            settle();
        }
    }

    __device__ static f4 row_products(int lane, int row, const uint16_t (&rows)[N][kChunk][KP + 8], int c, f4 x) {
        f4 product;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            float y = 0.0f;
#pragma unroll
            for (int n = N - 1; n >= 0; --n) y += to_float(bf16{rows[n][row + s][place_of(16 * c + (lane & 15))]});
            product[s] = y * x[s];
        }
        return product;
    }

    // dq = y + N k and N^T q into dk; or M k + M^T k into dk = y.
    template <bool kDo>
    __device__ void last_products(int lane, int wave, const ChunkRows<E, KP>& rows, GradientTriangles<E, KP>& tri,
                                  f4 (&dk)[KP / 16]) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            u4 a[3];
            if (2 * m <= wave) {
                operand_triangle<3>(lane, triangle<kDo>(tri), wave, m, a);
                add_products(lane, a, rows.k, m, y);
            }
            if (2 * m + 1 >= wave) {
                operand_transpose<3>(lane, triangle<kDo>(tri), wave, m, a);
                add_products(lane, a, left_rows<kDo>(rows), m, dk);
            }
        }
    }
};

template <class E, int KP>
__global__ __launch_bounds__((64 * kGradientWaves<E, KP>), 2) void delta_gradients_kernel(RuleParams P) {
    constexpr int N = kPlanes<E>, kWaves = kGradientWaves<E, KP>;
    constexpr bool kBoth = kWaves == 4;                      // a wave has both kinds of terms
    constexpr int kPieces = 8 * KP / (64 * kWaves), kRowsOfU = 8 / kWaves;
    constexpr int kDown = 8 * kWaves;                        // rows that the workgroup's pieces are of
    extern __shared__ char lds_bytes[];
    auto& lds = *reinterpret_cast<GradientLds<E, KP>*>(lds_bytes);
    auto& rows = lds.of.rows;
    const ChunkGates& gates = lds.rest.gates;
    const int wave = wave_of_workgroup() & 3;
    const bool of_do = kBoth || wave_of_workgroup() < 4, of_dr = kBoth || !of_do;
    int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int64_t sequence = blockIdx.x / static_cast<uint32_t>(P.n_chunks);
    const int chunk = static_cast<int>(blockIdx.x % static_cast<uint32_t>(P.n_chunks));
    const int64_t env = sequence / P.r.value_heads;
    const int head = static_cast<int>(sequence % P.r.value_heads);
    const int K = P.r.key_dim, V = P.r.value_dim;
    const int64_t t0 = static_cast<int64_t>(chunk) * kChunk;
    const int tokens = tokens_of(P, chunk);

    const int64_t kv = static_cast<int64_t>(K) * V, inner = sequence * (P.n_chunks - 1);
    const float* S = chunk > 0 ? P.r.states + (inner + chunk - 1) * kv
                               : P.r.initial_state ? P.r.initial_state + sequence * kv : nullptr;
    const float* dS = chunk + 1 < P.n_chunks ? P.dstates + (inner + chunk) * kv
                                              : P.d.grad_final_state ? P.d.grad_final_state + sequence * kv : nullptr;
    const int64_t rows_at = (sequence * P.r.steps + t0) * V;
    const uint32_t row_bytes = 4 * V, grad_row_bytes = static_cast<uint32_t>(P.d.grad_out_stride[1]) * sizeof(E);
    const Buffer from_s = buffer_of(S, S ? K * row_bytes : 0), from_ds = buffer_of(dS, dS ? K * row_bytes : 0);
    const Buffer from_u = buffer_of(P.r.updates + rows_at, tokens * row_bytes);
    const Buffer from_dr = buffer_of(P.rgrads + rows_at, tokens * row_bytes);
    const Buffer from_grad = buffer_of(at<E>(P.d.grad_out, P.d.grad_out_stride, env, t0, head),
                                       (tokens - 1) * grad_row_bytes + V * sizeof(E));
    const int piece_row = threadIdx.x >> 3, piece_column = (threadIdx.x & 7) * 4;
    const int slot = (piece_row & 15) + 16 * ((threadIdx.x & 7) >> 1), half = threadIdx.x & 1;
    const int my_token = 16 * wave + col;  // of the wave's tile of tokens, as an operand's row

    Part<float, 4> next_s[kPieces], next_ds[kPieces], next_u[kRowsOfU];
    Part<float, 8> next_dr;
    Part<E, 8> next_do;
    const auto fetch = [&](int v0) {
        const int c = v0 + piece_column;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int row = piece_row + kDown * i, valid = row < K ? V - c : 0;
            if (S) next_s[i].load(from_s, row * row_bytes + 4 * c, valid, P.wide_state);
            if (dS) next_ds[i].load(from_ds, row * row_bytes + 4 * c, valid, P.wide_state);
        }
#pragma unroll
        for (int i = 0; i < kRowsOfU; ++i) {
            const int row = piece_row + kDown * i;
            next_u[i].load(from_u, row * row_bytes + 4 * c, row < tokens ? V - c : 0, P.wide_state);
        }
        const int valid = my_token < tokens ? V - v0 - 8 * g : 0;
        if (of_do) next_do.load(from_grad, my_token * grad_row_bytes + (v0 + 8 * g) * sizeof(E), valid, P.wide_do);
        if (of_dr) next_dr.load(from_dr, my_token * row_bytes + 4 * (v0 + 8 * g), valid, P.wide_state);
    };
    fetch(0);
    GatesFetch of_gates;
    if (wave_of_workgroup() == kWaves - 1) of_gates.fetch(P, env, head, t0, tokens);
    if constexpr (kRowsStay<E, KP>) ChunkFetch<E, KP, 64 * kWaves, true>::load(P, rows, env, head, t0, tokens);
    if (wave_of_workgroup() == kWaves - 1) of_gates.put(lds.rest.gates);
    GradientTerms<E, KP> terms, others;
    GradientTerms<E, KP>& terms_dr = kBoth ? others : terms;  // with eight waves a wave has one kind
    f4 w[KP / 16];
    terms.clear();
    if constexpr (kBoth) others.clear();
#pragma unroll
    for (int c = 0; c < KP / 16; ++c) w[c] = f4{0, 0, 0, 0};
    float dot = 0.0f;
    for (int v0 = 0; v0 < V; v0 += 32) {
        if (v0 > 0) __syncthreads();
        float a[4], x[8];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int tile = (piece_row + kDown * i) >> 4;
            if (S) {
                next_s[i].floats(a);
                stage_part(lds.stage.s[tile], slot, half, a);
            }
            if (dS) {
                next_ds[i].floats(a);
                stage_part(lds.stage.ds[tile], slot, half, a);
                if (S)
#pragma unroll
                    for (int n = 0; n < 4; ++n) dot += float_of(next_s[i].words[0][n]) * a[n];
            }
        }
#pragma unroll
        for (int i = 0; i < kRowsOfU; ++i) {
            next_u[i].floats(a);
            stage_part(lds.stage.u[(piece_row + kDown * i) >> 4], slot, half, a);
        }
        u4 a_do[N], a_dr[3];
        if (of_do) {
            next_do.floats(x);
            split8(x, a_do);
        }
        if (of_dr) {
            next_dr.floats(x);
            split8(x, a_dr);
        }
        __syncthreads();
        if (v0 + 32 < V) fetch(v0 + 32);
        settle();
        if (of_dr) terms_dr.products(lane, wave, lds.stage, S, a_dr);
        if (of_do) {
            terms.products(lane, wave, lds.stage, S, a_do);
            if (dS) {
                u4 a_u[3], b[3];
                staged_operand(lane, lds.stage.u[wave], a_u);
#pragma unroll
                for (int c = 0; c < KP / 16; ++c) {
                    staged_operand(lane, lds.stage.ds[c], b);
                    w[c] = mma(a_u, b, w[c]);
                    settle();
                }
            }
        }
    }
    dot = sum_tokens(sum16(dot));
    if (lane == 0) lds.rest.dot_part[threadIdx.x >> 6] = dot;
    __syncthreads();
    if constexpr (!kRowsStay<E, KP>) {
        ChunkFetch<E, KP, 64 * kWaves, true>::load(P, rows, env, head, t0, tokens);
        __syncthreads();
    }

    // The triangles N and M; the sums over their rows and columns.
    lane = fresh_lane(), col = lane & 15, g = lane >> 4;
    const int row = 16 * wave + 4 * g;
    if (of_do) {
        terms.template make_triangle<true>(lane, wave, rows, gates, lds.tri, P.r.scale);
        terms.template close_rows<true>(lane, wave, rows, gates, P.r.scale);
        const f4 f = four(gates.f, row), beta = four(gates.beta, row);
        f4 kw = {0, 0, 0, 0};
        if (dS)
#pragma unroll
            for (int c = 0; c < KP / 16; ++c) {
                kw = kw + terms.row_products(lane, row, rows.k, c, w[c]);
                w[c] = beta * f * w[c];
                settle();
            }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const float own = sum16(terms.row_sum[s]), left = f[s] * sum16(kw[s]);
            if (col == 0) {
                lds.rest.g_row[0][row + s] = own - beta[s] * left;
                lds.rest.beta_row[row + s] = left;
            }
        }
    }
    if (of_dr) {
        terms_dr.template make_triangle<false>(lane, wave, rows, gates, lds.tri, P.r.scale);
        terms_dr.template close_rows<false>(lane, wave, rows, gates, P.r.scale);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const float own = sum16(terms_dr.row_sum[s]);
            if (col == 0) lds.rest.g_row[1][row + s] = own;
        }
    }
    __syncthreads();
    if (wave_of_workgroup() == 0) {
        float dbeta = lds.rest.beta_row[lane], dG = lds.rest.g_row[0][lane] + lds.rest.g_row[1][lane];
        const float f_all = sum_tokens(sum16(gates.beta[lane] * dbeta));  // (before the triangles' parts)
#pragma unroll
        for (int n = 0; n < kWaves; ++n) {
            dbeta += lds.tri.beta_part[n][lane];
            dG -= lds.tri.g_part[n][lane];
        }
        if (lane == 63) {
            const float keep = gates.e[63];
            dG += f_all;
            float all = 0.0f;
#pragma unroll
            for (int n = 0; n < kWaves; ++n) all += lds.rest.dot_part[n];
            if (keep != 0.0f) dG += keep * all;
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const float later = __shfl_down(dG, d);
            dG += lane + d < 64 ? later : 0.0f;
        }
        if (lane < tokens) {
            const int before = lane > 0 ? gates.episode[lane - 1] : 0;
            const int64_t to = (env * P.r.steps + t0 + lane) * P.r.value_heads + head;
            P.d.d_g[to] = gates.episode[lane] != before ? 0.0f : dG;
            P.d.d_beta[to] = dbeta;
        }
    }

    lane = fresh_lane();
    if (of_do) terms.template last_products<true>(lane, wave, rows, lds.tri, w);
    if (of_dr) terms_dr.template last_products<false>(lane, wave, rows, lds.tri, terms_dr.y);
    if constexpr (kBoth) {
#pragma unroll
        for (int c = 0; c < KP / 16; ++c) w[c] = w[c] + others.y[c];
    } else {
        __syncthreads();  // the rows are done with: do's part of dk goes to the waves that have dr's
        if (of_do)
#pragma unroll
            for (int c = 0; c < KP / 16; ++c) lds.of.exchange[wave][c][lane] = w[c];
        __syncthreads();
        if (of_dr)
#pragma unroll
            for (int c = 0; c < KP / 16; ++c) w[c] = terms_dr.y[c] + lds.of.exchange[wave][c][lane];
    }
    const int left = tokens - 16 * wave;  // rows of the wave's tile
    if (left <= 0) return;
    const int64_t token = env * P.r.steps + t0 + 16 * wave;
    if (P.group == 1) {
        const int64_t to = (token * P.r.key_heads + head) * K, stride = static_cast<int64_t>(P.r.key_heads) * K;
        if (of_do) store_tiles<E, KP>(static_cast<E*>(P.d.d_q) + to, stride, left, K, terms.y);
        if (of_dr) store_tiles<E, KP>(static_cast<E*>(P.d.d_k) + to, stride, left, K, w);
    } else {
        const int64_t to = (token * P.r.value_heads + head) * K, stride = static_cast<int64_t>(P.r.value_heads) * K;
        if (of_do) store_tiles<float, KP>(P.dq_heads + to, stride, left, K, terms.y);
        if (of_dr) store_tiles<float, KP>(P.dk_heads + to, stride, left, K, w);
    }
}

// A key head's gradients are the sum of its value heads', in their order (no atomics: the same
// result every time). Bound by memory: 16 us for 74 MB at 2 x 4001 steps, 8 heads of 128 (4.6 TB/s).
template <class E>
__global__ __launch_bounds__(256) void delta_join_heads_kernel(RuleParams P, int64_t count) {
    const int K = P.r.key_dim;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < count; i += gridDim.x * 256ll) {
        const int64_t row = i / K;
        const int64_t from = row * P.group * K + i % K;
        float q = 0.0f, k = 0.0f;
        for (int n = 0; n < P.group; ++n) {
            q += P.dq_heads[from + static_cast<int64_t>(n) * K];
            k += P.dk_heads[from + static_cast<int64_t>(n) * K];
        }
        static_cast<E*>(P.d.d_q)[i] = from_float<E>(q);
        static_cast<E*>(P.d.d_k)[i] = from_float<E>(k);
    }
}

int launched(const char* what) {
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return set_error(NAVI_POLICY_E_LAUNCH, "%s: kernel launch failed: %s", what, hipGetErrorString(err));
    return NAVI_POLICY_OK;
}

int blocks_of(const navi_delta_rule& r, int columns) {
    const int each = r.dtype == NAVI_POLICY_F32 && r.key_dim > 64 ? kWalkColumns<float, 128> : kWalkColumns<bf16, 64>;
    return (columns + each - 1) / each;
}

int64_t chunks_of(int64_t steps) { return (steps + kChunk - 1) / kChunk; }

// Segments of a walk, at most 16: one where workgroups of 64 columns for whole walks fill half of the
// card's 256 CUs (192 sequences of 4096 steps, one head of 64, forward: 349 us in 1, 385 in 2; 128:
// 274 in 4, 286 in 2); else as many as give each CU a workgroup, of four chunks or more, for the join
// takes about a third of a chunk for each. A second workgroup to a CU gives less and needs
// segments of eight chunks. 2 x 4001 steps, 8 heads of 128: 410 us forward and back in 8 segments, 437
// in 15; 16384 steps, 16 heads of 128, forward: 371 us in 16, 387 in 8.
int segments_of(const navi_delta_rule& r) {
    const int64_t blocks = std::max<int64_t>(1, r.envs * r.value_heads * ((r.value_dim + 63) / 64)), chunks = chunks_of(r.steps);
    if (blocks > 128) return 1;
    const int64_t most = std::max(std::min(256 / blocks, chunks / 4), chunks / 8);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({512 / blocks, most, 16})));
}

int64_t segment_floats(const navi_delta_rule& r) {
    return r.envs * r.value_heads * (segments_of(r) - 1) * (static_cast<int64_t>(r.key_dim) * r.value_dim + r.key_dim * r.key_dim);
}

template <class E, int KP, bool kBack, bool kSummary>
int walk(const RuleParams& P, unsigned segments, hipStream_t stream) {
    constexpr size_t lds = sizeof(ScanLds<E, KP>);
    const int64_t blocks = (P.r.envs * P.r.value_heads + 7) / 8 * 8 * (kSummary ? P.summary_blocks : P.blocks);
    const dim3 grid(static_cast<unsigned>(blocks), 1, segments), threads(kWalkThreads<E, KP>);
    if constexpr (kBack)
        hipLaunchKernelGGL((delta_reverse_kernel<E, KP, kSummary>), grid, threads, lds, stream, P);
    else
        hipLaunchKernelGGL((delta_forward_kernel<E, KP, kSummary>), grid, threads, lds, stream, P);
    return launched("the gated delta rule");
}

template <class E, int KP, bool kBack>
int walk_all(const RuleParams& P, hipStream_t stream) {
    const unsigned segments = static_cast<unsigned>(P.n_segments);
    if (segments > 1) {
        int code = walk<E, KP, kBack, true>(P, segments - 1, stream);
        if (code != NAVI_POLICY_OK) return code;
        if (segments > 2) {
            const dim3 grid(static_cast<unsigned>(P.r.envs * P.r.value_heads), (P.r.value_dim + 15) / 16);
            hipLaunchKernelGGL(delta_join_kernel<KP>, grid, dim3(256), 0, stream, P);
            code = launched("the gated delta rule");
            if (code != NAVI_POLICY_OK) return code;
        }
    }
    return walk<E, KP, kBack, false>(P, segments, stream);
}

template <class E, int KP>
int forward(const RuleParams& P, hipStream_t stream) {
    if (P.n_chunks > 0) {
        hipLaunchKernelGGL((delta_triangles_kernel<E, KP>), dim3(static_cast<unsigned>(P.r.envs * P.r.value_heads * P.n_chunks)),
                           dim3(256), sizeof(TriangleLds<E, KP>), stream, P);
        const int code = launched("navi_delta_forward");
        if (code != NAVI_POLICY_OK) return code;
    }
    return walk_all<E, KP, false>(P, stream);
}

template <class E, int KP>
int backward(const RuleParams& P, hipStream_t stream) {
    int code = walk_all<E, KP, true>(P, stream);
    if (code != NAVI_POLICY_OK) return code;
    hipLaunchKernelGGL((delta_gradients_kernel<E, KP>), dim3(static_cast<unsigned>(P.r.envs * P.r.value_heads * P.n_chunks)),
                       dim3(64 * kGradientWaves<E, KP>), sizeof(GradientLds<E, KP>), stream, P);
    code = launched("navi_delta_backward");
    if (code != NAVI_POLICY_OK || P.group == 1) return code;
    const int64_t count = P.r.envs * P.r.steps * P.r.key_heads * P.r.key_dim;
    hipLaunchKernelGGL(delta_join_heads_kernel<E>, dim3(static_cast<unsigned>(std::min<int64_t>((count + 255) / 256, 8192))),
                       dim3(256), 0, stream, P, count);
    return launched("navi_delta_backward");
}

template <class E>
int run(const RuleParams& P, bool back, hipStream_t stream) {
    if (P.r.key_dim <= 64) return back ? backward<E, 64>(P, stream) : forward<E, 64>(P, stream);
    return back ? backward<E, 128>(P, stream) : forward<E, 128>(P, stream);
}

int run_typed(const RuleParams& P, bool back, hipStream_t stream) {
    if (P.r.dtype == NAVI_POLICY_F32) return run<float>(P, back, stream);
    if (P.r.dtype == NAVI_POLICY_BF16) return run<bf16>(P, back, stream);
    return run<f16>(P, back, stream);
}

// Whether the rows of steps lie one after another, 64 of them within reach of a buffer access
// (the bytes from one to the next times 64, and a row, stay below 2^31).
constexpr int64_t kFarthest = INT32_MAX / kChunk - 65536 * 4;
bool rows_apart(const int64_t (&stride)[3], int64_t bytes, int64_t dim) {
    return stride[1] >= dim && stride[1] <= kFarthest / bytes;
}

// Wide buffer accesses need addresses of whole 4-byte words, and rows that end between them.
bool wide_columns(const void* p, const int64_t (&stride)[3], int64_t bytes, int64_t dim) {
    return reinterpret_cast<uintptr_t>(p) % 4 == 0 && dim % 8 == 0 && stride[0] * bytes % 4 == 0 && stride[1] * bytes % 4 == 0 &&
           stride[2] * bytes % 4 == 0;
}

bool wide_rows(const void* p, const int64_t (&stride)[3], int64_t bytes, int64_t dim) {
    return aligned16(p) && dim % 8 == 0 && stride[0] * bytes % 16 == 0 && stride[1] * bytes % 16 == 0 &&
           stride[2] * bytes % 16 == 0;
}

}  // namespace

// Sizes that every form needs; 1 where there is nothing to do.
int check_rule(const navi_delta_rule* r) {
    if (!r) return set_error(NAVI_POLICY_E_ARG, "rule must be non-null");
    if (r->dtype < NAVI_POLICY_F32 || r->dtype > NAVI_POLICY_F16)
        return set_error(NAVI_POLICY_E_ARG, "dtype must be float32, bfloat16 or float16");
    if (r->key_heads <= 0 || r->value_heads <= 0 || r->value_heads % r->key_heads != 0)
        return set_error(NAVI_POLICY_E_ARG, "value_heads must be a positive multiple of key_heads");
    if (r->key_dim <= 0 || r->key_dim > NAVI_POLICY_MAX_KEY_DIM)
        return set_error(NAVI_POLICY_E_ARG, "key_dim must be in [1, %d]", NAVI_POLICY_MAX_KEY_DIM);
    if (r->value_dim <= 0 || r->value_dim > 65536) return set_error(NAVI_POLICY_E_ARG, "value_dim must be in [1, 65536]");
    if (r->envs < 0 || r->steps < 0) return set_error(NAVI_POLICY_E_ARG, "envs and steps must not be negative");
    if (r->envs > INT32_MAX / r->value_heads || r->steps > INT32_MAX)
        return set_error(NAVI_POLICY_E_ARG, "envs * value_heads and steps must be below 2^31");
    if (r->envs == 0) return 1;
    if (r->steps > 0 && (!r->q || !r->k || !r->v || !r->g || !r->beta || !r->out))
        return set_error(NAVI_POLICY_E_ARG, "q, k, v, g, beta and out must be non-null");
    const int64_t bytes = r->dtype == NAVI_POLICY_F32 ? 4 : 2;
    if (!aligned(bytes, r->q, r->k, r->v, r->out) ||
        !aligned(4, r->g, r->beta, r->initial_state, r->final_state, r->states, r->updates))
        return set_error(NAVI_POLICY_E_ARG, "arrays must be aligned to their elements");
    return NAVI_POLICY_OK;
}

// Workgroups read the inputs in any order, so what is written shares no memory with them: out
// but with v number for number (whose reader writes them), final_state in the recurrent form but
// with initial_state (the same).
int check_apart(const navi_delta_rule* r, bool in_place) {
    if (r->envs == 0) return NAVI_POLICY_OK;
    const int64_t bytes = r->dtype == NAVI_POLICY_F32 ? 4 : 2, V = r->value_dim, K = r->key_dim;
    const int64_t row = r->value_heads * V, state = r->value_heads * K * V;
    const auto of = [&](const void* p, int64_t heads, int64_t dim, const int64_t(&s)[3], int64_t each) {
        return r->steps > 0 && p ? extent_of(p, {r->envs, r->steps, heads, dim}, {s[0], s[1], s[2], 1}, each) : Extent{0, 0};
    };
    const auto of_state = [&](const float* p) { return p ? extent_of(p, {r->envs, 1, 1, state}, {state, 0, 0, 1}, 4) : Extent{0, 0}; };
    const Extent out = of(r->out, r->value_heads, V, {r->steps * row, row, V}, bytes), final_state = of_state(r->final_state);
    const bool own = r->out == r->v && (r->value_heads == 1 || r->v_stride[2] == V) && (r->steps == 1 || r->v_stride[1] == row) &&
                     (r->envs == 1 || r->v_stride[0] == r->steps * row);
    const Extent inputs[] = {
        of(r->q, r->key_heads, K, r->q_stride, bytes), of(r->k, r->key_heads, K, r->k_stride, bytes),
        of(r->g, r->value_heads, 1, r->g_stride, 4), of(r->beta, r->value_heads, 1, r->beta_stride, 4),
        of(r->starts, 1, 1, {r->starts_stride[0], r->starts_stride[1], 0}, 1)};
    bool fine = apart(out, final_state);
    for (const Extent& x : inputs) fine = fine && apart(out, x) && apart(final_state, x);
    const Extent v = of(r->v, r->value_heads, V, r->v_stride, bytes), initial = of_state(r->initial_state);
    fine = fine && (own || apart(out, v)) && apart(out, initial) && apart(final_state, v);
    fine = fine && ((in_place && r->final_state == r->initial_state) || apart(final_state, initial));
    return fine ? NAVI_POLICY_OK : set_error(NAVI_POLICY_E_ARG, "out or the state after shares memory with what is read");
}

namespace {

int setup(const navi_delta_rule* r, bool back, RuleParams& P) {
    const int code = check_rule(r);
    if (code != NAVI_POLICY_OK) return code;
    P.r = *r;
    P.group = r->value_heads / r->key_heads;
    P.n_chunks = static_cast<int32_t>(chunks_of(r->steps));
    P.blocks = blocks_of(*r, r->value_dim);
    P.summary_blocks = blocks_of(*r, (r->value_dim + 15) / 16 * 16 + r->key_dim);
    P.n_segments = segments_of(*r);
    const int64_t bytes = r->dtype == NAVI_POLICY_F32 ? 4 : 2;
    if (r->envs * r->value_heads * chunks_of(r->steps) > INT32_MAX)
        return set_error(NAVI_POLICY_E_ARG, "envs * value_heads * chunks must be below 2^31");
    const int64_t sequences = r->envs * r->value_heads, walks = (sequences + 7) / 8 * 8 * std::max(P.blocks, P.n_segments > 1 ? P.summary_blocks : 0);
    const int walk_threads = r->dtype == NAVI_POLICY_F32 && r->key_dim > 64 ? kWalkThreads<float, 128> : kWalkThreads<bf16, 64>;
    const int chunk_threads = !back ? 256 : 64 * (r->dtype == NAVI_POLICY_F16 && r->key_dim <= 64 ? kGradientWaves<f16, 64> : kGradientWaves<bf16, 64>);
    if (!launchable(walks, walk_threads) || !launchable(sequences * P.n_chunks, chunk_threads))
        return set_error(NAVI_POLICY_E_ARG, "envs * value_heads * chunks or * value_dim is too large (a launch has fewer than 2^32 threads)");
    if (P.n_chunks > 0 && (!r->matrices || !aligned16(r->matrices)))
        return set_error(NAVI_POLICY_E_ARG, "matrices must be non-null and 16-byte aligned");
    if (r->value_heads > kFarthest / 4 / std::max(r->value_dim, r->key_dim))
        return set_error(NAVI_POLICY_E_ARG, "value_heads * value_dim or value_heads * key_dim is too large");
    if (r->steps == 1) {  // (the stride of an axis of one may be anything)
        P.r.q_stride[1] = P.r.k_stride[1] = r->key_dim;
        P.r.v_stride[1] = r->value_dim;
    }
    if (!(rows_apart(P.r.q_stride, bytes, r->key_dim) && rows_apart(P.r.k_stride, bytes, r->key_dim) &&
          rows_apart(P.r.v_stride, bytes, r->value_dim)) && r->steps > 0)
        return set_error(NAVI_POLICY_E_ARG, "the steps of q, k and v overlap or lie too far apart");
    P.wide_qk = wide_rows(r->q, P.r.q_stride, bytes, r->key_dim) && wide_rows(r->k, P.r.k_stride, bytes, r->key_dim);
    P.wide_v = wide_columns(r->v, P.r.v_stride, bytes, r->value_dim);
    P.wide_out = reinterpret_cast<uintptr_t>(r->out) % 4 == 0 && r->value_dim % 4 == 0;
    return NAVI_POLICY_OK;
}

float* place_segments(RuleParams& P, float* at) {
    const int64_t slots = P.r.envs * P.r.value_heads * (P.n_segments - 1);
    P.segment_states = at;
    P.segment_matrices = at + slots * P.r.key_dim * P.r.value_dim;
    return P.segment_matrices + slots * P.r.key_dim * P.r.key_dim;
}

}  // namespace
}  // namespace navi_policy

using namespace navi_policy;

extern "C" int navi_delta_forward(const navi_delta_rule* rule, void* stream) {
    RuleParams P{};
    const int code = setup(rule, false, P);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : NAVI_POLICY_OK;
    if (!rule->states != !rule->updates && P.n_chunks > 1)
        return set_error(NAVI_POLICY_E_ARG, "states and updates are saved together or not at all");
    if (P.n_chunks == 0 && !rule->final_state) return NAVI_POLICY_OK;
    if (P.n_segments > 1 && (!rule->scratch || !aligned16(rule->scratch)))
        return set_error(NAVI_POLICY_E_ARG, "scratch must be non-null and 16-byte aligned");
    const int shared = check_apart(rule, false);
    if (shared != NAVI_POLICY_OK) return shared;
    place_segments(P, static_cast<float*>(rule->scratch));
    return run_typed(P, false, as_stream(stream));
}

extern "C" int64_t navi_delta_scratch(const navi_delta_rule* rule) {
    const int code = check_rule(rule);
    if (code < 0) return code;
    return 4 * segment_floats(*rule);
}

extern "C" int64_t navi_delta_workspace(const navi_delta_rule* rule) {
    const int code = check_rule(rule);
    if (code < 0) return code;
    const int64_t sequences = rule->envs * rule->value_heads, steps = rule->steps;
    const int64_t inner = std::max<int64_t>(0, chunks_of(steps) - 1);
    const int64_t states = sequences * inner * rule->key_dim * rule->value_dim;
    const int64_t rows = sequences * steps * rule->value_dim;
    const int64_t heads = rule->value_heads > rule->key_heads ? sequences * steps * rule->key_dim : 0;
    const auto rounded = [](int64_t n) { return (n + 3) / 4 * 4; };
    return 4 * (rounded(states) + rounded(rows) + 2 * rounded(heads) + segment_floats(*rule));
}

extern "C" int navi_delta_backward(const navi_delta_rule* rule, const navi_delta_gradients* gradients, void* stream) {
    RuleParams P{};
    const int code = setup(rule, true, P);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : NAVI_POLICY_OK;
    if (!gradients) return set_error(NAVI_POLICY_E_ARG, "gradients must be non-null");
    P.d = *gradients;
    if (rule->steps == 0) return set_error(NAVI_POLICY_E_ARG, "the backward pass needs at least one step");
    if (!P.d.grad_out || !P.d.d_q || !P.d.d_k || !P.d.d_v || !P.d.d_g || !P.d.d_beta || !P.d.workspace)
        return set_error(NAVI_POLICY_E_ARG, "grad_out, the gradients and workspace must be non-null");
    if (!rule->updates || (P.n_chunks > 1 && !rule->states))
        return set_error(NAVI_POLICY_E_ARG, "the backward pass needs the forward pass's states and updates");
    const int64_t sequences = rule->envs * rule->value_heads;
    if (!aligned16(P.d.workspace)) return set_error(NAVI_POLICY_E_ARG, "workspace must be 16-byte aligned");
    const auto rounded = [](int64_t n) { return (n + 3) / 4 * 4; };
    P.dstates = static_cast<float*>(P.d.workspace);
    P.rgrads = P.dstates + rounded(sequences * (P.n_chunks - 1) * rule->key_dim * rule->value_dim);
    P.dq_heads = P.rgrads + rounded(sequences * rule->steps * rule->value_dim);
    P.dk_heads = P.dq_heads + rounded(P.group > 1 ? sequences * rule->steps * rule->key_dim : 0);
    place_segments(P, P.dk_heads + rounded(P.group > 1 ? sequences * rule->steps * rule->key_dim : 0));
    const int64_t bytes = rule->dtype == NAVI_POLICY_F32 ? 4 : 2;
    if (!aligned(bytes, P.d.grad_out, P.d.d_q, P.d.d_k, P.d.d_v) ||
        !aligned(4, P.d.grad_final_state, P.d.d_g, P.d.d_beta, P.d.d_initial_state))
        return set_error(NAVI_POLICY_E_ARG, "arrays must be aligned to their elements");
    if (rule->steps == 1) P.d.grad_out_stride[1] = rule->value_dim;
    if (!rows_apart(P.d.grad_out_stride, bytes, rule->value_dim))
        return set_error(NAVI_POLICY_E_ARG, "the steps of grad_out overlap or lie too far apart");
    P.wide_state = rule->value_dim % 8 == 0;
    P.wide_do = wide_columns(P.d.grad_out, P.d.grad_out_stride, bytes, rule->value_dim);
    return run_typed(P, true, as_stream(stream));
}
