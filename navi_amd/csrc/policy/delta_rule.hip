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

template <class E>
__device__ inline f4 to_floats(const E (&x)[4]) {
    return f4{to_float(x[0]), to_float(x[1]), to_float(x[2]), to_float(x[3])};
}

__device__ inline f4 four(const float (&x)[kChunk], int row) { return *reinterpret_cast<const f4*>(&x[row]); }

// x * factor, 0 where the factor is 0 whatever x is: a state that an episode's start clears.
__device__ inline f4 gated(f4 x, f4 factor) {
    f4 y;
#pragma unroll
    for (int s = 0; s < 4; ++s) y[s] = factor[s] == 0.0f ? 0.0f : x[s] * factor[s];
    return y;
}

__device__ inline int tokens_of(const RuleParams& P, int chunk) {
    const int64_t left = P.r.steps - static_cast<int64_t>(chunk) * kChunk;
    return static_cast<int>(left < kChunk ? left : kChunk);
}

// The triangles and gates of every chunk, which need no state: a workgroup each.
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
    load_rows<E, KP>(P, lds.rows, env, head, t0, tokens);
    if (wave == 0) load_gates(P, lds.gates, env, head, t0, tokens);
    __syncthreads();
    if (threadIdx.x < kChunk) {
        to.e[threadIdx.x] = lds.gates.e[threadIdx.x];
        to.fb[threadIdx.x] = lds.gates.f[threadIdx.x] * lds.gates.beta[threadIdx.x];
    }
    make_triangles<E, KP>(lds, to, P.r.scale, wave);
}

// What reaches the output alone is rounded with it: for 16-bit outputs, two planes (2^-16)
// of S, P and u there are far below that rounding (2^-9 and 2^-12).
template <class E>
inline constexpr int kOutPlanes = sizeof(E) == 4 ? 3 : 2;

template <class E, int KP, int NP>
struct ScanLds {
    ChunkRows<E, KP> rows;
    Triangle<3> x;
    Triangle<NP> p;
    float gates[2][kChunk];  // E, F beta
};

template <int N>
__device__ inline void first_planes(const u4 (&from)[3], u4 (&to)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) to[n] = from[n];
}

template <int KP>
__device__ inline void load_state(const Columns<float>& at, const float* from, int K, f4 (&state)[KP / 16]) {
    at.load<KP / 16>(at.rows(from, from ? K : 0), [&](int c, int s, float x) { state[c][s] = x; });
}

template <int KP>
__device__ inline void store_state(const Columns<float>& at, float* to, int K, const f4 (&state)[KP / 16]) {
    at.store<KP / 16>(at.rows(to, K), [&](int c, int s) { return state[c][s]; });
}

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
__device__ inline void times_triangle(const Triangle<N>& t, const u4 (&b)[2][NB], f4 (&x)[4]) {
    u4 a[4][N];
#pragma unroll
    for (int i = 0; i < 4; ++i) operand_triangle<N>(t, i, 0, a[i]);
    mma_each<4>(a, b[0], x);
    u4 below[2][N];
    f4 y[2] = {x[2], x[3]};
#pragma unroll
    for (int i = 0; i < 2; ++i) operand_triangle<N>(t, 2 + i, 1, below[i]);
    mma_each<2>(below, b[1], y);
    x[2] = y[0];
    x[3] = y[1];
}

template <int N, int NB>
__device__ inline void times_transpose(const Triangle<N>& t, const u4 (&b)[2][NB], f4 (&x)[4]) {
    u4 a[4][N];
#pragma unroll
    for (int j = 0; j < 4; ++j) operand_transpose<N>(t, j, 1, a[j]);
    mma_each<4>(a, b[1], x);
    u4 left[2][N];
    f4 y[2] = {x[0], x[1]};
#pragma unroll
    for (int j = 0; j < 2; ++j) operand_transpose<N>(t, j, 0, left[j]);
    mma_each<2>(left, b[0], y);
    x[0] = y[0];
    x[1] = y[1];
}

// Columns of rows in LDS times b, added to four tiles of a state from tile c on.
template <int N, int kPitch, int NB, int kCount>
__device__ inline void add_columns(const uint16_t (&rows)[N][kChunk][kPitch], int c, const u4 (&b)[2][NB], f4 (&state)[kCount]) {
    f4 x[4] = {state[c], state[c + 1], state[c + 2], state[c + 3]};
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        u4 a[4][N];
#pragma unroll
        for (int n = 0; n < 4; ++n) operand_columns(rows, c + n, m, a[n]);
        mma_each<4>(a, b[m], x);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) state[c + n] = x[n];
}

// A wave holds 16 columns of the state as results of products (KP / 16 tiles), a workgroup
// kThreads / 64 such columns of one head; it walks the chunks with the state in registers.
// The state is the second operand of S^T k without a move: its tiles hold the contracted axis
// in the order of results, which the other operand is read in as well.
template <class E, int KP, int kThreads, bool kSummary>
__global__ __launch_bounds__(kThreads) void delta_forward_kernel(RuleParams P) {
    constexpr int N = kPlanes<E>, NP = kOutPlanes<E>;
    extern __shared__ char lds_bytes[];
    auto& lds = *reinterpret_cast<ScanLds<E, KP, NP>*>(lds_bytes);
    const int wave = wave_of_workgroup(), g = (threadIdx.x & 63) >> 4;
    const int64_t sequence = blockIdx.x;
    const int64_t env = sequence / P.r.value_heads;
    const int head = static_cast<int>(sequence % P.r.value_heads);
    const int K = P.r.key_dim, V = P.r.value_dim;
    const Walk walk = Walk::of<kSummary>(P, sequence, (blockIdx.y * (kThreads / 64) + wave) * 16, P.r.initial_state,
                                         P.r.final_state);
    const int first = walk.first;
    const ChunkMatrices* matrices = reinterpret_cast<const ChunkMatrices*>(P.r.matrices) + sequence * P.n_chunks;
    const E* v = at<E>(P.r.v, P.r.v_stride, env, 0, head) + first;
    const Columns<E> rows_v(P.r.v_stride[1], walk.unit ? 0 : V - first),
        rows_out(static_cast<int64_t>(P.r.value_heads) * V, V - first);
    const Columns<float> rows_state(walk.columns, walk.columns - first);

    f4 state[KP / 16];
    walk.begin_state<KP>(rows_state, K, state);

    ChunkFetch<E, KP, kThreads, !kSummary> next;
    E v_next[4][4];
    const auto fetch = [&](int chunk) {
        const int64_t t0 = static_cast<int64_t>(chunk) * kChunk;
        next.fetch(P, matrices[chunk], env, head, t0, tokens_of(P, chunk));
        rows_v.template load<4>(rows_v.rows(v + t0 * P.r.v_stride[1], tokens_of(P, chunk)),
                                [&](int i, int s, E x) { v_next[i][s] = x; });
    };
    if (walk.begin < walk.end) fetch(walk.begin);
    for (int chunk = walk.begin; chunk < walk.end; ++chunk) {
        const int64_t t0 = static_cast<int64_t>(chunk) * kChunk;
        const int tokens = tokens_of(P, chunk);
        if (chunk > walk.begin) __syncthreads();
        next.template put<NP>(P, lds.rows, lds.x, lds.p, lds.gates, env, head, t0, tokens);
        f4 values[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) values[i] = to_floats(v_next[i]);
        __syncthreads();
        if (chunk + 1 < walk.end) fetch(chunk + 1);
        if (!walk.working) continue;

        if (!kSummary && P.r.states && chunk > 0)
            store_state<KP>(rows_state, P.r.states + (sequence * (P.n_chunks - 1) + chunk - 1) * K * V + first, K, state);
        f4 u[4], o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = o[i] = f4{0, 0, 0, 0};
        if (chunk > walk.begin || walk.from || walk.unit) {
#pragma unroll
            for (int m = 0; m < KP / 32; ++m) {
                u4 b[3], a[4][N];
                split8(state[2 * m], state[2 * m + 1], b);
#pragma unroll
                for (int i = 0; i < 4; ++i) operand_rows_as_results(lds.rows.k, 16 * i, m, a[i]);
                mma_each<4>(a, b, u);
                if constexpr (!kSummary) {
                    u4 b_out[NP];
                    first_planes(b, b_out);
#pragma unroll
                    for (int i = 0; i < 4; ++i) operand_rows_as_results(lds.rows.q, 16 * i, m, a[i]);
                    mma_each<4>(a, b_out, o);
                }
            }
        }
        u4 r[2][3];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            f4 x[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int i = 2 * m + n;
                const f4 e = four(lds.gates[0], 16 * i + 4 * g);
                x[n] = values[i] - gated(u[i], e);
                o[i] = P.r.scale * gated(o[i], e);
                u[i] = f4{0, 0, 0, 0};
            }
            split8(x[0], x[1], r[m]);
        }
        times_triangle<3>(lds.x, r, u);
        if (!kSummary && P.r.updates)
            rows_state.store<4>(rows_state.rows(P.r.updates + (sequence * P.r.steps + t0) * V + first, tokens),
                                [&](int i, int s) { return u[i][s]; });
        // The state first: the next chunk waits for it.
        const float keep = lds.gates[0][kChunk - 1];
#pragma unroll
        for (int m = 0; m < 2; ++m)
            split8(u[2 * m] * four(lds.gates[1], 32 * m + 4 * g), u[2 * m + 1] * four(lds.gates[1], 32 * m + 16 + 4 * g), r[m]);
#pragma unroll
        for (int c = 0; c < KP / 16; ++c) state[c] = gated(state[c], f4{keep, keep, keep, keep});
#pragma unroll
        for (int c = 0; c < KP / 16; c += 4) add_columns(lds.rows.k, c, r, state);
        if constexpr (!kSummary) {
            u4 w[2][NP];
#pragma unroll
            for (int m = 0; m < 2; ++m) split8(u[2 * m], u[2 * m + 1], w[m]);
            times_triangle<NP>(lds.p, w, o);
            rows_out.template store<4>(
                rows_out.rows(static_cast<E*>(P.r.out) + ((env * P.r.steps + t0) * P.r.value_heads + head) * V + first, tokens),
                [&](int i, int s) { return from_float<E>(o[i][s]); });
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
// dS and dr go to memory for delta_gradients_kernel.
template <class E, int KP, int kThreads, bool kSummary>
__global__ __launch_bounds__(kThreads) void delta_reverse_kernel(RuleParams P) {
    constexpr int N = kPlanes<E>;
    extern __shared__ char lds_bytes[];
    auto& lds = *reinterpret_cast<ScanLds<E, KP, 3>*>(lds_bytes);
    const int wave = wave_of_workgroup(), g = (threadIdx.x & 63) >> 4;
    const int64_t sequence = blockIdx.x;
    const int64_t env = sequence / P.r.value_heads;
    const int head = static_cast<int>(sequence % P.r.value_heads);
    const int K = P.r.key_dim, V = P.r.value_dim;
    const Walk walk = Walk::of<kSummary>(P, sequence, (blockIdx.y * (kThreads / 64) + wave) * 16, P.d.grad_final_state,
                                         P.d.d_initial_state);
    const int first = walk.first;
    const ChunkMatrices* matrices = reinterpret_cast<const ChunkMatrices*>(P.r.matrices) + sequence * P.n_chunks;
    const E* grad = at<E>(P.d.grad_out, P.d.grad_out_stride, env, 0, head) + first;
    const Columns<E> rows_grad(P.d.grad_out_stride[1], walk.unit ? 0 : V - first),
        rows_v(static_cast<int64_t>(P.r.value_heads) * V, V - first);
    const Columns<float> rows_state(walk.columns, walk.columns - first);

    f4 dstate[KP / 16];
    walk.begin_state<KP>(rows_state, K, dstate);

    ChunkFetch<E, KP, kThreads, true> next;
    E grad_next[4][4];
    const auto fetch = [&](int chunk) {
        const int64_t t0 = static_cast<int64_t>(chunk) * kChunk;
        next.fetch(P, matrices[chunk], env, head, t0, tokens_of(P, chunk));
        rows_grad.template load<4>(rows_grad.rows(grad + t0 * P.d.grad_out_stride[1], tokens_of(P, chunk)),
                                   [&](int i, int s, E x) { grad_next[i][s] = x; });
    };
    const int last = P.n_chunks - 1;
    if (walk.begin < walk.end) fetch(last - walk.begin);
    for (int step = walk.begin; step < walk.end; ++step) {
        const int chunk = last - step;
        const int64_t t0 = static_cast<int64_t>(chunk) * kChunk;
        const int tokens = tokens_of(P, chunk);
        if (step > walk.begin) __syncthreads();
        next.template put<3>(P, lds.rows, lds.x, lds.p, lds.gates, env, head, t0, tokens);
        f4 dO[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) dO[i] = to_floats(grad_next[i]);
        __syncthreads();
        if (step + 1 < walk.end) fetch(chunk - 1);
        if (!walk.working) continue;

        if (!kSummary && step > 0)
            store_state<KP>(rows_state, P.dstates + (sequence * (P.n_chunks - 1) + chunk) * K * V + first, K, dstate);
        f4 du[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) du[i] = f4{0, 0, 0, 0};
        if (step > walk.begin || walk.from || walk.unit) {
#pragma unroll
            for (int m = 0; m < KP / 32; ++m) {
                u4 b[3], a[4][N];
                split8(dstate[2 * m], dstate[2 * m + 1], b);
#pragma unroll
                for (int i = 0; i < 4; ++i) operand_rows_as_results(lds.rows.k, 16 * i, m, a[i]);
                mma_each<4>(a, b, du);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) du[i] = du[i] * four(lds.gates[1], 16 * i + 4 * g);
        }
        {
            u4 raw[2][N];
#pragma unroll
            for (int m = 0; m < 2; ++m) split8(dO[2 * m], dO[2 * m + 1], raw[m]);
            times_transpose<3>(lds.p, raw, du);
        }
        u4 b[2][3];
#pragma unroll
        for (int m = 0; m < 2; ++m) split8(du[2 * m], du[2 * m + 1], b[m]);
#pragma unroll
        for (int j = 0; j < 4; ++j) du[j] = f4{0, 0, 0, 0};
        times_transpose<3>(lds.x, b, du);  // dr
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
            for (int c = 0; c < KP / 16; ++c) dstate[c] = gated(dstate[c], f4{keep, keep, keep, keep});
#pragma unroll
            for (int m = 0; m < 2; ++m) split8(du[2 * m], du[2 * m + 1], b[m]);
#pragma unroll
            for (int c = 0; c < KP / 16; c += 4) add_columns(lds.rows.k, c, b, dstate);
#pragma unroll
            for (int m = 0; m < 2; ++m) split8(dO[2 * m], dO[2 * m + 1], b[m]);
#pragma unroll
            for (int c = 0; c < KP / 16; c += 4) add_columns(lds.rows.q, c, b, dstate);
        }
    }
    if (walk.to && walk.working) store_state<KP>(rows_state, walk.to + first, K, dstate);
}

// The states before the segments but the first, one after another, from what the summary left
// of each: S <- M S + N with N the state that it makes of zeros (of the given state, for
// segment 0) and M its matrix. Takes N's place. A workgroup holds 64 columns; M's planes go
// through LDS.
template <int KP>
__global__ __launch_bounds__(256) void delta_join_kernel(RuleParams P) {
    extern __shared__ char lds_bytes[];
    auto& m_planes = *reinterpret_cast<uint16_t(*)[KP / 16][KP / 32][3][64][8]>(lds_bytes);
    const int wave = wave_of_workgroup();
    const int64_t sequence = blockIdx.x;
    const int first = (blockIdx.y * 4 + wave) * 16;
    const int K = P.r.key_dim, V = P.r.value_dim;
    const int64_t kv = static_cast<int64_t>(K) * V, slots = sequence * (P.n_segments - 1);
    const Columns<float> rows_state(V, V - first);
    f4 state[KP / 16], next[KP / 16];
    load_state<KP>(rows_state, P.segment_states + slots * kv + first, K, state);
    // of a segment while the one before it is computed: its N, and an operand's parts of its M (a
    // lane holds columns 4 g and 16 + 4 g on of 32, in the order of results)
    constexpr int kParts = KP * KP / 8 / 256;
    f4 part[kParts][2];
    const bool wide = K % 4 == 0;
    const auto fetch = [&](int segment) {
        const Buffer matrix = buffer_of(P.segment_matrices + (slots + segment) * K * K, 4 * K * K);
        load_state<KP>(rows_state, P.segment_states + (slots + segment) * kv + first, K, next);
#pragma unroll
        for (int n = 0; n < kParts; ++n) {
            const int at = threadIdx.x + 256 * n, lane = at & 63, m = (at >> 6) % (KP / 32), c = (at >> 6) / (KP / 32);
            const int row = 16 * c + (lane & 15);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int column = 32 * m + 4 * (lane >> 4) + 16 * h;
                const uint32_t offset = 4 * (row * K + column);
                if (wide) {
                    part[n][h] = __builtin_bit_cast(f4, buffer_load16(matrix, row < K && column < K ? offset : kOutside));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        part[n][h][i] = buffer_load<float>(matrix, row < K && column + i < K ? offset + 4 * i : kOutside);
                }
            }
        }
    };
    if (P.n_segments > 2) fetch(1);
    for (int segment = 1; segment + 1 < P.n_segments; ++segment) {
        if (segment > 1) __syncthreads();
#pragma unroll
        for (int n = 0; n < kParts; ++n) {
            const int at = threadIdx.x + 256 * n;
            u4 plane[3];
            split8(part[n][0], part[n][1], plane);
#pragma unroll
            for (int i = 0; i < 3; ++i) *reinterpret_cast<u4*>(m_planes[(at >> 6) / (KP / 32)][(at >> 6) % (KP / 32)][i][at & 63]) = plane[i];
        }
        f4 x[KP / 16];
#pragma unroll
        for (int c = 0; c < KP / 16; ++c) x[c] = next[c];
        __syncthreads();
        if (segment + 2 < P.n_segments) fetch(segment + 1);
#pragma unroll
        for (int m = 0; m < KP / 32; ++m) {
            u4 b[3];
            split8(state[2 * m], state[2 * m + 1], b);
#pragma unroll
            for (int c = 0; c < KP / 16; c += 4) {
                u4 a[4][3];
                f4 y[4] = {x[c], x[c + 1], x[c + 2], x[c + 3]};
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                        a[n][i] = *reinterpret_cast<const u4*>(m_planes[c + n][m][i][threadIdx.x & 63]);
                mma_each<4>(a, b, y);
#pragma unroll
                for (int n = 0; n < 4; ++n) x[c + n] = y[n];
            }
        }
#pragma unroll
        for (int c = 0; c < KP / 16; ++c) state[c] = x[c];
        store_state<KP>(rows_state, P.segment_states + (slots + segment) * kv + first, K, state);
    }
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
template <class E, int KP>
struct GradientLds {
    union {
        struct {
            uint16_t s[KP / 16][3][64][8], ds[KP / 16][3][64][8];  // 32 columns of S and dS as operands
            uint16_t u[4][3][64][8];                                // and of u
        } stage;
        struct {
            ChunkRows<E, KP> rows;
            Triangle<kOutPlanes<E>> n, m;  // (they reach dq and dk alone)
        };
    };
    ChunkGates gates;
    float beta_part[16][kChunk], g_part[16][kChunk], beta_row[kChunk], g_row[kChunk], f_row[kChunk];
    float dot_part[4];
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

// Eight numbers of a row from `offset` bytes on: in 16-byte loads where rows are multiples of
// eight, else one by one, those from `valid` on as zeros.
template <class T>
struct Eight {
    static constexpr int kWords = sizeof(T) == 4 ? 2 : 1;
    u4 words[kWords];

    __device__ void load(Buffer from, uint32_t offset, int valid, bool wide) {
        if (wide) {
            const uint32_t lane = valid > 0 ? offset : kOutside;
#pragma unroll
            for (int w = 0; w < kWords; ++w) words[w] = buffer_load16(from, lane + 16 * w);
            return;
        }
        uint32_t x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const T y = buffer_load<T>(from, i < valid ? offset + i * sizeof(T) : kOutside);
            if constexpr (sizeof(T) == 4)
                x[i] = bits_of(y);
            else
                x[i] = __builtin_bit_cast(uint16_t, y);
        }
#pragma unroll
        for (int i = 0; i < 4 * kWords; ++i)
            words[i / 4][i % 4] = kWords == 2 ? x[i] : x[2 * i % 8] | x[(2 * i + 1) % 8] << 16;
    }

    __device__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (kWords == 2)
                x[i] = float_of(words[i / 4][i % 4]);
            else
                x[i] = to_float(__builtin_bit_cast(T, static_cast<uint16_t>(words[0][i / 2] >> (16 * (i % 2)))));
        }
    }
};

// The inputs of 32 columns of V: of S, dS and u for the workgroup, of do and dr for the wave.
template <class E, int KP>
struct GradientFetch {
    static constexpr int kPieces = KP / 64;
    Eight<float> s[kPieces], ds[kPieces], u, dr;
    Eight<E> grad;
};

template <class E, int KP>
__global__ __launch_bounds__(256, KP == 64 ? 3 : 1) void delta_gradients_kernel(RuleParams P) {
    constexpr int N = kPlanes<E>, NP = kOutPlanes<E>;
    extern __shared__ char lds_bytes[];
    auto& lds = *reinterpret_cast<GradientLds<E, KP>*>(lds_bytes);
    const int lane = threadIdx.x & 63, wave = wave_of_workgroup();
    const int col = lane & 15, g = lane >> 4;
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
    const int piece_row = threadIdx.x >> 2, piece_column = (threadIdx.x & 3) * 8;
    const int my_token = 16 * wave + col;  // of the wave's tile of tokens, as an operand's row

    GradientFetch<E, KP> next;
    const auto fetch = [&](int v0) {
        const int c = v0 + piece_column;
#pragma unroll
        for (int i = 0; i < KP / 64; ++i) {
            const uint32_t offset = (piece_row + 64 * i) * row_bytes + 4 * c;
            const int valid = piece_row + 64 * i < K ? V - c : 0;
            if (S) next.s[i].load(from_s, offset, valid, P.wide_state);
            if (dS) next.ds[i].load(from_ds, offset, valid, P.wide_state);
        }
        next.u.load(from_u, piece_row * row_bytes + 4 * c, piece_row < tokens ? V - c : 0, P.wide_state);
        const int valid = my_token < tokens ? V - v0 - 8 * g : 0;
        next.dr.load(from_dr, my_token * row_bytes + 4 * (v0 + 8 * g), valid, P.wide_state);
        next.grad.load(from_grad, my_token * grad_row_bytes + (v0 + 8 * g) * sizeof(E), valid, P.wide_do);
    };
    fetch(0);
    if (wave == 0) load_gates(P, lds.gates, env, head, t0, tokens);
    f4 y[KP / 16], z[KP / 16], w[KP / 16], h[4], rr[4];
#pragma unroll
    for (int c = 0; c < KP / 16; ++c) y[c] = z[c] = w[c] = f4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = rr[j] = f4{0, 0, 0, 0};
    float dot = 0.0f;
    for (int v0 = 0; v0 < V; v0 += 32) {
        if (v0 > 0) __syncthreads();
        float a[8], b[8];
        u4 plane[3];
#pragma unroll
        for (int i = 0; i < KP / 64; ++i) {
            const int tile = (piece_row >> 4) + 4 * i, slot = (piece_row & 15) + 16 * (threadIdx.x & 3);
            if (S) {
                next.s[i].floats(a);
                split8(a, plane);
#pragma unroll
                for (int n = 0; n < 3; ++n) *reinterpret_cast<u4*>(lds.stage.s[tile][n][slot]) = plane[n];
            }
            if (dS) {
                next.ds[i].floats(b);
                split8(b, plane);
#pragma unroll
                for (int n = 0; n < 3; ++n) *reinterpret_cast<u4*>(lds.stage.ds[tile][n][slot]) = plane[n];
            }
            if (S && dS)
#pragma unroll
                for (int n = 0; n < 8; ++n) dot += a[n] * b[n];
        }
        next.u.floats(a);
        split8(a, plane);
#pragma unroll
        for (int n = 0; n < 3; ++n)
            *reinterpret_cast<u4*>(lds.stage.u[piece_row >> 4][n][(piece_row & 15) + 16 * (threadIdx.x & 3)]) = plane[n];
        u4 a_do[N], a_dr[3], a_u[3];
        next.grad.floats(a);
        split8(a, a_do);
        next.dr.floats(a);
        split8(a, a_dr);
        __syncthreads();
        if (v0 + 32 < V) fetch(v0 + 32);
        if (dS) {
#pragma unroll
            for (int n = 0; n < 3; ++n) a_u[n] = *reinterpret_cast<const u4*>(lds.stage.u[wave][n][lane]);
        }
#pragma unroll
        for (int c = 0; c < KP / 16; ++c) {
            u4 x[3];
            if (S) {
#pragma unroll
                for (int n = 0; n < 3; ++n) x[n] = *reinterpret_cast<const u4*>(lds.stage.s[c][n][lane]);
                y[c] = mma(a_do, x, y[c]);
                z[c] = mma(a_dr, x, z[c]);
            }
            if (dS) {
#pragma unroll
                for (int n = 0; n < 3; ++n) x[n] = *reinterpret_cast<const u4*>(lds.stage.ds[c][n][lane]);
                w[c] = mma(a_u, x, w[c]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > wave) continue;
            u4 x[3];
#pragma unroll
            for (int n = 0; n < 3; ++n) x[n] = *reinterpret_cast<const u4*>(lds.stage.u[j][n][lane]);
            h[j] = mma(a_do, x, h[j]);
            rr[j] = mma(a_dr, x, rr[j]);
        }
    }
    dot = sum16(dot);
    dot += __shfl_xor(dot, 16);
    dot += __shfl_xor(dot, 32);
    if (lane == 0) lds.dot_part[wave] = dot;
    __syncthreads();
    load_rows<E, KP>(P, lds.rows, env, head, t0, tokens);
    __syncthreads();

    // The triangles N and M; the sums over their rows and columns.
    const int row = 16 * wave + 4 * g;
    f4 row_sum = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float beta_sum = 0.0f, g_sum = 0.0f;
        if (j <= wave) {
            f4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m < KP / 32; ++m) {
                u4 a[N], b[N];
                operand_rows(lds.rows.k, 16 * j, m, b);
                operand_rows(lds.rows.k, 16 * wave, m, a);
                kk = mma(a, b, kk);
                operand_rows(lds.rows.q, 16 * wave, m, a);
                qk = mma(a, b, qk);
            }
            const int column = 16 * j + col;
            const float hi = lds.gates.hi[column], lo = lds.gates.lo[column], beta = lds.gates.beta[column];
            const int episode = lds.gates.episode[column];
            f4 n, mm;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const bool below = row + s > column, on = row + s >= column;
                const float d = on ? decay(lds.gates, row + s, hi, lo, episode) : 0.0f;
                const float ph = P.r.scale * d * h[j][s];
                const float rd = below ? rr[j][s] * d : 0.0f;
                n[s] = on ? ph * beta : 0.0f;
                mm[s] = -rd * beta;
                const float pair = below ? n[s] * qk[s] + mm[s] * kk[s] : 0.0f;
                beta_sum += on ? ph * qk[s] - rd * kk[s] : 0.0f;
                g_sum += pair;
                row_sum[s] += pair;
            }
            store_slot<NP>(lds.n, tile_of(wave, j), lane, n);
            store_slot<NP>(lds.m, tile_of(wave, j), lane, mm);
        }
        lds.beta_part[4 * wave + g][16 * j + col] = beta_sum;
        lds.g_part[4 * wave + g][16 * j + col] = g_sum;
    }
    const f4 e = four(lds.gates.e, row), f = four(lds.gates.f, row), beta = four(lds.gates.beta, row);
    f4 qy = {0, 0, 0, 0}, kz = {0, 0, 0, 0}, kw = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < KP / 16; ++c) {
        y[c] = P.r.scale * gated(y[c], e);
        z[c] = gated(z[c], e);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            float qx = 0.0f, kx = 0.0f;
#pragma unroll
            for (int n = N - 1; n >= 0; --n) {
                qx += to_float(bf16{lds.rows.q[n][row + s][16 * c + col]});
                kx += to_float(bf16{lds.rows.k[n][row + s][16 * c + col]});
            }
            qy[s] += qx * y[c][s];
            kz[s] += kx * z[c][s];
            kw[s] += kx * w[c][s];
        }
        z[c] = beta * f * w[c] - z[c];  // dk's part
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const float own = sum16(row_sum[s] + qy[s] - kz[s]), left = f[s] * sum16(kw[s]);
        if (col == 0) {
            lds.beta_row[row + s] = left;
            lds.f_row[row + s] = beta[s] * left;
            lds.g_row[row + s] = own - beta[s] * left;
        }
    }
    __syncthreads();
    if (wave == 0) {
        float dbeta = lds.beta_row[lane], dG = lds.g_row[lane], f_all = lds.f_row[lane];
#pragma unroll
        for (int n = 0; n < 16; ++n) {
            dbeta += lds.beta_part[n][lane];
            dG -= lds.g_part[n][lane];
        }
        f_all = sum16(f_all);
        f_all += __shfl_xor(f_all, 16);
        f_all += __shfl_xor(f_all, 32);
        if (lane == 63) {
            const float keep = lds.gates.e[63];
            dG += f_all;
            if (keep != 0.0f)
                dG += keep * ((lds.dot_part[0] + lds.dot_part[1]) + (lds.dot_part[2] + lds.dot_part[3]));
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const float later = __shfl_down(dG, d);
            dG += lane + d < 64 ? later : 0.0f;
        }
        if (lane < tokens) {
            const int before = lane > 0 ? lds.gates.episode[lane - 1] : 0;
            const int64_t to = (env * P.r.steps + t0 + lane) * P.r.value_heads + head;
            P.d.d_g[to] = lds.gates.episode[lane] != before ? 0.0f : dG;
            P.d.d_beta[to] = dbeta;
        }
    }

    // dq (in y) and dk (in z).
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const bool left = 2 * m <= wave, below = 2 * m + 1 >= wave;
        u4 n_left[NP], m_left[NP], n_below[NP], m_below[NP];
        if (left) {
            operand_triangle<NP>(lds.n, wave, m, n_left);
            operand_triangle<NP>(lds.m, wave, m, m_left);
        }
        if (below) {
            operand_transpose<NP>(lds.n, wave, m, n_below);
            operand_transpose<NP>(lds.m, wave, m, m_below);
        }
#pragma unroll
        for (int c = 0; c < KP / 16; ++c) {
            u4 b[N];
            operand_columns(lds.rows.k, c, m, b);
            if (left) {
                y[c] = mma(n_left, b, y[c]);
                z[c] = mma(m_left, b, z[c]);
            }
            if (below) {
                z[c] = mma(m_below, b, z[c]);
                operand_columns(lds.rows.q, c, m, b);
                z[c] = mma(n_below, b, z[c]);
            }
        }
    }
    const int left = tokens - 16 * wave;  // rows of the wave's tile
    if (left <= 0) return;
    if (P.group == 1) {
        const int64_t to = ((env * P.r.steps + t0 + 16 * wave) * P.r.key_heads + head) * K;
        const int64_t stride = static_cast<int64_t>(P.r.key_heads) * K;
        store_tiles<E, KP>(static_cast<E*>(P.d.d_q) + to, stride, left, K, y);
        store_tiles<E, KP>(static_cast<E*>(P.d.d_k) + to, stride, left, K, z);
    } else {
        const int64_t to = ((env * P.r.steps + t0 + 16 * wave) * P.r.value_heads + head) * K;
        const int64_t stride = static_cast<int64_t>(P.r.value_heads) * K;
        store_tiles<float, KP>(P.dq_heads + to, stride, left, K, y);
        store_tiles<float, KP>(P.dk_heads + to, stride, left, K, z);
    }
}

// A key head's gradients are the sum of its value heads', in their order.
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

// Columns of a head that a workgroup takes: up to 64, or up to 128 where the head has more.
int columns_of(int value_dim) { return value_dim <= 64 ? 64 : 128; }

int blocks_of(int value_dim) { return (value_dim + columns_of(value_dim) - 1) / columns_of(value_dim); }

// Walks in segments: 0 workgroups of a whole walk are too few to fill the card's 256 CUs, and
// the chunks enough that the summary pass and the join (about as long as four chunks) pay.
int segments_of(int64_t sequences, int value_dim, int64_t chunks) {
    const int64_t blocks = sequences * blocks_of(value_dim);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({256 / std::max<int64_t>(1, blocks), chunks / 4, 16})));
}

int64_t segment_floats(int64_t sequences, int key_dim, int value_dim, int segments) {
    return sequences * (segments - 1) * (static_cast<int64_t>(key_dim) * value_dim + key_dim * key_dim);
}

template <class E, int KP, int kThreads, bool kBack, bool kSummary>
int walk(const RuleParams& P, dim3 grid, hipStream_t stream) {
    constexpr size_t lds = sizeof(ScanLds<E, KP, kBack ? 3 : kOutPlanes<E>>);
    if constexpr (kBack)
        hipLaunchKernelGGL((delta_reverse_kernel<E, KP, kThreads, kSummary>), grid, dim3(kThreads), lds, stream, P);
    else
        hipLaunchKernelGGL((delta_forward_kernel<E, KP, kThreads, kSummary>), grid, dim3(kThreads), lds, stream, P);
    return launched("the gated delta rule");
}

template <class E, int KP, bool kBack>
int walk_all(const RuleParams& P, hipStream_t stream) {
    const unsigned sequences = static_cast<unsigned>(P.r.envs * P.r.value_heads);
    const unsigned segments = static_cast<unsigned>(P.n_segments);
    if (segments > 1) {
        const int columns = (P.r.value_dim + 15) / 16 * 16 + P.r.key_dim;
        int code = walk<E, KP, 256, kBack, true>(P, dim3(sequences, (columns + 63) / 64, segments - 1), stream);
        if (code != NAVI_POLICY_OK) return code;
        if (segments > 2) {
            hipLaunchKernelGGL(delta_join_kernel<KP>, dim3(sequences, (P.r.value_dim + 63) / 64), dim3(256),
                               KP * KP * 6, stream, P);
            code = launched("the gated delta rule");
            if (code != NAVI_POLICY_OK) return code;
        }
    }
    const dim3 grid(sequences, blocks_of(P.r.value_dim), segments);
    return columns_of(P.r.value_dim) == 64 ? walk<E, KP, 256, kBack, false>(P, grid, stream)
                                           : walk<E, KP, 512, kBack, false>(P, grid, stream);
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
                       dim3(256), sizeof(GradientLds<E, KP>), stream, P);
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

int64_t chunks_of(int64_t steps) { return (steps + kChunk - 1) / kChunk; }

// Whether the rows of steps lie one after another, 64 of them within reach of a buffer access
// (the bytes from one to the next times 64, and a row, stay below 2^31).
constexpr int64_t kFarthest = INT32_MAX / kChunk - 65536 * 4;
bool rows_apart(const int64_t (&stride)[3], int64_t bytes, int64_t dim) {
    return stride[1] >= dim && stride[1] <= kFarthest / bytes;
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
    return NAVI_POLICY_OK;
}

namespace {

int setup(const navi_delta_rule* r, RuleParams& P) {
    const int code = check_rule(r);
    if (code != NAVI_POLICY_OK) return code;
    P.r = *r;
    P.group = r->value_heads / r->key_heads;
    P.n_chunks = static_cast<int32_t>(chunks_of(r->steps));
    P.n_segments = segments_of(r->envs * r->value_heads, r->value_dim, P.n_chunks);
    const int64_t bytes = r->dtype == NAVI_POLICY_F32 ? 4 : 2;
    if (r->envs * r->value_heads * chunks_of(r->steps) > INT32_MAX)
        return set_error(NAVI_POLICY_E_ARG, "envs * value_heads * chunks must be below 2^31");
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
    const int code = setup(rule, P);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : NAVI_POLICY_OK;
    if (!rule->states != !rule->updates && P.n_chunks > 1)
        return set_error(NAVI_POLICY_E_ARG, "states and updates are saved together or not at all");
    if (P.n_chunks == 0 && !rule->final_state) return NAVI_POLICY_OK;
    if (P.n_segments > 1 && (!rule->scratch || !aligned16(rule->scratch)))
        return set_error(NAVI_POLICY_E_ARG, "scratch must be non-null and 16-byte aligned");
    place_segments(P, static_cast<float*>(rule->scratch));
    return run_typed(P, false, as_stream(stream));
}

extern "C" int64_t navi_delta_scratch(const navi_delta_rule* rule) {
    const int code = check_rule(rule);
    if (code < 0) return code;
    const int64_t sequences = rule->envs * rule->value_heads;
    return 4 * segment_floats(sequences, rule->key_dim, rule->value_dim,
                              segments_of(sequences, rule->value_dim, chunks_of(rule->steps)));
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
    const int64_t segments = segment_floats(sequences, rule->key_dim, rule->value_dim,
                                            segments_of(sequences, rule->value_dim, chunks_of(steps)));
    return 4 * (rounded(states) + rounded(rows) + 2 * rounded(heads) + segments);
}

extern "C" int navi_delta_backward(const navi_delta_rule* rule, const navi_delta_gradients* gradients, void* stream) {
    RuleParams P{};
    const int code = setup(rule, P);
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
    if (rule->steps == 1) P.d.grad_out_stride[1] = rule->value_dim;
    if (!rows_apart(P.d.grad_out_stride, bytes, rule->value_dim))
        return set_error(NAVI_POLICY_E_ARG, "the steps of grad_out overlap or lie too far apart");
    // (16-byte buffer loads need addresses of whole 4-byte words)
    P.wide_state = rule->value_dim % 8 == 0;
    P.wide_do = P.wide_state && reinterpret_cast<uintptr_t>(P.d.grad_out) % 4 == 0 &&
                P.d.grad_out_stride[0] * bytes % 4 == 0 && P.d.grad_out_stride[1] * bytes % 4 == 0 &&
                P.d.grad_out_stride[2] * bytes % 4 == 0;
    return run_typed(P, true, as_stream(stream));
}
