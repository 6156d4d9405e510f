// qk_norm.hip — norms of queries and keys for each head and the rotation by position, one
// pass over each row; the backward pass, one pass over the rows and their gradients.
//
// y = x inv w, inv = 1 / sqrt(sum x^2 [/ D] + eps), then z = rotation(y). Backward, with
// dy = the inverse rotation of dz: dx = inv dy w - x inv^3 sum(dy w x) [/ D], dw = sum over
// rows of dy x inv. Bound by memory: a row is read and written once. 1024 x 128 steps, 4 + 4 heads of
// 64, bfloat16: forward 70 us for 268 MB (3.8 TB/s), backward 101 us for 403 MB (4.0 TB/s).
#include <algorithm>
#include <climits>

#include "policy_common.hpp"

namespace navi_policy {
namespace {

constexpr int kMaxBlocks = 2048;    // workgroups of a launch for each of q and k; they stride over the rows
constexpr int kWeightBlocks = 512;  // where a pass sums weight gradients: rows of partial sums

// n / d for n < 2^31 by one multiplication: with 2^(l-1) < d <= 2^l, m = floor(2^(31+l) / d) + 1
// exceeds 2^(31+l) / d by at most 1 = 2^l / 2^l, so the product's error stays under n / 2^31 < 1
// part in d.
struct Divisor {
    uint32_t d, m, shift;
};

Divisor divisor_of(int64_t d) {
    if (d <= 1) return Divisor{1, 0, 0};
    int l = 0;
    while ((int64_t{1} << l) < d) ++l;
    return Divisor{static_cast<uint32_t>(d), static_cast<uint32_t>((uint64_t{1} << (31 + l)) / d + 1), static_cast<uint32_t>(l - 1)};
}

__device__ inline uint32_t divide(uint32_t n, Divisor by) { return by.m == 0 ? n : __umulhi(n, by.m) >> by.shift; }

struct Side {  // of the queries or of the keys
    const void* x;
    const void* grad;
    void* out;  // y, or dx
    const float* weight;
    float* d_weight;
    float* partial;  // [blocks][D]
    int64_t x_stride[3], grad_stride[3];
    int64_t rows;
    int32_t heads;
    int32_t x_dense, grad_dense;  // rows one after another
    Divisor by_heads;
};

struct NormParams {
    Side side[2];
    int64_t steps, positions_end, positions_stride[2];
    const void* positions;
    const float* cos;
    const float* sin;
    float eps, share;  // the sum of squares is multiplied by `share`
    int32_t dim, pairs, interleaved, positions_wide, blocks;
    int32_t small;  // rows below 2^31
    int32_t positions_dense;
    Divisor by_steps;
};

struct Row {
    int64_t x, grad;  // offsets
    int64_t position;
};

// Where a row is. Its env, step and head are asked for only where rows are not one after another
// (all conditions are the launch's: scalar branches).
template <bool kBack>
__device__ inline Row row_of(const NormParams& P, const Side& s, int64_t r) {
    Row at{r * P.dim, r * P.dim, 0};
    const bool scattered = !s.x_dense || (kBack && !s.grad_dense);
    if (!scattered && P.pairs == 0) return at;
    int64_t token, env, step;
    int32_t head;
    if (P.small) {
        const uint32_t row = static_cast<uint32_t>(r), t = divide(row, s.by_heads), e = divide(t, P.by_steps);
        head = static_cast<int32_t>(row - t * s.by_heads.d);
        token = t;
        env = e;
        step = t - e * P.by_steps.d;
    } else {
        token = r / s.heads;
        head = static_cast<int32_t>(r - token * s.heads);
        env = token / P.steps;
        step = token - env * P.steps;
    }
    if (!s.x_dense) at.x = env * s.x_stride[0] + step * s.x_stride[1] + head * s.x_stride[2];
    if (kBack && !s.grad_dense) at.grad = env * s.grad_stride[0] + step * s.grad_stride[1] + head * s.grad_stride[2];
    if (P.pairs == 0) return at;
    at.position = step;
    if (P.positions) {
        const int64_t offset = P.positions_dense ? token : env * P.positions_stride[0] + step * P.positions_stride[1];
        at.position = P.positions_wide ? static_cast<const int64_t*>(P.positions)[offset]
                                       : static_cast<const int32_t*>(P.positions)[offset];
    }
    return at;
}

template <class E>
__device__ inline void load_eight(const E* from, float (&x)[8]) {
    union {
        u4 words[sizeof(E) == 4 ? 2 : 1];
        E elements[8];
    } got;
    got.words[0] = *reinterpret_cast<const u4*>(from);
    if constexpr (sizeof(E) == 4) got.words[1] = *reinterpret_cast<const u4*>(from + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(got.elements[i]);
}

template <class E>
__device__ inline void store_eight(E* to, const float (&x)[8]) {
    union {
        u4 words[sizeof(E) == 4 ? 2 : 1];
        E elements[8];
    } put;
#pragma unroll
    for (int i = 0; i < 8; ++i) put.elements[i] = from_float<E>(x[i]);
    *reinterpret_cast<u4*>(to) = put.words[0];
    if constexpr (sizeof(E) == 4) *reinterpret_cast<u4*>(to + 4) = put.words[1];
}

// The rotation of eight numbers of a row at element e by its position: its angles, asked for
// with the row itself, then applied (back: the opposite angles). Pairs and e are multiples of 8
// (of pairs of neighbours, 4). `turned`: 0 none, 1 by its angles, 2 by a position that the tables
// do not have.
__device__ inline void load_turn(const NormParams& P, const Row& at, int e, bool inside, float (&c)[8], float (&s)[8], int& turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = s[i] = 0.0f;
    turned = 0;
    if (!inside || e >= 2 * P.pairs) return;
    turned = at.position >= 0 && at.position < P.positions_end ? 1 : 2;
    const int pair = P.interleaved ? e / 2 : e >= P.pairs ? e - P.pairs : e;
    const int64_t table = (turned == 1 ? at.position * P.pairs : 0) + pair;
    const f4 c0 = *reinterpret_cast<const f4*>(P.cos + table), s0 = *reinterpret_cast<const f4*>(P.sin + table);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = c0[i], s[i] = s0[i];
    if (P.interleaved) return;
    const f4 c1 = *reinterpret_cast<const f4*>(P.cos + table + 4), s1 = *reinterpret_cast<const f4*>(P.sin + table + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[4 + i] = c1[i], s[4 + i] = s1[i];
}

template <bool kBack>
__device__ inline void apply_turn(const NormParams& P, int e, const float (&c)[8], const float (&s)[8], int turned, float (&x)[8]) {
    if (P.pairs == 0) return;
    if (P.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float sine = kBack ? -s[i] : s[i], a = x[2 * i], b = x[2 * i + 1];
            if (turned) {
                x[2 * i] = turned == 1 ? a * c[i] - b * sine : __builtin_nanf("");
                x[2 * i + 1] = turned == 1 ? b * c[i] + a * sine : __builtin_nanf("");
            }
        }
        return;
    }
    const bool second = e >= P.pairs;
    const int apart = P.pairs / 8, lane = threadIdx.x & 63;
    const int other = turned ? (second ? lane - apart : lane + apart) : lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = __shfl(x[i], other);
        if (turned) x[i] = turned == 1 ? x[i] * c[i] + (second != kBack ? y : -y) * s[i] : __builtin_nanf("");
    }
}

template <int kLanes>
__device__ inline float sum_row(float x) {
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) x += __shfl_xor(x, d);
    return x;
}

// Rows of eight numbers a lane, kLanes lanes a row (a power of two, at least D / 8). Backward
// takes two rows of a lane at once, so that the loads of both are on their way; forward, which
// waits for less, does better with more waves (1024 x 128 steps, 4 + 4 heads of 64, bfloat16: 69 us
// with one, 90 with two; backward 115 and 101).
template <class E, int kLanes, bool kBack>
__global__ __launch_bounds__(256) void qk_norm_kernel(NormParams P) {
    const Side& S = P.side[blockIdx.y];
    const int lane = threadIdx.x & 63, e = (lane & (kLanes - 1)) * 8;
    const bool inside = e < P.dim;
    constexpr int kRows = 64 / kLanes, kAtOnce = kBack ? 2 : 1;  // of a wave
    const int64_t stride = static_cast<int64_t>(gridDim.x) * 4 * kRows * kAtOnce;
    float weight[8], sum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        weight[i] = S.weight && inside ? S.weight[e + i] : 1.0f;
        sum[i] = 0.0f;
    }
    for (int64_t r0 = (blockIdx.x * 4ll + (threadIdx.x >> 6)) * kRows * kAtOnce; r0 < S.rows; r0 += stride) {
        float x[kAtOnce][8] = {}, dz[kAtOnce][8] = {};
        Row at[kAtOnce];
        float c[kAtOnce][8], s[kAtOnce][8];
        int turned[kAtOnce];
        bool valid[kAtOnce];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            const int64_t r = r0 + n * kRows + lane / kLanes;
            valid[n] = inside && r < S.rows;
            at[n] = row_of<kBack>(P, S, r < S.rows ? r : 0);  // (positions first: loads return in order)
        }
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            if (valid[n]) load_eight(static_cast<const E*>(S.x) + at[n].x + e, x[n]);
            if (kBack && valid[n]) load_eight(static_cast<const E*>(S.grad) + at[n].grad + e, dz[n]);
        }
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) load_turn(P, at[n], e, inside, c[n], s[n], turned[n]);
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            float square = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) square += x[n][i] * x[n][i];
            const float inv = rsqrtf(sum_row<kLanes>(square) * P.share + P.eps);
            float y[8];
            if constexpr (!kBack) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[n][i] * inv * weight[i];
                apply_turn<false>(P, e, c[n], s[n], turned[n], y);
            } else {
                apply_turn<true>(P, e, c[n], s[n], turned[n], dz[n]);
                float dot = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[n][i] *= inv;
                    sum[i] += valid[n] ? dz[n][i] * x[n][i] : 0.0f;
                    dz[n][i] *= weight[i];
                    dot += dz[n][i] * x[n][i];
                }
                dot = sum_row<kLanes>(dot) * P.share;
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = inv * (dz[n][i] - x[n][i] * dot);
            }
            if (valid[n]) store_eight(static_cast<E*>(S.out) + (r0 + n * kRows + lane / kLanes) * P.dim + e, y);
        }
    }
    if (kBack && S.partial) {
        __shared__ float part[4][kLanes * 8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int d = kLanes; d < 64; d *= 2) sum[i] += __shfl_xor(sum[i], d);
            if (lane < kLanes) part[threadIdx.x >> 6][e + i] = sum[i];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < P.dim; i += 256)
            S.partial[static_cast<int64_t>(blockIdx.x) * P.dim + i] = (part[0][i] + part[1][i]) + (part[2][i] + part[3][i]);
    }
}

// The same for any sizes and alignments: a wave a row, the row in LDS. Far from memory's rate where
// rows are short: most lanes of a wave have no number, and its two barriers a row tie four rows
// together. bfloat16, 268 MB read and written forward, 403 back: head dimension 40 with 10 pairs 1028
// and 1459 us (0.26 TB/s; 47 us forward without a rotation, by the kernel above), 80 with 20 pairs 580
// and 858, 1000 without a rotation 169 and 369 (1.6 and 1.1 TB/s).
template <class E, bool kBack>
__global__ __launch_bounds__(256) void qk_norm_any_kernel(NormParams P) {
    constexpr int kEach = NAVI_POLICY_MAX_NORM_DIM / 64;
    __shared__ float row[4][NAVI_POLICY_MAX_NORM_DIM];
    const Side& S = P.side[blockIdx.y];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float sum[kEach] = {};
    const int64_t rounds = (S.rows + gridDim.x * 4ll - 1) / (gridDim.x * 4ll);
    for (int64_t n = 0; n < rounds; ++n) {
        const int64_t r = (n * gridDim.x + blockIdx.x) * 4 + wave;
        const bool valid = r < S.rows;
        const Row at = row_of<kBack>(P, S, valid ? r : 0);
        const E* from = static_cast<const E*>(S.x) + at.x;
        const bool known = at.position >= 0 && at.position < P.positions_end;
        const float* cosine = P.cos + (known ? at.position * P.pairs : 0);
        const float* sine = P.sin + (known ? at.position * P.pairs : 0);
        float x[kEach], square = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int e = lane + 64 * i;
            x[i] = valid && e < P.dim ? to_float(from[e]) : 0.0f;
            square += x[i] * x[i];
        }
        const float inv = rsqrtf(sum_row<64>(square) * P.share + P.eps);
        const E* grad = kBack ? static_cast<const E*>(S.grad) + at.grad : nullptr;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int e = lane + 64 * i;
            if (e >= P.dim) continue;
            if constexpr (kBack)
                row[wave][e] = valid ? to_float(grad[e]) : 0.0f;
            else
                row[wave][e] = x[i] * inv * (S.weight ? S.weight[e] : 1.0f);
        }
        __syncthreads();
        float y[kEach], dot = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int e = lane + 64 * i;
            y[i] = 0.0f;
            if (e >= P.dim) continue;
            y[i] = row[wave][e];
            if (e < 2 * P.pairs) {
                const int pair = P.interleaved ? e / 2 : e < P.pairs ? e : e - P.pairs;
                const bool second = P.interleaved ? (e & 1) : e >= P.pairs;
                const int other = P.interleaved ? e ^ 1 : second ? e - P.pairs : e + P.pairs;
                const float b = row[wave][other];
                y[i] = known ? y[i] * cosine[pair] + (second != kBack ? b : -b) * sine[pair] : __builtin_nanf("");
            }
            if constexpr (kBack) {
                sum[i] += valid ? y[i] * (x[i] * inv) : 0.0f;
                y[i] *= S.weight ? S.weight[e] : 1.0f;
                dot += y[i] * (x[i] * inv);
            }
        }
        if constexpr (kBack) {
            dot = sum_row<64>(dot) * P.share;
#pragma unroll
            for (int i = 0; i < kEach; ++i) y[i] = inv * (y[i] - x[i] * inv * dot);
        }
        if (valid)
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (lane + 64 * i < P.dim)
                    static_cast<E*>(S.out)[r * P.dim + lane + 64 * i] = from_float<E>(y[i]);
        __syncthreads();
    }
    if (kBack && S.partial) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (lane + 64 * i < P.dim) row[wave][lane + 64 * i] = sum[i];
        __syncthreads();
        for (int i = threadIdx.x; i < P.dim; i += 256)
            S.partial[static_cast<int64_t>(blockIdx.x) * P.dim + i] = (row[0][i] + row[1][i]) + (row[2][i] + row[3][i]);
    }
}

// Weight gradients from the workgroups' sums, in their order: eight numbers of a row at a
// time over 32 threads, so that the reads of one thread are few.
__global__ __launch_bounds__(256) void qk_norm_weights_kernel(NormParams P) {
    const Side& S = P.side[blockIdx.y];
    if (!S.partial) return;
    __shared__ float part[32][8];
    const int i = blockIdx.x * 8 + (threadIdx.x & 7), first = threadIdx.x >> 3;
    float sum = 0.0f;
    if (i < P.dim)
        for (int b = first; b < P.blocks; b += 32) sum += S.partial[static_cast<int64_t>(b) * P.dim + i];
    part[first][threadIdx.x & 7] = sum;
    __syncthreads();
    if (threadIdx.x < 8 && i < P.dim) {
        sum = 0.0f;
        for (int b = 0; b < 32; ++b) sum += part[b][threadIdx.x];
        S.d_weight[i] = sum;
    }
}

template <class E, bool kBack>
void launch(const NormParams& P, bool wide, dim3 grid, hipStream_t stream) {
    if (!wide)
        hipLaunchKernelGGL((qk_norm_any_kernel<E, kBack>), grid, dim3(256), 0, stream, P);
    else if (P.dim <= 32)
        hipLaunchKernelGGL((qk_norm_kernel<E, 4, kBack>), grid, dim3(256), 0, stream, P);
    else if (P.dim <= 64)
        hipLaunchKernelGGL((qk_norm_kernel<E, 8, kBack>), grid, dim3(256), 0, stream, P);
    else if (P.dim <= 128)
        hipLaunchKernelGGL((qk_norm_kernel<E, 16, kBack>), grid, dim3(256), 0, stream, P);
    else if (P.dim <= 256)
        hipLaunchKernelGGL((qk_norm_kernel<E, 32, kBack>), grid, dim3(256), 0, stream, P);
    else
        hipLaunchKernelGGL((qk_norm_kernel<E, 64, kBack>), grid, dim3(256), 0, stream, P);
}

int lanes_of(int dim) { return dim <= 32 ? 4 : dim <= 64 ? 8 : dim <= 128 ? 16 : dim <= 256 ? 32 : 64; }

bool wide_rows(const void* p, const int64_t (&stride)[3], int64_t bytes) {
    return aligned16(p) && stride[0] * bytes % 16 == 0 && stride[1] * bytes % 16 == 0 && stride[2] * bytes % 16 == 0;
}

// Whether rows lie one after another (the stride of an axis of one says nothing).
bool dense(const int64_t (&stride)[3], const navi_qk_norm_args* a, int64_t heads) {
    return (heads == 1 || stride[2] == a->head_dim) && (a->steps == 1 || stride[1] == heads * a->head_dim) &&
           (a->envs == 1 || stride[0] == a->steps * heads * a->head_dim);
}

int check(const navi_qk_norm_args* a) {
    if (!a) return set_error(NAVI_POLICY_E_ARG, "args must be non-null");
    if (a->dtype < NAVI_POLICY_F32 || a->dtype > NAVI_POLICY_F16)
        return set_error(NAVI_POLICY_E_ARG, "dtype must be float32, bfloat16 or float16");
    if (a->norm != NAVI_POLICY_NORM_RMS && a->norm != NAVI_POLICY_NORM_L2)
        return set_error(NAVI_POLICY_E_ARG, "norm must be rms or l2");
    if (a->head_dim <= 0 || a->head_dim > NAVI_POLICY_MAX_NORM_DIM)
        return set_error(NAVI_POLICY_E_ARG, "head_dim must be in [1, %d]", NAVI_POLICY_MAX_NORM_DIM);
    if (a->query_heads < 0 || a->key_heads < 0 || a->envs < 0 || a->steps < 0)
        return set_error(NAVI_POLICY_E_ARG, "sizes must not be negative");
    if (a->pairs < 0 || 2 * a->pairs > a->head_dim) return set_error(NAVI_POLICY_E_ARG, "2 * pairs must be in [0, head_dim]");
    if (a->pairs > 0 && (!a->cos || !a->sin || a->positions_end <= 0))
        return set_error(NAVI_POLICY_E_ARG, "a rotation needs cos and sin");
    if (!aligned(4, a->cos, a->sin, a->partial) || !aligned(a->positions_wide ? 8 : 4, a->positions))
        return set_error(NAVI_POLICY_E_ARG, "arrays must be aligned to their elements");
    if (!(a->eps >= 0.0f)) return set_error(NAVI_POLICY_E_ARG, "eps must not be negative");
    return NAVI_POLICY_OK;
}

int run(const navi_qk_norm_args* a, bool back, hipStream_t stream) {
    const int code = check(a);
    if (code != NAVI_POLICY_OK) return code;
    NormParams P{};
    const int64_t tokens = a->envs * a->steps;
    P.side[0] = Side{a->q, a->grad_q, back ? a->d_q : a->q_out, a->q_weight, a->d_q_weight, nullptr, {}, {}, tokens * a->query_heads, a->query_heads, 0, 0, divisor_of(a->query_heads)};
    P.side[1] = Side{a->k, a->grad_k, back ? a->d_k : a->k_out, a->k_weight, a->d_k_weight, nullptr, {}, {}, tokens * a->key_heads, a->key_heads, 0, 0, divisor_of(a->key_heads)};
    const int64_t bytes = a->dtype == NAVI_POLICY_F32 ? 4 : 2;
    const bool inside_lanes = a->interleaved ? a->pairs % 4 == 0 : a->pairs % 8 == 0;
    bool wide = a->head_dim <= 512 && a->head_dim % 8 == 0 && inside_lanes && aligned16(a->cos) && aligned16(a->sin);
    int64_t most = 0;
    for (int i = 0; i < 2; ++i) {
        Side& s = P.side[i];
        std::copy(i ? a->k_stride : a->q_stride, (i ? a->k_stride : a->q_stride) + 3, s.x_stride);
        std::copy(i ? a->grad_k_stride : a->grad_q_stride, (i ? a->grad_k_stride : a->grad_q_stride) + 3, s.grad_stride);
        most = std::max(most, s.rows);
        s.x_dense = dense(s.x_stride, a, s.heads);
        s.grad_dense = dense(s.grad_stride, a, s.heads);
        if (s.rows == 0) continue;
        if (!s.x || !s.out || (back && !s.grad)) return set_error(NAVI_POLICY_E_ARG, "q, k, their gradients and outputs must be non-null");
        if (!aligned(bytes, s.x, s.out) || (back && !aligned(bytes, s.grad)) || !aligned(4, s.weight, s.d_weight))
            return set_error(NAVI_POLICY_E_ARG, "arrays must be aligned to their elements");
        wide = wide && wide_rows(s.x, s.x_stride, bytes) && aligned16(s.out) && (!back || wide_rows(s.grad, s.grad_stride, bytes));
    }
    P.steps = a->steps;
    P.positions = a->positions;
    P.positions_stride[0] = a->positions_stride[0];
    P.positions_stride[1] = a->positions_stride[1];
    P.positions_wide = a->positions_wide;
    P.positions_dense = (a->steps == 1 || a->positions_stride[1] == 1) && (a->envs == 1 || a->positions_stride[0] == a->steps);
    P.positions_end = a->positions_end;
    P.cos = a->cos;
    P.sin = a->sin;
    P.eps = a->eps;
    P.dim = a->head_dim;
    P.share = a->norm == NAVI_POLICY_NORM_RMS ? static_cast<float>(1.0 / a->head_dim) : 1.0f;
    P.pairs = a->pairs;
    P.interleaved = a->interleaved;
    const bool weights = back && (a->d_q_weight || a->d_k_weight);
    if (weights && !a->partial) return set_error(NAVI_POLICY_E_ARG, "weight gradients need partial");
    if (most == 0 && !weights) return NAVI_POLICY_OK;
    P.small = most < INT32_MAX && a->steps < INT32_MAX;
    P.by_steps = divisor_of(a->steps);
    const int64_t rows_of_block = wide ? (back ? 8 : 4) * (64 / lanes_of(a->head_dim)) : 4;
    const int64_t blocks = (most + rows_of_block - 1) / rows_of_block;
    P.blocks = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(blocks, weights ? kWeightBlocks : kMaxBlocks)));
    if (weights) {
        if (a->d_q_weight) P.side[0].partial = a->partial;
        if (a->d_k_weight) P.side[1].partial = a->partial + static_cast<int64_t>(kWeightBlocks) * a->head_dim;
    }
    const dim3 grid(static_cast<unsigned>(P.blocks), 2);
    if (a->dtype == NAVI_POLICY_F32)
        back ? launch<float, true>(P, wide, grid, stream) : launch<float, false>(P, wide, grid, stream);
    else if (a->dtype == NAVI_POLICY_BF16)
        back ? launch<bf16, true>(P, wide, grid, stream) : launch<bf16, false>(P, wide, grid, stream);
    else
        back ? launch<f16, true>(P, wide, grid, stream) : launch<f16, false>(P, wide, grid, stream);
    if (weights)
        hipLaunchKernelGGL(qk_norm_weights_kernel, dim3((a->head_dim + 7) / 8, 2), dim3(256), 0, stream, P);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess)
        return set_error(NAVI_POLICY_E_LAUNCH, "navi_qk_norm: kernel launch failed: %s", hipGetErrorString(err));
    return NAVI_POLICY_OK;
}

}  // namespace
}  // namespace navi_policy

extern "C" int navi_qk_norm(const navi_qk_norm_args* args, void* stream) {
    return navi_policy::run(args, false, navi_policy::as_stream(stream));
}

extern "C" int navi_qk_norm_backward(const navi_qk_norm_args* args, void* stream) {
    return navi_policy::run(args, true, navi_policy::as_stream(stream));
}

extern "C" int64_t navi_qk_norm_workspace(const navi_qk_norm_args* args) {
    const int code = navi_policy::check(args);
    return code != NAVI_POLICY_OK ? code : 8ll * navi_policy::kWeightBlocks * args->head_dim;
}
