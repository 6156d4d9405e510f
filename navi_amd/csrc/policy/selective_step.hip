// selective_step.hip — the selective state space scan token by token, the state in registers: one
// frame of every environment while acting, and short runs.
//
// With the state S before a token, y = a S^T c + (beta (b . c) + d) x and S <- a S + beta b x^T: S is
// read once, updated and written once. A lane holds kRows consecutive rows of kColumns adjacent
// columns, eight lanes a row of 8 kColumns columns (128 bytes of float32), eight groups of them the
// state dimension; the products join by three exchanges between lanes, and waves share nothing. Bound by memory:
// 1024 environments of 8 heads of 128 x 64 take 92 us for 540 MB (5.9 TB/s), one environment 5.5 us, a trip there and back.
#include "policy_common.hpp"

namespace navi_policy {

int check_selective(const navi_selective_scan_args* a);
int check_selective_apart(const navi_selective_scan_args& a, bool in_place);

namespace {

struct StepParams {
    navi_selective_scan_args a;
    int32_t group;
    int32_t blocks;  // of 8 kColumns columns in a state
    int64_t units;   // waves' worth of work
    int32_t wide;    // rows of b and c that 16-byte loads can read
};

// A lane's part of a row of n numbers, zeros past its end.
template <class E, int kRows>
__device__ inline void load_rows(const E* row, int n, int first, bool wide, float (&x)[kRows]) {
    constexpr int kEach = 16 / sizeof(E);
    const Buffer from = buffer_of(row, n * sizeof(E));
    if (kRows % kEach == 0 && wide) {
        u4 words[(kRows + kEach - 1) / kEach];
#pragma unroll
        for (int w = 0; w < kRows / kEach; ++w) words[w] = buffer_load16(from, (first + w * kEach) * sizeof(E));
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const uint32_t word = words[i / kEach][i % kEach * sizeof(E) / 4];
            if constexpr (sizeof(E) == 4)
                x[i] = float_of(word);
            else
                x[i] = to_float(__builtin_bit_cast(E, static_cast<uint16_t>(word >> (16 * (i % 2)))));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) x[i] = to_float(buffer_load<E>(from, (first + i) * sizeof(E)));
}

template <class E, int kRows, int kColumns>
__global__ __launch_bounds__(256) void selective_step_kernel(StepParams P) {
    const int64_t unit = blockIdx.x * static_cast<int64_t>(blockDim.x >> 6) + wave_of_workgroup();
    if (unit >= P.units) return;
    const int lane = threadIdx.x & 63, first = (lane >> 3) * kRows;
    const int64_t sequence = unit / P.blocks;
    const int column = (static_cast<int>(unit % P.blocks) * 8 + (lane & 7)) * kColumns;
    const int64_t env = sequence / P.a.heads;
    const int head = static_cast<int>(sequence % P.a.heads), group = head / P.group;
    const int N = P.a.state_dim, V = P.a.head_dim;
    const bool inside = column < V;  // (kColumns divides V)
    const uint32_t row_bytes = 4 * V, state_bytes = N * row_bytes;
    const uint32_t offset = inside ? first * row_bytes + 4 * column : kOutside;

    float state[kRows][kColumns];
    const float* initial = P.a.initial_state;
    const Buffer from = buffer_of(initial ? initial + sequence * N * V : nullptr, initial ? state_bytes : 0);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if constexpr (kColumns == 4) {
            const f4 x = __builtin_bit_cast(f4, buffer_load16(from, offset + i * row_bytes));
#pragma unroll
            for (int c = 0; c < 4; ++c) state[i][c] = x[c];
        } else {
            state[i][0] = buffer_load<float>(from, offset + i * row_bytes);
        }
    }
    const E* b = static_cast<const E*>(P.a.b) + env * P.a.b_stride[0] + group * P.a.b_stride[2];
    const E* c = static_cast<const E*>(P.a.c) + env * P.a.c_stride[0] + group * P.a.c_stride[2];
    const E* x = static_cast<const E*>(P.a.x) + env * P.a.x_stride[0] + head * P.a.x_stride[2] + column;
    const float* dt = P.a.dt + env * P.a.dt_stride[0] + head * P.a.dt_stride[2];
    const float a = P.a.a[head], bias = P.a.dt_bias ? P.a.dt_bias[head] : 0.0f, d = P.a.d ? P.a.d[head] : 0.0f;
    E* out = static_cast<E*>(P.a.out) + (env * P.a.steps * P.a.heads + head) * V + column;
    for (int64_t t = 0; t < P.a.steps; ++t) {
        float key[kRows], query[kRows], value[kColumns];
        load_rows(b + t * P.a.b_stride[1], N, first, P.wide, key);
        load_rows(c + t * P.a.c_stride[1], N, first, P.wide, query);
#pragma unroll
        for (int n = 0; n < kColumns; ++n) value[n] = inside ? to_float(x[t * P.a.x_stride[1] + n]) : 0.0f;
        const float z = dt[t * P.a.dt_stride[1]] + bias;
        const float beta = fmaxf(z, 0.0f) + log1pf(expf(-fabsf(z)));
        float keep = expf(beta * a);
        if (P.a.starts && P.a.starts[env * P.a.starts_stride[0] + t * P.a.starts_stride[1]]) keep = 0.0f;
        if (keep == 0.0f) {  // whatever the state holds
#pragma unroll
            for (int i = 0; i < kRows; ++i)
#pragma unroll
                for (int n = 0; n < kColumns; ++n) state[i][n] = 0.0f;
        }
        float read[kColumns], own = 0.0f;
#pragma unroll
        for (int n = 0; n < kColumns; ++n) read[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            own += key[i] * query[i];
#pragma unroll
            for (int n = 0; n < kColumns; ++n) {
                read[n] += state[i][n] * query[i];
                state[i][n] = keep * state[i][n] + key[i] * (beta * value[n]);
            }
        }
#pragma unroll
        for (int s = 8; s < 64; s *= 2) {
            own += __shfl_xor(own, s);
#pragma unroll
            for (int n = 0; n < kColumns; ++n) read[n] += __shfl_xor(read[n], s);
        }
        if (lane < 8 && inside)
#pragma unroll
            for (int n = 0; n < kColumns; ++n)
                out[t * P.a.heads * V + n] = from_float<E>(keep * read[n] + (beta * own + d) * value[n]);
    }
    if (!P.a.final_state) return;
    const Buffer to = buffer_of(P.a.final_state + sequence * N * V, state_bytes);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if constexpr (kColumns == 4) {
            const float row[4] = {state[i][0], state[i][1], state[i][2], state[i][3]};
            buffer_store_four(to, offset + i * row_bytes, row);
        } else {
            buffer_store(to, offset + i * row_bytes, state[i][0]);
        }
    }
}

template <class E, int kRows, int kColumns>
int step(StepParams& P, hipStream_t stream) {
    P.blocks = (P.a.head_dim + 8 * kColumns - 1) / (8 * kColumns);
    P.units = P.a.envs * P.a.heads * P.blocks;
    const unsigned threads = P.units >= 4096 ? 256 : 64;  // few waves: each on a CU of its own
    const int64_t blocks = (P.units + threads / 64 - 1) / (threads / 64);
    if (!launchable(blocks, threads))
        return set_error(NAVI_POLICY_E_ARG, "navi_selective_step: too many envs, heads and columns (a launch has fewer than 2^32 threads)");
    hipLaunchKernelGGL((selective_step_kernel<E, kRows, kColumns>), dim3(static_cast<unsigned>(blocks)), dim3(threads), 0, stream, P);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess)
        return set_error(NAVI_POLICY_E_LAUNCH, "navi_selective_step: kernel launch failed: %s", hipGetErrorString(err));
    return NAVI_POLICY_OK;
}

template <class E, int kColumns>
int rows(StepParams& P, hipStream_t stream) {
    if (P.a.state_dim <= 32) return step<E, 4, kColumns>(P, stream);
    if (P.a.state_dim <= 64) return step<E, 8, kColumns>(P, stream);
    return step<E, 16, kColumns>(P, stream);
}

template <class E>
int columns(StepParams& P, hipStream_t stream) {
    const bool wide = P.a.head_dim % 4 == 0 && aligned16(P.a.initial_state) && aligned16(P.a.final_state);
    return wide ? rows<E, 4>(P, stream) : rows<E, 1>(P, stream);
}

}  // namespace
}  // namespace navi_policy

extern "C" int navi_selective_step(const navi_selective_scan_args* args, void* stream) {
    using namespace navi_policy;
    const int code = check_selective(args);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : NAVI_POLICY_OK;
    if (args->steps > 0 && !args->out) return set_error(NAVI_POLICY_E_ARG, "out must be non-null");
    const int shared = check_selective_apart(*args, true);
    if (shared != NAVI_POLICY_OK) return shared;
    StepParams P{};
    P.a = *args;
    P.group = args->heads / args->groups;
    const int64_t bytes = args->dtype == NAVI_POLICY_F32 ? 4 : 2;
    const auto wide = [&](const void* rows, const int64_t (&stride)[3]) {
        return aligned16(rows) && stride[0] * bytes % 16 == 0 && stride[1] * bytes % 16 == 0 && stride[2] * bytes % 16 == 0;
    };
    P.wide = args->state_dim * bytes % 16 == 0 && wide(args->b, args->b_stride) && wide(args->c, args->c_stride);
    if (args->dtype == NAVI_POLICY_F32) return columns<float>(P, as_stream(stream));
    if (args->dtype == NAVI_POLICY_BF16) return columns<bf16>(P, as_stream(stream));
    return columns<f16>(P, as_stream(stream));
}
