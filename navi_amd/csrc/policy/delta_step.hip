// delta_step.hip — the gated delta rule token by token, the state in registers: one frame of
// every environment while acting, and short runs.
//
// With the state S before a token, the two products S^T k and S^T q come from one pass over
// it: o = scale (a S^T q + beta (k . q) u), so S is read once, updated and written once.
// A lane holds kRows consecutive rows of kColumns adjacent columns, eight lanes a row of
// 8 kColumns columns (128 bytes of float32), eight groups of them the key dimension; the
// products join by three exchanges between lanes, and waves share nothing.
//
// Bound by the state's memory: 1024 environments, 4 heads of 128 x 128, read and write 537 MB in
// 90 to 94 us (5.8 TB/s; 109 with branches at the ends of rows and keys read number by number). 64
// environments, 4 heads of 64, and one of 8 heads of 128 take 5.7 us: a launch and one trip to memory.
#include "policy_common.hpp"

namespace navi_policy {

int check_rule(const navi_delta_rule* r);
int check_apart(const navi_delta_rule* r, bool in_place);

namespace {

struct StepParams {
    navi_delta_rule r;
    int32_t group;
    int32_t blocks;  // of 8 kColumns columns in a state
    int64_t units;   // waves' worth of work
    int32_t wide;    // rows of queries and keys that 16-byte loads can read
};

// A lane's part of a row of K numbers, zeros past its end.
template <class E, int kRows>
__device__ inline void load_rows(const E* row, int K, int first, bool wide, float (&x)[kRows]) {
    constexpr int kEach = 16 / sizeof(E);
    const Buffer from = buffer_of(row, K * sizeof(E));
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
__global__ __launch_bounds__(256) void delta_step_kernel(StepParams P) {
    const int64_t unit = blockIdx.x * static_cast<int64_t>(blockDim.x >> 6) + wave_of_workgroup();
    if (unit >= P.units) return;
    const int lane = threadIdx.x & 63, first = (lane >> 3) * kRows;
    const int64_t sequence = unit / P.blocks;
    const int column = (static_cast<int>(unit % P.blocks) * 8 + (lane & 7)) * kColumns;
    const int64_t env = sequence / P.r.value_heads;
    const int head = static_cast<int>(sequence % P.r.value_heads), key_head = head / P.group;
    const int K = P.r.key_dim, V = P.r.value_dim;
    const bool inside = column < V;  // (kColumns divides V)
    const uint32_t row_bytes = 4 * V, state_bytes = K * row_bytes;
    const uint32_t offset = inside ? first * row_bytes + 4 * column : kOutside;

    float state[kRows][kColumns];
    const float* initial = P.r.initial_state;
    const Buffer from = buffer_of(initial ? initial + sequence * K * V : nullptr, initial ? state_bytes : 0);
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
    const E* q = static_cast<const E*>(P.r.q) + env * P.r.q_stride[0] + key_head * P.r.q_stride[2];
    const E* k = static_cast<const E*>(P.r.k) + env * P.r.k_stride[0] + key_head * P.r.k_stride[2];
    const E* v = static_cast<const E*>(P.r.v) + env * P.r.v_stride[0] + head * P.r.v_stride[2] + column;
    const float* g = P.r.g + env * P.r.g_stride[0] + head * P.r.g_stride[2];
    const float* beta = P.r.beta + env * P.r.beta_stride[0] + head * P.r.beta_stride[2];
    E* out = static_cast<E*>(P.r.out) + (env * P.r.steps * P.r.value_heads + head) * V + column;
    for (int64_t t = 0; t < P.r.steps; ++t) {
        float key[kRows], query[kRows], x[kColumns];
        load_rows(k + t * P.r.k_stride[1], K, first, P.wide, key);
        load_rows(q + t * P.r.q_stride[1], K, first, P.wide, query);
#pragma unroll
        for (int c = 0; c < kColumns; ++c) x[c] = inside ? to_float(v[t * P.r.v_stride[1] + c]) : 0.0f;
        float a = expf(g[t * P.r.g_stride[1]]);
        const float b = beta[t * P.r.beta_stride[1]];
        if (P.r.starts && P.r.starts[env * P.r.starts_stride[0] + t * P.r.starts_stride[1]]) a = 0.0f;
        if (a == 0.0f) {  // whatever the state holds
#pragma unroll
            for (int i = 0; i < kRows; ++i)
#pragma unroll
                for (int c = 0; c < kColumns; ++c) state[i][c] = 0.0f;
        }
        float sk[kColumns], sq[kColumns], kq = 0.0f;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) sk[c] = sq[c] = 0.0f;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            kq += key[i] * query[i];
#pragma unroll
            for (int c = 0; c < kColumns; ++c) {
                sk[c] += state[i][c] * key[i];
                sq[c] += state[i][c] * query[i];
            }
        }
#pragma unroll
        for (int d = 8; d < 64; d *= 2) {
            kq += __shfl_xor(kq, d);
#pragma unroll
            for (int c = 0; c < kColumns; ++c) {
                sk[c] += __shfl_xor(sk[c], d);
                sq[c] += __shfl_xor(sq[c], d);
            }
        }
        float u[kColumns];
#pragma unroll
        for (int c = 0; c < kColumns; ++c) u[c] = b * (x[c] - a * sk[c]);
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int c = 0; c < kColumns; ++c) state[i][c] = a * state[i][c] + key[i] * u[c];
        if (lane < 8 && inside)
#pragma unroll
            for (int c = 0; c < kColumns; ++c)
                out[t * P.r.value_heads * V + c] = from_float<E>(P.r.scale * (a * sq[c] + kq * u[c]));
    }
    if (!P.r.final_state) return;
    const Buffer to = buffer_of(P.r.final_state + sequence * K * V, state_bytes);
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
    P.blocks = (P.r.value_dim + 8 * kColumns - 1) / (8 * kColumns);
    P.units = P.r.envs * P.r.value_heads * P.blocks;
    const unsigned threads = P.units >= 4096 ? 256 : 64;  // few waves: each on a CU of its own
    const int64_t blocks = (P.units + threads / 64 - 1) / (threads / 64);
    if (blocks > INT32_MAX) return set_error(NAVI_POLICY_E_ARG, "navi_delta_step: too many envs, heads and columns");
    hipLaunchKernelGGL((delta_step_kernel<E, kRows, kColumns>), dim3(static_cast<unsigned>(blocks)), dim3(threads), 0, stream, P);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess)
        return set_error(NAVI_POLICY_E_LAUNCH, "navi_delta_step: kernel launch failed: %s", hipGetErrorString(err));
    return NAVI_POLICY_OK;
}

template <class E, int kColumns>
int rows(StepParams& P, hipStream_t stream) {
    if (P.r.key_dim <= 32) return step<E, 4, kColumns>(P, stream);
    if (P.r.key_dim <= 64) return step<E, 8, kColumns>(P, stream);
    return step<E, 16, kColumns>(P, stream);
}

template <class E>
int columns(StepParams& P, hipStream_t stream) {
    const bool wide = P.r.value_dim % 4 == 0 && aligned16(P.r.initial_state) && aligned16(P.r.final_state);
    return wide ? rows<E, 4>(P, stream) : rows<E, 1>(P, stream);
}

}  // namespace
}  // namespace navi_policy

extern "C" int navi_delta_step(const navi_delta_rule* rule, void* stream) {
    using namespace navi_policy;
    const int code = check_rule(rule);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : NAVI_POLICY_OK;
    if (rule->states || rule->updates) return set_error(NAVI_POLICY_E_ARG, "the recurrent form saves no states or updates");
    const int shared = check_apart(rule, true);
    if (shared != NAVI_POLICY_OK) return shared;
    StepParams P{};
    P.r = *rule;
    P.group = rule->value_heads / rule->key_heads;
    const int64_t bytes = rule->dtype == NAVI_POLICY_F32 ? 4 : 2;
    const auto wide = [&](const void* rows, const int64_t (&stride)[3]) {
        return aligned16(rows) && stride[0] * bytes % 16 == 0 && stride[1] * bytes % 16 == 0 && stride[2] * bytes % 16 == 0;
    };
    P.wide = rule->key_dim * bytes % 16 == 0 && wide(rule->q, rule->q_stride) && wide(rule->k, rule->k_stride);
    if (rule->dtype == NAVI_POLICY_F32) return columns<float>(P, as_stream(stream));
    if (rule->dtype == NAVI_POLICY_BF16) return columns<bf16>(P, as_stream(stream));
    return columns<f16>(P, as_stream(stream));
}
