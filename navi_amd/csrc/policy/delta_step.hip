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
// 104 to 111 us (5.0 TB/s). 64 environments, 4 heads of 64, take 6.5 us: a launch and one trip
// to memory.
#include "policy_common.hpp"

namespace navi_policy {

int check_rule(const navi_delta_rule* r);

namespace {

struct StepParams {
    navi_delta_rule r;
    int32_t group;
    int32_t blocks;  // of 8 kColumns columns in a state
    int64_t units;   // waves' worth of work
};

template <class E, int kRows, int kColumns>
__global__ __launch_bounds__(256) void delta_step_kernel(StepParams P) {
    const int64_t unit = blockIdx.x * static_cast<int64_t>(blockDim.x >> 6) + (threadIdx.x >> 6);
    if (unit >= P.units) return;
    const int lane = threadIdx.x & 63, first = (lane >> 3) * kRows;
    const int64_t sequence = unit / P.blocks;
    const int column = (static_cast<int>(unit % P.blocks) * 8 + (lane & 7)) * kColumns;
    const int64_t env = sequence / P.r.value_heads;
    const int head = static_cast<int>(sequence % P.r.value_heads), key_head = head / P.group;
    const int K = P.r.key_dim, V = P.r.value_dim;
    const bool inside = column < V;  // (kColumns divides V)
    const int64_t offset = sequence * K * V + column;

    float state[kRows][kColumns];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
#pragma unroll
        for (int c = 0; c < kColumns; ++c) state[i][c] = 0.0f;
        if (P.r.initial_state && inside && first + i < K) {
            const float* from = P.r.initial_state + offset + static_cast<int64_t>(first + i) * V;
            if constexpr (kColumns == 4) {
                const f4 x = *reinterpret_cast<const f4*>(from);
#pragma unroll
                for (int c = 0; c < 4; ++c) state[i][c] = x[c];
            } else {
                state[i][0] = *from;
            }
        }
    }
    const E* q = static_cast<const E*>(P.r.q) + env * P.r.q_stride[0] + key_head * P.r.q_stride[2] + first;
    const E* k = static_cast<const E*>(P.r.k) + env * P.r.k_stride[0] + key_head * P.r.k_stride[2] + first;
    const E* v = static_cast<const E*>(P.r.v) + env * P.r.v_stride[0] + head * P.r.v_stride[2] + column;
    const float* g = P.r.g + env * P.r.g_stride[0] + head * P.r.g_stride[2];
    const float* beta = P.r.beta + env * P.r.beta_stride[0] + head * P.r.beta_stride[2];
    E* out = static_cast<E*>(P.r.out) + (env * P.r.steps * P.r.value_heads + head) * V + column;
    for (int64_t t = 0; t < P.r.steps; ++t) {
        float key[kRows], query[kRows], x[kColumns];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const bool valid = first + i < K;
            key[i] = valid ? to_float(k[t * P.r.k_stride[1] + i]) : 0.0f;
            query[i] = valid ? to_float(q[t * P.r.q_stride[1] + i]) : 0.0f;
        }
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
    if (P.r.final_state && inside)
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            if (first + i < K) {
                float* to = P.r.final_state + offset + static_cast<int64_t>(first + i) * V;
                if constexpr (kColumns == 4)
                    *reinterpret_cast<f4*>(to) = f4{state[i][0], state[i][1], state[i][2], state[i][3]};
                else
                    *to = state[i][0];
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
    StepParams P{};
    P.r = *rule;
    P.group = rule->value_heads / rule->key_heads;
    if (rule->dtype == NAVI_POLICY_F32) return columns<float>(P, as_stream(stream));
    if (rule->dtype == NAVI_POLICY_BF16) return columns<bf16>(P, as_stream(stream));
    return columns<f16>(P, as_stream(stream));
}
