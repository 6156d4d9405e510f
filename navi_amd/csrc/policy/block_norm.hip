// block_norm.hip — what stands between two blocks of a residual stream, in one pass over its rows:
// the norm after a block, its gate and scale, the sum with the stream, and the norm before the next.
//
//     n = y r post,  r = 1 / sqrt(mean y^2 + eps),   m = n silu(gate),   h = residual + scale m
//     normed = h q pre,  q = 1 / sqrt(mean h^2 + eps)
//
// Backward, with e = pre dnormed and the same r and q found again from the inputs:
//     dh = dstream + q e - h q^3 mean(e h)          (= dresidual)
//     dm = scale dh,  dgate = dm n silu'(gate),  f = post silu(gate) dm,  dy = r f - y r^3 mean(f y)
// and dscale, dpost, dpre sums over rows of dh m, dm silu(gate) y r, dnormed h q. The norm is that of
// the float32 sum, not of the stream as it is rounded. Bound by memory: each row of each array is
// read or written once, held in registers in between. 1024 x 128 rows of 256 in bfloat16 beside a
// float32 stream take 99 us (470 MB with a gate, 4.7 TB/s), backward 170 (3.9 to 4.4 TB/s with the sums' partials).
#include <algorithm>
#include <climits>

#include "policy_common.hpp"

namespace navi_policy {
namespace {

constexpr int kPartialBlocks = NAVI_POLICY_BLOCK_PARTIALS;

struct Rows {
    const void* p;
    int64_t stride[2];
    int32_t dense;  // rows one after another
};

struct BlockParams {
    navi_block_norm_args a;
    Rows y, residual, gate, grad_stream, grad_normed;
    int64_t rows;
    int32_t blocks;
    int32_t wide;  // rows that 16-byte accesses can
    float share;   // 1 / width
    Divisor by_steps;
};

__device__ inline float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// A row's numbers, lane by lane: vector v of a lane is 8 numbers at 8 (v kLanes + lane).
template <int kLanes, int kVecs>
struct RowOf {
    float x[kVecs][8];

    template <class E>
    __device__ void load(const BlockParams& P, const Rows& from, int64_t row, int lane) {
        int64_t offset = row * P.a.width;
        if (!from.dense) {
            const uint32_t env = divide(static_cast<uint32_t>(row), P.by_steps);
            offset = env * from.stride[0] + (row - static_cast<int64_t>(env) * P.by_steps.d) * from.stride[1];
        }
        const E* base = static_cast<const E*>(from.p) + offset;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const int at = 8 * (v * kLanes + lane);
            if (P.wide) {
                if (at < P.a.width) {
                    load_eight(base + at, x[v]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[v][i] = 0.0f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[v][i] = at + i < P.a.width ? to_float(base[at + i]) : 0.0f;
            }
        }
    }

    template <class E>
    __device__ void store(const BlockParams& P, void* to, int64_t row, int lane) const {
        E* base = static_cast<E*>(to) + row * P.a.width;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const int at = 8 * (v * kLanes + lane);
            if (P.wide) {
                if (at < P.a.width) store_eight(base + at, x[v]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (at + i < P.a.width) base[at + i] = from_float<E>(x[v][i]);
            }
        }
    }

    // A vector of weights, `other` without one.
    __device__ void load_vector(const BlockParams& P, const float* from, int lane, float other) {
#pragma unroll
        for (int v = 0; v < kVecs; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int at = 8 * (v * kLanes + lane) + i;
                x[v][i] = !from ? other : at < P.a.width ? from[at] : 0.0f;
            }
    }

    template <class F>
    __device__ void each(F f) {
#pragma unroll
        for (int v = 0; v < kVecs; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[v][i] = f(v, i);
    }

    template <class F>
    __device__ static float sum(F f) {
        float s[8] = {};
#pragma unroll
        for (int v = 0; v < kVecs; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += f(v, i);
        return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    }
};

// Sums over a row's lanes (of a wave, or of all four).
template <int kLanes>
__device__ inline float over_row(float x) {
#pragma unroll
    for (int d = 1; d < (kLanes < 64 ? kLanes : 64); d *= 2) x += __shfl_xor(x, d);
    if constexpr (kLanes == 256) {
        __shared__ float part[4];
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
        __syncthreads();
        x = (part[0] + part[1]) + (part[2] + part[3]);
    }
    return x;
}

template <class E, class R, int kLanes, int kVecs>
__global__ __launch_bounds__(256) void block_norm_kernel(BlockParams P) {
    using Row = RowOf<kLanes, kVecs>;
    constexpr int kRows = 256 / kLanes;
    const int lane = threadIdx.x % kLanes;
    Row post, pre, scale;
    post.load_vector(P, P.a.post_weight, lane, 1.0f);
    pre.load_vector(P, P.a.pre_weight, lane, 1.0f);
    scale.load_vector(P, P.a.scale, lane, 1.0f);
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * kRows; first < P.rows; first += static_cast<int64_t>(P.blocks) * kRows) {
        const int64_t row = first + threadIdx.x / kLanes;
        const bool inside = row < P.rows;  // (the others of the workgroup wait for the same barriers)
        const int64_t at = inside ? row : P.rows - 1;
        Row y, h, gate;
        y.template load<E>(P, P.y, at, lane);
        h.template load<R>(P, P.residual, at, lane);
        if (P.gate.p) gate.template load<E>(P, P.gate, at, lane);
        const float r = rsqrtf(over_row<kLanes>(Row::sum([&](int v, int i) { return y.x[v][i] * y.x[v][i]; })) * P.share + P.a.eps);
        h.each([&](int v, int i) {
            float m = y.x[v][i] * r * post.x[v][i];
            if (P.gate.p) m *= gate.x[v][i] * sigmoid(gate.x[v][i]);
            return h.x[v][i] + scale.x[v][i] * m;
        });
        const float q = rsqrtf(over_row<kLanes>(Row::sum([&](int v, int i) { return h.x[v][i] * h.x[v][i]; })) * P.share + P.a.eps);
        if (!inside) continue;
        h.template store<R>(P, P.a.stream, row, lane);
        y.each([&](int v, int i) { return h.x[v][i] * q * pre.x[v][i]; });
        y.template store<E>(P, P.a.normed, row, lane);
    }
}

template <class E, class R, int kLanes, int kVecs>
__global__ __launch_bounds__(256) void block_norm_backward_kernel(BlockParams P) {
    using Row = RowOf<kLanes, kVecs>;
    constexpr int kRows = 256 / kLanes;
    extern __shared__ float sums_lds[];
    const int lane = threadIdx.x % kLanes;
    Row post, pre, scale, d_post, d_pre, d_scale;
    post.load_vector(P, P.a.post_weight, lane, 1.0f);
    pre.load_vector(P, P.a.pre_weight, lane, 1.0f);
    scale.load_vector(P, P.a.scale, lane, 1.0f);
    d_post.each([](int, int) { return 0.0f; });
    d_pre.each([](int, int) { return 0.0f; });
    d_scale.each([](int, int) { return 0.0f; });
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * kRows; first < P.rows; first += static_cast<int64_t>(P.blocks) * kRows) {
        const int64_t row = first + threadIdx.x / kLanes;
        const bool inside = row < P.rows;
        const int64_t at = inside ? row : P.rows - 1;
        Row y, h, gate, dh, dn;
        y.template load<E>(P, P.y, at, lane);
        h.template load<R>(P, P.residual, at, lane);
        if (P.gate.p)
            gate.template load<E>(P, P.gate, at, lane);
        if (P.grad_stream.p)
            dh.template load<R>(P, P.grad_stream, at, lane);
        else
            dh.each([](int, int) { return 0.0f; });
        if (P.grad_normed.p)
            dn.template load<E>(P, P.grad_normed, at, lane);
        else
            dn.each([](int, int) { return 0.0f; });
        const float r = rsqrtf(over_row<kLanes>(Row::sum([&](int v, int i) { return y.x[v][i] * y.x[v][i]; })) * P.share + P.a.eps);
        y.each([&](int v, int i) { return y.x[v][i] * r; });
        const auto open = [&](int v, int i) { return P.gate.p ? gate.x[v][i] * sigmoid(gate.x[v][i]) : 1.0f; };
        h.each([&](int v, int i) { return h.x[v][i] + scale.x[v][i] * (y.x[v][i] * post.x[v][i] * open(v, i)); });
        const float q = rsqrtf(over_row<kLanes>(Row::sum([&](int v, int i) { return h.x[v][i] * h.x[v][i]; })) * P.share + P.a.eps);
        const float eh = over_row<kLanes>(Row::sum([&](int v, int i) { return dn.x[v][i] * pre.x[v][i] * h.x[v][i]; })) * P.share;
        const float mine = inside ? 1.0f : 0.0f;  // (rows that stand twice are summed once)
        if (P.a.d_pre_weight) d_pre.each([&](int v, int i) { return d_pre.x[v][i] + mine * (dn.x[v][i] * h.x[v][i] * q); });
        dh.each([&](int v, int i) {
            return dh.x[v][i] + q * (dn.x[v][i] * pre.x[v][i] - h.x[v][i] * (q * q * eh));
        });
        if (inside) dh.template store<R>(P, P.a.d_residual, row, lane);
        if (P.a.d_scale)
            d_scale.each([&](int v, int i) { return d_scale.x[v][i] + mine * (dh.x[v][i] * y.x[v][i] * post.x[v][i] * open(v, i)); });
        dh.each([&](int v, int i) { return dh.x[v][i] * scale.x[v][i]; });  // dm
        if (P.gate.p) {
            dn.each([&](int v, int i) {  // dgate
                const float z = gate.x[v][i], s = sigmoid(z);
                return dh.x[v][i] * y.x[v][i] * post.x[v][i] * (s + z * s * (1.0f - s));
            });
            if (inside && P.a.d_gate) dn.template store<E>(P, P.a.d_gate, row, lane);
            dh.each([&](int v, int i) { return dh.x[v][i] * open(v, i); });
        }
        if (P.a.d_post_weight) d_post.each([&](int v, int i) { return d_post.x[v][i] + mine * (dh.x[v][i] * y.x[v][i]); });
        dh.each([&](int v, int i) { return dh.x[v][i] * post.x[v][i]; });
        const float fy = over_row<kLanes>(Row::sum([&](int v, int i) { return dh.x[v][i] * y.x[v][i]; })) * P.share;
        y.each([&](int v, int i) { return r * (dh.x[v][i] - y.x[v][i] * fy); });
        if (inside) y.template store<E>(P, P.a.d_y, row, lane);
    }
    if (!P.a.partial) return;
    // The workgroup's rows together, then its row of partial sums.
    const Row* sums[3] = {&d_scale, &d_post, &d_pre};
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < kVecs; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) sums_lds[(v * 8 + i) * 256 + threadIdx.x] = sums[s]->x[v][i];
        __syncthreads();
        for (int n = threadIdx.x; n < P.a.width; n += 256) {
            const int v = n / (8 * kLanes), l = n / 8 % kLanes, i = n % 8;
            float sum = 0.0f;
            for (int g = 0; g < kRows; ++g) sum += sums_lds[(v * 8 + i) * 256 + g * kLanes + l];
            P.a.partial[(static_cast<int64_t>(blockIdx.x) * 3 + s) * P.a.width + n] = sum;
        }
    }
}

__global__ __launch_bounds__(1024) void block_norm_sums_kernel(BlockParams P) {
    const int column = blockIdx.x * kSumColumns + threadIdx.x % kSumColumns, columns = 3 * P.a.width;
    const float all = sum_of_column(P.a.partial, P.blocks, columns, column);
    if (threadIdx.x >= kSumColumns || column >= columns) return;
    float* to[3] = {P.a.d_scale, P.a.d_post_weight, P.a.d_pre_weight};
    float* at = to[column / P.a.width];
    if (at) at[column % P.a.width] = all;
}

int launched(const char* name) {
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return set_error(NAVI_POLICY_E_LAUNCH, "%s: kernel launch failed: %s", name, hipGetErrorString(err));
    return NAVI_POLICY_OK;
}

template <class E, class R, int kLanes, int kVecs>
int run(BlockParams& P, bool back, hipStream_t stream) {
    const int64_t blocks = (P.rows + 256 / kLanes - 1) / (256 / kLanes);
    // (backward: as many as leave a row of partial sums each)
    P.blocks = static_cast<int32_t>(std::min<int64_t>(blocks, back ? kPartialBlocks : 4096));
    if (!back) {
        hipLaunchKernelGGL((block_norm_kernel<E, R, kLanes, kVecs>), dim3(P.blocks), dim3(256), 0, stream, P);
        return launched("navi_block_norm");
    }
    const unsigned lds = P.a.partial ? kVecs * 8 * 256 * sizeof(float) : 0;
    hipLaunchKernelGGL((block_norm_backward_kernel<E, R, kLanes, kVecs>), dim3(P.blocks), dim3(256), lds, stream, P);
    if (P.a.partial) hipLaunchKernelGGL(block_norm_sums_kernel, dim3((3 * P.a.width + kSumColumns - 1) / kSumColumns), dim3(1024), 0, stream, P);
    return launched("navi_block_norm_backward");
}

template <class E, class R>
int sized(BlockParams& P, bool back, hipStream_t stream) {
    if (P.a.width <= 128) return run<E, R, 16, 1>(P, back, stream);
    if (P.a.width <= 256) return run<E, R, 32, 1>(P, back, stream);
    if (P.a.width <= 512) return run<E, R, 64, 1>(P, back, stream);
    if (P.a.width <= 1024) return run<E, R, 64, 2>(P, back, stream);
    if (P.a.width <= 2048) return run<E, R, 256, 1>(P, back, stream);
    if (P.a.width <= 4096) return run<E, R, 256, 2>(P, back, stream);
    return run<E, R, 256, 4>(P, back, stream);
}

int check(const navi_block_norm_args* a) {
    if (!a) return set_error(NAVI_POLICY_E_ARG, "args must be non-null");
    if (a->dtype < NAVI_POLICY_F32 || a->dtype > NAVI_POLICY_F16)
        return set_error(NAVI_POLICY_E_ARG, "dtype must be float32, bfloat16 or float16");
    if (a->stream_dtype != a->dtype && a->stream_dtype != NAVI_POLICY_F32)
        return set_error(NAVI_POLICY_E_ARG, "stream_dtype must be dtype or float32");
    if (a->width <= 0 || a->width > NAVI_POLICY_MAX_BLOCK_WIDTH)
        return set_error(NAVI_POLICY_E_ARG, "width must be in [1, %d]", NAVI_POLICY_MAX_BLOCK_WIDTH);
    if (!(a->eps >= 0.0f)) return set_error(NAVI_POLICY_E_ARG, "eps must not be negative");
    if (a->envs < 0 || a->steps < 0) return set_error(NAVI_POLICY_E_ARG, "envs and steps must not be negative");
    if (a->envs == 0 || a->steps == 0) return 1;
    if (a->envs > INT32_MAX / a->steps) return set_error(NAVI_POLICY_E_ARG, "envs * steps must be below 2^31");
    if (!a->y || !a->residual) return set_error(NAVI_POLICY_E_ARG, "y and residual must be non-null");
    const int64_t bytes = a->dtype == NAVI_POLICY_F32 ? 4 : 2, wide = a->stream_dtype == NAVI_POLICY_F32 ? 4 : 2;
    if (!aligned(bytes, a->y, a->gate, a->normed, a->grad_normed, a->d_y, a->d_gate) ||
        !aligned(wide, a->residual, a->stream, a->grad_stream, a->d_residual) ||
        !aligned(4, a->scale, a->post_weight, a->pre_weight, a->d_scale, a->d_post_weight, a->d_pre_weight, a->partial))
        return set_error(NAVI_POLICY_E_ARG, "arrays must be aligned to their elements");
    return NAVI_POLICY_OK;
}

Rows rows_of(const navi_block_norm_args& a, const void* p, const int64_t (&stride)[2]) {
    Rows r{p, {a.envs > 1 ? stride[0] : 0, a.steps > 1 ? stride[1] : 0}, 0};
    r.dense = (a.steps == 1 || stride[1] == a.width) && (a.envs == 1 || stride[0] == a.steps * a.width);
    return r;
}

int run_typed(const navi_block_norm_args* args, bool back, hipStream_t stream) {
    BlockParams P{};
    const navi_block_norm_args& a = P.a = *args;
    P.rows = a.envs * a.steps;
    P.share = 1.0f / a.width;
    P.by_steps = divisor_of(a.steps);
    P.y = rows_of(a, a.y, a.y_stride);
    P.residual = rows_of(a, a.residual, a.residual_stride);
    P.gate = rows_of(a, a.gate, a.gate_stride);
    if (back) {
        P.grad_stream = rows_of(a, a.grad_stream, a.grad_stream_stride);
        P.grad_normed = rows_of(a, a.grad_normed, a.grad_normed_stride);
    }
    const int64_t bytes = a.dtype == NAVI_POLICY_F32 ? 4 : 2, stream_bytes = a.stream_dtype == NAVI_POLICY_F32 ? 4 : 2;
    const auto wide = [](const Rows& r, int64_t each) {
        return !r.p || (aligned16(r.p) && r.stride[0] * each % 16 == 0 && r.stride[1] * each % 16 == 0);
    };
    P.wide = a.width % 8 == 0 && wide(P.y, bytes) && wide(P.gate, bytes) && wide(P.residual, stream_bytes) &&
             wide(P.grad_stream, stream_bytes) && wide(P.grad_normed, bytes) &&
             (back ? aligned(16, a.d_y, a.d_gate, a.d_residual) : aligned(16, a.normed, a.stream));
    if (a.dtype == NAVI_POLICY_F32) return sized<float, float>(P, back, stream);
    if (a.stream_dtype == NAVI_POLICY_F32)
        return a.dtype == NAVI_POLICY_BF16 ? sized<bf16, float>(P, back, stream) : sized<f16, float>(P, back, stream);
    return a.dtype == NAVI_POLICY_BF16 ? sized<bf16, bf16>(P, back, stream) : sized<f16, f16>(P, back, stream);
}

// Rows are read and written in any order: outputs share no memory with inputs, but the stream may
// take the place of its residual, and normed that of y, number for number (a row's lanes have read it).
int check_apart(const navi_block_norm_args& a) {
    const int64_t bytes = a.dtype == NAVI_POLICY_F32 ? 4 : 2, wide = a.stream_dtype == NAVI_POLICY_F32 ? 4 : 2, W = a.width;
    const auto rows = [&](const void* p, const int64_t(&s)[2], int64_t each) {
        return p ? extent_of(p, {a.envs, a.steps, W, 1}, {s[0], s[1], 1, 0}, each) : Extent{0, 0};
    };
    const int64_t dense[2] = {a.steps * W, W};
    const auto own = [&](const void* to, const void* p, const int64_t(&s)[2]) {
        return to == p && (a.envs == 1 || s[0] == dense[0]) && (a.steps == 1 || s[1] == W);
    };
    const auto vector = [&](const float* p) { return p ? extent_of(p, {W, 1, 1, 1}, {1, 0, 0, 0}, 4) : Extent{0, 0}; };
    const Extent stream = rows(a.stream, dense, wide), normed = rows(a.normed, dense, bytes);
    const Extent y = rows(a.y, a.y_stride, bytes), residual = rows(a.residual, a.residual_stride, wide);
    const Extent others[] = {rows(a.gate, a.gate_stride, bytes), vector(a.scale), vector(a.post_weight), vector(a.pre_weight)};
    bool fine = apart(stream, normed) && apart(stream, y) && apart(normed, residual);
    for (const Extent& r : others) fine = fine && apart(stream, r) && apart(normed, r);
    fine = fine && (own(a.stream, a.residual, a.residual_stride) || apart(stream, residual));
    fine = fine && (own(a.normed, a.y, a.y_stride) || apart(normed, y));
    return fine ? NAVI_POLICY_OK : set_error(NAVI_POLICY_E_ARG, "stream or normed shares memory with what is read");
}

}  // namespace
}  // namespace navi_policy

extern "C" int navi_block_norm(const navi_block_norm_args* args, void* stream) {
    using namespace navi_policy;
    const int code = check(args);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : NAVI_POLICY_OK;
    if (!args->stream || !args->normed) return set_error(NAVI_POLICY_E_ARG, "stream and normed must be non-null");
    const int shared = check_apart(*args);
    if (shared != NAVI_POLICY_OK) return shared;
    return run_typed(args, false, as_stream(stream));
}

extern "C" int64_t navi_block_norm_workspace(const navi_block_norm_args* args) {
    using namespace navi_policy;
    const int code = check(args);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : 0;
    return std::min<int64_t>(kPartialBlocks, args->envs * args->steps) * 3 * args->width * 4;
}

extern "C" int navi_block_norm_backward(const navi_block_norm_args* args, void* stream) {
    using namespace navi_policy;
    const int code = check(args);
    if (code < 0) return code;
    if (code != NAVI_POLICY_OK) return set_error(NAVI_POLICY_E_ARG, "the backward pass needs at least one row");
    if (!args->d_y || !args->d_residual) return set_error(NAVI_POLICY_E_ARG, "d_y and d_residual must be non-null");
    if ((args->d_scale || args->d_post_weight || args->d_pre_weight) && !args->partial)
        return set_error(NAVI_POLICY_E_ARG, "gradients of scale and weights need the workspace");
    return run_typed(args, true, as_stream(stream));
}
