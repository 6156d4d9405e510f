// causal_conv.hip — a short convolution over the last frames, channel by channel, and its
// gradients.
//
//     z[t] = bias + sum_k weight[taps - 1 - k] x[t - k]   (k < taps, t - k in t's episode),  y = act(z)
//
// with the window's inputs before the first step. Backward, dz = dy act'(z):
// dx[t] = sum_k weight[taps - 1 - k] dz[t + k] over t + k in t's episode, dweight and dbias sums
// over all tokens. A lane holds a piece of a row (16 bytes) and walks the tokens of a segment with
// the last inputs in registers, so an input is read once but for taps - 1 at each segment's ends.
// A token that begins an episode clears what is held of earlier inputs: nothing is multiplied by a
// zero, an infinity of another episode is not seen. Bound by memory and what hides its latency: 1024 x 128 steps of
// 384 channels in bfloat16 take 55 us forward (201 MB, 3.7 TB/s) and 94 backward (302 MB, 3.2 TB/s; two
// conversions, an exponential and 16 fused products a number of taps 4 beside).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "policy_common.hpp"

namespace navi_policy {
namespace {

constexpr int kBatch = 8, kBackBatch = 4;  // rows asked for at once
constexpr int kMaxTaps = NAVI_POLICY_MAX_TAPS;
constexpr int kPartialBlocks = NAVI_POLICY_CONV_PARTIALS;  // most workgroups' worth of sums a channel has

struct ConvParams {
    navi_causal_conv_args a;
    int32_t across, rows;    // of a workgroup: pieces of a row, and segments at once
    int32_t groups;          // pieces of a row
    int32_t across_blocks;   // workgroups that a row takes
    int32_t down_blocks;     // workgroups down the segments
    int32_t segment;         // tokens
    uint32_t items, segments;  // segments, of all envs and of one
    Divisor by_segments, by_across, by_across_blocks;
};

// Pieces of rows as they lie in memory.
template <class E, int kVec>
struct Piece {
    static constexpr int kBytes = kVec * sizeof(E);
    using Words = std::conditional_t<kBytes == 16, u4, std::conditional_t<kBytes == 8, u2, std::conditional_t<kBytes == 4, uint32_t, uint16_t>>>;
    Words words;

    __device__ void load(Buffer from, uint32_t offset) {
        if constexpr (kBytes == 16)
            words = buffer_load16(from, offset);
        else if constexpr (kBytes == 8)
            words = __builtin_bit_cast(u2, __builtin_amdgcn_raw_buffer_load_b64(from, offset, 0, 0));
        else if constexpr (kBytes == 4)
            words = __builtin_amdgcn_raw_buffer_load_b32(from, offset, 0, 0);
        else
            words = __builtin_amdgcn_raw_buffer_load_b16(from, offset, 0, 0);
    }
    __device__ void store(Buffer to, uint32_t offset) const {
        if constexpr (kBytes == 16)
            __builtin_amdgcn_raw_buffer_store_b128(words, to, offset, 0, 0);
        else if constexpr (kBytes == 8)
            __builtin_amdgcn_raw_buffer_store_b64(words, to, offset, 0, 0);
        else if constexpr (kBytes == 4)
            __builtin_amdgcn_raw_buffer_store_b32(words, to, offset, 0, 0);
        else
            __builtin_amdgcn_raw_buffer_store_b16(words, to, offset, 0, 0);
    }
    __device__ void clear() { words = Words{}; }
    __device__ void floats(float (&x)[kVec]) const {
        union {
            Words words;
            E elements[kVec];
        } got{words};
#pragma unroll
        for (int i = 0; i < kVec; ++i) x[i] = to_float(got.elements[i]);
    }
    __device__ void from(const float (&x)[kVec]) {
        union {
            Words words;
            E elements[kVec];
        } put;
#pragma unroll
        for (int i = 0; i < kVec; ++i) put.elements[i] = from_float<E>(x[i]);
        words = put.words;
    }
};

// 1 / (1 + e^-z): e^-z overflows to infinity for z below -88, and its reciprocal to 0.
__device__ inline float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// Rows [env][step][channels] of an array from an env on, and where a lane is in them: accesses by 32-bit
// offsets, kOutside for what is not there, without branches.
struct Lines {
    Buffer buffer;
    uint32_t lane, step;  // bytes: of the lane's env and channel, and from step to step

    __device__ Lines(const void* base, int64_t stride0, int64_t stride1, uint32_t bytes, uint32_t env0, uint32_t env, int32_t channel) {
        buffer = buffer_of(static_cast<const char*>(base) + env0 * stride0 * bytes, base ? 0x80000000u : 0u);
        lane = static_cast<uint32_t>((env - env0) * stride0 + channel) * bytes;
        step = static_cast<uint32_t>(stride1) * bytes;
    }
    __device__ uint32_t at(int32_t t, bool there) const { return there ? lane + static_cast<uint32_t>(t) * step : kOutside; }
};

// A thread's place: a piece of the channels, and segments from `item` on.
template <int kVec>
struct Place {
    uint32_t first, row, step;  // the workgroup's first segment, the thread's among them, segments from turn to turn
    int32_t channel, block, down;
    bool inside;

    __device__ explicit Place(const ConvParams& P) {
        down = static_cast<int32_t>(divide(blockIdx.x, P.by_across_blocks));
        block = static_cast<int32_t>(blockIdx.x) - down * P.across_blocks;
        row = divide(threadIdx.x, P.by_across);
        const int32_t group = block * P.across + static_cast<int32_t>(threadIdx.x - row * P.across);
        channel = group * kVec;
        first = down * P.rows;
        step = P.down_blocks * P.rows;
        inside = row < static_cast<uint32_t>(P.rows) && group < P.groups;
    }
};

// The inputs before a segment's first token, in its episode: held[k] is that of k + 1 tokens before.
template <class E, int kVec, int kTaps>
__device__ inline void begin_segment(const Lines& x, const Lines& window, const Lines& starts, int32_t t0, bool inside, Piece<E, kVec> (&held)[kTaps - 1]) {
    bool same = inside;  // no token after the one k + 1 before has begun an episode
#pragma unroll
    for (int k = 0; k < kTaps - 1; ++k) {
        const int32_t t = t0 - 1 - k;
        if (k > 0) same = same && __builtin_amdgcn_raw_buffer_load_b8(starts.buffer, starts.at(t + 1, t + 1 >= 0 && inside), 0, 0) == 0;
        Piece<E, kVec> before;
        held[k].load(x.buffer, x.at(t, t >= 0 && same));
        before.load(window.buffer, window.at(kTaps - 1 + t, t < 0 && same));
        held[k].words = t < 0 ? before.words : held[k].words;
    }
}

template <class E, int kVec, int kTaps>
__device__ inline void load_weights(const ConvParams& P, int32_t channel, bool inside, float (&weight)[kTaps][kVec], float (&bias)[kVec]) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        bias[i] = P.a.bias && inside ? P.a.bias[channel + i] : 0.0f;
#pragma unroll
        for (int k = 0; k < kTaps; ++k) weight[k][i] = inside ? P.a.weight[static_cast<int64_t>(channel + i) * kTaps + kTaps - 1 - k] : 0.0f;
    }
}

// z of a token from its input and those held.
template <class E, int kVec, int kTaps>
__device__ inline void convolve(const Piece<E, kVec>& x, const Piece<E, kVec> (&held)[kTaps - 1], const float (&weight)[kTaps][kVec],
                                const float (&bias)[kVec], float (&z)[kVec]) {
    float in[kVec];
    x.floats(in);
#pragma unroll
    for (int i = 0; i < kVec; ++i) z[i] = bias[i] + weight[0][i] * in[i];
#pragma unroll
    for (int k = 1; k < kTaps; ++k) {
        held[k - 1].floats(in);
#pragma unroll
        for (int i = 0; i < kVec; ++i) z[i] += weight[k][i] * in[i];
    }
}

template <class E, int kVec, int kTaps>
__device__ inline void push(const Piece<E, kVec>& x, Piece<E, kVec> (&held)[kTaps - 1]) {
#pragma unroll
    for (int k = kTaps - 2; k > 0; --k) held[k] = held[k - 1];
    held[0] = x;
}

template <class E, int kVec, int kTaps>
__global__ __launch_bounds__(256) void causal_conv_kernel(ConvParams P) {
    const Place<kVec> place(P);
    float weight[kTaps][kVec], bias[kVec];
    load_weights<E, kVec, kTaps>(P, place.channel, place.inside, weight, bias);
    const int64_t dense = static_cast<int64_t>(P.a.steps) * P.a.channels, kept = static_cast<int64_t>(kTaps - 1) * P.a.channels;
    const int32_t steps = static_cast<int32_t>(P.a.steps);
    for (uint32_t first = place.first; first < P.items; first += place.step) {
        const uint32_t item = first + place.row, env0 = divide(first, P.by_segments);
        const bool inside = place.inside && item < P.items;
        const uint32_t env = divide(inside ? item : first, P.by_segments);
        const int32_t t0 = static_cast<int32_t>((inside ? item : first) - env * P.segments) * P.segment;
        const int32_t t1 = t0 + P.segment < steps ? t0 + P.segment : steps;
        const Lines x(P.a.x, P.a.x_stride[0], P.a.x_stride[1], sizeof(E), env0, env, place.channel);
        const Lines starts(P.a.starts, P.a.starts_stride[0], P.a.starts_stride[1], 1, env0, env, 0);
        const Lines out(P.a.out, dense, P.a.channels, sizeof(E), env0, env, place.channel);
        const Lines window(P.a.window, kept, P.a.channels, sizeof(E), env0, env, place.channel);
        Piece<E, kVec> held[kTaps - 1];
        begin_segment<E, kVec, kTaps>(x, window, starts, t0, inside, held);
        for (int32_t t = t0; t < t1; t += kBatch) {
            Piece<E, kVec> row[kBatch];
            uint8_t start[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const bool there = inside && t + i < t1;
                row[i].load(x.buffer, x.at(t + i, there));
                start[i] = __builtin_amdgcn_raw_buffer_load_b8(starts.buffer, starts.at(t + i, there), 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (start[i])
#pragma unroll
                    for (int k = 0; k < kTaps - 1; ++k) held[k].clear();
                float z[kVec];
                convolve<E, kVec, kTaps>(row[i], held, weight, bias, z);
                if (P.a.activation == NAVI_POLICY_SILU)
#pragma unroll
                    for (int n = 0; n < kVec; ++n) z[n] *= sigmoid(z[n]);
                Piece<E, kVec> y;
                y.from(z);
                y.store(out.buffer, out.at(t + i, inside && t + i < t1));
                if (t + i < t1) push<E, kVec, kTaps>(row[i], held);
            }
        }
        if (P.a.window_out) {
            const Lines after(P.a.window_out, kept, P.a.channels, sizeof(E), env0, env, place.channel);
#pragma unroll
            for (int k = 0; k < kTaps - 1; ++k) held[k].store(after.buffer, after.at(kTaps - 2 - k, inside && t1 == steps));
        }
    }
}

// A lane's walk over a segment: `pending[k]` is what the input k tokens before has got so far.
template <class E, int kVec, int kTaps>
struct BackwardWalk {
    float weight[kTaps][kVec], bias[kVec];
    float sums[kTaps + 1][kVec];  // of dz x for each tap, and of dz
    float pending[kTaps][kVec];
    Piece<E, kVec> held[kTaps - 1];
    int since;  // tokens since the last start, as far as any tap asks

    template <bool kSums>
    __device__ void token(const Piece<E, kVec>& x, const Piece<E, kVec>& dy, bool start, bool silu) {
        since = start ? 0 : since < kTaps ? since + 1 : kTaps;
        if (start)
#pragma unroll
            for (int k = 0; k < kTaps - 1; ++k) held[k].clear();
        float z[kVec], dz[kVec];
        convolve<E, kVec, kTaps>(x, held, weight, bias, z);
        dy.floats(dz);
        if (silu)
#pragma unroll
            for (int n = 0; n < kVec; ++n) {
                const float s = sigmoid(z[n]);
                dz[n] *= s + z[n] * s * (1.0f - s);
            }
        if (since >= kTaps - 1) {
#pragma unroll
            for (int k = 0; k < kTaps; ++k)
#pragma unroll
                for (int n = 0; n < kVec; ++n) pending[k][n] += weight[k][n] * dz[n];
        } else {
#pragma unroll
            for (int k = 0; k < kTaps; ++k)
                if (k <= since)
#pragma unroll
                    for (int n = 0; n < kVec; ++n) pending[k][n] += weight[k][n] * dz[n];
        }
        if constexpr (kSums) {
            float in[kVec];
            x.floats(in);
#pragma unroll
            for (int n = 0; n < kVec; ++n) {
                sums[0][n] += dz[n] * in[n];
                sums[kTaps][n] += dz[n];
            }
#pragma unroll
            for (int k = 1; k < kTaps; ++k) {
                held[k - 1].floats(in);
#pragma unroll
                for (int n = 0; n < kVec; ++n) sums[k][n] += dz[n] * in[n];
            }
        }
        push<E, kVec, kTaps>(x, held);
    }

    // The oldest input has all that it gets.
    __device__ Piece<E, kVec> finish() {
        Piece<E, kVec> d;
        d.from(pending[kTaps - 1]);
#pragma unroll
        for (int k = kTaps - 1; k > 0; --k)
#pragma unroll
            for (int n = 0; n < kVec; ++n) pending[k][n] = pending[k - 1][n];
#pragma unroll
        for (int n = 0; n < kVec; ++n) pending[0][n] = 0.0f;
        return d;
    }
};

// Segments' inputs and dy once, with those of the taps - 1 tokens after each segment (whole segments but
// for an env's last, whose walk ends with its last token). Four numbers a lane, also of 16 bits: sums,
// weights and what is pending of eight would leave a SIMD one wave.
template <class E, int kVec, int kTaps>
__global__ __launch_bounds__(256, sizeof(E) == 4 ? 2 : 4) void causal_conv_backward_kernel(ConvParams P) {
    constexpr int kSums = kTaps + 1;
    extern __shared__ float sums_lds[];
    const Place<kVec> place(P);
    BackwardWalk<E, kVec, kTaps> w;
#pragma unroll
    for (int s = 0; s < kSums; ++s)
#pragma unroll
        for (int n = 0; n < kVec; ++n) w.sums[s][n] = 0.0f;
    load_weights<E, kVec, kTaps>(P, place.channel, place.inside, w.weight, w.bias);
    const bool silu = P.a.activation == NAVI_POLICY_SILU;
    const int64_t dense = static_cast<int64_t>(P.a.steps) * P.a.channels, kept = static_cast<int64_t>(kTaps - 1) * P.a.channels;
    const int32_t steps = static_cast<int32_t>(P.a.steps);
    for (uint32_t first = place.first; first < P.items; first += place.step) {
        const uint32_t item = first + place.row, env0 = divide(first, P.by_segments);
        const bool inside = place.inside && item < P.items;
        const uint32_t env = divide(inside ? item : first, P.by_segments);
        const int32_t t0 = static_cast<int32_t>((inside ? item : first) - env * P.segments) * P.segment;
        const int32_t t1 = t0 + P.segment < steps ? t0 + P.segment : steps;
        const int32_t last = t1 + kTaps - 1 < steps ? t1 + kTaps - 1 : steps;
        const Lines x(P.a.x, P.a.x_stride[0], P.a.x_stride[1], sizeof(E), env0, env, place.channel);
        const Lines dy(P.a.grad_out, P.a.grad_out_stride[0], P.a.grad_out_stride[1], sizeof(E), env0, env, place.channel);
        const Lines starts(P.a.starts, P.a.starts_stride[0], P.a.starts_stride[1], 1, env0, env, 0);
        const Lines dx(P.a.d_x, dense, P.a.channels, sizeof(E), env0, env, place.channel);
        const Lines window(P.a.window, kept, P.a.channels, sizeof(E), env0, env, place.channel);
        const Lines d_window(P.a.d_window, kept, P.a.channels, sizeof(E), env0, env, place.channel);
        const auto finish = [&](int32_t t) {
            const Piece<E, kVec> d = w.finish();
            d.store(dx.buffer, dx.at(t, inside && t >= t0 && t < t1));
        };
        begin_segment<E, kVec, kTaps>(x, window, starts, t0, inside, w.held);
#pragma unroll
        for (int k = 0; k < kTaps; ++k)
#pragma unroll
            for (int n = 0; n < kVec; ++n) w.pending[k][n] = 0.0f;
        w.since = kTaps;
        Piece<E, kVec> after[kTaps - 1], after_dy[kTaps - 1];  // the tokens after the segment
        uint8_t after_start[kTaps - 1];
#pragma unroll
        for (int k = 0; k < kTaps - 1; ++k) {
            const bool there = inside && t1 + k < last;
            after[k].load(x.buffer, x.at(t1 + k, there));
            after_dy[k].load(dy.buffer, dy.at(t1 + k, there));
            after_start[k] = __builtin_amdgcn_raw_buffer_load_b8(starts.buffer, starts.at(t1 + k, there), 0, 0);
        }
        for (int32_t t = t0; t < t1; t += kBackBatch) {
            Piece<E, kVec> row[kBackBatch], grad[kBackBatch];
            uint8_t start[kBackBatch];
#pragma unroll
            for (int i = 0; i < kBackBatch; ++i) {
                const bool there = inside && t + i < t1;
                row[i].load(x.buffer, x.at(t + i, there));
                grad[i].load(dy.buffer, dy.at(t + i, there));
                start[i] = __builtin_amdgcn_raw_buffer_load_b8(starts.buffer, starts.at(t + i, there), 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kBackBatch; ++i) {
                if (t + i >= t1) break;
                w.template token<true>(row[i], grad[i], start[i] != 0, silu);
                if (t == 0 && i < kTaps - 1 && P.a.d_window) {  // (what leaves before the first step)
                    const Piece<E, kVec> d = w.finish();
                    d.store(d_window.buffer, d_window.at(i, inside));
                } else {
                    finish(t + i - (kTaps - 1));
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kTaps - 1; ++k) {
            if (t1 + k >= last) break;
            w.template token<false>(after[k], after_dy[k], after_start[k] != 0, silu);
            finish(t1 + k - (kTaps - 1));
        }
        // What is left: inputs whose last readers are done, and those that the window after
        // the last step holds (pending[k + 1] is the input k + 1 tokens before `last`).
        if (P.a.grad_window) {
            const Lines grad_window(P.a.grad_window, kept, P.a.channels, sizeof(E), env0, env, place.channel);
#pragma unroll
            for (int k = 0; k < kTaps - 1; ++k) {
                Piece<E, kVec> g;
                g.load(grad_window.buffer, grad_window.at(kTaps - 2 - k, inside && last == steps && k <= w.since));
                float d[kVec];
                g.floats(d);
#pragma unroll
                for (int n = 0; n < kVec; ++n) w.pending[k + 1][n] += d[n];
            }
        }
#pragma unroll
        for (int k = 0; k < kTaps - 1; ++k) {
            const int32_t t = last - (kTaps - 1) + k;
            const Piece<E, kVec> d = w.finish();
            d.store(dx.buffer, dx.at(t, inside && t >= t0 && t < t1));
            d.store(d_window.buffer, d_window.at(kTaps - 1 + t, inside && t < 0 && t0 == 0));
        }
    }
    if (!P.a.partial) return;
    // The workgroup's segments together, then its row of partial sums.
#pragma unroll
    for (int s = 0; s < kSums; ++s)
#pragma unroll
        for (int n = 0; n < kVec; ++n) sums_lds[(s * kVec + n) * 256 + threadIdx.x] = w.sums[s][n];
    __syncthreads();
    for (int32_t i = threadIdx.x; i < P.across * kSums * kVec; i += 256) {
        const int32_t s = static_cast<int32_t>(divide(i, P.by_across)), c = i - s * P.across;
        const int32_t channel = (place.block * P.across + c) * kVec + s % kVec;
        if (place.block * P.across + c >= P.groups) continue;
        float sum = 0.0f;
        for (int32_t r = 0; r < P.rows; ++r) sum += sums_lds[s * 256 + r * P.across + c];
        P.a.partial[(static_cast<int64_t>(place.down) * kSums + s / kVec) * P.a.channels + channel] = sum;
    }
}

template <int kTaps>
__global__ __launch_bounds__(1024) void causal_conv_sums_kernel(ConvParams P) {
    const int32_t column = blockIdx.x * kSumColumns + threadIdx.x % kSumColumns, columns = (kTaps + 1) * P.a.channels;
    const float all = sum_of_column(P.a.partial, P.down_blocks, columns, column);
    if (threadIdx.x >= kSumColumns || column >= columns) return;
    const int32_t k = column / P.a.channels, channel = column % P.a.channels;
    if (k == kTaps) {
        if (P.a.d_bias) P.a.d_bias[channel] = all;
    } else if (P.a.d_weight) {
        P.a.d_weight[static_cast<int64_t>(channel) * kTaps + kTaps - 1 - k] = all;
    }
}

constexpr int64_t kMostBlocks = (1 << 24) - 1;  // of 256 threads: a launch has fewer than 2^32
constexpr int64_t kReach = int64_t{1} << 31;  // bytes that a workgroup's 32-bit offsets reach

// How a call is laid out. Segments are as long as leaves 2^16 lanes (of 2^18 that the card holds at
// once) their own; longer ones read fewer inputs twice, shorter ones fill the card. false: too large.
bool lay_out(ConvParams& P, int vec, bool back) {
    const navi_causal_conv_args& a = P.a;
    P.groups = a.channels / vec;
    P.across = std::min(P.groups, 256);
    P.across_blocks = (P.groups + P.across - 1) / P.across;
    P.segment = 64;
    while (P.segment > 8 && a.envs * ((a.steps + P.segment - 1) / P.segment) * P.groups < (1 << 16)) P.segment /= 2;
    const int64_t segments = std::max<int64_t>(1, (a.steps + P.segment - 1) / P.segment), items = a.envs * segments;
    // What a workgroup reaches from the first of its envs on: as many as it has rows, if that is near enough.
    const int64_t bytes = a.dtype == NAVI_POLICY_F32 ? 4 : 2;
    const auto reach = [&](int64_t envs) {
        const auto rows = [&](int64_t env, int64_t step) { return envs * std::abs(env) + a.steps * std::abs(step) + a.channels; };
        int64_t most = std::max(rows(a.x_stride[0], a.x_stride[1]), rows(a.steps * a.channels, a.channels));
        if (back) most = std::max(most, rows(a.grad_out_stride[0], a.grad_out_stride[1]));
        return std::max(most * bytes, a.starts ? rows(a.starts_stride[0], a.starts_stride[1]) : 0);
    };
    P.rows = 256 / P.across;
    if (reach((P.rows + segments - 1) / segments + 1) >= kReach) P.rows = 1;
    if (reach(0) >= kReach || items > INT32_MAX / 2) return false;
    P.items = static_cast<uint32_t>(items);
    P.segments = static_cast<uint32_t>(segments);
    const int64_t down = (items + P.rows - 1) / P.rows;
    const int64_t most = back ? std::max(1, kPartialBlocks / P.across_blocks) : kMostBlocks / P.across_blocks;
    P.down_blocks = static_cast<int32_t>(std::min(down, most));
    P.by_segments = divisor_of(segments);
    P.by_across = divisor_of(P.across);
    P.by_across_blocks = divisor_of(P.across_blocks);
    return true;
}

int check(const navi_causal_conv_args* a) {
    if (!a) return set_error(NAVI_POLICY_E_ARG, "args must be non-null");
    if (a->dtype < NAVI_POLICY_F32 || a->dtype > NAVI_POLICY_F16)
        return set_error(NAVI_POLICY_E_ARG, "dtype must be float32, bfloat16 or float16");
    if (a->taps < 2 || a->taps > kMaxTaps) return set_error(NAVI_POLICY_E_ARG, "taps must be in [2, %d]", kMaxTaps);
    if (a->channels <= 0 || a->channels > 65536) return set_error(NAVI_POLICY_E_ARG, "channels must be in [1, 65536]");
    if (a->activation != NAVI_POLICY_NONE && a->activation != NAVI_POLICY_SILU)
        return set_error(NAVI_POLICY_E_ARG, "activation must be none or silu");
    if (a->envs < 0 || a->steps < 0 || a->envs > INT32_MAX || a->steps > INT32_MAX || a->envs * std::max<int64_t>(a->steps, 1) > (int64_t{1} << 40))
        return set_error(NAVI_POLICY_E_ARG, "envs and steps must not be negative, and below 2^31 (2^40 together)");
    for (const int64_t (*stride)[2] : {&a->x_stride, &a->starts_stride, &a->grad_out_stride})
        if ((*stride)[0] < 0 || (*stride)[1] < 0) return set_error(NAVI_POLICY_E_ARG, "strides must not be negative");
    if (a->envs == 0) return 1;
    if (!a->weight || (a->steps > 0 && !a->x)) return set_error(NAVI_POLICY_E_ARG, "x and weight must be non-null");
    const int64_t bytes = a->dtype == NAVI_POLICY_F32 ? 4 : 2;
    if (!aligned(bytes, a->x, a->window, a->out, a->window_out, a->grad_out, a->grad_window, a->d_x, a->d_window) ||
        !aligned(4, a->weight, a->bias, a->d_weight, a->d_bias, a->partial))
        return set_error(NAVI_POLICY_E_ARG, "arrays must be aligned to their elements");
    return NAVI_POLICY_OK;
}

// Workgroups go in any order, so what is written shares no memory with what is read: but with a
// single step, where the lane that writes a number has read it, out may be x and window_out window.
int check_apart(const navi_causal_conv_args& a) {
    const int64_t bytes = a.dtype == NAVI_POLICY_F32 ? 4 : 2, C = a.channels, kept = a.taps - 1;
    const auto rows = [&](const void* p, const int64_t(&s)[2]) {
        return p && a.steps > 0 ? extent_of(p, {a.envs, a.steps, C, 1}, {s[0], s[1], 1, 0}, bytes) : Extent{0, 0};
    };
    const auto dense = [&](const void* p, int64_t n, int64_t each) {
        return p && n > 0 ? extent_of(p, {n, 1, 1, 1}, {1, 0, 0, 0}, each) : Extent{0, 0};
    };
    const Extent x = rows(a.x, a.x_stride), window = dense(a.window, a.envs * kept * C, bytes);
    const Extent out = dense(a.out, a.envs * a.steps * C, bytes), window_out = dense(a.window_out, a.envs * kept * C, bytes);
    const Extent others[] = {dense(a.weight, C * a.taps, 4), dense(a.bias, C, 4),
                             a.starts && a.steps > 0 ? extent_of(a.starts, {a.envs, a.steps, 1, 1}, {a.starts_stride[0], a.starts_stride[1], 0, 0}, 1) : Extent{0, 0}};
    bool fine = apart(out, window_out) && apart(out, window) && apart(window_out, x);
    for (const Extent& r : others) fine = fine && apart(out, r) && apart(window_out, r);
    const bool own = a.steps == 1 && a.out == a.x && (a.envs == 1 || a.x_stride[0] == C);
    fine = fine && (own || apart(out, x)) && ((a.steps <= 1 && a.window_out == a.window) || apart(window_out, window));
    return fine ? NAVI_POLICY_OK : set_error(NAVI_POLICY_E_ARG, "out or the window after shares memory with what is read");
}

int launched(const char* name) {
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return set_error(NAVI_POLICY_E_LAUNCH, "%s: kernel launch failed: %s", name, hipGetErrorString(err));
    return NAVI_POLICY_OK;
}

template <class E, int kVec, int kTaps>
int run(ConvParams& P, bool back, hipStream_t stream) {
    if (!lay_out(P, kVec, back))
        return set_error(NAVI_POLICY_E_ARG, "navi_causal_conv: an env's steps must lie within 2 GiB, and envs * steps / 8 below 2^30");
    const dim3 grid(static_cast<unsigned>(P.across_blocks * P.down_blocks));
    if constexpr (kVec == 1 || kVec * sizeof(E) == 16) {
        if (!back) {
            hipLaunchKernelGGL((causal_conv_kernel<E, kVec, kTaps>), grid, dim3(256), 0, stream, P);
            return launched("navi_causal_conv");
        }
    }
    if constexpr (kVec <= 4) {
        const unsigned lds = P.a.partial ? (kTaps + 1) * kVec * 256 * sizeof(float) : 0;
        hipLaunchKernelGGL((causal_conv_backward_kernel<E, kVec, kTaps>), grid, dim3(256), lds, stream, P);
        if (P.a.partial)
            hipLaunchKernelGGL((causal_conv_sums_kernel<kTaps>), dim3(((kTaps + 1) * P.a.channels + kSumColumns - 1) / kSumColumns), dim3(1024),
                               0, stream, P);
    }
    return launched("navi_causal_conv_backward");
}

// Whether rows are whole pieces of `piece` bytes at their addresses.
bool wide(const navi_causal_conv_args& a, bool back, int64_t piece) {
    const int64_t bytes = a.dtype == NAVI_POLICY_F32 ? 4 : 2;
    const auto rows = [&](const void* p, const int64_t(&s)[2]) {
        return aligned(piece, p) && s[0] * bytes % piece == 0 && s[1] * bytes % piece == 0;
    };
    const bool fine = a.channels * bytes % piece == 0 && rows(a.x, a.x_stride) && aligned(piece, a.window);
    if (!back) return fine && aligned(piece, a.out, a.window_out);
    return fine && rows(a.grad_out, a.grad_out_stride) && aligned(piece, a.d_x, a.d_window, a.grad_window);
}

template <class E, int kVec>
int tapped(ConvParams& P, bool back, hipStream_t stream) {
    if (P.a.taps == 2) return run<E, kVec, 2>(P, back, stream);
    if (P.a.taps == 3) return run<E, kVec, 3>(P, back, stream);
    return run<E, kVec, 4>(P, back, stream);
}

template <class E>
int typed(ConvParams& P, bool back, hipStream_t stream) {
    constexpr int kForward = 16 / sizeof(E);
    if (!back && wide(P.a, back, 16)) return tapped<E, kForward>(P, back, stream);
    if (back && wide(P.a, back, 4 * sizeof(E))) return tapped<E, 4>(P, back, stream);
    return tapped<E, 1>(P, back, stream);
}

int run_typed(const navi_causal_conv_args* args, bool back, hipStream_t stream) {
    ConvParams P{};
    P.a = *args;
    if (P.a.steps <= 1) P.a.x_stride[1] = P.a.grad_out_stride[1] = P.a.channels;  // (the stride of an axis of one may be anything)
    if (P.a.envs == 1) P.a.x_stride[0] = P.a.grad_out_stride[0] = 0;
    if (P.a.dtype == NAVI_POLICY_F32) return typed<float>(P, back, stream);
    if (P.a.dtype == NAVI_POLICY_BF16) return typed<bf16>(P, back, stream);
    return typed<f16>(P, back, stream);
}

}  // namespace
}  // namespace navi_policy

extern "C" int navi_causal_conv(const navi_causal_conv_args* args, void* stream) {
    using namespace navi_policy;
    const int code = check(args);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : NAVI_POLICY_OK;
    if (args->steps > 0 && !args->out) return set_error(NAVI_POLICY_E_ARG, "out must be non-null");
    if (args->steps == 0 && !args->window_out) return NAVI_POLICY_OK;
    const int shared = check_apart(*args);
    if (shared != NAVI_POLICY_OK) return shared;
    return run_typed(args, false, as_stream(stream));
}

extern "C" int64_t navi_causal_conv_workspace(const navi_causal_conv_args* args) {
    using namespace navi_policy;
    const int code = check(args);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : 0;
    const int64_t groups = args->channels / 4;  // (the fewest pieces of a row)
    const int64_t most = std::max<int64_t>(1, kPartialBlocks / std::max<int64_t>(1, (groups + 255) / 256));
    const int64_t down = std::min(most, args->envs * std::max<int64_t>(1, (args->steps + 7) / 8));
    return down * (args->taps + 1) * args->channels * 4;
}

extern "C" int navi_causal_conv_backward(const navi_causal_conv_args* args, void* stream) {
    using namespace navi_policy;
    const int code = check(args);
    if (code != NAVI_POLICY_OK) return code < 0 ? code : NAVI_POLICY_OK;
    if (args->steps == 0) return set_error(NAVI_POLICY_E_ARG, "the backward pass needs at least one step");
    if (!args->grad_out || !args->d_x) return set_error(NAVI_POLICY_E_ARG, "grad_out and d_x must be non-null");
    if ((args->d_weight || args->d_bias) && !args->partial)
        return set_error(NAVI_POLICY_E_ARG, "gradients of the weight and the bias need the workspace");
    return run_typed(args, true, as_stream(stream));
}
