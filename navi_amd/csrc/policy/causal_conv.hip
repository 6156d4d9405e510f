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
// zero, an infinity of another episode is not seen.
#include <algorithm>
#include <climits>

#include "policy_common.hpp"

namespace navi_policy {
namespace {

constexpr int kBatch = 8;          // rows asked for at once
constexpr int kMaxTaps = NAVI_POLICY_MAX_TAPS;
constexpr int kPartialBlocks = NAVI_POLICY_CONV_PARTIALS;  // most workgroups' worth of sums a channel has

struct ConvParams {
    navi_causal_conv_args a;
    int32_t groups;          // pieces of a row
    int32_t across, rows;    // of a workgroup: pieces, and segments at once
    int32_t across_blocks;   // workgroups that a row takes
    int32_t down_blocks;     // workgroups down the segments
    int32_t segment;         // tokens
    int64_t segments;        // of an env
};

// Pieces of rows as they lie in memory.
template <class E, int kVec>
struct Piece {
    u4 words;
    __device__ void load(const E* from) { words = *reinterpret_cast<const u4*>(from); }
    __device__ void store(E* to) const { *reinterpret_cast<u4*>(to) = words; }
    __device__ void clear() { words = u4{0, 0, 0, 0}; }
    __device__ void floats(float (&x)[kVec]) const {
        union {
            u4 words;
            E elements[kVec];
        } got{words};
#pragma unroll
        for (int i = 0; i < kVec; ++i) x[i] = to_float(got.elements[i]);
    }
    __device__ void from(const float (&x)[kVec]) {
        union {
            u4 words;
            E elements[kVec];
        } put;
#pragma unroll
        for (int i = 0; i < kVec; ++i) put.elements[i] = from_float<E>(x[i]);
        words = put.words;
    }
};

template <class E>
struct Piece<E, 1> {
    E element;
    __device__ void load(const E* from) { element = *from; }
    __device__ void store(E* to) const { *to = element; }
    __device__ void clear() { element = from_float<E>(0.0f); }
    __device__ void floats(float (&x)[1]) const { x[0] = to_float(element); }
    __device__ void from(const float (&x)[1]) { element = from_float<E>(x[0]); }
};

// 1 / (1 + e^-z): e^-z overflows to infinity for z below -88, and its reciprocal to 0.
__device__ inline float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// Where a thread works: a piece of the channels, and segments from `item` on.
struct Place {
    int32_t channel;
    int64_t item, step;
    bool inside;
};

template <int kVec>
__device__ inline Place place_of(const ConvParams& P) {
    const int32_t block = blockIdx.x % P.across_blocks, down = blockIdx.x / P.across_blocks;
    const int32_t c = threadIdx.x % P.across, r = threadIdx.x / P.across;
    const int32_t group = block * P.across + c;
    return Place{group * kVec, static_cast<int64_t>(down) * P.rows + r, static_cast<int64_t>(P.down_blocks) * P.rows,
                 r < P.rows && group < P.groups};
}

// The inputs before a segment's first token, in its episode: held[k] is that of k + 1 tokens before.
template <class E, int kVec, int kTaps>
__device__ inline void begin_segment(const ConvParams& P, int64_t env, int64_t t0, int32_t channel, Piece<E, kVec> (&held)[kTaps - 1]) {
    const E* x = static_cast<const E*>(P.a.x) + env * P.a.x_stride[0] + channel;
    const E* window = P.a.window ? static_cast<const E*>(P.a.window) + env * (kTaps - 1) * P.a.channels + channel : nullptr;
    bool same = true;  // no token after the one k + 1 before has begun an episode
#pragma unroll
    for (int k = 0; k < kTaps - 1; ++k) {
        held[k].clear();
        const int64_t t = t0 - 1 - k;
        if (k > 0 && t + 1 >= 0 && P.a.starts && P.a.starts[env * P.a.starts_stride[0] + (t + 1) * P.a.starts_stride[1]]) same = false;
        if (!same) continue;
        if (t >= 0)
            held[k].load(x + t * P.a.x_stride[1]);
        else if (window)
            held[k].load(window + (kTaps - 1 + t) * P.a.channels);
    }
}

template <class E, int kVec, int kTaps>
__device__ inline void load_weights(const ConvParams& P, int32_t channel, float (&weight)[kTaps][kVec], float (&bias)[kVec]) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        bias[i] = P.a.bias ? P.a.bias[channel + i] : 0.0f;
#pragma unroll
        for (int k = 0; k < kTaps; ++k) weight[k][i] = P.a.weight[static_cast<int64_t>(channel + i) * kTaps + kTaps - 1 - k];
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
    const Place at = place_of<kVec>(P);
    if (!at.inside) return;
    float weight[kTaps][kVec], bias[kVec];
    load_weights<E, kVec, kTaps>(P, at.channel, weight, bias);
    for (int64_t item = at.item; item < P.a.envs * P.segments; item += at.step) {
        const int64_t env = item / P.segments, t0 = (item - env * P.segments) * P.segment;
        const int64_t t1 = t0 + P.segment < P.a.steps ? t0 + P.segment : P.a.steps;
        const E* x = static_cast<const E*>(P.a.x) + env * P.a.x_stride[0] + at.channel;
        const uint8_t* starts = P.a.starts ? P.a.starts + env * P.a.starts_stride[0] : nullptr;
        E* out = static_cast<E*>(P.a.out) + env * P.a.steps * P.a.channels + at.channel;
        Piece<E, kVec> held[kTaps - 1];
        begin_segment<E, kVec, kTaps>(P, env, t0, at.channel, held);
        for (int64_t t = t0; t < t1; t += kBatch) {
            Piece<E, kVec> row[kBatch];
            bool start[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                start[i] = false;
                if (t + i < t1) {
                    row[i].load(x + (t + i) * P.a.x_stride[1]);
                    if (starts) start[i] = starts[(t + i) * P.a.starts_stride[1]] != 0;
                }
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (t + i >= t1) break;
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
                y.store(out + (t + i) * P.a.channels);
                push<E, kVec, kTaps>(row[i], held);
            }
        }
        if (P.a.window_out && t1 == P.a.steps) {
            E* to = static_cast<E*>(P.a.window_out) + env * (kTaps - 1) * P.a.channels + at.channel;
#pragma unroll
            for (int k = 0; k < kTaps - 1; ++k) held[k].store(to + (kTaps - 2 - k) * P.a.channels);
        }
    }
}

// A segment's lane walks its tokens and taps - 1 after them, dz of each once: `pending[k]` is what
// the input k tokens before has got so far.
template <class E, int kVec, int kTaps>
__global__ __launch_bounds__(256) void causal_conv_backward_kernel(ConvParams P) {
    constexpr int kSums = kTaps + 1;
    extern __shared__ float sums_lds[];
    const Place at = place_of<kVec>(P);
    float sums[kSums][kVec] = {};
    if (at.inside) {
        float weight[kTaps][kVec], bias[kVec];
        load_weights<E, kVec, kTaps>(P, at.channel, weight, bias);
        for (int64_t item = at.item; item < P.a.envs * P.segments; item += at.step) {
            const int64_t env = item / P.segments, t0 = (item - env * P.segments) * P.segment;
            const int64_t t1 = t0 + P.segment < P.a.steps ? t0 + P.segment : P.a.steps;
            const int64_t first = t0 == 0 ? -(kTaps - 1) : t0;  // the first segment has the window's gradients too
            const int64_t last = t1 + kTaps - 1 < P.a.steps ? t1 + kTaps - 1 : P.a.steps;
            const E* x = static_cast<const E*>(P.a.x) + env * P.a.x_stride[0] + at.channel;
            const E* dy = static_cast<const E*>(P.a.grad_out) + env * P.a.grad_out_stride[0] + at.channel;
            const uint8_t* starts = P.a.starts ? P.a.starts + env * P.a.starts_stride[0] : nullptr;
            E* dx = static_cast<E*>(P.a.d_x) + env * P.a.steps * P.a.channels + at.channel;
            E* d_window = P.a.d_window ? static_cast<E*>(P.a.d_window) + env * (kTaps - 1) * P.a.channels + at.channel : nullptr;
            Piece<E, kVec> held[kTaps - 1];
            begin_segment<E, kVec, kTaps>(P, env, t0, at.channel, held);
            float pending[kTaps][kVec] = {};
            int since = kTaps;  // tokens since the last start, as far as any tap asks
            const auto finish = [&](int64_t t) {  // the oldest has all that it gets
                if (t >= first && t < t1) {
                    Piece<E, kVec> d;
                    d.from(pending[kTaps - 1]);
                    if (t >= 0)
                        d.store(dx + t * P.a.channels);
                    else if (d_window)
                        d.store(d_window + (kTaps - 1 + t) * P.a.channels);
                }
#pragma unroll
                for (int k = kTaps - 1; k > 0; --k)
#pragma unroll
                    for (int n = 0; n < kVec; ++n) pending[k][n] = pending[k - 1][n];
#pragma unroll
                for (int n = 0; n < kVec; ++n) pending[0][n] = 0.0f;
            };
            for (int64_t t = t0; t < last; t += kBatch) {
                Piece<E, kVec> row[kBatch], grad[kBatch];
                bool start[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    start[i] = false;
                    if (t + i < last) {
                        row[i].load(x + (t + i) * P.a.x_stride[1]);
                        grad[i].load(dy + (t + i) * P.a.grad_out_stride[1]);
                        if (starts) start[i] = starts[(t + i) * P.a.starts_stride[1]] != 0;
                    }
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    if (t + i >= last) break;
                    since = start[i] ? 0 : since < kTaps ? since + 1 : kTaps;
                    if (start[i])
#pragma unroll
                        for (int k = 0; k < kTaps - 1; ++k) held[k].clear();
                    float z[kVec], dz[kVec];
                    convolve<E, kVec, kTaps>(row[i], held, weight, bias, z);
                    grad[i].floats(dz);
                    if (P.a.activation == NAVI_POLICY_SILU)
#pragma unroll
                        for (int n = 0; n < kVec; ++n) {
                            const float s = sigmoid(z[n]);
                            dz[n] *= s + z[n] * s * (1.0f - s);
                        }
#pragma unroll
                    for (int k = 0; k < kTaps; ++k)
                        if (k <= since)
#pragma unroll
                            for (int n = 0; n < kVec; ++n) pending[k][n] += weight[k][n] * dz[n];
                    if (t + i < t1) {
                        float in[kVec];
                        row[i].floats(in);
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
                    push<E, kVec, kTaps>(row[i], held);
                    finish(t + i - (kTaps - 1));
                }
            }
            // What is left: inputs whose last readers are done, and those that the window after
            // the last step holds (pending[k + 1] is the input k + 1 tokens before `last`).
            const E* grad_window = P.a.grad_window && last == P.a.steps
                                       ? static_cast<const E*>(P.a.grad_window) + env * (kTaps - 1) * P.a.channels + at.channel : nullptr;
#pragma unroll
            for (int k = 0; k < kTaps - 1; ++k) {
                if (!grad_window || k > since) continue;
                Piece<E, kVec> g;
                g.load(grad_window + (kTaps - 2 - k) * P.a.channels);
                float x[kVec];
                g.floats(x);
#pragma unroll
                for (int n = 0; n < kVec; ++n) pending[k + 1][n] += x[n];
            }
#pragma unroll
            for (int k = 0; k < kTaps - 1; ++k) finish(last - (kTaps - 1) + k);
        }
    }
    if (!P.a.partial) return;
    // The workgroup's segments together, then its row of partial sums.
#pragma unroll
    for (int s = 0; s < kSums; ++s)
#pragma unroll
        for (int n = 0; n < kVec; ++n) sums_lds[(s * kVec + n) * 256 + threadIdx.x] = sums[s][n];
    __syncthreads();
    const int32_t block = blockIdx.x % P.across_blocks, down = blockIdx.x / P.across_blocks;
    for (int32_t i = threadIdx.x; i < P.across * kSums * kVec; i += 256) {
        const int32_t c = i % P.across, s = i / P.across, channel = (block * P.across + c) * kVec + s % kVec;
        if (block * P.across + c >= P.groups) continue;
        float sum = 0.0f;
        for (int32_t r = 0; r < P.rows; ++r) sum += sums_lds[s * 256 + r * P.across + c];
        P.a.partial[(static_cast<int64_t>(down) * kSums + s / kVec) * P.a.channels + channel] = sum;
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

// How a call is laid out. Segments are as long as leaves 2^16 lanes (of 2^18 that the card holds at
// once) their own; longer ones read fewer inputs twice, shorter ones fill the card.
void lay_out(ConvParams& P, int vec, bool back) {
    const navi_causal_conv_args& a = P.a;
    P.groups = a.channels / vec;
    P.across = std::min(P.groups, 256);
    P.rows = 256 / P.across;
    P.across_blocks = (P.groups + P.across - 1) / P.across;
    P.segment = 64;
    while (P.segment > 8 && a.envs * ((a.steps + P.segment - 1) / P.segment) * P.groups < (1 << 16)) P.segment /= 2;
    P.segments = std::max<int64_t>(1, (a.steps + P.segment - 1) / P.segment);
    const int64_t down = (a.envs * P.segments + P.rows - 1) / P.rows;
    const int64_t most = back ? std::max(1, kPartialBlocks / P.across_blocks) : INT32_MAX / P.across_blocks;
    P.down_blocks = static_cast<int32_t>(std::min(down, most));
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
    lay_out(P, kVec, back);
    const int64_t blocks = static_cast<int64_t>(P.across_blocks) * P.down_blocks;
    if (blocks > INT32_MAX) return set_error(NAVI_POLICY_E_ARG, "navi_causal_conv: too many envs, steps and channels");
    if (!back) {
        hipLaunchKernelGGL((causal_conv_kernel<E, kVec, kTaps>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, P);
        return launched("navi_causal_conv");
    }
    const unsigned lds = P.a.partial ? (kTaps + 1) * kVec * 256 * sizeof(float) : 0;
    hipLaunchKernelGGL((causal_conv_backward_kernel<E, kVec, kTaps>), dim3(static_cast<unsigned>(blocks)), dim3(256), lds, stream, P);
    if (P.a.partial)
        hipLaunchKernelGGL((causal_conv_sums_kernel<kTaps>), dim3(((kTaps + 1) * P.a.channels + kSumColumns - 1) / kSumColumns), dim3(1024), 0,
                           stream, P);
    return launched("navi_causal_conv_backward");
}

bool wide(const navi_causal_conv_args& a, bool back) {
    const int64_t bytes = a.dtype == NAVI_POLICY_F32 ? 4 : 2;
    const auto rows = [&](const void* p, const int64_t(&s)[2]) {
        return aligned16(p) && s[0] * bytes % 16 == 0 && s[1] * bytes % 16 == 0;
    };
    bool fine = a.channels * bytes % 16 == 0 && rows(a.x, a.x_stride) && aligned16(a.window);
    if (!back) return fine && aligned16(a.out) && aligned16(a.window_out);
    return fine && rows(a.grad_out, a.grad_out_stride) && aligned16(a.d_x) && aligned16(a.d_window) && aligned16(a.grad_window);
}

template <class E>
int typed(ConvParams& P, bool back, hipStream_t stream) {
    const auto taps = [&](auto vec) {
        constexpr int kVec = decltype(vec)::value;
        if (P.a.taps == 2) return run<E, kVec, 2>(P, back, stream);
        if (P.a.taps == 3) return run<E, kVec, 3>(P, back, stream);
        return run<E, kVec, 4>(P, back, stream);
    };
    if (wide(P.a, back)) return taps(std::integral_constant<int, 16 / sizeof(E)>{});
    return taps(std::integral_constant<int, 1>{});
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
    const int64_t groups = args->channels * (args->dtype == NAVI_POLICY_F32 ? 4 : 2) / 16;  // (of 16 bytes: the fewest)
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
