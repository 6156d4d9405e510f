/*
 * navi_policy.h — C ABI of libnavi_policy.so: HIP kernels (gfx950) of the operators that
 * a policy with a memory runs over the tracer's observations, and of its training step.
 *
 * The reference's policy cores (projects/actor) are PyTorch modules; these entry points
 * have no kernel counterpart there. Every pointer is device memory unless noted, aligned to
 * its elements, or to more where that is noted. Launches are asynchronous on `stream`; no entry
 * point allocates device memory, waits for the device or keeps anything of a call. Each
 * returns NAVI_POLICY_OK or a negative code and leaves a message in navi_policy_last_error()
 * (thread-local).
 */
#ifndef NAVI_POLICY_H
#define NAVI_POLICY_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NAVI_POLICY_OK 0
#define NAVI_POLICY_E_ARG (-1)
#define NAVI_POLICY_E_LAUNCH (-2)

/* Element types of queries, keys, values, gradients. */
#define NAVI_POLICY_F32 0
#define NAVI_POLICY_BF16 1
#define NAVI_POLICY_F16 2

/* Largest key dimension of the gated delta rule, and head dimension of navi_qk_norm. */
#define NAVI_POLICY_MAX_KEY_DIM 128
#define NAVI_POLICY_MAX_NORM_DIM 1024
/* Tokens that the chunked form takes at once: saved states lie this far apart. */
#define NAVI_POLICY_CHUNK 64
/* Floats that a chunk's matrices take in navi_delta_rule.matrices. */
#define NAVI_POLICY_CHUNK_MATRICES 5248

/*
 * The gated delta rule. Per env b and value head h (key head h / (value_heads / key_heads)),
 * with the state S a key_dim x value_dim matrix of float32 and a_t = 0 at a token that
 * starts an episode, exp(g_t) elsewhere:
 *
 *     u_t = v_t - a_t S^T k_t,   S <- a_t S + beta_t k_t u_t^T,   o_t = scale S^T q_t
 *
 * q, k: [envs][steps][key_heads][key_dim] of `dtype`, v and out: [envs][steps][value_heads]
 * [value_dim] of it, g and beta: [envs][steps][value_heads] of float32, starts: [envs][steps]
 * of bytes (0 or not) or NULL. Strides are in elements, of the env, step and head axes; the
 * last axis is contiguous, and so are out and the states. g is meant to be <= 0; one of
 * -infinity (below -1e5) starts an episode as `starts` does. An initial state that a start at
 * the first step clears may hold anything. Other inputs are finite: in the chunked form a NaN
 * or infinity may reach every token of its chunk of 64 and what follows them. A launch has fewer than
 * 2^32 threads: envs x value_heads x chunks and envs x value_heads x ceil(value_dim / 64) stay below 2^24 (2^23
 * chunks backward, and 128 columns for 64, where a workgroup has 512 threads).
 */
typedef struct navi_delta_rule {
    int32_t dtype;              /* NAVI_POLICY_* of q, k, v, out and their gradients */
    int32_t key_heads, value_heads;
    int32_t key_dim, value_dim; /* 1 to NAVI_POLICY_MAX_KEY_DIM; 1 to 65536 */
    int64_t envs, steps;
    float scale;
    const void* q;
    const void* k;
    const void* v;
    int64_t q_stride[3], k_stride[3], v_stride[3];
    const float* g;
    const float* beta;
    int64_t g_stride[3], beta_stride[3];
    const uint8_t* starts;      /* or NULL */
    int64_t starts_stride[2];
    const float* initial_state; /* [envs][value_heads][key_dim][value_dim], or NULL for zeros */
    void* out;
    float* final_state;         /* as initial_state, or NULL; may be initial_state itself in
                                   navi_delta_step. Else it shares no memory with what is read, nor
                                   does out, which may be v itself (contiguous) */
    float* matrices; /* [envs * value_heads][chunks][NAVI_POLICY_CHUNK_MATRICES], 16-byte aligned:
                        written by navi_delta_forward, read again by the backward pass (not used by
                        navi_delta_step); chunks = ceil(steps / NAVI_POLICY_CHUNK) */
    void* scratch;   /* navi_delta_scratch bytes for navi_delta_forward alone, 16-byte aligned (NULL where
                        that is 0) */
    /* what the backward pass reads as well, or NULL both: */
    float* states;  /* [envs * value_heads][chunks - 1][key_dim][value_dim] the state before each
                       chunk but the first */
    float* updates; /* [envs * value_heads][steps][value_dim]: u */
} navi_delta_rule;

/* Chunked form: matrix products over chunks of 64 tokens, the states passed from one to the
 * next. For rollouts, and the forward pass of training. */
int navi_delta_forward(const navi_delta_rule* rule, void* stream);

/* Bytes of scratch that navi_delta_forward needs (0 but for long sequences of few heads);
 * negative for invalid sizes. */
int64_t navi_delta_scratch(const navi_delta_rule* rule);

/* Recurrent form: one token after another with the state in registers; for single tokens
 * and short runs. final_state may be initial_state (updated in place). Saves nothing for a
 * backward pass (states and updates must be NULL). */
int navi_delta_step(const navi_delta_rule* rule, void* stream);

/* Gradients (each contiguous in the layout of its input without gaps). */
typedef struct navi_delta_gradients {
    const void* grad_out;           /* of out, `dtype` */
    int64_t grad_out_stride[3];
    const float* grad_final_state;  /* contiguous, or NULL for zeros */
    void* d_q;
    void* d_k;
    void* d_v;
    float* d_g;
    float* d_beta;
    float* d_initial_state;         /* or NULL */
    void* workspace;                /* navi_delta_workspace bytes, 16-byte aligned */
} navi_delta_gradients;

/* Bytes of workspace that navi_delta_backward needs; negative for invalid sizes. */
int64_t navi_delta_workspace(const navi_delta_rule* rule);

/* Backward pass over what navi_delta_forward read and saved (rule->out and
 * rule->final_state are not read). */
int navi_delta_backward(const navi_delta_rule* rule, const navi_delta_gradients* gradients, void* stream);

/*
 * Norms of queries and keys for each head, with the position rotation in the same pass.
 * Per row x of head_dim numbers, y = x / sqrt(sum x^2 [/ head_dim] + eps) [* weight]; then
 * the first 2 * pairs numbers are rotated by the angles of the token's position p: with
 * c = cos[p][i], s = sin[p][i], (y_a, y_b) becomes (y_a c - y_b s, y_b c + y_a s), where
 * (a, b) = (i, i + pairs), or (2 i, 2 i + 1) with `interleaved`.
 * q: [envs][steps][query_heads][head_dim] with strides of the env, step and head axes, the
 * last one contiguous; k likewise; outputs contiguous. A position outside [0, positions_end)
 * gives NaN in the numbers that it would rotate.
 */
#define NAVI_POLICY_NORM_RMS 0 /* mean of squares */
#define NAVI_POLICY_NORM_L2 1  /* sum of squares */

typedef struct navi_qk_norm_args {
    int32_t dtype;
    int32_t norm;          /* NAVI_POLICY_NORM_* */
    int32_t query_heads, key_heads, head_dim;
    int32_t pairs;         /* rotated pairs, 0 for none */
    int32_t interleaved;
    int32_t positions_wide; /* positions are int64, else int32 */
    int64_t envs, steps;
    float eps;
    const void* q;
    const void* k;
    int64_t q_stride[3], k_stride[3];
    const float* q_weight; /* [head_dim] or NULL */
    const float* k_weight;
    const void* positions; /* [envs][steps] with strides, or NULL: a token's step */
    int64_t positions_stride[2];
    const float* cos;      /* [positions_end][pairs] */
    const float* sin;
    int64_t positions_end;
    void* q_out;
    void* k_out;
    /* the backward pass: gradients of q_out and k_out (strides as q's), q_out and k_out not
     * read; d_q and d_k contiguous; d_q_weight, d_k_weight [head_dim] or NULL, through
     * `partial`, navi_qk_norm_workspace bytes (NULL without them). */
    const void* grad_q;
    const void* grad_k;
    int64_t grad_q_stride[3], grad_k_stride[3];
    void* d_q;
    void* d_k;
    float* d_q_weight;
    float* d_k_weight;
    float* partial;
} navi_qk_norm_args;

int navi_qk_norm(const navi_qk_norm_args* args, void* stream);
int navi_qk_norm_backward(const navi_qk_norm_args* args, void* stream);
int64_t navi_qk_norm_workspace(const navi_qk_norm_args* args);

/*
 * The norm of all numbers of n_tensors tensors, sqrt(sum x^2), into norm[0], and the tensors
 * times min(1, max_norm / (norm + eps)) into `to`. A tensor may be scaled in place; otherwise what
 * is written shares no memory with what else is written or read.
 * from, to, counts and dtypes (NAVI_POLICY_*) are host arrays, read during the call; tensors
 * are contiguous and aligned to their elements. `partial`: NAVI_POLICY_NORM_PARTIALS floats.
 * Sums are taken in a fixed order: the same numbers give the same norm.
 */
#define NAVI_POLICY_NORM_PARTIALS 2048

int navi_clip_grad_norm(int32_t n_tensors, const void* const* from, void* const* to, const int64_t* counts,
                        const int32_t* dtypes, float max_norm, float eps, float* norm, float* partial, void* stream);

/*
 * A short convolution over the last frames, channel by channel:
 *
 *     z[t][c] = bias[c] + sum over k < taps of weight[c][taps - 1 - k] x[t - k][c],  out = act(z)
 *
 * where inputs before the first step come from `window` (zeros without one) and inputs of another
 * episode than t's (before the last of `starts` up to t) count as zeros, whatever they hold.
 * x: [envs][steps][channels] of `dtype` with strides of the env and step axes, the last one
 * contiguous; out, windows and d_x contiguous. window_out receives the last taps - 1 inputs (with
 * those of `window` where there are fewer steps), zeros in place of those of an earlier episode
 * than the last token's. Written arrays share no memory with read ones, but with a single step out
 * may be x and window_out window.
 */
#define NAVI_POLICY_MAX_TAPS 4
#define NAVI_POLICY_NONE 0
#define NAVI_POLICY_SILU 1 /* z / (1 + exp(-z)) */
#define NAVI_POLICY_CONV_PARTIALS 2048

typedef struct navi_causal_conv_args {
    int32_t dtype, channels;
    int32_t taps;       /* 2 to NAVI_POLICY_MAX_TAPS */
    int32_t activation; /* NAVI_POLICY_NONE or NAVI_POLICY_SILU */
    int64_t envs, steps;
    const void* x;
    int64_t x_stride[2];
    const float* weight; /* [channels][taps] */
    const float* bias;   /* [channels] or NULL */
    const uint8_t* starts; /* [envs][steps] or NULL */
    int64_t starts_stride[2];
    const void* window; /* [envs][taps - 1][channels] or NULL */
    void* out;
    void* window_out;   /* like window, or NULL */
    /* the backward pass (out and window_out are not read); what it writes shares no memory with anything else: */
    const void* grad_out;
    int64_t grad_out_stride[2];
    const void* grad_window; /* of window_out, contiguous, or NULL */
    void* d_x;
    float* d_weight;    /* or NULL, */
    float* d_bias;      /* or NULL, through */
    void* d_window;     /* or NULL */
    float* partial;     /* navi_causal_conv_workspace bytes (NULL without d_weight and d_bias) */
} navi_causal_conv_args;

int navi_causal_conv(const navi_causal_conv_args* args, void* stream);
int navi_causal_conv_backward(const navi_causal_conv_args* args, void* stream);
int64_t navi_causal_conv_workspace(const navi_causal_conv_args* args);

/*
 * What stands between two blocks of a residual stream. Per row of `width` numbers:
 *
 *     m = y / sqrt(mean y^2 + eps) post_weight silu(gate),   stream = residual + scale m,
 *     normed = stream / sqrt(mean stream^2 + eps) pre_weight     (of the sum before it is rounded)
 *
 * y, gate, normed: `dtype`, residual and stream: `stream_dtype` (dtype or float32); y, residual and
 * gate [envs][steps][width] with strides of the env and step axes, the last one contiguous; outputs
 * contiguous. gate, scale and the weights may be NULL (factors of 1). The outputs share no memory with each other or
 * the inputs, but stream may be residual and normed y, where those are contiguous.
 */
#define NAVI_POLICY_MAX_BLOCK_WIDTH 8192
#define NAVI_POLICY_BLOCK_PARTIALS 1024

typedef struct navi_block_norm_args {
    int32_t dtype, stream_dtype;
    int32_t width;
    float eps;
    int64_t envs, steps;
    const void* y;
    const void* residual;
    const void* gate; /* or NULL */
    int64_t y_stride[2], residual_stride[2], gate_stride[2];
    const float* scale;       /* [width] or NULL, */
    const float* post_weight; /* likewise, */
    const float* pre_weight;  /* likewise */
    void* stream;
    void* normed;
    /* the backward pass (stream and normed are not read); what it writes shares no memory with anything else: */
    const void* grad_stream; /* or NULL for zeros */
    const void* grad_normed; /* or NULL for zeros */
    int64_t grad_stream_stride[2], grad_normed_stride[2];
    void* d_y;
    void* d_residual;
    void* d_gate;         /* or NULL */
    float* d_scale;       /* or NULL, through */
    float* d_post_weight; /* or NULL, */
    float* d_pre_weight;  /* or NULL, */
    float* partial;       /* navi_block_norm_workspace bytes (NULL without those three) */
} navi_block_norm_args;

int navi_block_norm(const navi_block_norm_args* args, void* stream);
int navi_block_norm_backward(const navi_block_norm_args* args, void* stream);
int64_t navi_block_norm_workspace(const navi_block_norm_args* args);

/*
 * A selective state space scan. Per env and head h (of group h / (heads / groups)), with beta =
 * softplus(dt + dt_bias[h]), the state S a state_dim x head_dim matrix of float32, cleared (whatever it
 * holds) at a token that starts an episode:
 *
 *     S <- exp(beta a[h]) S + beta b x^T,   out = S^T c + d[h] x
 *
 * x and out: [envs][steps][heads][head_dim] of `dtype`, b and c: [envs][steps][groups][state_dim] of
 * it, dt: [envs][steps][heads] of float32, a, d and dt_bias: [heads]. Strides are in elements, of the
 * env, step and head (or group) axes; the last axis is contiguous, and so are out, the states and the
 * gradients. beta a is meant to be <= 0; below -1e5 it starts an episode as `starts` does. Other
 * inputs are finite: in the chunked form a NaN or infinity may reach every token of its chunk of
 * NAVI_POLICY_CHUNK and what follows them.
 *
 * A launch has fewer than 2^32 threads, 256 a workgroup: scans take envs (rounded up to 8 /
 * groups where there are more) x heads x ceil(head_dim / 64) workgroups below 2^24, backward also with state_dim for
 * head_dim, and envs x heads x chunks; single tokens a wave of 64 for each 32 columns of a head (8 where head_dim is not
 * a multiple of four or states are not aligned to 16 bytes), below 2^26.
 */
#define NAVI_POLICY_MAX_STATE_DIM 128 /* and head_dim */
#define NAVI_POLICY_MAX_HEADS 16384

typedef struct navi_selective_scan_args {
    int32_t dtype;
    int32_t heads, groups; /* heads: 1 to NAVI_POLICY_MAX_HEADS, a multiple of groups */
    int32_t state_dim, head_dim;
    int64_t envs, steps;
    const void* x;
    const void* b;
    const void* c;
    int64_t x_stride[3], b_stride[3], c_stride[3];
    const float* dt;
    int64_t dt_stride[3];
    const float* a;
    const float* d;       /* or NULL */
    const float* dt_bias; /* or NULL */
    const uint8_t* starts; /* [envs][steps] or NULL */
    int64_t starts_stride[2];
    const float* initial_state; /* [envs][heads][state_dim][head_dim], or NULL for zeros */
    void* out;
    float* final_state;   /* as initial_state, or NULL; may be initial_state itself in
                             navi_selective_step. Else it shares no memory with what is read, nor does
                             out, which there may be x itself (contiguous) */
    void* scratch;        /* navi_selective_scan_scratch bytes for navi_selective_scan, 16-byte aligned (NULL
                             where that is 0) */
    /* the backward pass (out, final_state and scratch are not read); what it writes shares no memory with anything
       else: */
    const void* grad_out;
    int64_t grad_out_stride[3];
    const float* grad_final_state; /* contiguous, or NULL for zeros */
    void* d_x;
    void* d_b;
    void* d_c;
    float* d_dt;
    float* d_a;           /* or NULL, */
    float* d_d;           /* or NULL, */
    float* d_dt_bias;     /* or NULL */
    float* d_initial_state; /* or NULL */
    void* workspace;      /* navi_selective_scan_workspace bytes, 16-byte aligned */
} navi_selective_scan_args;

/* Chunked form, for rollouts and training. */
int navi_selective_scan(const navi_selective_scan_args* args, void* stream);
int navi_selective_scan_backward(const navi_selective_scan_args* args, void* stream);
int64_t navi_selective_scan_scratch(const navi_selective_scan_args* args);
int64_t navi_selective_scan_workspace(const navi_selective_scan_args* args);

/* Recurrent form: one token after another with the state in registers; for single tokens and short
 * runs. Needs no scratch. */
int navi_selective_step(const navi_selective_scan_args* args, void* stream);

/*
 * Matrices made nearly orthogonal: X = G / (|G| + eps) with |G| the root of the sum of squares, then
 * `steps` times X <- a X + (b A + c A A) X with A = X X^T (X is G or its transpose, the one with no
 * more rows than columns), into `to` in G's orientation.
 * from: rows x cols numbers with the strides (in elements) of rows and columns, one of them 1; to:
 * any strides. Products are of two float16 each (22 bits), but for bfloat16 results of matrices with more
 * than 256 rows and columns of one (11 bits). A matrix may be written in its place; otherwise what is written shares
 * no memory with what else is written or read. `matrices` is a host array, read during the call.
 * Factors that can take singular values s past 7.9 before the last step, or |b s^2 + c s^4| past 62 in
 * one (from s = 1 on), are refused.
 */
typedef struct navi_orthogonalize_matrix {
    const void* from;
    void* to;
    int64_t rows, cols; /* at most 2^20 each, 2^31 numbers */
    int64_t from_stride[2], to_stride[2];
    int32_t from_dtype, to_dtype; /* NAVI_POLICY_* */
} navi_orthogonalize_matrix;

/* `workspace`: navi_orthogonalize_workspace bytes, 256-byte aligned. */
int navi_orthogonalize(int32_t count, const navi_orthogonalize_matrix* matrices, int32_t steps, float a, float b, float c,
                       float eps, void* workspace, void* stream);
int64_t navi_orthogonalize_workspace(int32_t count, const navi_orthogonalize_matrix* matrices);

/* Message of the last failure on the calling thread ("" if none). */
const char* navi_policy_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NAVI_POLICY_H */
