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
 * or infinity may reach every token of its chunk of 64 and what follows them.
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

/* Message of the last failure on the calling thread ("" if none). */
const char* navi_policy_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NAVI_POLICY_H */
