/*
 * inet_policy.h -- C ABI of the operators that a recurrent robot policy computes beside the engines
 * (libinet_policy.so, HIP kernels for gfx950): the delta-rule memory, the gated feed-forward and the block norms.
 *
 * One robot is one row of the batch (E envs x R robots of an engine). Conventions, as inet_nr.h: the caller owns every
 * device buffer and workspace; nothing is allocated and the host never waits; work goes on `stream`; every entry point
 * returns 0 or a negative INET_POLICY_E* code; sizes, types and pointers are checked before any launch; no entry point
 * throws. A batch, a window or a row count of zero is valid: what is written is then the state as it was and the weights'
 * gradients, zeros.
 */
#ifndef INET_POLICY_H
#define INET_POLICY_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define INET_POLICY_ABI_VERSION 1

#define INET_POLICY_OK 0
#define INET_POLICY_EINVAL (-1)
#define INET_POLICY_EUNSUPPORTED (-2)
#define INET_POLICY_ELAUNCH (-3)

/* element types */
#define INET_POLICY_F32 0
#define INET_POLICY_BF16 1
#define INET_POLICY_F16 2

#define INET_POLICY_MAX_HEAD 128      /* key and value sizes of a head */
#define INET_POLICY_MAX_WIDTH 8192    /* row length of the block norms */

/* activations of the gated feed-forward */
#define INET_POLICY_SILU 0
#define INET_POLICY_GELU 1            /* the tanh form */
#define INET_POLICY_RELU 2

/*
 * The gated delta rule. Per robot b and head h, with S a K x V matrix in 32 bits:
 *     S_t = d_t S_{t-1} + beta_t k_t (v_t - (d_t S_{t-1})^T k_t)^T       d_t = e^{g_t}, 0 where reset[b][t] is set
 *     o_t = scale S_t^T q_t
 * Value head h reads query and key head h / (H / Hk). A log-decay below -104 (whose exponential is 0 in 32 bits)
 * empties the memory as reset does. Element strides are given for batch, step and head; the last axis of q, k, v is
 * contiguous. o, the states and every gradient are contiguous: [B][T][heads][size], states [B][H][K][V].
 */
typedef struct InetDelta {
    int32_t B, T, Hk, H, K, V;
    int32_t dtype, gate_dtype;                  /* of q, k, v, o and their gradients; of g, beta and theirs (float32 ones
                                                   are of 32-bit grade whatever dtype is) */
    float scale;
    int32_t chunk;                              /* steps a chunk: inet_policy_delta_chunk(), for both directions */
    int64_t q_s[3], k_s[3], v_s[3], g_s[3], beta_s[3], reset_s[2];
    const void *q, *k, *v, *g, *beta;
    const uint8_t *reset;                       /* or NULL */
    const float *state;                         /* [B][H][K][V], or NULL: empty */
    void *o;
    float *state_out;                           /* may not overlap state */
    /* kept by the forward pass for the backward pass: the prediction errors v_t - (d_t S_{t-1})^T k_t, [B][T][H][V] (NULL:
       neither is kept), and the state at the start of each chunk but the first, [B][H][chunks - 1][K][V] (NULL where
       there is one chunk). The backward pass takes `state` too. */
    float *chunk_state, *err;
    void *work;                                 /* inet_policy_delta_work() bytes for the direction; err and chunk_state
                                                   have to be there too where that is more than 0 */
} InetDelta;

/* The backward pass: gradients of the inputs from those of o and of state_out (NULL: zero). */
typedef struct InetDeltaGrad {
    const void *d_o;
    const float *d_state_out;
    void *d_q, *d_k, *d_v, *d_g, *d_beta;
    float *d_state;                             /* or NULL: not wanted */
    /* workspaces: gradient of the state after each chunk but the last (as chunk_state), of the errors (as err; both NULL
       where there is one chunk), and where H > Hk the heads' own d_q and d_k in 32 bits, [2][B][T][H][K] */
    float *chunk_grad, *err_grad, *head_grad;
} InetDeltaGrad;

int32_t inet_policy_abi_version(void);
const char *inet_policy_build_info(void);

/* steps a chunk for a window's sizes and types, which are read from a (0: invalid or unsupported) */
int32_t inet_policy_delta_chunk(const InetDelta *a);
/* workspace of a window's forward or backward pass in bytes (sizes, type and chunk are read from a; -1: invalid) */
int64_t inet_policy_delta_work(const InetDelta *a, int32_t backward);
int32_t inet_policy_delta_forward(const InetDelta *a, void *stream);
int32_t inet_policy_delta_backward(const InetDelta *a, const InetDeltaGrad *d, void *stream);
/* one step, the state updated in place: T = 1, state_out is the state (state itself is ignored); strides of step unused */
int32_t inet_policy_delta_step(const InetDelta *a, void *stream);

/*
 * The gated feed-forward: y = act(x w_gate^T) * (x w_up^T), x [N][D], w_gate and w_up [F][D], y [N][F], bfloat16 or
 * float16, sums in 32 bits. Row strides in elements; columns contiguous.
 */
typedef struct InetFfn {
    int64_t N;
    int32_t D, F, dtype, act;
    int64_t x_s, w_gate_s, w_up_s, y_s;
    const void *x, *w_gate, *w_up;
    void *y;
    void *work;                                 /* inet_policy_ffn_work() bytes */
} InetFfn;

typedef struct InetFfnGrad {
    const void *d_y;                            /* [N][F], row stride d_y_s */
    int64_t d_y_s;
    void *d_x, *d_w_gate, *d_w_up;              /* contiguous; any may be NULL: not wanted */
} InetFfnGrad;

int64_t inet_policy_ffn_work(int64_t N, int32_t D, int32_t F, int32_t backward);
int32_t inet_policy_ffn_forward(const InetFfn *a, void *stream);
int32_t inet_policy_ffn_backward(const InetFfn *a, const InetFfnGrad *d, void *stream);

/*
 * Block norms: h = f / rms(f) * post_weight, y = x + scale * gate * h, n = y / rms(y) * pre_weight, with
 * rms(z) = sqrt(mean(z^2) + eps). Rows of D contiguous elements with row strides in elements.
 */
typedef struct InetNorm {
    int64_t N;
    int32_t D, dtype, gate_kind;                /* gate_kind 0: none, 1: one value a row, 2: one a value */
    float eps;                                  /* 0 or more */
    int64_t x_s, f_s, gate_s;
    const void *x, *f, *gate;                   /* f NULL: y = x (no block before) */
    const float *scale, *post_weight, *pre_weight;   /* [D] float32; scale NULL: 1; post_weight NULL: h = f;
                                                        pre_weight NULL: no n */
    void *y, *n;                                /* contiguous */
} InetNorm;

typedef struct InetNormGrad {
    const void *d_y, *d_n;                      /* contiguous [N][D]; NULL: zero */
    void *d_x, *d_f, *d_gate;                   /* contiguous */
    float *d_scale, *d_post_weight, *d_pre_weight;
    float *work;                                /* inet_policy_norm_work() bytes */
} InetNormGrad;

int64_t inet_policy_norm_work(int64_t N, int32_t D);
int32_t inet_policy_norm_forward(const InetNorm *a, void *stream);
int32_t inet_policy_norm_backward(const InetNorm *a, const InetNormGrad *d, void *stream);

#ifdef __cplusplus
}
#endif
#endif
