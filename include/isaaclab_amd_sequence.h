/*
 * isaaclab_amd -- C ABI of the sequence operators: the short causal convolution and the selective state space
 * recurrence of a policy's or an actuator's memory, over whole rollouts (forward and backward) and one environment step
 * at a time, and the clipping of gradients by their global norm.
 *
 * Nothing in the reference stands behind these calls: its recurrent models are torch modules inside the RL libraries.
 * The conventions of isaaclab_amd.h hold, except that activations may be 16 bit (ILX_F32 / ILX_BF16 / ILX_F16) and
 * strided: a tensor of activations is (batch, length, channels) with unit channel stride, `*_batch` and `*_time` are its
 * other two strides in elements, so a time-major rollout buffer is passed as it is.  Parameters, states and their
 * gradients are dense float32.  There are at most 2^23 channels and, in the recurrence, time strides are below 2^27
 * elements and a sequence has at most 2^31 - 4097 rows; a larger shape is refused (ILX_ESHAPE).
 *
 * `starts` (batch, length) bytes, non-zero where an episode begins: nothing from before that row reaches it or any later
 * row.  `lengths` (batch) int32: rows from lengths[b] on are not read, their outputs and gradients are written as zeros
 * and the state passes over them unchanged; values are clamped to [0, length].  Both may be NULL.
 *
 * Scratch memory is the caller's: the *_workspace functions say how many floats a call needs (0 if none).  The same
 * descriptor must be given to both; the contents need not survive the call.  Results do not depend on what it held, and no
 * sum's order depends on scheduling: two runs give the same bits.
 *
 * All arithmetic is in 32 bits.  Sums of parameters' gradients span at most 512 rows in 32 bits, longer ones are added in 64, and so
 * are those of grad_B and grad_C over blocks of 64 channels and the squares of a norm.  Inputs that are infinite or NaN make
 * what depends on them infinite or NaN, though not always the one of the two that the formula says (and grad_A, in which the
 * state behind the last row does not occur, may become NaN where that state is infinite).
 */
#ifndef ISAACLAB_AMD_SEQUENCE_H
#define ISAACLAB_AMD_SEQUENCE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ILX_F32 0
#define ILX_BF16 1
#define ILX_F16 2

#define ILX_CONV_MAX_WIDTH 8
#define ILX_SCAN_MAX_STATES 32
#define ILX_SCAN_BLOCK 8 /* rows between two saved states of a forward pass that a backward pass follows */

/* ---- short causal convolution ------------------------------------------------------------------
 * p[b,t,d] = bias[d] + sum_j weight[d, width-1-j] * x[b,t-j,d],  out = p or p * sigmoid(p).
 * Rows t < 0 are the carried state: state[b, width-1-i, d] is row -i.  `last` receives the last width-1 rows, those from
 * before the last start as zeros; it may be `state` itself only in the one-step call. */
typedef struct ilx_short_conv {
    const void* x;
    int64_t x_batch, x_time;
    const float* weight;   /* (channels, width) */
    const float* bias;     /* (channels), may be NULL */
    const float* state;    /* (batch, width-1, channels), may be NULL: zeros */
    const uint8_t* starts; /* may be NULL */
    int64_t starts_batch, starts_time;
    const int32_t* lengths; /* may be NULL */
    void* out;
    int64_t out_batch, out_time;
    float* last; /* (batch, width-1, channels), may be NULL */
    int64_t batch, length;
    int32_t channels, width;
    int32_t dtype; /* of x, out and their gradients */
    int32_t silu;
    /* backward only */
    const void* grad_out;
    int64_t grad_out_batch, grad_out_time;
    const float* grad_last; /* may be NULL */
    void* grad_x;
    int64_t grad_x_batch, grad_x_time;
    float* grad_weight; /* (channels, width) */
    float* grad_bias;   /* may be NULL */
    float* grad_state;  /* may be NULL */
    float* workspace;
    int64_t workspace_floats;
} ilx_short_conv;

int ilx_short_conv_forward(const ilx_short_conv* conv, void* stream);
int ilx_short_conv_workspace(const ilx_short_conv* conv, int64_t* floats); /* of the backward call */
int ilx_short_conv_backward(const ilx_short_conv* conv, void* stream);
/* one row per sequence (length is taken as 1, the time strides are not read, lengths must be NULL); the state is
 * updated in place */
int ilx_short_conv_step(const ilx_short_conv* conv, void* stream);

/* ---- selective state space recurrence -----------------------------------------------------------
 * dt = softplus(delta[b,t,d] + delta_bias[d])  (or the sum itself without `softplus`)
 * h[b,n,d] <- exp(dt * A[d,n]) * h[b,n,d] + dt * B[b,t,g,n] * x[b,t,d],   g = d / (channels / groups)
 * y = sum_n C[b,t,g,n] * h[b,n,d] + D[d] * x[b,t,d],   out = y or y * gate * sigmoid(gate).
 * The state is (batch, states, channels).  B and C are (batch, length, groups, states) with unit state stride and
 * `states` between groups. */
typedef struct ilx_state_space {
    const void* x;
    int64_t x_batch, x_time;
    const void* delta;
    int64_t delta_batch, delta_time;
    const void* gate; /* may be NULL */
    int64_t gate_batch, gate_time;
    const float* A; /* (channels, states) */
    const void* B;
    int64_t B_batch, B_time;
    const void* C;
    int64_t C_batch, C_time;
    const float* D;          /* (channels), may be NULL: 0 */
    const float* delta_bias; /* (channels), may be NULL: 0 */
    const float* state;      /* (batch, states, channels), may be NULL: zeros */
    const uint8_t* starts;
    int64_t starts_batch, starts_time;
    const int32_t* lengths;
    void* out;
    int64_t out_batch, out_time;
    float* last;  /* (batch, states, channels), may be NULL; may be `state` itself only in the one-step call */
    float* saved; /* (batch, ceil(length / ILX_SCAN_BLOCK), states, channels), may be NULL: the state ahead of every block,
                     written by forward, read by backward */
    int64_t batch, length;
    int32_t channels, states, groups;
    int32_t dtype;    /* of x, delta, gate, out and their gradients */
    int32_t bc_dtype; /* of B and C: dtype or ILX_F32 */
    int32_t softplus;
    /* backward only; the gradients of x, delta and gate have one pair of strides, those of B and C are dense */
    const void* grad_out;
    int64_t grad_out_batch, grad_out_time;
    const float* grad_last; /* may be NULL */
    void* grad_x;
    void* grad_delta;
    void* grad_gate; /* NULL exactly if gate is */
    int64_t grad_batch, grad_time;
    float* grad_A;          /* (channels, states) */
    void* grad_B;           /* (batch, length, groups, states) */
    void* grad_C;
    float* grad_D;          /* may be NULL */
    float* grad_delta_bias; /* may be NULL */
    float* grad_state;      /* may be NULL */
    float* workspace;
    int64_t workspace_floats;
} ilx_state_space;

int ilx_state_space_workspace(const ilx_state_space* scan, int backward, int64_t* floats);
int ilx_state_space_forward(const ilx_state_space* scan, void* stream);
int ilx_state_space_backward(const ilx_state_space* scan, void* stream);
/* one row per sequence, the state updated in place */
int ilx_state_space_step(const ilx_state_space* scan, void* stream);

/* ---- gradient norm and clipping -----------------------------------------------------------------
 * norm = (sum over all tensors of |g|^2)^(1/2) (norm_kind 0) or the largest |g| (norm_kind 1), written to `norm`; with
 * clip != 0 every tensor is then multiplied in place by min(1, max_norm / (norm + 1e-6)), in float32, rounded once.
 * Tensors are dense; their pointers, element counts and types are host arrays.  A norm that is not finite scales by what the
 * formula gives (infinity: zeros, and NaN where a gradient is infinite; NaN: NaN everywhere). */
int ilx_gradient_norm_workspace(const int64_t* sizes_host, int32_t count, int64_t* floats);
int ilx_gradient_norm(void* const* tensors_host, const int64_t* sizes_host, const int32_t* dtypes_host, int32_t count,
                      int32_t norm_kind, int32_t clip, float max_norm, float* norm, float* workspace, int64_t workspace_floats,
                      void* stream);

#ifdef __cplusplus
}
#endif

#endif
