/* libhdla_hip.so -- C ABI of the operators of a state space block: the short causal convolution, the selective state space scan, the norms around a block.
 *
 * Conventions are those of hdla_hip.h (device pointers, streams, workspaces, return codes), but that x, dt, z, B and C of the scan and x of the convolution may
 * lie at any address and with strides of their own.  dtype codes: HDLA_BF16, HDLA_FP32.  A batch of no sequences (B = N = 0) leaves zeros in the gradients of
 * parameters and touches nothing else. */
#ifndef HDLA_STATE_SPACE_H
#define HDLA_STATE_SPACE_H

#include "hdla_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HDLA_STATE_SPACE_VERSION 2
int hdla_state_space_version(void);   /* HDLA_STATE_SPACE_VERSION of the built library */

/* Short causal convolution over the tokens of each channel, W taps (2, 3 or 4), optionally followed by silu:
 *     p_t = bias + sum_j weight[., j] x_{t-W+1+j};   y_t = silu ? p_t sigmoid(p_t) : p_t
 * x [B, T, D] of `dtype`, at any address and with strides of its own (elements; the last one is 1); weight [D, W], bias [D] or NULL contiguous, each bf16 or fp32.
 * state, last, dstate, dlast [N, W - 1, D] of `dtype`: the inputs before a sequence's first token (NULL: zeros) and its last W - 1 (NULL: not wanted).
 * y, dy, dx [B, T, D] and the states are contiguous and 16-byte aligned.  cu_seqlens (device int64[N + 1], B = 1): packed sequences; rows of no sequence become zero.
 * hdla_short_conv_bwd: dbias NULL without bias, dstate NULL where it is not wanted; dweight, dbias in the type of weight, bias, summed in a fixed order through `workspace`
 * (hdla_short_conv_workspace_bytes() bytes, 16-byte aligned).  hdla_short_conv_step: T = 1, one token of each of N = B sequences; new_state may be state itself. */
typedef struct hdla_conv_dims {
    int32_t B, T, D, W, N;
    int32_t dtype, weight_dtype, bias_dtype, silu;
    int64_t x_batch, x_row;
    const int64_t* cu_seqlens;
} hdla_conv_dims;
int hdla_short_conv_fwd(const hdla_conv_dims* dims, const void* x, const void* weight, const void* bias, const void* state, void* y, void* last, void* stream);
size_t hdla_short_conv_workspace_bytes(const hdla_conv_dims* dims);
int hdla_short_conv_bwd(const hdla_conv_dims* dims, const void* x, const void* weight, const void* bias, const void* state, const void* dy, const void* dlast,
                        void* dx, void* dweight, void* dbias, void* dstate, void* workspace, size_t workspace_bytes, void* stream);
int hdla_short_conv_step(const hdla_conv_dims* dims, const void* x, const void* weight, const void* bias, const void* state, void* y, void* new_state, void* stream);

/* Selective state space scan.  Per channel d (of D, in G groups of neighbours) with S <= 64 states, group g = d / (D / G):
 *     delta_t = softplus(dt_t + dt_bias)  [or dt_t + dt_bias];   h_t = exp(delta_t A) h_{t-1} + delta_t x_t B_t;
 *     y_t = (C_t . h_t + D x_t) silu(z_t)
 * x, dt, z [B, T, D] and B, C [B, T, G, S] of `dtype`, at any address and with strides of their own (elements; the last one is 1); A [D, S], D [D], dt_bias [D]
 * contiguous, each bf16 or fp32; D, z, dt_bias may be NULL.  States [N, D, S] fp32.  y, dy and the gradients are contiguous, 16-byte aligned.
 * cu_seqlens (device int64[N + 1], B = 1): packed sequences; rows of no sequence become zero in y and in the gradients.
 * hdla_scan_fwd: h0 and ht may be NULL.  states (hdla_scan_states_bytes() bytes, 16-byte aligned, or NULL): the state that enters every 64th token (32nd where there are many sequences and channels), for hdla_scan_bwd;
 * workspace of hdla_scan_fwd_workspace_bytes() bytes (0 where there are no segments), 16-byte aligned.
 * hdla_scan_bwd: dht, dh0, dD, ddt_bias, dz NULL where there is none (dh0 NULL: not wanted).  dx, ddt, dz [B, T, D], dB, dC [B, T, G, S] of `dtype`,
 * dA, dD, ddt_bias in the type of A, D, dt_bias.  Sums are taken in a fixed order through `workspace` (hdla_scan_workspace_bytes() bytes, 16-byte aligned).
 * hdla_scan_step: T = 1, one token of each of N = B sequences; new_state may be state itself. */
typedef struct hdla_scan_dims {
    int32_t B, T, D, S, G, N;
    int32_t dtype, A_dtype, D_dtype, bias_dtype, softplus;
    int64_t x_batch, x_row, dt_batch, dt_row, z_batch, z_row, B_batch, B_row, B_group, C_batch, C_row, C_group;
    const int64_t* cu_seqlens;
} hdla_scan_dims;
size_t hdla_scan_states_bytes(const hdla_scan_dims* dims);
int hdla_scan_fwd(const hdla_scan_dims* dims, const void* x, const void* dt, const void* A, const void* B, const void* C, const void* D, const void* z,
                  const void* dt_bias, const float* h0, void* y, float* ht, void* states, size_t states_bytes, void* workspace, size_t workspace_bytes, void* stream);
size_t hdla_scan_fwd_workspace_bytes(const hdla_scan_dims* dims);
size_t hdla_scan_workspace_bytes(const hdla_scan_dims* dims);
int hdla_scan_bwd(const hdla_scan_dims* dims, const void* x, const void* dt, const void* A, const void* B, const void* C, const void* D, const void* z,
                  const void* dt_bias, const void* dy, const float* dht, const void* states, size_t states_bytes, void* dx, void* ddt, void* dA, void* dB,
                  void* dC, void* dD, void* dz, void* ddt_bias, float* dh0, void* workspace, size_t workspace_bytes, void* stream);
int hdla_scan_step(const hdla_scan_dims* dims, const void* x, const void* dt, const void* A, const void* B, const void* C, const void* D, const void* z,
                   const void* dt_bias, const float* state, void* y, float* new_state, void* stream);

/* The norms around a block with its gate and the residual stream.  Per row of E channels:
 *     p = post_norm ? x / rms(x) post_weight : x;   u = p act(gate);   r = residual + scale u;   y = r / rms(r) weight;   rms(v) = sqrt(mean v^2 + eps)
 * x, gate, y [rows, E] of `dtype`; residual, r of residual_dtype (bf16 or fp32 beside bf16, else fp32); weight, post_weight, scale [E], each bf16 or fp32 or NULL (ones; for the
 * scale `factor`); residual, gate may be NULL.  All contiguous, matrices 16-byte aligned.  E up to 4096.
 * hdla_block_norm_bwd: dy or dr NULL where nothing reaches that output; dresidual NULL without residual; dweight, dpost_weight, dscale in the types of weight, post_weight, scale, summed in
 * a fixed order through `workspace` (hdla_block_norm_workspace_bytes() bytes, 16-byte aligned). */
enum { HDLA_ACT_NONE = 0, HDLA_ACT_SIGMOID = 1, HDLA_ACT_SILU = 2 };
typedef struct hdla_block_norm_dims {
    int64_t rows;
    int32_t E, dtype, residual_dtype, weight_dtype, post_dtype, scale_dtype, act, post_norm;
    float factor, eps;
} hdla_block_norm_dims;
int hdla_block_norm_fwd(const hdla_block_norm_dims* dims, const void* x, const void* residual, const void* weight, const void* post_weight, const void* gate, const void* scale,
                        void* y, void* r, void* stream);
size_t hdla_block_norm_workspace_bytes(const hdla_block_norm_dims* dims);
int hdla_block_norm_bwd(const hdla_block_norm_dims* dims, const void* x, const void* residual, const void* weight, const void* post_weight, const void* gate, const void* scale,
                        const void* dy, const void* dr, void* dx, void* dresidual, void* dweight, void* dpost_weight, void* dgate, void* dscale, void* workspace,
                        size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
