/*
 * mmn_sequence.h -- C ABI of libmmn_hip.so, second part: operators that turn a sequence (coded events, tokens, a time series) into
 * features an encoder of the fusion chain can take.  Embedding lookup and its gradient, the causal depthwise convolution, the
 * selective scan; forward, backward, and the forms for one new step.
 *
 * Conventions as in mmn_hip.h: device pointers, a hipStream_t as void*, everything asynchronous on `stream` and capture-safe, no
 * allocation (workspaces come from the caller, 256-byte aligned), 0 or a negative MMN_ERR_* returned, nothing throws.  The caller's current device is
 * the tensors' device.  `type` is the element type of the data; parameters, states of the scan and all sums are 32-bit floats.
 * The reference has no counterpart (its recurrent encoders, multimodn/encoders/rnn_encoder.py and lstm_encoder.py, are torch modules).
 */
#ifndef MMN_SEQUENCE_H
#define MMN_SEQUENCE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MMN_SEQ_F32 0
#define MMN_SEQ_BF16 1
#define MMN_SEQ_F16 2
#define MMN_SEQ_MAX_STATES 32

/* out[r] = scale * table[ids[r]]; an id outside [0, vocab) gives zeros.  ids: int64 (ids64 = 1) or int32; rows < 2^31. */
int mmn_seq_embed(const void* ids, int ids64, const void* table, void* out, int64_t rows, int64_t vocab, int width, int type, float scale, void* stream);
/* out[v] = scale * sum over r with ids[r] = v, in the order of r, of grad[r]; every row of out is written.  rows and vocab < 2^31. */
size_t mmn_seq_embed_grad_bytes(int64_t rows, int64_t vocab, int width);
int mmn_seq_embed_grad(const void* ids, int ids64, const void* grad, void* out, int64_t rows, int64_t vocab, int width, int type, float scale,
                       void* ws, size_t ws_bytes, void* stream);

/* pre[t] = bias + sum_j w[channel][j] x[t - (taps-1) + j]; y = pre * logistic(pre) (silu) or pre.  Strides in elements, channels adjacent.
 * y, dx, state [batch][taps-1][width] and the other states are dense.  lengths (or NULL): steps of every row, clamped to [0, steps]. */
typedef struct mmn_seq_conv_desc {
    const void *x, *state;            /* state: inputs before step 0, or NULL for zeros */
    void *y, *state_out;              /* state_out: the last taps-1 inputs, or NULL */
    const float *weight, *bias;       /* [width][taps], [width] or NULL */
    const int32_t* lengths;
    const void *dy, *dstate_out;      /* backward; dstate_out or NULL */
    void *dx, *dstate;                /* dstate or NULL */
    float *dweight, *dbias;           /* [width][taps], then [width], in ONE buffer: dbias = dweight + width * taps */
    int64_t batch, x_row, x_step, dy_row, dy_step;
    int32_t steps, width, taps, silu, type, reserved;
} mmn_seq_conv_desc;
int mmn_seq_conv(const mmn_seq_conv_desc* c, void* stream);
size_t mmn_seq_conv_grad_bytes(const mmn_seq_conv_desc* c);
int mmn_seq_conv_grad(const mmn_seq_conv_desc* c, void* ws, size_t ws_bytes, void* stream);
/* one step: x [batch][width] (row stride x_row), state -> state_out (may be the same buffer) */
int mmn_seq_conv_step(const mmn_seq_conv_desc* c, void* stream);

/* dt = softplus(dt_raw + dt_bias); h = exp(dt a) h + dt x b; y = (sum_n c h + d x) * silu(z).  a [width][states], b and c
 * [batch][steps][groups][states] (states adjacent), the rest [batch][steps][width] (channels adjacent) with the given strides; y, dx,
 * ddt, dz, db, dc, states [batch][width][states] dense.  The step strides of x, dt, z, dy are from width to 2^23, those of one step or
 * none are not used.  d, dt_bias, z, lengths, state, state_out may be NULL. */
typedef struct mmn_seq_scan_desc {
    const void *x, *dt, *b, *c, *z;
    const float *a, *d, *dt_bias, *state;
    const int32_t* lengths;
    void* y;
    float *state_out, *marks;         /* marks: what a backward pass needs (mmn_seq_scan_marks floats), or NULL */
    const void* dy;                   /* backward */
    const float* dstate_out;
    void *dx, *ddt, *db, *dc, *dz;
    float *dparams, *dstate;          /* dparams: [width][states] da, then [width] dd, then [width] d(dt_bias) */
    int64_t batch, x_row, x_step, dt_row, dt_step, b_row, b_step, b_group, c_row, c_step, c_group, z_row, z_step, dy_row, dy_step;
    int32_t steps, width, groups, states, softplus, type;
} mmn_seq_scan_desc;
size_t mmn_seq_scan_marks(const mmn_seq_scan_desc* s);
size_t mmn_seq_scan_bytes(const mmn_seq_scan_desc* s, int backward);
int mmn_seq_scan(const mmn_seq_scan_desc* s, void* ws, size_t ws_bytes, void* stream);
int mmn_seq_scan_grad(const mmn_seq_scan_desc* s, void* ws, size_t ws_bytes, void* stream);
int mmn_seq_scan_step(const mmn_seq_scan_desc* s, void* stream);

/* dx [rows][width] = dpre [rows][hidden] times weight [hidden][width], all 32-bit and dense, hidden <= 128: the gradient that leaves the
 * fusion chain at an encoder's input, from its first hidden layer's pre-activation gradients (mmn_debug_buffer kind 7). */
int mmn_seq_input_grad(const float* dpre, const float* weight, float* dx, int64_t rows, int hidden, int width, void* stream);

#ifdef __cplusplus
}
#endif
#endif
