/*
 * roaster_mixer.h -- the recurrent layers from the residual stream to the residual
 * stream, for any number of rows: the root-mean-square norm (with the residual's
 * addition, over whole rows or over heads with a gate, its output in f32 or in
 * 8 bits), the matrix product in 8-bit integers for the projections, and the
 * selective state space scan with its short causal convolution
 * (model.c:252-323, 1282-1347 for one token, 1604-1660 for a prompt's chunk;
 * the norms and the residual model.c:1349-1358).
 *
 * Conventions as in roaster_attn.h: row-major, device pointers, strides in
 * elements, calls ordered on the library's stream (roaster_stream), ROASTER_OK
 * or a negative ROASTER_E* with the message in roaster_last_error().  Argument
 * structures are host memory, read within the call.  Sizes, alignments and
 * overlaps are checked by the call (ROASTER_EINVAL, nothing launched).  No call
 * allocates, copies to the host or waits: after roaster_init all of them can be
 * captured into a HIP graph on roaster_stream.  Two calls, or two captured graphs,
 * that may run at the same time need outputs, states and workspaces of their own.
 */
#ifndef ROASTER_MIXER_H
#define ROASTER_MIXER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- norm ------------------------------------------------------------------- */
/* For every row:
 *   v = x, or with res: res += x in place and v = res
 *   y = v * rsqrt(mean(v^2) + eps) * weight, the mean over each `group` elements
 *       (group = 0: y = v)
 *   y = y * gate * sigmoid(gate)                                (with a gate)
 * and y in f32, in 8 bits, or both:
 *   q = y * 127 / max|y|, rounded to nearest even, and q_scale = max|y| / 127
 * A row whose largest |y| is below 2^-119 has scale and values 0; a row with an
 * infinite or NaN y has scale NaN and values 0.  Sums are in f32.  A row's results
 * are the same whatever the other rows.  A row whose squares pass f32's range gives
 * zeros.  y may be x (with the same stride); nothing else may overlap.
 * rows = 0 does nothing. */
typedef struct {
    int rows;                 /* 0 .. 2^20 */
    int cols;                 /* a multiple of 4, up to 16384 */
    int group;                /* cols; a power of two, 16 .. 256, that divides cols (a head); or 0 */
    const float *x;           /* all f32 tensors 16-byte aligned, strides multiples of 4, at most 2^32 */
    size_t x_row;
    float *res;               /* or NULL */
    size_t res_row;           /* at least cols, as y_row and q_row */
    const float *weight;      /* [group], or NULL: ones */
    const float *gate;        /* or NULL */
    size_t gate_row;
    float eps;
    float *y;                 /* or NULL */
    size_t y_row;
    int8_t *q;                /* or NULL; 4-byte aligned, stride a multiple of 4 (of 16 for roaster_matmul_i8) */
    size_t q_row;
    float *q_scale;           /* [rows], where q is given */
} RoasterNorm;

int roaster_norm(const RoasterNorm *norm);

/* ---- matrix product in 8-bit integers ---------------------------------------- */
/* A matrix in 8 bits with a scale for each row (output channel): weight = value * scale.
 * data holds the values in the order in which the products read them (rows padded
 * to 32, columns to 128), written by roaster_i8_pack. */
typedef struct {
    void  *data;              /* roaster_i8_bytes bytes, 16-byte aligned */
    float *scale;             /* [rows] */
    int    rows;              /* 1 .. 2^20 */
    int    cols;              /* a multiple of 16, 16 .. 65536 */
} RoasterI8;

/* Bytes of data; host only.  0 for bad sizes. */
size_t roaster_i8_bytes(int rows, int cols);

#define ROASTER_I8_FROM_F32 0    /* f32 [rows][cols], 16-byte aligned */
#define ROASTER_I8_FROM_Q4K 1    /* rows of Q4_K super-blocks; cols a multiple of 256 */
#define ROASTER_I8_FROM_Q6K 2    /* rows of Q6_K super-blocks; cols a multiple of 256 */
#define ROASTER_I8_FROM_I8  3    /* int8 [rows][cols], 16-byte aligned, scale as the caller has filled it */

/* Once for a matrix on the device.  Of f32 and quantised rows the largest becomes 127
 * (scale = max / 127, value = weight * 127 / max, rounded to nearest even; a row below 2^-119
 * has scale and values 0, one with an infinite or NaN weight scale NaN and values 0).
 * W, data and scale must not overlap. */
int roaster_i8_pack(const void *W, int from, const RoasterI8 *to);

/* y[t][r] = x_scale[t] * scale[r] * sum_c x[t][c] * value[r][c]
 * for rows tokens x of 8-bit values (roaster_norm's q and q_scale).  The sums are exact
 * (32-bit integers); the product with the two scales, which are multiplied first, is rounded as
 * f32.  An infinite or NaN scale reaches its row or channel alone.  Outputs must not overlap inputs.  rows = 0 does
 * nothing. */
typedef struct {
    int rows;                 /* 0 .. 2^20 */
    const int8_t *x;          /* [rows][w->cols], 16-byte aligned */
    size_t x_row;             /* a multiple of 16, at most 2^32 */
    const float *x_scale;     /* [rows] */
    float *y;                 /* [rows][w->rows] */
    size_t y_row;             /* at least w->rows, at most 2^32 */
} RoasterMatmulI8;

int roaster_matmul_i8(const RoasterMatmulI8 *mm, const RoasterI8 *w);

/* ---- selective state space scan with its short causal convolution ------------- */
/* One layer's states of n_req requests.  Both are the requests' own: request r's lie at index r,
 * and the request whose next token has position 0 starts from zeros whatever they hold. */
typedef struct {
    int n_req;                /* 1 .. 2048 */
    int k_heads, v_heads;     /* v_heads a multiple of k_heads, at most 256; value head h uses key head h / (v_heads / k_heads) */
    int k_dim, v_dim;         /* 64 or 128 each */
    int taps;                 /* of the convolution, 2 .. 4 */
    float *conv;              /* [n_req][taps][channels]: entry p % taps is the input of position p */
    float *state;             /* [n_req][v_heads][v_dim][k_dim] */
} RoasterSsmState;            /* both 16-byte aligned */

#define ROASTER_SCAN_DELTA 0  /* gated delta rule, as the model's recurrent layers have it */
#define ROASTER_SCAN_STATE 1  /* the same without the correction: scalar decay, step and input */

/* One step of all requests: request r's new tokens are rows first[r] .. first[r + 1] - 1, in order
 * (roaster_kv_plan's first and row_pos).  Of each row, its channels being
 * [queries k_heads * k_dim][keys k_heads * k_dim][values v_heads * v_dim]:
 *   c = silu(conv_b + sum_j conv_w[.][j] * x of position pos - (taps - 1) + j)     (zero before position 0)
 *   q, k, v = c, and per value head
 *   dt = softplus(a + dt_bias),  d = exp(a_coef * dt)
 *   DELTA:  q, k = q / sqrt(sum q^2 + eps), k / sqrt(sum k^2 + eps),  beta = sigmoid(b)
 *           S = d S;  S += beta (v - S k) k^T          S of [v_dim][k_dim]
 *   STATE:  S = d S + dt v k^T
 *   out = scale * S q  (+ skip * v)
 * Rows from first[n_req] on stay as they were, and so do the states of requests without new
 * tokens.  States, sums and decays are in f32 (sums of a_coef * dt in 64 bits).  Of requests of many
 * tokens 64 are taken at a time, by products whose operands have 22 bits and none below 2^-30 of the largest
 * |v| (STATE: |dt v| |k|) and row of S among them and the 64 tokens before: within eight times the error of the
 * same steps in f32 and 2^-26 of those.  A query or key whose sum of squares passes f32's range is a zero vector (DELTA);
 * with eps = 0 those whose sum is 0 in f32 give NaN.
 * Infinite or NaN inputs reach their request's rows from their own on, and its states, and no
 * other's.  a_coef * dt must be finite; where it is positive a prompt goes token by token.
 * A request whose rows are not within 0 .. rows, whose position is negative or that has more than
 * `most` new tokens is left out, its rows NaN where they are within 0 .. rows and its states as they
 * were, and reported by roaster_sync (ROASTER_EINVAL).  Requests' rows must not overlap (those of a
 * plan never do): rows that several claim are any of theirs, and what does not fit the workspace is
 * left out like this.  What kernels run goes by rows, most, n_req and v_heads and by each request's
 * own number of tokens; last bits of a row depend on them, and are the same for the same call.
 * rows = 0 does nothing. */
typedef struct {
    int rows;                 /* 0 .. 262144 */
    int most;                 /* new tokens of a request at most, 1 .. rows: 1 a decode step */
    int mode;                 /* ROASTER_SCAN_* */
    const float *x;           /* [rows][channels], 16-byte aligned, stride a multiple of 4, at most 2^32 */
    size_t x_row;
    const float *a;           /* [rows][v_heads] */
    size_t a_row;             /* at most 2^32, as b_row */
    const float *b;           /* [rows][v_heads], read for DELTA alone */
    size_t b_row;
    const float *conv_w;      /* [channels][taps], the last tap for the row's own input; 16-byte aligned */
    const float *conv_b;      /* [channels], or NULL */
    const float *a_coef;      /* [v_heads] */
    const float *dt_bias;     /* [v_heads], or NULL */
    const float *skip;        /* [v_heads], or NULL */
    float scale, eps;
    const int *first;         /* [n_req + 1] */
    const int *row_pos;       /* [rows]; that of each request's first row is read */
    float *out;               /* [rows][v_heads][v_dim], 16-byte aligned */
    size_t out_row;           /* at least v_heads * v_dim, a multiple of 4, at most 2^32 */
    void *ws;                 /* 16-byte aligned, at least roaster_ssm_ws_bytes */
    size_t ws_bytes;
} RoasterSsmScan;

/* Workspace of a call with so many rows and new tokens of a request (one for more of both
 * serves as well); host only.  0 for bad arguments. */
size_t roaster_ssm_ws_bytes(int rows, int most, const RoasterSsmState *state);
int roaster_ssm_scan(const RoasterSsmScan *scan, const RoasterSsmState *state);

#ifdef __cplusplus
}
#endif
#endif
