/* pvder_sequence.h -- C ABI of the sequence operators of the agents (libpvder_sequence.so): attention that decays with
 * distance, over whole windows and for single env steps, and the gated residual add between two norms.
 *
 * Conventions of pvder_hip.h: plain device pointers, a hipStream_t, asynchronous, allocation-free (workspaces come from the
 * caller); 0 / PVDER_EINVAL (-10001) / -hipError_t.  Nothing is launched when a call is refused.  Strides count elements;
 * the last dimension of every tensor has stride 1 unless a field says otherwise.  All offsets are 64-bit.  A launch has fewer than
 * 2^32 threads: rows (B, N) beyond that are taken in several launches, heads of one row and pieces of T are refused. */
#ifndef PVDER_SEQUENCE_H
#define PVDER_SEQUENCE_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { PVDER_SEQ_F32 = 0, PVDER_SEQ_BF16 = 1 };
enum { PVDER_SEQ_MAX_HEAD = 128, PVDER_SEQ_MAX_SCANS = 3, PVDER_SEQ_MAX_WIDTH = 8192, PVDER_SEQ_MAX_TOKEN_STRIDE = 1 << 26,
       PVDER_SEQ_MAX_TOKENS = 1 << 30 };

/* One scan over the tokens of every (batch row b, head h): a state S of [dk, dv], fp32.
 *   forward :  R_t = g S_(t-1);  o_t = a_read R_t^T q_t + a_intra (q_t . k_t) v_t;  S_t = R_t + a_write k_t v_t^T
 *   reverse :  S is what the later tokens left, the weight g comes behind the token and not before it:
 *              o_t = a_read S_(t+1)^T q_t + a_intra (q_t . k_t) v_t;  S_t = g (S_(t+1) + a_write k_t v_t^T)
 * With a_intra = a_read * a_write the forward form is o_t = a_read S_t^T q_t.  The three gradients of an attention are scans of its inputs
 * in other places:  dq = scan(do, v, k),  dk = reverse scan(v, do, q),  dv = reverse scan(k, q, do). */
typedef struct pvder_seq_scan {
    const void *q, *k, *v;          /* [B, T, H, dk], [B, T, H, dk], [B, T, H, dv] */
    void *o;                        /* [B, T, H, dv]; rows at and behind lengths[b] are written as zeros */
    int64_t q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h, o_b, o_t, o_h;   /* q_t .. o_t: a row's length .. PVDER_SEQ_MAX_TOKEN_STRIDE bytes */
    const float *s_in;              /* state that comes in, NULL: zeros; element (i, j) of (b, h) at b s_b + h s_h + i s_k + j s_v */
    float *s_out;                   /* state that goes out, NULL: not wanted; same strides */
    int64_t s_b, s_h, s_k, s_v;     /* s_k, s_v >= 0, dk s_k + dv s_v < 2^29 */
    const float *kept;              /* NULL, or the workspace that an earlier run left: see below */
    float a_read, a_write, a_intra;
    int32_t dk, dv, reverse;        /* dk, dv: 16 bytes of elements (8 bf16, 4 fp32) .. PVDER_SEQ_MAX_HEAD */
    int32_t transpose_of;           /* 0, or 1 + the number of an earlier scan of this call: see below */
} pvder_seq_scan;

typedef struct pvder_seq_attn {
    pvder_seq_scan scan[PVDER_SEQ_MAX_SCANS];
    const float *log_decay;         /* [H]: g = exp(min(log_decay, 0)); NaN counts as 0 */
    const uint8_t *starts;          /* NULL or [B, T], != 0: an episode starts at this token, nothing before it counts */
    const int32_t *lengths;         /* NULL or [B]: tokens of each row, taken into 0 .. T */
    float *workspace;               /* pvder_seq_attn_plan() floats, 16-byte aligned; NULL when that is 0 */
    int64_t starts_b, starts_t;
    int32_t B, T, H, n_scans, dtype, segments;   /* segments: as pvder_seq_attn_plan() set it, at most T / 64 */
} pvder_seq_attn;

/* Sets a->segments, the pieces of T that run side by side, by B, T, H, n_scans, dtype and the scans' dk, dv, kept and transpose_of alone
 * (no pointer is followed), and returns the floats of workspace that they need (0: none); < 0: PVDER_EINVAL.
 *
 * With several pieces a run first works out the state that comes into each, and leaves these states in the workspace.  A scan whose k is
 * another's v and whose v is its k, in the same direction and with the same a_write, has that scan's states, transposed.  They are read
 * instead of worked out again if the other is named: transpose_of in the same call, or, as kept, the workspace of an earlier run of that
 * scan alone, with the same B, T, H, dtype, starts, lengths and (transposed) s_in.  Where a scan has kept, segments goes into the plan
 * as the earlier run had it, and is left so, or set to 1: all of T in one piece then, and kept is not read. */
int64_t pvder_seq_attn_plan(pvder_seq_attn *a);
int pvder_seq_attn_run(const pvder_seq_attn *a, void *stream);

/* One token of every row n and head h:  S = g S + k v^T (S taken as zeros where starts[n] != 0 or g is 0),  o = scale S^T q.  The state is
 * updated in place; `state` is contiguous [N, H, dk, dv]. */
typedef struct pvder_seq_step {
    const void *q, *k, *v;          /* [N, H, dk], [N, H, dk], [N, H, dv] */
    void *o;                        /* [N, H, dv] */
    int64_t q_n, q_h, k_n, k_h, v_n, v_h, o_n, o_h;
    float *state;
    const float *log_decay;         /* as above */
    const uint8_t *starts;          /* NULL or [N] */
    int64_t starts_n;
    int32_t N, H, dk, dv, dtype;
    float scale;
} pvder_seq_step;
int pvder_seq_step_run(const pvder_seq_step *a, void *stream);

/* The residual stream between two blocks:  h' = h + scale * sigmoid(gate) * y / rms(y) * post,   x = h' / rms(h') * pre,
 * rms(z) = sqrt(mean z^2 + eps), row by row; all sums in fp32, x from the unrounded h'. */
typedef struct pvder_seq_norm {
    const void *h, *y, *gate;       /* [rows, width]; gate NULL: 1 instead of the sigmoid */
    int64_t h_r, y_r, gate_r;       /* row strides */
    const float *post, *pre, *scale;    /* [width]; scale NULL: 1 */
    void *h_out, *x_out;            /* forward: contiguous [rows, width] */
    float *stats;                   /* [rows, 2]: 1 / rms(y), 1 / rms(h'); written by the forward pass (NULL: not wanted), read by the backward */
    const void *dh, *dx;            /* backward: gradients of h' and x, [rows, width]; NULL: zeros */
    int64_t dh_r, dx_r;
    void *dh_out, *dy_out, *dgate_out;      /* backward: contiguous [rows, width]; dgate_out only with gate */
    float *dparam;                  /* backward: [3, width], gradients of post, pre, scale; NULL: not wanted */
    float *workspace;               /* backward: pvder_seq_norm_workspace() floats; NULL when that is 0 */
    int64_t rows;
    int32_t width, dtype;
    float eps;
} pvder_seq_norm;
int64_t pvder_seq_norm_workspace(const pvder_seq_norm *a);      /* by rows, width, dtype and whether dparam is wanted */
int pvder_seq_norm_forward(const pvder_seq_norm *a, void *stream);
int pvder_seq_norm_backward(const pvder_seq_norm *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* PVDER_SEQUENCE_H */
