/*
 * flare_b200_mixers.h - the causal token mixers of libflare_b200.so beside FLARE: the short causal convolution and the
 * selective state space scan, for whole sequences (with gradients), prompts and single tokens.
 *
 * Conventions are those of flare_b200.h: device pointers, sizes, an int status; launches on the given stream; no call
 * allocates or synchronises; workspaces come from the caller (sizes from *_workspace_bytes, 256-byte aligned).
 * Token tensors are [B, N, ...] with contiguous innermost dimension and strides in ELEMENTS; any stride and alignment is
 * taken (16-byte aligned rows of a multiple of 8 elements are read in wide pieces, others element by element).
 *
 * Packed rows: `documents` [B, N] int32 (NULL: every row is one document).  A document is a run of equal ids; a token
 * with a negative id is padding: it takes no part, its outputs and gradients are 0.  Padded prompts: `lengths` [B] int32
 * (NULL: N each): tokens from lengths[b] on are padding in the same sense and leave the carried state as it is.
 */
#ifndef FLARE_B200_MIXERS_H_
#define FLARE_B200_MIXERS_H_

#include "flare_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

enum flare_activation { FLARE_IDENTITY = 0, FLARE_SILU = 1 };

/*
 * y[t, c] = act(bias[c] + sum_{j < W} weight[c, W - 1 - j] x[t - j, c]), the taps inside the token's document; in front
 * of a row lie the W - 1 rows of `state_in` (oldest first), zeros without one.  W is 2, 3 or 4.
 * documents and states exclude one another.
 */
typedef struct flare_conv_args {
  const void* x;            /* [B, N, C] */
  const void* weight;       /* [C, W] contiguous, weight_dtype */
  const void* bias;         /* [C] contiguous, weight_dtype; may be NULL */
  const int32_t* documents; /* [B, N] contiguous or NULL */
  const int32_t* lengths;   /* [B] or NULL */
  const void* state_in;     /* [B, W - 1, C] contiguous, dtype; may be NULL */
  void* state_out;          /* the same; may be NULL; not the buffer of state_in */
  void* y;                  /* [B, N, C] contiguous */
  const void* dy;           /* backward: [B, N, C] */
  void* dx;                 /* backward: [B, N, C] contiguous */
  void* dweight;            /* backward: [C, W] contiguous, weight_dtype */
  void* dbias;              /* backward: [C], weight_dtype; may be NULL */
  void* workspace;          /* backward only */
  size_t workspace_bytes;
  int32_t B, N, C, W;
  int64_t x_stride_b, x_stride_n, dy_stride_b, dy_stride_n;
  int32_t dtype, weight_dtype, activation;
} flare_conv_args_t;

int flare_conv_forward(const flare_conv_args_t* args, flare_stream_t stream);
/* no states and no lengths */
size_t flare_conv_backward_workspace_bytes(const flare_conv_args_t* args);
int flare_conv_backward(const flare_conv_args_t* args, flare_stream_t stream);
/* One token: x, y [B, C] (x_stride_b; N, documents and lengths are ignored).  state_out [B, W - 1, C] is read and updated
 * in place; state_in is ignored. */
int flare_conv_decode(const flare_conv_args_t* args, flare_stream_t stream);

/*
 * Selective scan, C channels with S states each (S is 8, 16 or 32):
 *   delta = softplus?(dt + dt_bias);  h[t] = exp(delta A) h[t-1] + delta b[t] x[t];  y[t] = (sum_s c[t, s] h[t, s] + D x[t]) silu?(z[t])
 * b and c are shared by the C / G channels of a group.  h starts at `state_in` (zeros without one) and at zero with every
 * document.  documents and states exclude one another.
 */
typedef struct flare_scan_args {
  const void* x;            /* [B, N, C] */
  const void* dt;           /* [B, N, C] */
  const void* z;            /* [B, N, C] or NULL: no gate */
  const void* b;            /* [B, N, G, S] */
  const void* c;            /* [B, N, G, S] */
  const float* A;           /* [C, S] contiguous */
  const float* D;           /* [C] or NULL */
  const float* dt_bias;     /* [C] or NULL */
  const int32_t* documents; /* [B, N] contiguous or NULL */
  const int32_t* lengths;   /* [B] or NULL */
  const float* state_in;    /* [B, C, S] contiguous or NULL */
  float* state_out;         /* the same; not the buffer of state_in */
  void* y;                  /* [B, N, C] contiguous */
  float* keep;              /* flare_scan_keep_bytes(args): the states that the backward starts from; forward: may be NULL */
  const void* dy;           /* backward: [B, N, C] */
  void* dx;                 /* backward: [B, N, C] contiguous, like ddt and dz */
  void* ddt;
  void* dz;                 /* with z only */
  void* db;                 /* [B, N, G, S] contiguous, like dc */
  void* dc;
  float* dA;                /* [C, S] */
  float* dD;                /* [C]; may be NULL */
  float* ddt_bias;          /* [C]; may be NULL */
  void* workspace;
  size_t workspace_bytes;
  int32_t B, N, C, S, G;
  int64_t x_stride_b, x_stride_n, dt_stride_b, dt_stride_n, z_stride_b, z_stride_n;
  int64_t b_stride_b, b_stride_n, b_stride_g, c_stride_b, c_stride_n, c_stride_g, dy_stride_b, dy_stride_n;
  int32_t dtype;       /* of x, dt, z, b, c, y, dy and their gradients */
  int32_t dt_softplus; /* 0: delta = dt + dt_bias */
} flare_scan_args_t;

size_t flare_scan_keep_bytes(const flare_scan_args_t* args);
size_t flare_scan_forward_workspace_bytes(const flare_scan_args_t* args);
int flare_scan_forward(const flare_scan_args_t* args, flare_stream_t stream);
/* no states and no lengths; `keep` as the forward of the same problem left it */
size_t flare_scan_backward_workspace_bytes(const flare_scan_args_t* args);
int flare_scan_backward(const flare_scan_args_t* args, flare_stream_t stream);
/* One token: x, dt, z, y [B, C], b, c [B, G, S] (the strides along n, N, documents and lengths are ignored).  state_out is
 * read and updated in place; state_in is ignored. */
int flare_scan_decode(const flare_scan_args_t* args, flare_stream_t stream);

/* sizeof(flare_conv_args_t / flare_scan_args_t) for which = 0 / 1 (other values: 0) */
size_t flare_mixers_abi_sizeof(int which);

#ifdef __cplusplus
}
#endif
#endif /* FLARE_B200_MIXERS_H_ */
