/*
 * flare_b200_mixers.h - the causal token mixers of libflare_b200.so beside FLARE: the short causal convolution and the
 * selective state space scan and softmax attention, for whole sequences (with gradients), prompts and single tokens.
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
  const float* A;           /* [C, S] contiguous, 16-byte aligned like the states */
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

/*
 * Causal attention of H query heads over J key / value heads (H a multiple of J, head h reads h / (H / J)) of width D (a
 * multiple of 8, at most 128), bf16 or fp16.  The score of the query at position i for the key at position j is
 *   cap tanh(scale <q, k> / cap) - slopes[h] |i - j|          (cap = 0: scale <q, k>, at most 1024; slopes NULL: no bias)
 * and token i sees the keys j <= i of its document, with `window` > 0 only j > i - window; where `prefix` [B, N] (bytes,
 * non-zero: true) holds for the first tokens of a document, all tokens of the document see those.  Without a key in
 * sight, or without a score above -infinity, y and all gradients are 0.
 *
 * Whole sequences (cached = NULL): Nk = Nq.  Prompts behind a cache (`cached` [B] int32: tokens that it holds): k and v are the
 * caches [B, Nk, J, D] with the new tokens in place (flare_attention_append), the Nq queries of row b lie at positions
 * cached[b] + i; lengths [B] (or NULL) as above; documents exclude `cached`, and there is no backward.
 */
typedef struct flare_attention_args {
  const void* q;            /* [B, Nq, H, D] */
  const void* k;            /* [B, Nk, J, D] */
  const void* v;            /* [B, Nk, J, D] */
  void* y;                  /* [B, Nq, H, D] contiguous */
  float* lse;               /* [B, H, Nq rounded up to 128]: minus log2 of the softmax denominators, for the backward; may be NULL */
  void* plan;               /* flare_attention_plan_bytes(args), 256-byte aligned: who sees whom, left by the forward for the backward; NULL: formed again */
  const int32_t* documents; /* [B, Nq] contiguous or NULL */
  const uint8_t* prefix;    /* [B, Nq] contiguous or NULL */
  const int32_t* cached;    /* [B] or NULL */
  const int32_t* lengths;   /* [B] or NULL */
  const float* slopes;      /* [H] or NULL */
  const void* dy;           /* backward: [B, Nq, H, D] */
  void* dq;                 /* [B, Nq, H, D] contiguous */
  void* dk;                 /* [B, Nk, J, D] contiguous, like dv */
  void* dv;
  void* workspace;
  size_t workspace_bytes;
  int32_t B, Nq, Nk, H, J, D;
  int64_t q_stride_b, q_stride_n, q_stride_h, k_stride_b, k_stride_n, k_stride_h, v_stride_b, v_stride_n, v_stride_h;
  int64_t dy_stride_b, dy_stride_n, dy_stride_h; /* all strides multiples of 8 elements and positive, pointers 16-byte aligned */
  float scale, cap;
  int32_t window; /* 0: none */
  int32_t dtype;
} flare_attention_args_t;

size_t flare_attention_plan_bytes(const flare_attention_args_t* args);
size_t flare_attention_forward_workspace_bytes(const flare_attention_args_t* args);
int flare_attention_forward(const flare_attention_args_t* args, flare_stream_t stream);
/* y, lse and (if given) plan as the forward of the same problem left them */
size_t flare_attention_backward_workspace_bytes(const flare_attention_args_t* args);
int flare_attention_backward(const flare_attention_args_t* args, flare_stream_t stream);

/*
 * Caches: k_cache, v_cache [B, L, J, D] (contiguous rows of D, strides in elements), written in place.
 * append: new_k[b, t] goes to position cached[b] + t for t < lengths[b] (NULL: N); positions outside [0, L) are left out.
 * decode: one token per row, q, y [B, H, D], new_k, new_v [B, J, D].  The row's keys are the first cached[b] of its cache and the
 * new one, which is written to position cached[b].  A row whose position lies outside [0, L) is idle: y = 0, nothing is written.
 * At most 65 535 rows in either.
 */
typedef struct flare_cache_args {
  const void* q;
  const void* new_k;
  const void* new_v;
  void* k_cache;
  void* v_cache;
  void* y;                /* [B, H, D] contiguous */
  const int32_t* cached;  /* [B]; append: NULL: 0 */
  const int32_t* lengths; /* [B] or NULL; append only */
  const float* slopes;    /* [H] or NULL */
  void* workspace;        /* decode */
  size_t workspace_bytes;
  int32_t B, N, H, J, D, L;
  int64_t q_stride_b, q_stride_h;
  int64_t new_k_stride_b, new_k_stride_n, new_k_stride_h, new_v_stride_b, new_v_stride_n, new_v_stride_h;
  int64_t k_stride_b, k_stride_n, k_stride_h, v_stride_b, v_stride_n, v_stride_h; /* of the caches; multiples of 8, like the others */
  float scale, cap;
  int32_t window;
  int32_t dtype;
} flare_cache_args_t;

int flare_attention_append(const flare_cache_args_t* args, flare_stream_t stream);
size_t flare_attention_decode_workspace_bytes(const flare_cache_args_t* args);
int flare_attention_decode(const flare_cache_args_t* args, flare_stream_t stream);

/* sizeof(flare_conv_args_t / flare_scan_args_t / flare_attention_args_t / flare_cache_args_t) for which = 0..3 (other values: 0) */
size_t flare_mixers_abi_sizeof(int which);

#ifdef __cplusplus
}
#endif
#endif /* FLARE_B200_MIXERS_H_ */
