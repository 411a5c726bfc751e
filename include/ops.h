/* SPDX-License-Identifier: Unlicense */

/* Generic tensor operations of the matcher networks, on one MI355X.
 *
 * The API is the reference's (ops.h:8-164 of i.coregistration.opencl),
 * signature for signature, so that the model drivers and the kernel
 * check call it unchanged; behind it are hand-written gfx950 kernels
 * (fp32 MFMA GEMM and implicit-GEMM convolution, flash attention,
 * wave-reduction norms, vectorised element-wise kernels).
 *
 * Tensors are float32, channel-major (C, H, W) for image-like data and
 * token-major (tokens, channels) for sequences. Offsets are in floats.
 * Every call checks on the host that each element it will touch lies
 * inside its buffers (cl_mem carries the byte size) and that element
 * counts passed to kernels stay below 2^31; a violation is a fatal
 * error naming the operation, before anything is launched. */

#ifndef ICOREG_OPS_H
#define ICOREG_OPS_H

#include "hip_backend.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Activations, applied after the bias (ops.h:8-13). */
#define ACT_NONE 0
#define ACT_GELU 1 /* Exact (erf) GELU. */
#define ACT_RELU 2
#define ACT_LEAKY 3 /* LeakyReLU with the given negative slope. */
#define ACT_GELU_TANH 4

/* Largest attention head dimension of ops_attention (ops.h:16). */
#define OPS_MAX_HEAD_DIM 128

/* ops.h:21-30. No kernel objects: every operation launches a typed HIP
 * kernel. scratch / scratch_bytes / im2col_bytes are kept for the
 * callers that read them; the implicit-GEMM convolution needs no
 * unfold scratch, so im2col_bytes bounds nothing here. */
struct ops {
    struct ocl_backend *ocl;
    cl_mem scratch;
    size_t scratch_bytes, im2col_bytes;
};

/* One GEMM operand: buffer, element offset, leading dimension and the
 * two batch strides (ops.h:34-39). Batch b of nb = nb0 * nb1 uses
 * (b / nb1) * s0 + (b % nb1) * s1. */
struct opnd {
    cl_mem buf;
    cl_long off;
    cl_int ld;
    cl_long s0, s1;
};

struct opnd ops_mat(cl_mem buf, long off, int ld);
struct opnd ops_bmat(cl_mem buf, long off, int ld, long s0, long s1);

void ops_init(struct ops *o, struct ocl_backend *ocl);
void ops_free(struct ops *o);

/* Per-name kernel times accumulated when ocl->profile is set (HIP events
 * around every launch, the stream synchronised after each), printed by
 * ops_report (ops.c:25-67). */
void ops_report(void);

/* Batched C = act(alpha * A * op(B) + bias) + R over nb = nb0 * nb1
 * products; bias per column, or per row with biasrow set; R NULL for no
 * residual, else it has C's layout (ldc, strides) from element offset
 * roff and may alias C. transb: B stored N x K (PyTorch Linear weight),
 * else K x N. ops.h:54-60. */
void ops_gemm(struct ops *o, int M, int N, int K, struct opnd A, struct opnd B,
              int transb, struct opnd C, int nb, int nb1, cl_mem bias,
              int biasrow, cl_mem R, long roff, float alpha, int act,
              float slope);

/* Token-major Y[rows, out] = act(X[rows, in] W^T + b) (+ Y when
 * residual), W the PyTorch [out, in] weight. ops.h:64-66. */
void ops_linear(struct ops *o, int rows, int in, int out, cl_mem X, long xoff,
                cl_mem W, cl_mem b, cl_mem Y, long yoff, int act, float slope,
                int residual);

/* 1x1 convolution: W (K, C) times X (C, HW) into Y (K, HW), bias per
 * output channel. ops.h:70-71. */
void ops_conv1x1(struct ops *o, cl_mem X, long xoff, int C, int HW, cl_mem W,
                 cl_mem b, int K, cl_mem Y, long yoff, int act, float slope);

/* Geometry of a 2D convolution or pooling window (ops.h:74-76). */
struct conv_geom {
    int kh, kw, sy, sx, py, px, dy, dx, groups;
};

/* Square kernel k, stride s, padding p, dilation 1, one group. */
struct conv_geom ops_geom(int k, int s, int p);

/* Output size of a convolution along one axis. */
int ops_conv_out(int n, int k, int s, int p, int d);

/* in (C, H, W) into out (K, Ho, Wo), weights (K, C / groups, kh, kw).
 * mean/rstd/alpha (NULL for none) normalise and gate every input value,
 * prelu((x - mean[c]) * rstd[c], alpha[c]), before the zero padding, as
 * DISK's blocks (ops.h:84-92). One group, 3 x 3 or 5 x 5, stride 1
 * or 2: direct fp32 MFMA kernel on LDS input patches; other one-group
 * geometries: implicit-GEMM fp32 MFMA kernel; grouped: a direct
 * kernel. */
void ops_conv2d(struct ops *o, cl_mem in, int C, int H, int W, cl_mem w,
                cl_mem b, int K, const struct conv_geom *g, cl_mem mean,
                cl_mem rstd, cl_mem alpha, int act, float slope, cl_mem out);

/* Extension with no counterpart in the reference: ops_conv2d over nb
 * images stored in_stride / out_stride floats apart (the two images of
 * a tile pair), in one launch; the same weights, bias and input
 * normalisation for every image. */
void ops_conv2d_batch(struct ops *o, int nb, cl_mem in, long in_stride, int C,
                      int H, int W, cl_mem w, cl_mem b, int K,
                      const struct conv_geom *g, cl_mem mean, cl_mem rstd,
                      cl_mem alpha, int act, float slope, cl_mem out,
                      long out_stride);

/* Instance statistics of (C, HW): mean and 1 / sqrt(biased var + eps)
 * per channel. ops.h:96-97. */
void ops_chan_stats(struct ops *o, cl_mem x, int C, int HW, float eps,
                    cl_mem mean, cl_mem rstd);

/* Y = act((X - mean) * rstd * g + b) per channel; mean (with rstd), g, b
 * may each be NULL. Y may alias X. ops.h:101-103. */
void ops_chan_affine(struct ops *o, cl_mem X, cl_mem Y, int C, int HW,
                     cl_mem mean, cl_mem rstd, cl_mem g, cl_mem b, int act,
                     float slope);

void ops_prelu(struct ops *o, cl_mem X, cl_mem Y, int C, int HW, cl_mem alpha);
void ops_act(struct ops *o, cl_mem X, cl_mem Y, long n, int act, float slope);

/* Row LayerNorm of rows x C (token-major), g/b NULL for none; Y may
 * alias X. ops.h:109-110. */
void ops_layernorm(struct ops *o, long rows, int C, cl_mem X, cl_mem Y,
                   cl_mem g, cl_mem b, float eps, int act, float slope);

/* In-place softmax(scale * x) over rows of L. ops.h:113. */
void ops_softmax_rows(struct ops *o, cl_mem S, long rows, int L, float scale);

/* O = softmax(scale Q K^T) V per head, nh heads of d <= 128 channels,
 * head h at columns h * d of token-major rows; kmask (Nk bytes, 0 =
 * ignore the key) may be NULL; a query with no key left gets zeros.
 * ops.h:119-121. */
void ops_attention(struct ops *o, struct opnd Q, struct opnd K, struct opnd V,
                   struct opnd O, int Nq, int Nk, int nh, int d, float scale,
                   cl_mem kmask);

/* ops_attention that allocates nothing: the key-split partials go to a
 * fixed 24 MiB device array (one per GPU, held until the process ends)
 * instead of the ops work buffer, which ops_attention grows with
 * hipMalloc. No counterpart in the reference; for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving
 * loops). Same results as ops_attention. A problem whose partials
 * exceed 24 MiB is a fatal error (RoMa's ViT attention, the largest on
 * the path, needs 20.3 MB). The array costs 24 MiB of device memory per
 * process on every GPU where the library is loaded, called or not.
 * Every call on one GPU shares the array: calls that overlap on one GPU
 * (other streams or threads) race. */
void ops_attention_noalloc(struct ops *o, struct opnd Q, struct opnd K,
                           struct opnd V, struct opnd O, int Nq, int Nk, int nh,
                           int d, float scale, cl_mem kmask);

/* ops_attention on nb independent problems in one launch, problem i's Q,
 * K, V and O starting bq, bk, bv, bo floats after problem i - 1's (kmask
 * shared). No counterpart in the reference, which loops over the images
 * of a pair with one attention launch each (eloftr.c:405-449,
 * roma.c:692-713). */
void ops_attention_batch(struct ops *o, int nb, struct opnd Q, long bq,
                         struct opnd K, long bk, struct opnd V, long bv,
                         struct opnd O, long bo, int Nq, int Nk, int nh, int d,
                         float scale, cl_mem kmask);

/* Rotary encoding in place on rows x (nh heads of d) of X (row stride
 * ld, offset off), row r at table row r % npos of cs (npos x d / 2
 * (cos, sin) pairs). interleaved: pairs (2f, 2f + 1), else (f, f + d/2).
 * ops.h:127-128. */
void ops_rope(struct ops *o, cl_mem X, long off, int ld, long rows, int nh,
              int d, int npos, cl_mem cs, int interleaved);

/* ---- Long token sequences and large tiles --------------------------------
 * Extensions with no counterpart in the reference, for transformer layers on
 * more tokens than the networks here were trained on: products in 8-bit
 * integers, rotary positions computed from the tokens' coordinates,
 * attention over the blocks of keys that a cheap score selects, norms that
 * leave 8-bit codes, keys and values kept in 8 bits, and attention within a
 * window. They
 * allocate nothing and leave the ops work buffer alone: what they need for
 * themselves is the caller's `work` buffer, of the size that the call's
 * _work_bytes function gives (0 where the sizes are invalid), 16-byte
 * aligned, its content of no meaning between calls. The size never falls as
 * tokens, keys, channels in or listed blocks grow: a buffer for the longest
 * call serves the shorter ones. Calls that may overlap on the device
 * (recorded graphs replayed side by side among them) need work buffers of
 * their own. */

/* 8-bit codes and scales of rows of C floats, row r at float xoff + r ldx of
 * X: with a = max |x|, S[r] = a / 127 and code(x) = x (127 / a) in float32,
 * rounded to the nearest integer, ties to even, so that x = code S within
 * S / 2. A row with a < 2^-100 counts as zero (S = 0); a row with a value
 * that is not finite gets S = NaN, codes 0. Row r of Q starts at byte r
 * ops_q8_pitch(C) (C rounded up to 64), zeros behind the C codes. Q 16-byte
 * aligned; X, Q and S apart. The same call makes the codes of a PyTorch
 * [out, in] weight (rows = out, C = in). */
int ops_q8_pitch(int C);
void ops_quant_rows(struct ops *o, long rows, int C, cl_mem X, long xoff,
                    int ldx, cl_mem Q, cl_mem S);

/* Y = act((XS[i] WS[j]) sum_k XQ[i][k] WQ[j][k] + b[j]) + R, token-major: XQ,
 * XS rows tokens, WQ, WS out channels as ops_quant_rows makes them, in <=
 * 2^17 of both, the sum exact in 32-bit integers, the product of the two
 * scales rounded to float32 first (its range ends at 2^128, and bits are lost
 * under 2^-126). Row i of Y starts at float
 * yoff + i ldy; b and R NULL for none, R with Y's row stride from roff, and
 * it may be Y itself, any other overlap of Y is an error. */
void ops_linear_qq(struct ops *o, int rows, int in, int out, cl_mem XQ,
                   cl_mem XS, cl_mem WQ, cl_mem WS, cl_mem b, cl_mem R,
                   long roff, cl_mem Y, long yoff, int ldy, int act,
                   float slope);

/* ops_quant_rows of the float tokens X, then ops_linear_qq. */
size_t ops_linear_q8_work_bytes(int rows, int in);
void ops_linear_q8(struct ops *o, int rows, int in, int out, cl_mem X,
                   long xoff, int ldx, cl_mem WQ, cl_mem WS, cl_mem b,
                   cl_mem R, long roff, cl_mem Y, long yoff, int ldy, int act,
                   float slope, cl_mem work);

/* Frequencies (radians a position) of the rot / 2 pairs for ops_rope_pos, on
 * the host: pair p belongs to coordinate p % axes and is the k-th, k = p /
 * axes, of its n = rot / axes channels; trained frequency w = base^(-2 k /
 * n). For coordinates beyond the trained ones, factor > 1 stretches them:
 * ROPE_LINEAR all alike (w / factor), ROPE_REBASE by the base (base
 * factor^(n / (n - 2))), ROPE_PARTS only pairs that turn few times over the
 * `trained` positions: w (g + (1 - g) / factor), g = (trained w / 2 pi -
 * slow) / (fast - slow) held to 0 .. 1. rot a multiple of 2 axes. */
#define ROPE_TRAINED 0
#define ROPE_LINEAR 1
#define ROPE_REBASE 2
#define ROPE_PARTS 3
void ops_rope_freqs(double *freq, int rot, int axes, double base, int kind,
                    double factor, double trained, double slow, double fast);

/* Rotary encoding by coordinates of two tensors (queries and keys; nh2 = 0
 * for one) of rows x (nh heads of d): the first rot channels of each head are
 * turned, pair p by the angle pos[row axes + p % axes] freq[p] (pos: int32,
 * freq: rot / 2 doubles; the angle in 64 bits), and multiplied by mult; the
 * others are copied. ROPE_INTERLEAVED: pairs (2 p, 2 p + 1), else (p, p + rot
 * / 2). ROPE_INVERSE: by the negative angle, the gradient of the forward
 * call. Xi to Yi, rows at the operands' offsets and ld (packed projections);
 * Yi may be Xi (same offset and ld), any other overlap of an output is an
 * error (rows side by side in one packed buffer do not overlap). rot 0 ..
 * min(d, 2048), even; axes 1 .. 4. */
#define ROPE_INTERLEAVED 1
#define ROPE_INVERSE 2
void ops_rope_pos(struct ops *o, long rows, int d, int rot, int axes,
                  cl_mem pos, cl_mem freq, float mult, int flags,
                  struct opnd X1, struct opnd Y1, int nh1, struct opnd X2,
                  struct opnd Y2, int nh2);

/* Attention over selected blocks of bs = 16, 32, 64 or 128 keys, the last one
 * shorter: nh query heads on nhk key heads (nh a multiple; query head h on
 * key head h / (nh / nhk)) of d <= 128 channels, head h at columns h d.
 *
 * ops_block_index: codes KC and scales KS of blocks b0 .. b0 + nb - 1, block
 * b, key head h at row b nhk + h: the mean of the block's kept keys (kmask:
 * Nk bytes, 0 = leave the key out, or NULL), rounded to float32 and coded as
 * by ops_quant_rows; scale -1 where no key is kept. An index that is kept
 * with a growing sequence has its last blocks made again. ops_key_blocks:
 * the number of blocks of Nk keys. */
int ops_key_blocks(int Nk, int bs);
void ops_block_index(struct ops *o, struct opnd K, int Nk, int nhk, int d,
                     int bs, cl_mem kmask, int b0, int nb, cl_mem KC,
                     cl_mem KS);

/* SEL[(query nh + head) top + i], int32: the blocks with the top (1 .. 64)
 * largest scores KS (q . KC), q the query's 8-bit codes, best first, ties to
 * the lower block, NaN above all numbers, -1 behind the last block that keeps
 * a key. The sum of the codes' products is exact: the same selection from
 * every kernel. No kernel needs work here: the size is 0, work may be NULL. */
size_t ops_block_select_work_bytes(int Nq, int nh, int nblk, int top);
void ops_block_select(struct ops *o, struct opnd Q, int Nq, int nh, int nhk,
                      int d, cl_mem KC, cl_mem KS, int nblk, int top,
                      cl_mem SEL, cl_mem work);

/* O = softmax(scale Q K^T) V over the kept keys of each query and head's
 * listed blocks (SEL as above; entries that are no block are skipped, a block
 * listed twice counts once). No key left: zeros. A NaN among the kept scores
 * makes the row NaN; what left-out keys and values hold does not matter; a
 * key's weight under 2^-126 of the row's largest may count as zero, and sums of
 * values from 2^115 on may pass float32's range before they are divided. O
 * may be Q (same offset and ld), any other overlap of O is an error. */
size_t ops_attention_blocks_work_bytes(int Nq, int Nk, int nh, int nhk, int d,
                                       int bs, int top);
void ops_attention_blocks(struct ops *o, struct opnd Q, struct opnd K,
                          struct opnd V, struct opnd O, int Nq, int Nk, int nh,
                          int nhk, int d, int bs, int top, cl_mem SEL,
                          float scale, cl_mem kmask, cl_mem work);

/* H = X + R and Y = H g / sqrt(mean(H^2) + eps), token-major, rows at the
 * operands' offsets and ld: the mean of a row's squares in 64 bits, the
 * root's reciprocal i rounded to float32, Y = (H i) g with both products
 * rounded, so that the codes are the same from every kernel. R.buf NULL: H is
 * X; g (C floats) NULL: ones; eps > 0. Outputs, any of them NULL but not all:
 * H, Y, and Y's 8-bit codes Q with their scales S as ops_quant_rows makes them
 * (both or none), which ops_linear_qq takes. H and Y may each be X or R (same
 * offset and ld), any other overlap of an output is an error. */
void ops_rms_norm(struct ops *o, long rows, int C, struct opnd X,
                  struct opnd R, cl_mem g, float eps, struct opnd H,
                  struct opnd Y, cl_mem Q, cl_mem S);

/* Keys and values kept in 8 bits, in pages of `page` = 16, 32, 64 or 128
 * tokens: page p, key head h, place t at row (p nhk + h) page + t of the codes
 * kc and vc (ops_cache_pitch(d) bytes a row: d rounded up to 16, zeros behind
 * the d <= 128 codes; 16-byte aligned) and of the scales ks and vs (floats).
 * Codes and scale of a token and head are those of ops_quant_rows. */
struct ops_cache {
    cl_mem kc, vc, ks, vs;
    cl_int pages, page, nhk, d;
};

/* The sequences of a call, all in device memory and not looked at by the
 * host. Rows start[b] .. start[b + 1] - 1 (int32, n + 1 of them, not falling)
 * of the token-major operands are the last ones of sequence b, of which len[b]
 * (int32) tokens are kept once the call's are: row start[b] + i is its
 * position len[b] - (start[b + 1] - start[b]) + i. Position i is place i % page
 * of page table[b ldt + i / page] (int32). A position that is negative or
 * behind the table, or whose entry is no page (-1: given back), is not kept.
 * Rows before start[0] and behind start[n] belong to no sequence. */
struct ops_seqs {
    cl_mem start, len, table;
    cl_int n, ldt;
};

/* ops_cache_write: the rows' keys K and values V (nhk heads of d, head h at
 * columns h d) to their places; rows without one are left out, places that no
 * row has stay as they are. Two rows of a call must not have one place: which
 * of them it keeps, and whether codes and scale are of the same, is not said.
 * ops_cache_read: code times scale of the rows' positions to K and V (either
 * may have no buffer), zeros where nothing is kept; rows of no sequence stay
 * as they are. rows: those of the operands; start is held to 0 .. rows. */
int ops_cache_pitch(int d);
void ops_cache_write(struct ops *o, const struct ops_cache *c,
                     const struct ops_seqs *s, int rows, struct opnd K,
                     struct opnd V);
void ops_cache_read(struct ops *o, const struct ops_cache *c,
                    const struct ops_seqs *s, int rows, struct opnd K,
                    struct opnd V);

/* O = softmax(scale Q K^T) V within a window: query i, at position q0 + i,
 * sees the keys j <= q0 + i + right of those with j >= q0 + i - left or j <
 * sinks (left, right < 0: no limit; right = 0: no later key; sinks >= 0: the
 * first keys stay visible), and of those the kept ones (kmask: Nk bytes, 0 =
 * leave the key out, or NULL). nh query heads on nhk key heads of d <= 128 as
 * for ops_attention_blocks. No key left: zeros. A NaN among the seen scores
 * makes the row NaN; what unseen keys and values hold does not matter; a key's
 * weight under 2^-126 of the row's largest may count as zero, and sums of
 * values from 2^115 on may pass float32's range before they are divided.
 * Sums, maxima and outputs are float32's. What enters the products may be
 * rounded: queries, keys and values to 22 bits or to 2^-39 of their row and
 * head's largest, but not to what moves a score log2 e by more than 2^-20
 * beyond the 22 bits; a weighted value to 2^-23 of itself or to 2^-35 of the
 * largest value among the keys up to the row's last, but not to more than 2^-20
 * of the row and head's largest output. So a channel of the values that is far
 * below (2^-15) the others of its row and head keeps fewer bits than those; in
 * calls of few rows (16 a key head and sequence) nothing is rounded to less
 * than float32. O may be Q (same offset and ld), any
 * other overlap of O is an error. work: what a call needs while it runs; calls
 * that may run at once, recorded ones too, have one each. */
size_t ops_attention_window_work_bytes(int Nq, int nh, int d);
void ops_attention_window(struct ops *o, struct opnd Q, struct opnd K,
                          struct opnd V, struct opnd O, int Nq, int Nk, int nh,
                          int nhk, int d, int q0, int left, int right,
                          int sinks, float scale, cl_mem kmask, cl_mem work);

/* The same over a cache, right = 0: each row's query (nh heads of the
 * cache's d, nh a multiple of its nhk) over the kept positions of its own
 * sequence. Rows of no sequence stay as they are in O. A row's own key is
 * seen like any other, so the call follows the rows' ops_cache_write. */
size_t ops_attention_cache_work_bytes(int rows, int nh, int d);
void ops_attention_cache(struct ops *o, const struct ops_cache *c,
                         const struct ops_seqs *s, int rows, struct opnd Q,
                         struct opnd O, int nh, int left, int sinks,
                         float scale, cl_mem work);

/* Bilinear resampling of in (C, h, w) into channels coff.. of out
 * (*, H, W). align_corners 0: scale > 0 gives source step 1 / scale,
 * scale 0 the size ratio. ops.h:133-134. */
void ops_resize(struct ops *o, cl_mem in, int C, int h, int w, cl_mem out,
                int H, int W, int coff, int align_corners, float scale);

/* Bilinear sampling of in (C, H, W) at n normalised (x, y) points of
 * grid into out (C, n), zero padding. ops.h:138-139. */
void ops_grid_sample(struct ops *o, cl_mem in, int C, int H, int W, cl_mem grid,
                     int n, int align_corners, cl_mem out);

/* F.unfold of in (C, H, W) into out (C * kh * kw, Ho * Wo). */
void ops_unfold(struct ops *o, cl_mem in, int C, int H, int W,
                const struct conv_geom *g, cl_mem out);

/* 2x2 / stride 2 average pooling. */
void ops_avgpool2(struct ops *o, cl_mem in, int C, int H, int W, cl_mem out);

/* k x k pooling, stride s, padding p: maximum (padding ignored) or
 * average (padding counted). */
void ops_pool2d(struct ops *o, cl_mem in, int C, int H, int W, int k, int s,
                int p, int max, cl_mem out);

/* (B, R, C) to (B, C, R). */
void ops_transpose(struct ops *o, cl_mem in, cl_mem out, int B, int R, int C);

/* out = alpha * a + beta * b[i % bmod] (b NULL: alpha * a); out may alias
 * a. */
void ops_axpby(struct ops *o, cl_mem out, cl_mem a, float alpha, cl_mem b,
               float beta, long n, long bmod);

/* Fold an eval-mode BatchNorm into the preceding convolution's weights w
 * (K x per) and bias b (K floats, in: the convolution's bias or zeros),
 * in double precision on the host. ops.h:162-164. */
void ops_fold_bn(float *w, float *b, int K, long per, const float *gamma,
                 const float *beta, const float *mean, const float *var,
                 float eps);

#ifdef __cplusplus
}
#endif

#endif /* ICOREG_OPS_H */
