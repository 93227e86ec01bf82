/*
 * bert_amd.h — additive extensions of the drop-in library (not in the
 * reference ABI; the reference consumers never need them).
 *
 * They exist for three callers:
 *   - bench.py / tests: device-resident batch evaluation on a caller-chosen
 *     HIP stream (inputs already in HBM, nothing copied, no sync);
 *   - multi-GPU: choose the devices a context is replicated on (the
 *     reference ABI has no device argument; SURVEY.md §8(b) "No device
 *     argument");
 *   - tooling: the deterministic synthetic GGUF generator and per-kernel
 *     timing.
 * All functions are C-ABI, take plain pointers and sizes, never throw, and
 * return 0 on success / negative on error (message via bert_amd_last_error).
 */
#ifndef BERT_AMD_H
#define BERT_AMD_H

#include <stdint.h>

#include "bert.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Load a GGUF and replicate its weights on the given HIP devices (ordinals as
   seen by this process).  n_devices <= 0: all visible devices, or the list in
   env BERT_AMD_DEVICES="0,1,...".  Returns NULL on error. */
BERT_API struct bert_ctx *bert_amd_load(const char *fname, const int32_t *devices, int32_t n_devices);

/* bert_amd_load with options: "key=value" items separated by ';' (NULL or ""
   = none).  Every key's default may come from the environment
   (BERT_AMD_<KEY> in upper case), which is read once, inside this call; the
   string overrides it.  Load-time keys (they shape the device weights):
     "i8"       Q4 projections on the int8-MFMA GEMMs: "0" none, "all", or a
                list of up, o, down joined by '+' (default: up+o+down for Q4_0
                at n_embd 384, up+down for Q4_1 there, up otherwise)
     "qkva_ntw" the fused QKV + attention kernel: 0 producer / consumer
                waves on an int8 QKV copy (Q4_0, head dim 32, n_embd 384;
                elsewhere 1), 1 | 2 head-pair units per main loop of the
                head-pair kernel, -1 (default) 0 where it exists, else 2
     "q41bf"    Q4_1 on the int8 GEMMs: the per-block scale products d_w d_a
                and m_w s_a as exact bf16 partial products on the bf16 MFMA
                (kernels.h W_Q4_1B) instead of the f32 MFMA: 1 every int8
                projection, 0 none, -1 (default) all but the 384-wide FFN-down
                + LayerNorm kernel (where they cost more than they save)
     "emb_raw"  1 (default): the word-embedding table stays in its GGUF row
                format on the device (dequantised in the embedding kernel as
                ggml's get_rows does); 0: an f32 copy.  Same results
   and every bert_amd_set_option key below.  Returns NULL on error (an unknown
   key or a bad value included). */
BERT_API struct bert_ctx *bert_amd_load_opts(const char *fname, const int32_t *devices, int32_t n_devices,
                                             const char *options);

BERT_API int32_t bert_amd_n_devices(struct bert_ctx *ctx);

/* hparams: [n_vocab, n_max_tokens, n_embd, n_intermediate, n_head, n_layer, weight ggml type] */
BERT_API int32_t bert_amd_hparams(struct bert_ctx *ctx, int32_t *out7);

/* Device-resident evaluation on replica `slot` (index into the context's
   device list), enqueued on `hip_stream` (a hipStream_t; NULL = HIP's null
   stream, i.e. torch's default stream).  Asynchronous: returns after
   enqueueing; every kernel and workspace fill runs on `hip_stream`.  Takes
   the context's lock (one eval at a time per context, like bert_eval_batch).
     d_tokens   : int32, packed token ids of all sentences (device memory)
     d_offsets  : int32[n_seqs+1], prefix offsets into d_tokens (device memory)
     h_offsets  : the same offsets in host memory (used for grid sizing)
     d_out      : float[n_seqs * n_embd] (device memory), L2-normalised
   Workspace is grown on demand (allocation happens outside any capture when
   the caller warms up with the largest batch first). */
BERT_API int32_t bert_amd_eval_device(struct bert_ctx *ctx, int32_t slot, const int32_t *d_tokens,
                                      const int32_t *d_offsets, const int32_t *h_offsets, int32_t n_seqs,
                                      float *d_out, void *hip_stream);

/* Per-kernel-class timing with HIP events on the launch stream.
   enable != 0 turns it on for subsequent evals (adds event records between
   launches; never used inside bench.py's timed region). */
BERT_API int32_t bert_amd_profile_enable(struct bert_ctx *ctx, int32_t enable);
/* Copies up to max_entries: names (NUL-separated into names_buf), total ms
   and launch counts since enable.  Returns the number of entries. */
BERT_API int32_t bert_amd_profile_read(struct bert_ctx *ctx, char *names_buf, int32_t names_len, float *total_ms,
                                       int32_t *counts, int32_t max_entries);

/* Deterministic synthetic BERT GGUF (see csrc/synth.cpp).
   ftype: 0 = f32, 1 = f16, 2 = Q4_0, 3 = Q4_1 (2-D *.weight tensors). */
BERT_API int bert_amd_synth_model(const char *path, int32_t n_vocab, int32_t n_max_tokens, int32_t n_embd,
                                  int32_t n_intermediate, int32_t n_head, int32_t n_layer, int32_t ftype,
                                  uint64_t seed, float w_std);

/* Tokenizer without a model/GPU (tests, tooling): runs the native WordPiece
   tokenizer configured by an HF tokenizer.json string.  frame == 0: the content
   ids of Encode(text) (at most n_max_tokens); frame != 0: bert_tokenize's
   [CLS] ... [SEP] framing with the given special ids.  Returns the count. */
BERT_API int32_t bert_amd_tokenize_json(const char *tokenizer_json, const char *text, int32_t *tokens,
                                        int32_t n_max_tokens, int32_t frame, int32_t cls_id, int32_t sep_id,
                                        int32_t pad_id);

/* Test hook: the embeddings + LayerNorm stage alone (reference
   bert.cpp:865-898) on a host batch (packed ids + offsets[n_seqs+1]), on
   replica 0.  Copies back X (f32 [M][n_embd], the LayerNorm output) and the
   first GEMM's activation format of it: q [M][n_embd] (int8 for Q4 models,
   fp16 / f32 for F16 / F32) and d [M][n_embd/32] (fp16 for Q4_0, f32 for
   Q4_1; may be NULL).  Lets tests pin the integer stage bit-exactly against
   the oracle's quantiser. */
BERT_API int32_t bert_amd_debug_embed(struct bert_ctx *ctx, const int32_t *tokens, const int32_t *offsets,
                                      int32_t n_seqs, float *X_out, void *q_out, void *d_out);

/* Test hook: the whole pipeline on a host batch (replica 0, one row group,
   the kernels bert_eval_batch would pick for it under the context's options),
   copying back the residual stream after every stage: X_out f32
   [n_layer + 1][M][n_embd] (stage 0 = embeddings + LayerNorm, reference
   bert.cpp:865-898; stage l + 1 = the output of encoder layer l,
   bert.cpp:900-993) and its activation form as bert_amd_debug_embed's q / d,
   per stage.  Lets tests pin parity layer by layer against the oracle. */
BERT_API int32_t bert_amd_debug_layers(struct bert_ctx *ctx, const int32_t *tokens, const int32_t *offsets,
                                       int32_t n_seqs, float *X_out, void *q_out, void *d_out);

/* Rows (tokens, padded to the 128-row tile) the device workspace of replica
   `slot` currently holds; -1 on a bad argument.  Lets callers and tests see
   that bert_encode_batch's n_batch_size bounds the working set. */
BERT_API int64_t bert_amd_workspace_rows(struct bert_ctx *ctx, int32_t slot);

/* Per-context pipeline options (defaults, then bert_amd_load_opts /
   BERT_AMD_<KEY> at load; this call changes them afterwards):
     "split" 0 | 1     run large fused batches as two row groups on two streams
     "pack"  -1 | 0 | 1 pack short sentences into shared fused-kernel tiles
                        when it pays (-1, default) / never / always
     "fuse_min" n >= 0 batches of fewer than n sentences (default 48) run the
                        unfused QKV GEMM + attention pair instead of the fused
                        kernel (lower latency for small batches)
     "unfused" 0 | 1    1: every batch on the QKV GEMM + attention pair (A/B
                        checks; default 0)
     "small_rows" n >= 0 batches of at most n padded rows (default 2048; one
                        sentence is 128) run the int8 GEMMs in 32-row tiles
                        (Q4_0, K <= 3072, <= 512 rows: the K loop split
                        over 12-16 waves; latency of small batches; 0 = never)
     "small_qkva" 0 | 1  1 (default): small batches (<= small_rows, <= 2048 rows) whose
                        sentences all have <= 64 tokens (Q4_0, n_embd 384, head
                        dim 32) run each head's int8 QKV and its attention in one
                        kernel (same results; one launch less per layer)
     "nt_x" 0 | 1        1 (default): the 384-wide projection + LayerNorm kernel
                        stores X with the nontemporal cache policy (all but the
                        last layer's X, which the pooling reads next), so the
                        weights its tiles re-read stay in L2; 0 plain stores
     "graph_seqs" n >= 0 host batches of at most n sentences (and fewer than
                        fuse_min) replay a captured HIP graph of their launches
                        (default 0: measured no faster)
     "encode_lanes" n >= 1 bert_encode_batch: lanes per device, each a host
                        thread with its own workspace and streams (default 2;
                        BERT_AMD_ENCODE_LANES)
     "encode_merge" n >= 1 bert_encode_batch: consecutive n_batch_size slices a
                        lane evaluates as one ragged batch (default 16;
                        BERT_AMD_ENCODE_MERGE; 1 = one slice per GPU batch),
                        merged only up to "encode_merge_rows" sentences
                        (default 256; BERT_AMD_ENCODE_MERGE_ROWS).  At most
                        lanes x max(n_batch_size, min(merge x n_batch_size,
                        merge_rows)) sentences are in flight per device
   Results are identical under every setting. */
BERT_API int32_t bert_amd_set_option(struct bert_ctx *ctx, const char *key, int32_t value);

/* Reads an option back into *value: every bert_amd_set_option key, plus the
   load-time choices as resolved for this model — "qkva_ntw" (0, 1 or 2),
   "i8_qkv", "i8_up", "i8_o", "i8_down" (1 when that Q4 projection runs on
   the int8-MFMA GEMMs: for QKV, the producer / consumer kernel's int8 copy
   and its unfused int8 twin), "q41bf" (the load option: -1 auto, 0, 1) and
   "q41bf_qkv", "q41bf_o", "q41bf_up", "q41bf_down" (1 when that Q4_1
   projection's int8 GEMM takes its scale products on the bf16 MFMA,
   W_Q4_1B).  Lets bench.py price each kernel on the
   arithmetic it runs.  Returns 0, or -2 on an unknown key. */
BERT_API int32_t bert_amd_get_option(struct bert_ctx *ctx, const char *key, int32_t *value);

/* How bert_eval_batch splits a batch over n_replicas devices: contiguous
   sentence slices balanced by token count, slice r = [cut[r], cut[r+1]),
   cut[0] = 0, cut[n_replicas] = n_seqs (cut has n_replicas + 1 entries).
   Pure host function (no device needed); lets tests check balance and
   coverage.  Returns 0, or -1 on invalid arguments. */
BERT_API int32_t bert_amd_shard_cuts(int32_t n_seqs, const int32_t *n_tokens, int32_t n_replicas, int32_t *cut);

/* ---------------------------------------------------------------------------
   Operators around the encoder, on device tensors of the caller: a dense layer
   and its gradients (a trained head or adapter on the embeddings), the lookup
   of token rows and its gradient, and the AdamW step that trains them.

   All of them run asynchronously on `hip_stream` (a hipStream_t; NULL = the
   null stream of `device`), allocate nothing, copy nothing to or from the host
   and may be captured into a HIP graph.  `device` is the HIP device that the
   tensors and the stream belong to; the caller's current device is left as it
   was.  Where a call takes a workspace, the caller gives device memory of at
   least the bytes its *_workspace function names, 16-byte aligned; the call may
   write all of it and keeps nothing in it for the next, so calls that may run
   at the same time (two streams, two graphs) need one each.  Rows of a matrix
   are `ld*` elements apart (at least its width; 0 for an input: the one row
   again for every row); nothing is written between them.  Results do not
   depend on the launch: the same inputs give the same bits.  Outputs and the
   workspace must not overlap inputs or each other unless a call says so (columns
   of one wider matrix do not overlap).  Each returns 0; or -1, an invalid
   argument, without having launched anything; or -3, a HIP error of this call's
   own, after which a part of it may have run: what it writes (an optimizer's
   weights and moments too) is then undefined (message via bert_amd_last_error). */

/* element types of the operators' tensors (ggml's numbers, as in the model files) */
enum bert_amd_type {
    BERT_AMD_F32 = 0,
    BERT_AMD_F16 = 1,
    BERT_AMD_Q4_0 = 2,
    BERT_AMD_Q4_1 = 3,
    BERT_AMD_BF16 = 30
};

/* activations; GELU is the tanh form the encoder's feed-forward layer uses,
   GELU_ERF z/2 (1 + erf(z / sqrt 2)), SILU z / (1 + exp(-z)) */
enum bert_amd_act {
    BERT_AMD_ACT_NONE = 0,
    BERT_AMD_ACT_RELU = 1,
    BERT_AMD_ACT_GELU = 2,
    BERT_AMD_ACT_GELU_ERF = 3,
    BERT_AMD_ACT_SILU = 4,
    BERT_AMD_ACT_TANH = 5
};

/* Dense layer: z = x W^T + bias, y = act(z) + residual.
     type     : F32, F16 or BF16, of x, w, residual, y and z; sums are f32, each
                output is rounded once
     x, w     : [M][K], [N][K]; bias: f32 [N] or NULL; residual: [M][N] or NULL
                (may be y itself, with ldr = ldy)
     y        : [M][N]; z: [M][N] or NULL: the pre-activation, kept for
                bert_amd_linear_backward
   M = 0 does nothing; M <= 2^30, 1 <= N, K < 2^22, and none of M N, M K and N K
   over 2^34.
   The workspace takes copies of x and w where their rows are not 16-byte pieces
   throughout: `aligned` != 0 says that both begin on 16 bytes and their row
   strides are multiples of 16 bytes (and under 2^21 elements). */
BERT_API int64_t bert_amd_linear_workspace(int32_t type, int64_t M, int32_t N, int32_t K, int32_t aligned);
BERT_API int32_t bert_amd_linear(int32_t device, int32_t type, int32_t act, int64_t M, int32_t N, int32_t K,
                                 const void *x, int64_t ldx, const void *w, int64_t ldw, const float *bias,
                                 const void *residual, int64_t ldr, void *y, int64_t ldy, void *z, int64_t ldz,
                                 void *workspace, int64_t workspace_bytes, void *hip_stream);

/* Its gradients from dy [M][N] (the residual's gradient is dy itself):
   dz = dy act'(z), dx = dz W [M][K], dw = dz^T x [N][K], dbias = the sum of dz
   over the rows, f32 [N].  z is not read (and may be NULL) for act NONE; it may
   be any [M][N] values.  Any of dx, dw, dbias may be NULL: not computed.  F16
   and BF16 round dz to the type before the two products (F16: to an infinity past
   65504), but not for M <= 8 with N <= 8192, nor where dz, dx or dw has at most
   4096 elements.  M = 0 gives zero dw and dbias.  `aligned` as above, of dy, x and w. */
BERT_API int64_t bert_amd_linear_backward_workspace(int32_t type, int32_t act, int64_t M, int32_t N, int32_t K,
                                                    int32_t aligned);
BERT_API int32_t bert_amd_linear_backward(int32_t device, int32_t type, int32_t act, int64_t M, int32_t N, int32_t K,
                                          const void *dy, int64_t lddy, const void *z, int64_t ldz, const void *x,
                                          int64_t ldx, const void *w, int64_t ldw, void *dx, int64_t lddx, void *dw,
                                          int64_t lddw, float *dbias, void *workspace, int64_t workspace_bytes,
                                          void *hip_stream);

/* Token rows: out[i] = scale * table[ids[i]], in f32, rounded once to out_type
   (F32, F16 or BF16).  An id outside [0, n_rows) gives a row of zeros (unlike
   the encoder's own gather, whose ids are tokens of a checked batch).
     table    : [n_rows][width] of table_type, F32, F16, BF16 or a GGUF's Q4_0 or
                Q4_1 rows (width a multiple of 32; a block's values as ggml's
                get_rows gives them), ld_table_bytes between rows
     out      : [n][width]
   n <= 2^30, width < 2^22. */
BERT_API int32_t bert_amd_lookup(int32_t device, int32_t table_type, int32_t out_type, int64_t n, int32_t n_rows,
                                 int32_t width, const void *table, int64_t ld_table_bytes, const int32_t *ids,
                                 float scale, void *out, int64_t ldo, void *hip_stream);

/* The table's gradient: dtable[v] = scale * (sum of dout[i] over the i with
   ids[i] = v), f32, in one fixed order of i; every row is written, unused ones
   as zero.  accumulate != 0 adds it to dtable instead and leaves unused rows
   untouched.  Ids outside [0, n_rows) and pad_id (-1: none) have no gradient.
     dout     : [n][width] of type F32, F16 or BF16; dtable: f32 [n_rows][width]
   n <= 2^28, n_rows <= 2^30, width < 2^20. */
BERT_API int64_t bert_amd_lookup_grad_workspace(int64_t n, int32_t n_rows, int32_t width);
BERT_API int32_t bert_amd_lookup_grad(int32_t device, int32_t type, int64_t n, int32_t n_rows, int32_t width,
                                      const void *dout, int64_t ldd, const int32_t *ids, float scale, int32_t pad_id,
                                      int32_t accumulate, float *dtable, int64_t ldt, void *workspace,
                                      int64_t workspace_bytes, void *hip_stream);

/* The word-embedding table of replica `slot` as bert_amd_lookup takes it (rows
   contiguous); it belongs to the context, until bert_free, and is read-only.  `type` is the
   file's row type, or F32 where the context keeps an f32 copy ("emb_raw" 0). */
BERT_API int32_t bert_amd_word_table(struct bert_ctx *ctx, int32_t slot, const void **table, int32_t *type,
                                     int32_t *n_rows, int32_t *width, int32_t *device);

/* One tensor of an AdamW step: n f32 weights p (updated), their gradient, and
   the moments (updated; all zero before step 1).  state_bits 32: m and v are
   f32 [n].  state_bits 8: codes, one byte each, [n], and the f32 scales
   m_scale, v_scale [(n + 255) / 256] of each 256 elements.  copy: n updated
   weights rounded to copy_type, or NULL. */
struct bert_amd_adamw_tensor {
    float *p;
    const void *grad;
    void *m, *v;
    float *m_scale, *v_scale;
    void *copy;
    int64_t n;
    double weight_decay;
};

/* One step over n_tensors tensors (a host array, not kept):
     m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2,
     p = p (1 - lr weight_decay)
         - lr / (1 - beta1^step) m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
   in f32.  g is grad (grad_type F32, F16 or BF16) times *grad_scale (one f32 in
   device memory; NULL: 1).  8-bit states store m and sqrt(v) as small floats,
   rounded up or down at random by `seed`, another one each step (unused with 32
   bits).  An infinity or NaN in g makes its weight and moments NaN, with 8-bit
   states the moments of its whole block of 256.  n <= 2^34; what is
   written must not overlap, nor a gradient lie in it (copies of the same
   gradient are fine).  Captured in a graph, step, lr and seed are those of the
   capture. */
BERT_API int32_t bert_amd_adamw(int32_t device, int32_t n_tensors, const struct bert_amd_adamw_tensor *tensors,
                                int32_t state_bits, int32_t grad_type, int32_t copy_type, double lr, double beta1,
                                double beta2, double eps, int64_t step, uint32_t seed, const float *grad_scale,
                                void *hip_stream);

/* 8-bit moments as f32 values: m_out, v_out [n] (either may be NULL). */
BERT_API int32_t bert_amd_adamw_moments(int32_t device, int64_t n, const void *m, const float *m_scale, const void *v,
                                        const float *v_scale, float *m_out, float *v_out, void *hip_stream);

BERT_API const char *bert_amd_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* BERT_AMD_H */
