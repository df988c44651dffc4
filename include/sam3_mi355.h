/*
 * sam3_mi355.h -- C-ABI of the MI355X (gfx950) backend for sam3.cpp's
 * quantized-matmul hot path.
 *
 * sam3.cpp builds ggml graphs and hands them to a backend
 * (sam3_graph_compute -> ggml_backend_graph_compute, sam3.cpp:1019-1030).
 * The nodes on the image-encoder hot path are MUL_MAT with F16/Q8_0/Q4_0/Q4_1
 * weights against F32 activations (sam3.cpp:3742,3783,3796,3799 for the SAM3
 * ViT; 4321,4349,4406,4451,4454 for SAM2 Hiera), FLASH_ATTN_EXT
 * (sam3.cpp:3778, 4399) and, for the explicit attention form, MUL_MAT(K,Q) /
 * SOFT_MAX / MUL_MAT(V^T,KQ) (sam3.cpp:8584-8589).  This header exposes one
 * entry point per such node, taking the ggml tensor layout fields (type, ne,
 * nb, data) so a ggml backend's graph_compute can forward node->src[i] and
 * the node itself unchanged.
 *
 * Conventions (ggml's): ne[0] is the contiguous dimension, nb[] are byte
 * strides, quantized rows are ne[0]/32 consecutive blocks.  All data pointers
 * are device pointers owned by the caller.  Calls enqueue work on the
 * context's HIP stream and return without waiting, like a backend's async
 * graph compute; mi355_synchronize() waits.  Nothing aborts: errors come back
 * as mi355_status values (the reference style, CLAUDE.md:62).
 */
#ifndef SAM3_MI355_H
#define SAM3_MI355_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* enum ggml_type ids used on this path (sam3.cpp:3246-3252). */
typedef enum {
    MI355_TYPE_F32 = 0,
    MI355_TYPE_F16 = 1,
    MI355_TYPE_Q4_0 = 2,
    MI355_TYPE_Q4_1 = 3,
    MI355_TYPE_Q8_0 = 8,
    MI355_TYPE_Q8_1 = 9,
} mi355_type;

/* enum ggml_status values, plus two refinements of FAILED. */
typedef enum {
    MI355_STATUS_INVALID_ARG = -4, /* shape/stride/pointer the op definition rejects */
    MI355_STATUS_UNSUPPORTED = -3, /* valid ggml op this backend does not implement */
    MI355_STATUS_ALLOC_FAILED = -2,
    MI355_STATUS_FAILED = -1,      /* a HIP runtime error */
    MI355_STATUS_SUCCESS = 0,
    MI355_STATUS_ABORTED = 1,
} mi355_status;

/* Activation-quantizer variant: ggml-cpu's from_float for Q8_0/Q8_1 exists as
 * the x86 SIMD routine (id = 127/amax, round half to even) and the scalar
 * _ref routine (id = 1/(amax/127), round half away).  mul_mat uses X86. */
typedef enum {
    MI355_ACT_X86 = 0,
    MI355_ACT_REF = 1,
} mi355_act_variant;

/* Version of this interface: 2 added the layout field of mi355_tensor (the
 * former padding word, which callers must now set to 0, e.g. by
 * zero-initializing the struct) and prepared weights.  A binding compiled
 * against one version checks mi355_abi_version() at load. */
#define MI355_ABI_VERSION 2
int mi355_abi_version(void);

/* The layout fields of a ggml_tensor (ggml.h struct ggml_tensor: type, ne,
 * nb, data).  data is a device pointer.  layout is MI355_LAYOUT_GGML (0, the
 * bytes ggml defines for type/ne/nb) except for a weight prepared by
 * mi355_weight_prepare (MI355_LAYOUT_INT8); any other value is rejected
 * (MI355_STATUS_INVALID_ARG) by every entry point. */
typedef enum {
    MI355_LAYOUT_GGML = 0,
    MI355_LAYOUT_INT8 = 1,
} mi355_layout;
typedef struct mi355_tensor {
    int32_t type;
    int32_t layout;
    int64_t ne[4];
    int64_t nb[4];
    void* data;
} mi355_tensor;

typedef struct mi355_context mi355_context;

/* Backend init: replaces ggml_backend_metal_init()/ggml_backend_cpu_init()
 * at sam3.cpp:3278-3292.  stream is a hipStream_t owned by the caller, or
 * NULL for the device's default (null) stream. */
mi355_status mi355_context_create(int device, void* stream, mi355_context** out);
void mi355_context_free(mi355_context* ctx);
/* Blocks until all work enqueued on the context's stream is done
 * (ggml_backend_synchronize). */
mi355_status mi355_synchronize(mi355_context* ctx);
/* ggml_status_to_string, used by sam3_graph_compute (sam3.cpp:1025-1027). */
const char* mi355_status_to_string(mi355_status status);
/* Text of the last error seen by this context ("" if none). */
const char* mi355_last_error(const mi355_context* ctx);
/* Reserve the context's scratch workspace (bytes); mul_mat grows it on
 * demand otherwise.  Replaces ggml-cpu's per-graph wdata buffer. */
mi355_status mi355_reserve_workspace(mi355_context* ctx, size_t bytes);
/* Workspace bytes mul_mat needs for these operands: the most over the
 * MUL_MAT routes (mi355_context_set_mmq_kernel). */
size_t mi355_mul_mat_workspace_size(const mi355_tensor* src0, const mi355_tensor* src1);

/* ---- Device buffers (the ggml-backend buffer calls around a graph) ---------
 * A buffer is one device allocation on the context's device, owned by the
 * caller until mi355_buffer_free.  It stands in for
 * ggml_backend_alloc_ctx_tensors (sam3.cpp:3320, the model's weights) and for
 * the graph allocator's buffer (ggml_gallocr_alloc_graph, sam3.cpp:6101-6115);
 * mi355_buffer_place puts a tensor at an offset in it (ggml_tallocr_alloc),
 * offsets being multiples of mi355_buffer_alignment().  The byte layouts are
 * ggml's, so tensor bytes read from a .ggml file or written by ggml-cpu are
 * used as they are. */
typedef struct mi355_buffer mi355_buffer;
size_t mi355_buffer_alignment(void);
mi355_status mi355_buffer_alloc(mi355_context* ctx, size_t size, mi355_buffer** out);
/* ggml_backend_buffer_free: waits for the device's work before freeing. */
void mi355_buffer_free(mi355_buffer* buf);
void* mi355_buffer_base(const mi355_buffer* buf);
size_t mi355_buffer_size(const mi355_buffer* buf);
/* Sets t->data = base + offset after checking that ggml_nbytes(t) bytes fit. */
mi355_status mi355_buffer_place(const mi355_buffer* buf, size_t offset, mi355_tensor* t);
/* ggml_nbytes of t's layout (0 for an empty tensor or an unknown type); for
 * a prepared weight (MI355_LAYOUT_INT8) the bytes of its prepared form. */
size_t mi355_tensor_nbytes(const mi355_tensor* t);
/* ggml_backend_buffer_clear. */
mi355_status mi355_buffer_clear(mi355_context* ctx, mi355_buffer* buf, uint8_t value);
/* ggml_backend_tensor_set / _get / _memset (sam3.cpp:3156-3179, 6117): bytes
 * [offset, offset + size) of the tensor's data, bounds-checked against
 * ggml_nbytes(t); ordered after the work already on the context's stream, and
 * returning when the host side is done (set: data may be reused; get: data
 * has arrived). */
mi355_status mi355_tensor_set(mi355_context* ctx, const mi355_tensor* t, const void* data, size_t offset, size_t size);
mi355_status mi355_tensor_get(mi355_context* ctx, const mi355_tensor* t, void* data, size_t offset, size_t size);
mi355_status mi355_tensor_memset(mi355_context* ctx, const mi355_tensor* t, uint8_t value, size_t offset, size_t size);

/* ---- MUL_MAT (ggml_mul_mat, sam3.cpp:3742,3783,3796,3799) ----------------
 * dst[N, M, b2, b3] = src0[K, N, a2, a3]^T . src1[K, M, b2, b3], with
 * b2 % a2 == 0, b3 % a3 == 0 (src0 broadcast by the ratio).
 * src0: F16, Q8_0, Q4_0 or Q4_1, rows contiguous (nb[0] = type size).
 * src1: F32 (any strides) or, with F16 src0, F16.  dst: F32, nb[0] = 4.
 * src1 may also hold the rows already quantized (mi355_rms_norm,
 * mi355_quantize_rows): Q8_0 with Q8_0 / Q4_0 weights, Q8_1 with Q4_1 ones, in
 * 2-D products; the same bits as with the finite F32 rows they were made of,
 * always by the int8 kernel (up to about 64 rows F32 rows have faster ways).
 * Q8_0/Q4_0 quantize src1 to Q8_0 and Q4_1 to Q8_1 (x86 variant) exactly as
 * ggml-cpu's from_float, then combine exact int32 block dots in fp32.  F16
 * converts src1 to F16 (round to nearest even) and accumulates in fp32. */
/* The mi355_supports_* queries are ggml_backend_supports_op for each node
 * kind: 1 when the entry point accepts these operands (no GPU work, no
 * context), 0 otherwise.  sam3.cpp runs each graph on a single backend
 * (sam3.cpp:3278-3292), so a graph builder checks every node before
 * choosing this one. */
int mi355_supports_mul_mat(const mi355_tensor* src0, const mi355_tensor* src1, const mi355_tensor* dst);
mi355_status mi355_mul_mat(mi355_context* ctx, const mi355_tensor* src0, const mi355_tensor* src1,
                           const mi355_tensor* dst);

/* ---- Prepared weights (the counterpart of ggml's "extra" buffer types, such
 * as ggml-cpu's, which repack Q4_0 weights into an interleaved layout when
 * ggml_backend_tensor_set uploads them; sam3.cpp uploads each weight once,
 * sam3.cpp:3156-3179).  A 2-D Q8_0 / Q4_0 / Q4_1 weight is repacked once into
 * the int8 MUL_MAT layout (quants as int8 rows, block scales in separate
 * arrays), so MUL_MATs with it skip the per-call repack.
 * mi355_weight_prepared_nbytes: bytes of the prepared form of w (0: w is not
 *   a 2-D Q8_0 / Q4_0 / Q4_1 weight with K % 32 == 0).
 * mi355_weight_prepare: repacks w (ggml layout, device data) into dst
 *   (256-byte aligned, dst_size >= the prepared bytes, not overlapping w) on
 *   the context's stream, and describes the result in *out: w's type and ne,
 *   layout MI355_LAYOUT_INT8, nb of a contiguous ggml tensor, data = dst.
 *   mi355_mul_mat and mi355_mul_mat_noalloc take *out as src0 and give the
 *   same bits as with w; the buffer and tensor calls copy it as bytes; every
 *   other op rejects it (MI355_STATUS_INVALID_ARG). */
size_t mi355_weight_prepared_nbytes(const mi355_tensor* w);
mi355_status mi355_weight_prepare(mi355_context* ctx, const mi355_tensor* w, void* dst, size_t dst_size,
                                  mi355_tensor* out);

/* ---- MUL_MAT without allocation (no counterpart in the reference; for
 * callers that cannot allocate device memory: code under HIP graph capture,
 * tight serving loops, harnesses that forbid hipMalloc) ----------------------
 * The same operation, checks and kernels as mi355_mul_mat, with the same
 * results.  Its scratch (the converted src1, split-K partial sums, the
 * 4-byte-pitch weight copy) lives in a fixed device array of
 * MI355_NOALLOC_SCRATCH_BYTES per GPU, held from library load until the
 * process ends, instead of the context's workspace; the call allocates and
 * frees nothing and records no timing events.  Operands whose plan on the
 * context's current route (mi355_context_set_mmq_kernel; under MI355_MMQ_AUTO
 * the int8 one, MI355_MMQ_F16 for ggml-layout Q4_1) needs more scratch than
 * that are rejected with MI355_STATUS_UNSUPPORTED, also where AUTO prefers a
 * route that needs less; where it prefers one that needs more than the array
 * holds, the call takes the former.  F32 weights need no scratch.  The most
 * any route needs, mi355_mul_mat_workspace_size, bounds it from above.  Every call on
 * one GPU uses that GPU's one array: calls through one context serialize on
 * its stream, and a call through another context first makes its stream
 * wait on an event the device's previous call recorded (each context creates
 * its event when it is created).  Under stream capture no event is waited on
 * or recorded: the caller orders the launches of captured graphs.  Host
 * threads sharing one context must serialize their calls. */
#define MI355_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)
mi355_status mi355_mul_mat_noalloc(mi355_context* ctx, const mi355_tensor* src0, const mi355_tensor* src1,
                                   const mi355_tensor* dst);

/* ---- activation quantize (ggml-cpu type_traits[vec_dot_type].from_float,
 * the src1 conversion step of MUL_MAT; quantize_row_q8_0/q8_1, F16 convert).
 * Converts every row (ne[0] elements, rows over ne[1..3]) of the F32 tensor
 * src into dst as contiguous ggml rows of type (Q8_0, Q8_1 or F16): row r at
 * dst + r*row_size.  variant selects the from_float flavour. */
mi355_status mi355_quantize_rows(mi355_context* ctx, int type, int variant, const mi355_tensor* src, void* dst);

/* ---- weight quantize (ggml_quantize_chunk(type, src, dst, 0, nrows,
 * n_per_row, NULL), examples/quantize.cpp:244-245: the _ref row quantizers
 * quantize_row_q8_0_ref / q4_0_ref / q4_1_ref).  Every row of the F32 or F16
 * tensor src (F16 widened to F32 exactly first, as sam3_quantize_model does
 * at quantize.cpp:227-237) -> dst as contiguous ggml rows of type (Q8_0, Q4_0
 * or Q4_1), row r at dst + r*row_size; dst 2-byte aligned. */
mi355_status mi355_quantize_weights(mi355_context* ctx, int type, const mi355_tensor* src, void* dst);

/* ---- Block-dot inspection (no ggml counterpart; test hook) ---------------
 * isums[b2][b3..][m][n][blk] = exact int32 block dots of the quantized
 * operands that mi355_mul_mat would combine, computed by the same MFMA
 * kernel.  src0 Q8_0/Q4_0/Q4_1; isums is a device buffer of
 * M*N*(K/32)*b2*b3 int32. */
mi355_status mi355_mul_mat_block_dots(mi355_context* ctx, const mi355_tensor* src0, const mi355_tensor* src1,
                                      int32_t* isums);

/* ---- SOFT_MAX (ggml_soft_max_ext(a, NULL, scale, 0.0f), sam3.cpp:8586) ----
 * Row-wise softmax of scale*src over ne[0]; F32 in/out, any row strides. */
int mi355_supports_soft_max_ext(const mi355_tensor* src, const mi355_tensor* mask, float max_bias,
                                const mi355_tensor* dst);
mi355_status mi355_soft_max_ext(mi355_context* ctx, const mi355_tensor* src, const mi355_tensor* mask,
                                float scale, float max_bias, const mi355_tensor* dst);

/* ---- FLASH_ATTN_EXT (ggml_flash_attn_ext(q,k,v,NULL,scale,0,0),
 * sam3.cpp:3778 ViT, 4399 Hiera) --------------------------------------------
 * q [D, n_q, n_head, B], k [D, n_kv, n_head_kv, B], v [Dv, n_kv, n_head_kv, B]
 * (F32 or F16, any strides: the ViT passes V as a permuted view,
 * sam3.cpp:3767); dst [Dv, n_head, n_q, B] F32 contiguous.  D = Dv in
 * {64, 96, 128}.  mask must be NULL, max_bias and logit_softcap 0. */
int mi355_supports_flash_attn_ext(const mi355_tensor* q, const mi355_tensor* k, const mi355_tensor* v,
                                  const mi355_tensor* mask, float max_bias, float logit_softcap,
                                  const mi355_tensor* dst);
mi355_status mi355_flash_attn_ext(mi355_context* ctx, const mi355_tensor* q, const mi355_tensor* k,
                                  const mi355_tensor* v, const mi355_tensor* mask, float scale, float max_bias,
                                  float logit_softcap, const mi355_tensor* dst);

/* ---- Transformer layers around the quantized products ------------------------
 * The nodes between the MUL_MATs of a layer that keeps its tokens in a cache: a
 * decoder, or the memory a video model attends to.  The reference runs such
 * layers on ggml's general backends (its text encoder, sam3.cpp:3928-4069, and
 * the tracker's memory attention, sam3.cpp:9062-9660); these entry points have
 * ggml's tensor layouts, with device pointers for the int32 operands. */

/* ggml_add, ggml_rms_norm, ggml_mul and the next MUL_MAT's from_float in one
 * pass over the rows: h = x + add (add NULL: h = x), sum = h (sum NULL: not
 * kept), dst = h / sqrt(mean(h^2) + eps) * w (w device F32 [ne0], NULL: no
 * weight).  x, add and sum: F32 or F16, the same type and ne; dst: F32, F16,
 * Q8_0 or Q8_1 (the x86 from_float, bit for bit mi355_quantize_rows of the F32
 * dst; a row with a NaN has NaN scales), the same ne.
 * Rows of ne0 <= 32768 contiguous elements, any row strides; ne0 % 32 == 0 for
 * Q8_0 and Q8_1.  h and every later step are fp32 as ggml's nodes are (the sum
 * of squares in double); sum and F16 outputs round once, and the norm is
 * h's before that rounding.  sum may be x or add, and dst x, add or sum, as
 * the same tensor; any other overlap is not allowed. */
int mi355_supports_rms_norm(const mi355_tensor* x, const mi355_tensor* add, const mi355_tensor* sum,
                            const mi355_tensor* dst);
mi355_status mi355_rms_norm(mi355_context* ctx, const mi355_tensor* x, const mi355_tensor* add, const float* w,
                            float eps, const mi355_tensor* sum, const mi355_tensor* dst);

/* ggml's to_float, the counterpart of mi355_quantize_rows: contiguous ggml rows
 * src of type (Q8_0, Q8_1, Q4_0 or Q4_1) -> every row of the F32 or F16 tensor
 * dst (nb[0] contiguous, any row strides).  F16 rounds the F32 value once. */
mi355_status mi355_dequantize_rows(mi355_context* ctx, int type, const void* src, const mi355_tensor* dst);

/* Rotary positions over one to four axes (ggml_rope_multi; sam3_apply_rope's
 * axial rotation is two axes with restart).  src, dst [ne0, n_head, n_tokens,
 * batch], F32 or F16, the same type and ne, rows contiguous, any other strides;
 * dst may be src.  The first n_dims elements of a head turn in pairs, the others
 * are copied.  pos: device int32 [axes][batch][n_tokens], axes being the axes up
 * to the last with pairs.  Pair i turns by
 *   pos[axis(i)] * freq_scale * freq_base ^ (-e / size),
 * restart 0: e = i, size = n_dims / 2 (the axes share the frequencies out);
 * restart 1: e = i's place among its axis's pairs, size = sections[axis].
 * sections: pairs of each axis, n_dims / 2 in all; MI355_ROPE_CONSECUTIVE: the
 * first sections[0] pairs have axis 0, and so on; MI355_ROPE_INTERLEAVED (three
 * axes): pair i has axis i % 3 = a for a = 1, 2 while i < 3 sections[a], and axis 0
 * otherwise.  Angles are taken modulo a turn in 64-bit fixed point: at the ends of
 * int32 a position's is good to 2^-30 of a turn (freq_scale up to 2 pi and
 * freq_base away from one), below fp32's own step.  inverse 1 turns back (the
 * gradient). */
typedef enum { MI355_ROPE_ADJACENT = 0, MI355_ROPE_HALVES = 1 } mi355_rope_pairs; /* (2i, 2i+1); (i, i + n_dims/2) */
typedef enum { MI355_ROPE_CONSECUTIVE = 0, MI355_ROPE_INTERLEAVED = 1 } mi355_rope_order;
typedef struct mi355_rope_params {
    int32_t n_dims; /* even, 2 .. 256, at most ne0 */
    int32_t pairs;  /* mi355_rope_pairs */
    int32_t order;  /* mi355_rope_order */
    int32_t restart;
    int32_t inverse;
    int32_t sections[4];
    float freq_base; /* > 0 */
    float freq_scale;
} mi355_rope_params;
int mi355_supports_rope_multi(const mi355_tensor* src, const mi355_rope_params* p, const mi355_tensor* dst);
mi355_status mi355_rope_multi(mi355_context* ctx, const mi355_tensor* src, const int32_t* pos,
                              const mi355_rope_params* p, const mi355_tensor* dst);

/* A cache of keys and values in 8 bits, in blocks of block_tokens tokens that
 * sequences hold through a table.  Block b, head h is block_tokens rows of
 * head_dim bytes at k + ((b * n_head_kv + h) * block_tokens) * head_dim (v alike),
 * with one F32 scale at k_scale[b * n_head_kv + h]: byte u stands for
 * (u - 128) * scale.  All device memory of the caller's, of any initial content;
 * k and v 16-byte aligned.  Scales are not negative. */
typedef struct mi355_kv_cache {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    int32_t n_blocks;
    int32_t n_head_kv;
    int32_t block_tokens; /* 16, 32, 64 or 128 */
    int32_t head_dim;     /* 64, 96 or 128 */
} mi355_kv_cache;
/* n_seq sequences in it: token t of sequence s is row t % block_tokens of block
 * table[s * max_blocks + t / block_tokens]; n_kv[s] is its length, the tokens of
 * the call included (taken as 0 below 0, and as max_blocks * block_tokens above
 * that).  Device int32.  A block id outside 0 .. n_blocks - 1 is never followed:
 * its tokens are not written, not read and not attended to. */
typedef struct mi355_kv_seqs {
    const int32_t* table;
    const int32_t* n_kv;
    int32_t n_seq;
    int32_t max_blocks;
} mi355_kv_seqs;

/* Writes the last n_new[s] tokens of every sequence s (device int32; NULL: all
 * n_tokens): row i of k and v [head_dim, n_tokens, n_head_kv, n_seq] (F32 or
 * F16, the same type, rows contiguous, any other strides) becomes token
 * n_kv[s] - n_new[s] + i (none before token 0); rows from n_new[s] on are not
 * read.  Per block and
 * head, with top the largest magnitude among its new elements:
 *   scale = top / 127, or max(scale, top / 127) where the block keeps tokens
 *           before the first new one;
 *   byte  = 128 + x / scale rounded to nearest, ties to even, within 1 .. 255
 *           (scale 0: 128); kept tokens whose scale grew are rounded anew from
 *           the values they stood for.
 * A NaN or infinity makes its block's scale NaN or infinite and the block's
 * values with it, until it is written from its first row again.  Among the blocks
 * that one call writes, of all sequences, each may stand once. */
mi355_status mi355_kv_cache_write(mi355_context* ctx, const mi355_kv_cache* cache, const mi355_kv_seqs* seqs,
                                  const mi355_tensor* k, const mi355_tensor* v, const int32_t* n_new);
/* Reads tokens back as (byte - 128) * scale in fp32, F16 rounded once: row i of
 * k and v [head_dim, n_tokens, n_head_kv, n_seq] (F32 or F16, as above; either may
 * be NULL) takes token pos[s * n_tokens + i] of sequence s (device int32; NULL:
 * token i).  Rows whose token is outside 0 .. n_kv[s] - 1 are left as they are. */
mi355_status mi355_kv_cache_read(mi355_context* ctx, const mi355_kv_cache* cache, const mi355_kv_seqs* seqs,
                                 const int32_t* pos, const mi355_tensor* k, const mi355_tensor* v);
/* FLASH_ATTN_EXT over the cache.  q [head_dim, n_q, n_head, n_seq] and dst
 * [head_dim, n_head, n_q, n_seq], each F32 or F16, rows contiguous, any other
 * strides; n_head a multiple of n_head_kv (query head h reads head
 * h / (n_head / n_head_kv)).  Sequence s has n_q[s] queries (device int32; NULL: all
 * n_q); rows of dst from n_q[s] on are left as they are.  Query i stands at position
 * p = n_kv[s] - n_q[s] + i and attends to tokens t < n_kv[s], with causal t <= p,
 * and with window > 0 t > p - window; a query that attends to nothing gives zeros,
 * one that sees a token of a block whose scales are not both finite gives NaN.
 * Scores, softmax and outputs accumulate in fp32.  An F16 q enters the matrix
 * products as it is and an F32 q as two halves (22 bits); the probabilities enter
 * as F16 for an F16 dst and as two halves for an F32 dst, each times its block's
 * value scale; the fp32 sum of an F16 dst is of these halves, and of the unrounded
 * probabilities where a block's scale is far below others'.  The cache's bytes
 * are exact in F16.  dst overlaps nothing that the call reads.
 * mi355_kv_cache_attn_workspace_size: bytes of the context's workspace that these
 * sizes need (0: none); a call grows it on demand, except under stream capture,
 * where it has to be there (mi355_reserve_workspace).  Graphs captured from one context
 * share its workspace: replay them one after another. */
int mi355_supports_kv_cache_attn(const mi355_kv_cache* cache, const mi355_kv_seqs* seqs, const mi355_tensor* q,
                                 const mi355_tensor* dst);
size_t mi355_kv_cache_attn_workspace_size(const mi355_context* ctx, const mi355_kv_cache* cache,
                                          const mi355_kv_seqs* seqs, const mi355_tensor* q, int32_t window);
mi355_status mi355_kv_cache_attn(mi355_context* ctx, const mi355_kv_cache* cache, const mi355_kv_seqs* seqs,
                                 const mi355_tensor* q, const int32_t* n_q, float scale, int causal, int32_t window,
                                 const mi355_tensor* dst);

/* ggml_rms_norm and ggml_mul of every head of the queries and of the keys, and
 * ggml_rope_multi of both, in one pass:
 *   dst = turned(x / sqrt(mean over ne0 of x^2 + eps) * w)
 * q [ne0, n_head, n_tokens, batch] and k [ne0, n_head_kv, n_tokens, batch] (either
 * may be NULL, with its output), F32 or F16, both the same type; q_dst and k_dst of the
 * same ne, F32 or F16, both the same type; rows of ne0 <= 256 contiguous elements, any
 * other strides, so that q and k may be parts of one product's rows.  q_w, k_w:
 * device F32 [ne0] or NULL.  pos and p as mi355_rope_multi's; elements past n_dims are
 * normed and not turned.  Every step is fp32, F16 outputs round once.  An output may be
 * its source, as the same tensor; any other overlap is not allowed. */
int mi355_supports_qk_norm_rope(const mi355_tensor* q, const mi355_tensor* k, const mi355_rope_params* p,
                                const mi355_tensor* q_dst, const mi355_tensor* k_dst);
mi355_status mi355_qk_norm_rope(mi355_context* ctx, const mi355_tensor* q, const mi355_tensor* k, const float* q_w,
                                const float* k_w, float eps, const int32_t* pos, const mi355_rope_params* p,
                                const mi355_tensor* q_dst, const mi355_tensor* k_dst);

/* A cache of keys and values in 4 bits, in blocks as mi355_kv_cache's, with an fp16
 * scale d for each 32 elements of a token and head: nibble u stands for (u - 8) d.
 * Row t of block b, head h is head_dim / 2 bytes at k + ((b * n_head_kv + h) *
 * block_tokens + t) * head_dim / 2 (v alike): 32-bit words of eight elements, element
 * 2 i in nibble i (bits 4 i on) and element 2 i + 1 in nibble i + 4.  Scales, with
 * G = head_dim / 32: k_scale[((b * n_head_kv + h) * block_tokens + t) * G + group] and
 * v_scale[((b * n_head_kv + h) * G + group) * block_tokens + t].  A scale has eight
 * significant bits and a magnitude up to 8160, so that every value is an fp16 number, or
 * is NaN, and then all scales of that token and head are.  All device memory of the
 * caller's, of any initial content where no sequence has tokens; k and v 16-byte aligned, scales 8-byte. */
typedef struct mi355_kv_cache4 {
    uint8_t* k;
    uint8_t* v;
    uint16_t* k_scale;
    uint16_t* v_scale;
    int32_t n_blocks;
    int32_t n_head_kv;
    int32_t block_tokens; /* 16, 32, 64 or 128 */
    int32_t head_dim;     /* 64, 96 or 128 */
} mi355_kv_cache4;

/* As mi355_kv_cache_write.  Of each 32 elements of a token and head, with ext the one
 * farthest from zero (the positive one of two):
 *   d = -ext / 8 rounded to eight significant bits, then to fp16 (to nearest, ties to even; one zero);
 *   nibble = 8 + x / d rounded to nearest, ties to even, within 0 .. 15 (d 0: 8).
 * A NaN, an infinity or a d beyond 8160 (magnitudes of 65408 and more) makes all scales of its token
 * and head NaN, keys' and values'.  Tokens do not touch one another.  Among the tokens that
 * one call writes, of all sequences, each place of the cache may stand once. */
mi355_status mi355_kv_cache4_write(mi355_context* ctx, const mi355_kv_cache4* cache, const mi355_kv_seqs* seqs,
                                   const mi355_tensor* k, const mi355_tensor* v, const int32_t* n_new);
/* As mi355_kv_cache_read: (nibble - 8) * d, exact in F32 and in F16. */
mi355_status mi355_kv_cache4_read(mi355_context* ctx, const mi355_kv_cache4* cache, const mi355_kv_seqs* seqs,
                                  const int32_t* pos, const mi355_tensor* k, const mi355_tensor* v);
/* As mi355_kv_cache_attn, over the cache's exact values: a query that attends to
 * nothing gives zeros, one that sees a token with NaN scales NaN.  lse (device F32
 * [n_seq][n_q][n_head], or NULL) takes log sum exp(scale q . k) over the tokens that the
 * query sees, -inf where there is none; rows from n_q[s] on are left as they are.
 * Scores are fp32, and hold a fraction up to magnitudes of 2^23: the softmax of larger ones means nothing.
 * Queries and probabilities enter the products as there; lse's fp32 sum is of the unrounded probabilities.
 * mi355_kv_cache4_attn_workspace_size as mi355_kv_cache_attn_workspace_size. */
int mi355_supports_kv_cache4_attn(const mi355_kv_cache4* cache, const mi355_kv_seqs* seqs, const mi355_tensor* q,
                                  const mi355_tensor* dst);
size_t mi355_kv_cache4_attn_workspace_size(const mi355_context* ctx, const mi355_kv_cache4* cache,
                                           const mi355_kv_seqs* seqs, const mi355_tensor* q, int32_t window);
mi355_status mi355_kv_cache4_attn(mi355_context* ctx, const mi355_kv_cache4* cache, const mi355_kv_seqs* seqs,
                                  const mi355_tensor* q, const int32_t* n_q, float scale, int causal, int32_t window,
                                  const mi355_tensor* dst, float* lse);
/* What an attention looked at: adds to sums[s][h][t] (device F32 [n_seq][n_head_kv]
 * [max_blocks * block_tokens]) the softmax weight of token t, exp(scale q . k - lse),
 * summed over the queries that see it and the heads of key head h's group.  lse as
 * mi355_kv_cache4_attn gave it for the same queries, scale, causal and window.  Places of
 * tokens that no query sees are left as they are.  Queries enter as the attention's; weights and sums are fp32, those
 * of every 1024 rows (queries and heads) by themselves first.  The same call gives the same bits.
 * mi355_kv_cache4_weights_workspace_size as the attention's. */
size_t mi355_kv_cache4_weights_workspace_size(const mi355_context* ctx, const mi355_kv_cache4* cache,
                                              const mi355_kv_seqs* seqs, const mi355_tensor* q, int32_t window);
mi355_status mi355_kv_cache4_weights(mi355_context* ctx, const mi355_kv_cache4* cache, const mi355_kv_seqs* seqs,
                                     const mi355_tensor* q, const int32_t* n_q, const float* lse, float scale,
                                     int causal, int32_t window, float* sums);
/* Brings sequences down to n_keep[s] tokens (device int32, within 0 .. max_keep; NULL: max_keep) where they
 * have more: each head keeps, of its n = n_kv[s] tokens, the last `recent`, the
 * first `first` (as many as n_keep[s] leaves), and of the others those with the largest
 * sums, the lower token of equal ones (a NaN is the smallest number; tokens of blocks that are not
 * there come last).  Kept tokens move together in place, in their order, from place 0 on;
 * keys keep the positions that they were turned by.  Places from n_out[s] on are left as they are.  Outputs:
 *   n_out[s] = min(n, n_keep[s]), the sequence's length from now on;
 *   kept[s][h][j] (int32 [n_seq][n_head_kv][max_keep]): where token j stood, the others left as they are;
 *   sums_out[s][h][..] (as sums): the kept tokens' sums, then zeros up to n, the others left as they are.
 * A kept token whose block is not there leaves a NaN key in its place; one that moves to such a block is
 * lost.  No output may overlap an input.  Sequences share no blocks. */
mi355_status mi355_kv_cache4_evict(mi355_context* ctx, const mi355_kv_cache4* cache, const mi355_kv_seqs* seqs,
                                   const float* sums, const int32_t* n_keep, int32_t max_keep, int32_t first,
                                   int32_t recent, float* sums_out, int32_t* kept, int32_t* n_out);

/* ---- SAM3 ViT image encoder ----------------------------------------------
 * The graph sam3_build_vit_graph builds (sam3.cpp:3836-3853) run on this
 * backend: the prefix (patch embedding, tiled pos_embed, ln_pre;
 * sam3.cpp:3810-3834) and sam3_vit_block_forward (sam3.cpp:3714-3805), with
 * the memory-bound ggml nodes around each MUL_MAT / FLASH_ATTN_EXT fused
 * into single passes that keep ggml's per-node fp32 rounding.
 * Activations x are device F32 [grid*grid][E] in image token order
 * (ggml [E, W, H, 1]).  All weight pointers are device pointers. */
typedef struct mi355_vit_hparams {
    int32_t embed_dim;   /* E (1024) */
    int32_t num_heads;   /* 16; head size E / num_heads in {64, 96, 128} */
    int32_t mlp_dim;     /* 4736 */
    int32_t window_size; /* 24 */
    int32_t grid;        /* tokens per image side: img_size / patch_size (72) */
    int32_t patch_size;  /* 14 */
    int32_t pos_grid;    /* side of pos_embed at pretrained resolution (24), tiled over the grid */
    float eps;           /* LayerNorm eps (1e-5) */
} mi355_vit_hparams;

typedef struct mi355_vit_block {
    /* linear weights [in, out] (ggml ne), F16 / Q8_0 / Q4_0 / Q4_1 (or F32) */
    mi355_tensor qkv_w, proj_w, fc1_w, fc2_w;
    const float* norm1_w;
    const float* norm1_b;
    const float* qkv_b;
    const float* proj_b;
    const float* norm2_w;
    const float* norm2_b;
    const float* fc1_b;
    const float* fc2_b;
    const float* freqs_cis; /* [N][head_dim/2][2] (cos, sin); N = window_size^2, or grid^2 if global; NULL: no RoPE */
    int32_t is_global;      /* 0: attention inside window_size^2 windows (ggml_win_part) */
} mi355_vit_block;

/* Device bytes the encoder keeps for its activations (allocated on first use). */
size_t mi355_vit_workspace_size(const mi355_vit_hparams* hp);
/* x = ln_pre(conv2d_p(image) + tile(pos_embed)): image device F32 [3][H][W]
 * with H = W = grid * patch_size; patch_w [P, P, 3, E] F32 or F16. */
mi355_status mi355_vit_prefix(mi355_context* ctx, const mi355_vit_hparams* hp, const float* image,
                              const mi355_tensor* patch_w, const float* pos_embed, const float* ln_pre_w,
                              const float* ln_pre_b, float* x);
/* x = sam3_vit_block_forward(x) in place. */
mi355_status mi355_vit_block_forward(mi355_context* ctx, const mi355_vit_hparams* hp, const mi355_vit_block* blk,
                                     float* x);
/* The whole encoder: prefix, then n_blocks blocks; x: [grid*grid][E] output. */
mi355_status mi355_vit_encode(mi355_context* ctx, const mi355_vit_hparams* hp, const float* image,
                              const mi355_tensor* patch_w, const float* pos_embed, const float* ln_pre_w,
                              const float* ln_pre_b, const mi355_vit_block* blocks, int n_blocks, float* x);

/* The fused node groups the encoder runs, for use by other graph builders
 * and for testing each against ggml's node sequence:
 * - layer_norm: y[row(r)] = ggml_add(ggml_mul(ggml_norm(x[r] (+ add[r']), eps), w), b)
 *   (sam3_layer_norm, sam3.cpp:1041-1051); add (optional) is added first,
 *   row r' = r, or (y%add_grid)*add_grid + x%add_grid when add_grid > 0
 *   (ggml_repeat of pos_embed, sam3.cpp:3820-3826); row(r) is r, or its
 *   ggml_win_part row when window > 0 (sam3.cpp:3734).  w, b may be NULL. */
mi355_status mi355_vit_layer_norm(mi355_context* ctx, const float* x, const float* add, int add_grid, const float* w,
                                  const float* b, float* y, int64_t rows, int E, int grid, int window, float eps);
/* qkv [M][3E] (+ bias) -> Q, K (RoPE applied, sam3_apply_rope) and V as
 * fp16 [M/N][NH][N][HD] (the FLASH_ATTN_EXT operand layout of
 * sam3.cpp:3742-3778); rope [N][HD/2][2] or NULL. */
mi355_status mi355_vit_qkv_rope(mi355_context* ctx, const float* qkv, const float* bias, const float* rope, void* q,
                                void* k, void* v, int64_t M, int N, int n_heads, int head_dim);
/* x[r] = x[r] + (p[row(r)] + b): proj bias, ggml_win_unpart (window > 0) and
 * the residual add (sam3.cpp:3783-3791). */
mi355_status mi355_vit_proj_residual(mi355_context* ctx, float* x, const float* p, const float* b, int64_t rows, int E,
                                     int grid, int window);
/* h = ggml_gelu_erf(h + b) over rows of n (sam3.cpp:3796-3797). */
mi355_status mi355_vit_bias_gelu(mi355_context* ctx, float* h, const float* b, int64_t rows, int n);
/* x = x + (f + b) over rows of n (sam3.cpp:3799-3802). */
mi355_status mi355_vit_bias_residual(mi355_context* ctx, float* x, const float* f, const float* b, int64_t rows, int n);

/* ---- SAM2 Hiera image encoder ---------------------------------------------
 * sam2_build_hiera_graph (sam3.cpp:4466-4535) on this backend: patch
 * embedding (conv 7x7, stride 4, pad 3, + bias) + pos_embed, then the blocks
 * of sam2_hiera_block_forward (sam3.cpp:4299-4461) with the per-block
 * metadata of sam2_precompute_hiera_metadata (sam3.cpp:1680-1746).
 * Activations are device F32 [S*S][C] in image token order (ggml [C, S, S]). */
typedef struct mi355_hiera_hparams {
    int32_t img_size;       /* 1024 */
    int32_t embed_dim;      /* 96 for Hiera-tiny */
    int32_t num_heads;      /* 1 */
    int32_t stages[4];      /* blocks per stage {1, 2, 7, 2} */
    int32_t q_pool;         /* stage transitions with Q pooling (3) */
    int32_t window_spec[4]; /* {8, 4, 14, 7} */
    int32_t global_idx[8];  /* blocks with global attention {5, 7, 9} */
    int32_t n_global;
    float eps;              /* LayerNorm eps (1e-6) */
} mi355_hiera_hparams;

typedef struct mi355_hiera_block {
    mi355_tensor qkv_w, proj_w, fc1_w, fc2_w;
    mi355_tensor dim_proj_w; /* data NULL for blocks that keep their width */
    const float* norm1_w;
    const float* norm1_b;
    const float* qkv_b;
    const float* proj_b;
    const float* norm2_w;
    const float* norm2_b;
    const float* fc1_b;
    const float* fc2_b;
    const float* dim_proj_b;
} mi355_hiera_block;

/* Per-block metadata as the reference derives it: width in/out, heads,
 * window size (0 = global) and Q pooling. */
typedef struct mi355_hiera_block_info {
    int32_t dim_in, dim_out, num_heads, window_size, q_stride, stage;
} mi355_hiera_block_info;
int mi355_hiera_n_blocks(const mi355_hiera_hparams* hp);
mi355_status mi355_hiera_block_info_get(const mi355_hiera_hparams* hp, int block_index, mi355_hiera_block_info* out);
/* Device bytes the encoder keeps for its activations (allocated on first use). */
size_t mi355_hiera_workspace_size(const mi355_hiera_hparams* hp);
/* One block: x [S*S][dim_in] -> x_out [S'*S'][dim_out], S' = S/2 with Q pooling.
 * x_out must not overlap x. */
mi355_status mi355_hiera_block_forward(mi355_context* ctx, const mi355_hiera_hparams* hp, int block_index,
                                       const mi355_hiera_block* blk, const float* x, int spatial, float* x_out);
/* x = conv2d(image, patch_w, stride 4, pad 3) + patch_b + pos_embed, the patch
 * embedding mi355_hiera_encode starts from (sam3.cpp:4473-4494: ggml_conv_2d =
 * im2col + F32 mul_mat, + bias, + pos_embed): image device F32 [3][img][img],
 * patch_w [7, 7, 3, E] F32 or F16, patch_b [E], pos_embed and x [S0*S0][E]
 * token-major (S0 = img/4). */
mi355_status mi355_hiera_prefix(mi355_context* ctx, const mi355_hiera_hparams* hp, const float* image,
                                const mi355_tensor* patch_w, const float* patch_b, const float* pos_embed, float* x);
/* The whole backbone: image device F32 [3][img][img]; patch_w [7, 7, 3, E]
 * F32 or F16, patch_b [E], pos_embed [S0*S0][E] (S0 = img/4).  stage_out[s]
 * (device [S_s*S_s][C_s], or NULL) receive the output of each stage's last
 * block, which writes it there directly; the next stage reads it from there, so
 * the maps must not overlap one another. */
mi355_status mi355_hiera_encode(mi355_context* ctx, const mi355_hiera_hparams* hp, const float* image,
                                const mi355_tensor* patch_w, const float* patch_b, const float* pos_embed,
                                const mi355_hiera_block* blocks, int n_blocks, float* const stage_out[4]);

/* sam2_compute_pos_embed (sam3.cpp:4076-4157) on the device: the pos_embed
 * that mi355_hiera_encode adds, out [H*W][E] token-major (ggml [E, W, H]) =
 * bicubic(bkg -> H x W; Keys a = -0.75, half-pixel centres, border-clamped
 * taps, as torch's bicubic with align_corners=False) + the window table tiled
 * modulo ws.  bkg [E][bkg_h][bkg_w] and win [E][ws][ws] are device F32 in the
 * raw byte order of "hiera.pos_embed" ([bkg_w, bkg_h, E, 1]) and
 * "hiera.pos_embed_window" ([ws, ws, E, 1]).  For SAM2.1 Hiera at 1024:
 * bkg 7x7, ws 8, H = W = 256. */
mi355_status mi355_hiera_pos_embed(mi355_context* ctx, const float* bkg, int E, int bkg_h, int bkg_w, const float* win,
                                   int ws, int H, int W, float* out);

/* ---- SAM3 SimpleFPN neck ----------------------------------------------------
 * sam3_build_neck_graph (sam3.cpp:3867-3925) on this backend.  Activations
 * are device F32 token-major [H*W][C] (ggml [C, W, H]): the ViT output the
 * neck reads (vit_out [E, W, H]) and the four maps it writes (the reference's
 * out[i] after its final cont(permute(.., 1, 2, 0, 3))) are exactly the
 * reference's layouts.  Kernels are the registered ggml tensors
 * (sam3.cpp:2566-2600): conv-transpose [2, 2, Cout, Cin], conv [1, 1, Cin,
 * Cout] and [3, 3, Cin, Cout], F32 or F16 (F32 under quantized ftypes: their
 * ne0 of 1, 2 or 3 is not a block multiple), contiguous; biases F32.
 * Numerics per op as ggml-cpu: conv-transpose with the kernel cast to F16 and
 * the input converted to F16; conv_2d with the activations in the kernel's
 * type; f32 accumulation; f32 bias adds; GELU-erf after scale 0's first
 * conv-transpose. */
typedef struct mi355_neck_scale {
    const mi355_tensor* deconv1_w; /* scales 0 and 1: [2, 2, C1, E] */
    const float* deconv1_b;
    const mi355_tensor* deconv2_w; /* scale 0: [2, 2, D, C1] */
    const float* deconv2_b;
    const mi355_tensor* conv1x1_w; /* [1, 1, Cin, D] */
    const float* conv1x1_b;
    const mi355_tensor* conv3x3_w; /* [3, 3, D, D] */
    const float* conv3x3_b;
} mi355_neck_scale;
/* Device bytes the neck keeps in the context for a G x G grid of E channels. */
size_t mi355_neck_workspace_size(int E, int G, const mi355_neck_scale scales[4]);
/* out[0] [(4G)^2][D], out[1] [(2G)^2][D], out[2] [G^2][D], out[3] [(G/2)^2][D]
 * from x [G^2][E]; G even.  Scale 0: conv-transpose + GELU, conv-transpose,
 * 1x1, 3x3; scale 1: conv-transpose, 1x1, 3x3; scale 2: 1x1, 3x3; scale 3:
 * 2x2 max-pool, 1x1, 3x3; every conv adds its bias. */
mi355_status mi355_sam3_neck(mi355_context* ctx, const float* x, int E, int G, const mi355_neck_scale scales[4],
                             float* const out[4]);
/* The neck's node groups on token-major activations, for other graph builders:
 * ggml_conv_transpose_2d_p0(w [2, 2, Cout, Cin], x, 2) + bias (+ ggml_gelu_erf
 * when gelu): x [H*W][Cin] -> y [(2H)*(2W)][Cout]; */
mi355_status mi355_neck_deconv(mi355_context* ctx, const mi355_tensor* w, const float* b, const float* x, int H, int W,
                               int gelu, float* y);
/* ggml_conv_2d_sk_p0 (w [1, 1, Cin, Cout]) or ggml_conv_2d_s1_ph (w [3, 3, Cin,
 * Cout]) + bias: x [H*W][Cin] -> y [H*W][Cout]; */
mi355_status mi355_neck_conv(mi355_context* ctx, const mi355_tensor* w, const float* b, const float* x, int H, int W,
                             float* y);
/* ggml_pool_2d(MAX, 2, 2, 2, 2, 0, 0): x [H*W][C] -> y [(H/2)*(W/2)][C]. */
mi355_status mi355_neck_maxpool(mi355_context* ctx, const float* x, int H, int W, int C, float* y);

/* ---- Model files (sam3.cpp's .ggml format) ----------------------------------
 * sam3_load_model / sam3_load_tensors (sam3.cpp:3095-3348): a header (magic
 * "sam3" 0x73616D33 version 3, or "sam2" 0x73616D32 version 1; ftype; tensor
 * count), the hyperparameters as int32 fields (sam3_load_hparams 1481-1524,
 * sam2_load_hparams 1568-1630; SAM2 files with the Hiera backbone only), then
 * per tensor: n_dims, name length, ggml type, ne[0..n_dims), name, zero
 * padding to a 32-byte file offset, and the raw ggml rows.  Opening indexes the
 * records; data is read when a tensor is loaded. */
typedef struct mi355_model_file mi355_model_file;
typedef struct mi355_model_tensor_info {
    const char* name;   /* valid while the file is open */
    int32_t type;       /* ggml type id: 0 F32, 1 F16, 2 Q4_0, 3 Q4_1, 8 Q8_0 */
    int32_t n_dims;
    int64_t ne[4];      /* ggml order, unused dims 1 */
    uint64_t offset;    /* file offset of the data (32-byte aligned) */
    uint64_t nbytes;    /* data bytes */
} mi355_model_tensor_info;
mi355_status mi355_model_file_open(const char* path, mi355_model_file** out);
void mi355_model_file_close(mi355_model_file* f);
/* Text of the last open/query error (the calls without a context). */
const char* mi355_model_file_last_error(void);
mi355_status mi355_model_file_header(const mi355_model_file* f, uint32_t* magic, int32_t* version, int32_t* ftype,
                                     int32_t* n_tensors);
/* The hyperparameter fields in file order; returns their count (or -1). */
int mi355_model_file_hparams(const mi355_model_file* f, const int32_t** values);
/* Index of the tensor called name, or -1. */
int mi355_model_file_find(const mi355_model_file* f, const char* name);
mi355_status mi355_model_file_tensor(const mi355_model_file* f, int index, mi355_model_tensor_info* out);
/* Device bytes of tensor index loaded as dst_type (0 when no conversion exists):
 * the file's own type, F32 (from F16 or by dequantizing Q8_0/Q4_0/Q4_1), or F16
 * (from F32) - the conversions sam3_load_tensors applies (sam3.cpp:3150-3185). */
size_t mi355_model_file_load_bytes(const mi355_model_file* f, int index, int32_t dst_type);
/* Tensor data -> device memory dst (dst_bytes >= mi355_model_file_load_bytes),
 * converted on the GPU when dst_type differs.  Synchronous. */
mi355_status mi355_model_file_load(mi355_context* ctx, const mi355_model_file* f, int index, int32_t dst_type,
                                   void* dst, size_t dst_bytes);

/* A SAM3 file's ViT backbone in device memory: the tensors sam3_register_tensors
 * declares for it (sam3.cpp:2530-2560: "vit.patch_embed.proj.weight",
 * "vit.pos_embed", "vit.ln_pre.*", "vit.blocks.N.*"), weights in the file's
 * weight type when their rows are whole blocks and F32 otherwise, as the
 * reference registers them; the hyperparameters of mi355_vit_encode derived as
 * sam3_load_hparams does.  Quantized linear weights (Q8_0 / Q4_0 / Q4_1) are
 * handed out prepared (mi355_weight_prepare).  The tables stay valid until
 * mi355_vit_weights_free. */
typedef struct mi355_vit_weights mi355_vit_weights;
mi355_status mi355_vit_weights_load(mi355_context* ctx, const mi355_model_file* f, mi355_vit_weights** out);
void mi355_vit_weights_free(mi355_vit_weights* w);
mi355_status mi355_vit_weights_get(const mi355_vit_weights* w, mi355_vit_hparams* hp, const mi355_vit_block** blocks,
                                   int* n_blocks, const mi355_tensor** patch_w, const float** pos_embed,
                                   const float** ln_pre_w, const float** ln_pre_b);

/* sam3_quantize_model (examples/quantize.cpp:20-331): copies the .ggml file
 * in_path to out_path with the header's ftype set to qtype (Q4_0, Q4_1 or
 * Q8_0) and every tensor that the reference quantizes rewritten by
 * mi355_quantize_weights: 2-D or higher, ne0 a multiple of 32, F32 or F16,
 * and not one of the embedding / table names the reference keeps (token_embed,
 * pos_embed, freqs_cis, ...).  Header, hyperparameters (SAM3; SAM2 including
 * the EdgeTAM extension), the other tensors and any bytes after the last
 * tensor are copied unchanged; records are re-padded to 32-byte offsets.
 * stats (may be NULL) receives the reference's summary counts.  Errors:
 * unknown magic / bad arguments INVALID_ARG, unsupported version or tensor type
 * UNSUPPORTED, I/O FAILED; unlike the reference a truncated input is an error,
 * not a silently shortened output. */
typedef struct mi355_quantize_stats {
    int32_t n_quantized, n_total;
    int64_t size_org;  /* F32-equivalent bytes of every tensor */
    int64_t size_new;  /* data bytes written */
} mi355_quantize_stats;
mi355_status mi355_model_quantize(mi355_context* ctx, const char* in_path, const char* out_path, int32_t qtype,
                                  mi355_quantize_stats* stats);

/* A SAM2 file's Hiera backbone in device memory: the tensors sam3_register_tensors
 * declares for it (sam3.cpp:1800-1840: "hiera.patch_embed.*", "hiera.pos_embed",
 * "hiera.pos_embed_window", "hiera.blocks.N.*" with ".proj.*" at stage
 * transitions), weights in the file's weight type when their rows are whole
 * blocks and F32 otherwise; the hyperparameters of sam2_load_hparams
 * (sam3.cpp:1568-1590); pos_embed [S0*S0][E] (S0 = img/4) computed by
 * mi355_hiera_pos_embed from the two tables; quantized linear weights
 * prepared (mi355_weight_prepare).  Everything mi355_hiera_encode takes besides
 * the image; valid until mi355_hiera_weights_free. */
typedef struct mi355_hiera_weights mi355_hiera_weights;
mi355_status mi355_hiera_weights_load(mi355_context* ctx, const mi355_model_file* f, mi355_hiera_weights** out);
void mi355_hiera_weights_free(mi355_hiera_weights* w);
mi355_status mi355_hiera_weights_get(const mi355_hiera_weights* w, mi355_hiera_hparams* hp,
                                     const mi355_hiera_block** blocks, int* n_blocks, const mi355_tensor** patch_w,
                                     const float** patch_b, const float** pos_embed);

/* Fusion in the encoder runners (no counterpart in the reference, whose graph
 * always materialises f32 activations; on by default).  When on, the passes
 * that feed a MUL_MAT with Q8_0/Q4_0/Q4_1 or F16 weights (LayerNorm, bias+GELU,
 * the attention output) write its activation operand (the same from_float
 * quantization ggml applies to those f32 rows), and the GEMMs run the
 * following node group in their epilogue (bias + residual with the window
 * unpartition; the ViT's qkv split + RoPE).  Off gives the unfused sequence
 * of node groups, for parity checks: both produce the same bits. */
mi355_status mi355_context_set_fusion(mi355_context* ctx, int enable);
/* The skinny MUL_MAT kernel (no counterpart in the reference; on by default):
 * on the fp16 route (MI355_MMQ_F16, and ggml-layout weights behind the
 * encoders' fused operands), quantized GEMMs with K <= 128 over at least 4096
 * activation rows (SAM2 Hiera's stage-1 projections, K = 96) run on a kernel
 * that keeps the whole weight matrix in LDS and streams the activation rows;
 * it computes every output with the tiled kernel's instruction sequence, so
 * both give the same bits.  On the int8 route (prepared weights, and Q8_0 /
 * Q4_0 under MI355_MMQ_AUTO) the same shapes (N % 4 == 0, no K split) run on
 * an int8 skinny kernel that keeps each wavefront's activation fragments in
 * registers and reads the small weight matrix from L2, again bit-identical to
 * the tiled int8 kernel, and MUL_MATs of at most 64 F32 activation rows with
 * K <= 512 on one that quantizes the rows itself.  Off routes all to the tiled
 * kernels (for comparisons). */
mi355_status mi355_context_set_skinny(mi355_context* ctx, int enable);

/* The kernel behind 2-D MUL_MATs with Q8_0 / Q4_0 / Q4_1 weights in the
 * ggml layout (no counterpart in the reference).  All give the same bits: the
 * exact int32 block sums combined as acc = fma(isum, d_a * d_w, acc) in block
 * order.
 * - MI355_MMQ_F16: fp16 MFMAs over the quants as exact halves, weights used in
 *   their ggml rows and decoded in registers;
 * - MI355_MMQ_INT8: src1 quantized to one-byte quants, weights repacked into
 *   int8 rows with separate scale arrays on each call, block sums on
 *   v_mfma_i32_32x32x32_i8;
 * - MI355_MMQ_AUTO (the default): the faster per call with the repack counted:
 *   MI355_MMQ_INT8, except for few activation rows over a large weight, and
 *   for Q4_1 with K <= 128, few rows and large grids with a long K.
 * Prepared weights always take the int8 kernel; other MUL_MATs keep their
 * own kernels. */
typedef enum {
    MI355_MMQ_F16 = 0,
    MI355_MMQ_INT8 = 1,
    MI355_MMQ_AUTO = 2,
} mi355_mmq_kernel;
mi355_status mi355_context_set_mmq_kernel(mi355_context* ctx, int kernel);

/* ---- Kernel timing --------------------------------------------------------
 * The device-side counterpart of the reference's timing around graph compute
 * (std::chrono, sam3.cpp:6122-6135) and of its per-op micro-bench
 * (tests/test_metal_profile.cpp:22-69).  While enabled, every kernel launch
 * of the context is bracketed by HIP events on its stream;
 * mi355_profile_collect waits for them and folds the elapsed times into
 * per-kernel totals, returning the number of distinct kernels (or <0). */
mi355_status mi355_profile_enable(mi355_context* ctx, int enable);
int mi355_profile_collect(mi355_context* ctx);
mi355_status mi355_profile_get(mi355_context* ctx, int index, const char** name, int* launches, double* total_ms);
void mi355_profile_reset(mi355_context* ctx);

#ifdef __cplusplus
}
#endif
#endif /* SAM3_MI355_H */
