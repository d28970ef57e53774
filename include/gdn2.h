/*
 * gdn2.h -- C ABI of the MI355X (gfx950) GDN-2 chunked linear-attention library
 * (libgdn2_hip.so).
 *
 * The library replaces the device side of the reference's Python API:
 *   gdn2_pallas_forward(q,k,v,w,b,g,scale,h0=None)          gdn2_fwd.py:400-424
 *   gdn2_pallas_forward_trainable(q,k,v,w,b,g,scale,h0=None) gdn2_pipeline.py:143-159
 * whose forward is kernels A-D (gdn2_fwd.py:142-397) and whose custom_vjp
 * backward is B1-B5 (gdn2_bwd.py:32-375, assembled at gdn2_pipeline.py:70-137).
 *
 * Conventions
 *  - Tensors are dense row-major.  q,k,v,w,b,g,out and all gradients are
 *    (B, T, H, D); states h0, h_final, dh_final, dh0 are (B, H, D, D) indexed
 *    [b][h][dk][dv] (gdn2_fwd.py:342,355-357).  out, h_final, dh0 are float32
 *    (gdn2_fwd.py:163-165,342); gradients come back in the input dtype
 *    (gdn2_pipeline.py:129-135).
 *  - Every pointer is caller-owned device memory, 16-byte aligned.  No entry
 *    point allocates: the caller sizes the workspace with the *_workspace_bytes
 *    functions.  Work is enqueued on `stream` (a hipStream_t; NULL = default
 *    stream) and the call returns without synchronising.
 *  - Return value 0 on success, a negative GDN2_ERR_* code otherwise;
 *    gdn2_strerror() names it.  Invalid shapes are rejected before any launch.
 *  - No mutable global state beyond the per-thread timing request of
 *    gdn2_set_launch_events and the clip bound of gdn2_set_clip: calls on
 *    different streams may run concurrently provided their workspaces do not
 *    overlap.
 */
#ifndef GDN2_H_
#define GDN2_H_

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types (in_dtype applies to q,k,v,w,b and the gradients). */
#define GDN2_F32  0
#define GDN2_BF16 1  /* bfloat16 data and bfloat16 MFMA operands (inference) */
/* bfloat16 q,k,v,w,b and gradients, float32 arithmetic, residuals and MFMA
 * operands: the float32 path on bfloat16 inputs, as the reference's training
 * path upcasts every input before any arithmetic (gdn2_fwd.py:100-103,
 * gdn2_bwd.py:130-142) -- without float32 copies of the inputs or gradients.
 * Chunk 64 only; the workspace is sized as for GDN2_F32. */
#define GDN2_BF16_F32 2

/* Error codes. */
#define GDN2_OK                0
#define GDN2_ERR_HEAD_DIM     -1  /* D not in {64,128,256};
                                     ref asserts D==128, gdn2_fwd.py:145, gdn2_bwd.py:348 */
#define GDN2_ERR_SEQ_LEN      -2  /* T % BT != 0; ref asserts, gdn2_fwd.py:146 */
#define GDN2_ERR_CHUNK        -3  /* BT not in {64,128}, or BT=128 with float32 arithmetic or D=256 */
#define GDN2_ERR_DTYPE        -4  /* unknown dtype code; GDN2_BF16 in the backward */
#define GDN2_ERR_NULL         -5  /* required pointer is NULL */
#define GDN2_ERR_ALIGN        -6  /* pointer not 16-byte aligned */
#define GDN2_ERR_WORKSPACE    -7  /* workspace smaller than *_workspace_bytes() */
#define GDN2_ERR_SHAPE        -8  /* B<1, H<1, T<0, or sizes overflow (elements,
                                     or workgroups of a launch past 2^31) */
#define GDN2_ERR_LAUNCH       -9  /* HIP launch failure */
#define GDN2_ERR_FLAGS       -10  /* invalid flag combination */
#define GDN2_ERR_SCRATCH     -11  /* gdn2_fwd_noalloc: workload needs more than its scratch */

/* Library version string, e.g. "0.1.0". */
const char* gdn2_version(void);

/* Static description of an error code (never NULL). */
const char* gdn2_strerror(int code);

/* Host-only shape/dtype check (no GPU needed).  Mirrors the reference's
 * trace-time assertions gdn2_fwd.py:145-146 and gdn2_bwd.py:348-349. */
int gdn2_validate(int B, int T, int H, int D, int BT, int in_dtype, int g_dtype);

/* Bytes of workspace gdn2_fwd needs for an inference call (flags 0).  With
 * GDN2_FWD_SAVE_A (gdn2_fwd_workspace_bytes_ex) the workspace holds the
 * per-chunk residuals (WY factors, chunk states, v_new) that gdn2_bwd reads;
 * after an inference call its contents are unspecified.  Where the state scan
 * forms the outputs itself (bfloat16 inputs at D = 128 and 256, float32 at
 * D = 64), the chunk states and v_new never leave the GPU's on-chip memory and
 * the inference workspace has no room for them. */
size_t gdn2_fwd_workspace_bytes(int B, int T, int H, int D, int BT, int in_dtype);

/* gdn2_fwd flags. */
#define GDN2_FWD_SAVE_A 1  /* also keep A = (I + Akk)^{-1} in ws, needed by gdn2_bwd */
/* q,k,w,b,g are given before their activations, which the forward applies as it
 * reads them: q,k <- q,k / max(|.|_2, 1e-12) over D, w,b <- sigmoid, g <-
 * -softplus(g) -- the caller's preparation step of BASELINE's input
 * distributions, fused into the forward.  Inference only: not with
 * GDN2_FWD_SAVE_A (the backward reads the activated inputs). */
#define GDN2_FWD_RAW_INPUTS 2
/* Segments of the state scan (bits 8-15; 0 = automatic).  Long sequences with
 * few (b,h) pairs split the serial chunk recurrence into S segments scanned in
 * parallel and chained by their affine transitions (the sequence-parallel
 * design of the reference's kernel D, gdn2_fwd.py:338-366).  The chaining is
 * exact while the +-CLIP clip of the carried state (gdn2_fwd.py:358) does not
 * bind; the segmented passes flag any state clip that binds, and a flagged call
 * reruns the scan serially on the device (no host round trip), so the result
 * is the serial one either way.  n is clamped to [1, T/BT]; a forced count
 * needs gdn2_fwd_workspace_bytes_ex's workspace. */
#define GDN2_FWD_SEGMENTS(n) (((n) & 0xff) << 8)
/* Accept T % BT != 0: the last chunk of each sequence holds T % BT tokens and
 * is padded inside the kernels with neutral tokens (k = q = 0, g = 0; the state
 * passes through them unchanged), so out and h_final equal the forward over the
 * T real tokens.  Without this flag T % BT != 0 is GDN2_ERR_SEQ_LEN, as the
 * reference asserts (gdn2_fwd.py:146).  gdn2_fwd_workspace_bytes_ex with the
 * same flag sizes the workspace.  Not for gdn2_bwd (its inputs are whole
 * chunks: a caller pads with zero tokens, which leaves every result unchanged). */
#define GDN2_FWD_PARTIAL_CHUNK 4

/* As gdn2_fwd_workspace_bytes, for the segment count `flags` selects.  No
 * counterpart in the reference (its scan is serial); used to force a count. */
size_t gdn2_fwd_workspace_bytes_ex(int B, int T, int H, int D, int BT, int in_dtype, int flags);

/* Forward: replaces gdn2_pallas_forward (gdn2_fwd.py:400-424), kernels A-D.
 * h0 may be NULL (zero initial state, gdn2_fwd.py:403-404).  out (B,T,H,D)
 * and h_final (B,H,D,D) are float32.  flags: 0 for inference, GDN2_FWD_SAVE_A
 * when gdn2_bwd will consume ws (the trainable forward, gdn2_pipeline.py:64-67).
 * Inference with bfloat16 inputs at D = 128 and 256 (and float32 at D = 64)
 * runs two kernels: the state scan forms the outputs itself. */
int gdn2_fwd(void* stream, int B, int T, int H, int D, int BT, int in_dtype, int g_dtype,
             const void* q, const void* k, const void* v, const void* w, const void* b,
             const void* g, const float* h0, float scale, float* out, float* h_final,
             void* ws, size_t ws_bytes, int flags);

/* Test hook: as gdn2_fwd, and additionally writes A = (I + Akk)^{-1}
 * (kernel B's output, gdn2_fwd.py:246-260) as float32 (B,H,N,BT,BT) to a_out.
 * The workspace keeps every residual tile (h_c and v_new included), so it
 * takes gdn2_fwd_workspace_bytes_ex(..., GDN2_FWD_SAVE_A) bytes (or
 * GDN2_FWD_SAVE_A | GDN2_FWD_PARTIAL_CHUNK when T % BT != 0). */
int gdn2_fwd_debug(void* stream, int B, int T, int H, int D, int BT, int in_dtype,
                   int g_dtype, const void* q, const void* k, const void* v,
                   const void* w, const void* b, const void* g, const float* h0,
                   float scale, float* out, float* h_final, void* ws, size_t ws_bytes,
                   float* a_out);

/* Timing hook.  For the next gdn2_fwd / gdn2_fwd_debug / gdn2_bwd call made
 * on the calling host thread, record events[0] (hipEvent_t) on the call's
 * stream before its first kernel and events[i] after its i-th kernel stage,
 * for i < n.  The request is consumed by that call (also when it fails).
 * gdn2_fwd has 3 stages (fwd_prep, the state scan, fwd_out); where the scan
 * forms the outputs the third stage launches nothing.  Returns 0. */
int gdn2_set_launch_events(void* const* events, int n);

/* Saturation bound of every stage sanitize (x -> clip(nan_to_num(x)) to
 * [-clip, clip]), the reference's module constant CLIP (gdn2_fwd.py:33, 1e4 by
 * default), which its README overrides after import (README.md:87-92), for
 * every kernel this library launches on the current device from now on.
 * Synchronous (a copy into constant memory): call it with none of this
 * library's work in flight on the device and outside graph capture.  Returns
 * GDN2_ERR_SHAPE for a bound that is not finite and positive. */
int gdn2_set_clip(float clip);

/* Bytes of workspace gdn2_bwd needs in addition to the forward workspace. */
size_t gdn2_bwd_workspace_bytes(int B, int T, int H, int D, int BT, int in_dtype);

/* Backward: replaces _gdn2_core_bwd (gdn2_pipeline.py:70-137), kernels B1-B5.
 * fwd_ws must hold the residuals of a gdn2_fwd call with GDN2_FWD_SAVE_A on
 * the same inputs, h0 and scale (the reference recomputes them,
 * gdn2_pipeline.py:77-83; a caller that kept no residuals re-runs gdn2_fwd
 * first).  BT must be 64.  dh_final and h0 may be NULL (zero).  dq,dk,dv,dw,db
 * are in_dtype, dg is g_dtype, dh0 is float32 (B,H,D,D); all gradients are
 * sanitized as gdn2_pipeline.py:129-135.  in_dtype is GDN2_F32 or GDN2_BF16_F32:
 * the arithmetic and the residuals in fwd_ws are float32, as the reference
 * upcasts every input before any arithmetic (gdn2_fwd.py:100-103,
 * gdn2_bwd.py:130-142; gdn2_pipeline.py:129-135); GDN2_BF16_F32 reads bfloat16
 * inputs and writes bfloat16 gradients.  in_dtype = GDN2_BF16 (bfloat16
 * residuals, whose rounding puts gradients contracted against a unit dh_final
 * outside the bfloat16 tolerance) is GDN2_ERR_DTYPE, and
 * gdn2_bwd_workspace_bytes returns 0 for it.
 * Launches 4 kernels at D <= 128 (see gdn2_set_launch_events); at D = 256 the
 * per-chunk products run as separate launches (the launch marks still bracket
 * the same four stages). */
int gdn2_bwd(void* stream, int B, int T, int H, int D, int BT, int in_dtype, int g_dtype,
             const void* q, const void* k, const void* v, const void* w, const void* b,
             const void* g, const float* h0, float scale, const float* dout,
             const float* dh_final, void* dq, void* dk, void* dv, void* dw, void* db,
             void* dg, float* dh0, const void* fwd_ws, size_t fwd_ws_bytes, void* ws,
             size_t ws_bytes);

/* Variable-length batch.  No reference counterpart: the reference takes
 * equal-length sequences with T % BT == 0 (gdn2_fwd.py:145-146).  num_seqs
 * sequences are packed along T in (1,T,H,D) inputs; each is chunked on its
 * own -- its last chunk may be short and is padded inside the kernels with
 * neutral tokens -- and scanned from its own h0[s] ((num_seqs,H,D,D), may be
 * NULL) to h_final[s] ((num_seqs,H,D,D)).  Device tables (int32):
 * cu_chunks[num_seqs+1], sequence s owning chunks [cu_chunks[s],
 * cu_chunks[s+1]) of the packed chunk list; chunk_start[total_chunks+1], the
 * first token row of each chunk, chunk_start[total_chunks] = T.  Table values
 * are clamped in the kernels (no access outside the buffers).  flags: 0,
 * GDN2_FWD_RAW_INPUTS, or GDN2_FWD_SAVE_A when gdn2_bwd_varlen will consume ws. */
size_t gdn2_fwd_varlen_workspace_bytes(int total_chunks, int H, int D, int BT, int in_dtype);
int gdn2_fwd_varlen(void* stream, int num_seqs, const int* cu_chunks, const int* chunk_start,
                    int total_chunks, int T, int H, int D, int BT, int in_dtype, int g_dtype,
                    const void* q, const void* k, const void* v, const void* w, const void* b,
                    const void* g, const float* h0, float scale, float* out, float* h_final,
                    void* ws, size_t ws_bytes, int flags);

/* Backward of a variable-length batch.  No reference counterpart (see
 * gdn2_fwd_varlen).  Every sequence must occupy whole chunks: the packed
 * inputs are (1, total_chunks*BT, H, D), sequence s owning chunks
 * [cu_chunks[s], cu_chunks[s+1]); a caller pads each sequence with zero tokens
 * (neutral: its results and gradients are unchanged).  fwd_ws holds the
 * residuals of gdn2_fwd_varlen with GDN2_FWD_SAVE_A on the same inputs, with
 * chunk_start[c] = c*BT.  dh_final and dh0 are (num_seqs,H,D,D) float32
 * (dh_final may be NULL); gradients as gdn2_bwd.  BT must be 64. */
size_t gdn2_bwd_varlen_workspace_bytes(int total_chunks, int H, int D, int BT, int in_dtype);
int gdn2_bwd_varlen(void* stream, int num_seqs, const int* cu_chunks, int total_chunks, int H,
                    int D, int BT, int in_dtype, int g_dtype, const void* q, const void* k,
                    const void* v, const void* w, const void* b, const void* g, const float* h0,
                    float scale, const float* dout, const float* dh_final, void* dq, void* dk,
                    void* dv, void* dw, void* db, void* dg, float* dh0, const void* fwd_ws,
                    size_t fwd_ws_bytes, void* ws, size_t ws_bytes);

/* Forward that allocates nothing: gdn2_fwd's kernels with the workspace in a
 * fixed device array of the library (GDN2_NOALLOC_SCRATCH_BYTES per GPU, held
 * until the process ends).  No counterpart in the reference: it is for callers
 * that cannot allocate device memory (code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc).  Arguments as gdn2_fwd
 * without ws / ws_bytes; flags: GDN2_FWD_RAW_INPUTS, GDN2_FWD_PARTIAL_CHUNK,
 * GDN2_FWD_SEGMENTS(n) -- GDN2_FWD_SAVE_A is GDN2_ERR_FLAGS (the residuals would
 * not survive the next call).  A workload whose inference workspace exceeds the
 * scratch returns GDN2_ERR_SCRATCH before any launch (128 MiB: about 97 k
 * token-heads B*T*H for bfloat16 inputs at chunk 128 and D = 128, e.g.
 * B = 1, T = 8192, H = 11).
 * All calls on one GPU share its scratch: calls that overlap on one GPU (other
 * streams, other threads) race and must be serialised by the caller. */
#define GDN2_NOALLOC_SCRATCH_BYTES ((size_t)128 << 20)
int gdn2_fwd_noalloc(void* stream, int B, int T, int H, int D, int BT, int in_dtype,
                     int g_dtype, const void* q, const void* k, const void* v, const void* w,
                     const void* b, const void* g, const float* h0, float scale, float* out,
                     float* h_final, int flags);

/* Single-token recurrent step on the (B,H,D,D) float32 state, for serving:
 * the reference has no decode entry; this is gdn2_pallas_forward with T = 1
 * (gdn2_fwd.py:400-424), i.e. one chunk of one token, on the state layout of
 * h0 / h_final (gdn2_fwd.py:342).  q,k,v,w,b,g are (B,H,D) (one token of the
 * (B,T,H,D) inputs); h_in may be NULL (zero state) and may equal h_out (update
 * in place); out (B,H,D) float32.  Dtypes as gdn2_fwd; no chunk size applies.
 * One kernel (see gdn2_set_launch_events). */
int gdn2_decode(void* stream, int B, int H, int D, int in_dtype, int g_dtype, const void* q,
                const void* k, const void* v, const void* w, const void* b, const void* g,
                float scale, const float* h_in, float* h_out, float* out);

/* ---- The forward's stages one at a time ------------------------------------
 * The reference's module-level kernels, for callers that run or inspect them
 * separately.  Float32 arithmetic and float32 outputs in the reference's
 * (B,H,N,BT,.) layouts; chunk 64 only (GDN2_ERR_CHUNK otherwise); in_dtype
 * GDN2_F32, or GDN2_BF16 / GDN2_BF16_F32 for bfloat16 inputs (computed in float32,
 * as the reference upcasts, gdn2_fwd.py:100-103,266-272); T % 64 == 0.
 * gdn2_fwd runs the same mathematics fused. */

/* Kernel A: replaces build_chunk_scores_pallas (gdn2_fwd.py:142-170).  q,k,b,g
 * (B,T,H,D); aqk = scale * causal scores, akk = strictly lower (b k) k scores,
 * each (B,H,N,64,64) float32, zero above the diagonal. */
int gdn2_chunk_scores(void* stream, int B, int T, int H, int D, int BT, int in_dtype,
                      int g_dtype, const void* q, const void* k, const void* b,
                      const void* g, float scale, float* aqk, float* akk);

/* Kernel B: replaces wy_solve_pallas (gdn2_fwd.py:246-260).  a = (I + akk)^{-1}
 * for nchunks tiles of 64 x 64 float32 ([nchunks][64][64]); only the strictly
 * lower part of akk is read. */
int gdn2_wy_solve(void* stream, long long nchunks, int BT, const float* akk, float* a);

/* Kernel C: replaces recompute_wy_pallas (gdn2_fwd.py:298-330).  Inputs
 * (B,T,H,D) and a given a (B,H,N,64,64); w_pseudo = a (b k e^gc), u = a (w v),
 * kg, qg (B,H,N,64,D) and gc_last (B,H,N,D), float32. */
int gdn2_recompute_wy(void* stream, int B, int T, int H, int D, int BT, int in_dtype,
                      int g_dtype, const void* q, const void* k, const void* v,
                      const void* w, const void* b, const void* g, const float* a,
                      float* w_pseudo, float* u, float* kg, float* qg, float* gc_last);

/* Workspace bytes of gdn2_chunk_combine (N chunks per sequence). */
size_t gdn2_chunk_combine_workspace_bytes(int B, int N, int H, int D, int BT);

/* Kernel D: replaces gdn2_inter_chunk_combine and
 * gdn2_inter_chunk_combine_with_state (gdn2_fwd.py:338-397).  Per-chunk float32
 * tiles as kernels A and C give them: aqk (B,H,N,64,64), w_pseudo, u, kg, qg
 * (B,H,N,64,D), gc_last (B,H,N,D); h0 may be NULL.  out is (B, N*64, H, D) (the
 * token layout of gdn2_fwd; the reference returns it per chunk), h_final
 * (B,H,D,D).  h_pre_all (B,H,N,D,D), the state entering each chunk, and
 * v_new_all (B,H,N,64,D) are written when not NULL. */
int gdn2_chunk_combine(void* stream, int B, int N, int H, int D, int BT, const float* aqk,
                       const float* w_pseudo, const float* u, const float* kg,
                       const float* qg, const float* gc_last, const float* h0, float scale,
                       float* out, float* h_final, float* h_pre_all, float* v_new_all,
                       void* ws, size_t ws_bytes);

/* ---- The backward's stages one at a time -----------------------------------
 * The reference's backward module functions (gdn2_bwd.py:32-342), float32 on
 * the reference's chunk layouts (B,H,N,64,.), chunk 64 (GDN2_ERR_CHUNK
 * otherwise), D in {64, 128, 256}.  Each takes a device workspace of
 * gdn2_bwd_stage_workspace_bytes(stage, ...) bytes for its layout copies (none
 * for the reverse cumsum).  gdn2_bwd runs the same mathematics fused. */
#define GDN2_STAGE_DHU 1   /* gdn2_bwd_dhu */
#define GDN2_STAGE_DAV 2   /* gdn2_bwd_dav */
#define GDN2_STAGE_WY 3    /* gdn2_bwd_wy_dqkg */
#define GDN2_STAGE_INTRA 4 /* gdn2_bwd_intra */
size_t gdn2_bwd_stage_workspace_bytes(int stage, int B, int N, int H, int D, int BT);

/* B1: replaces gdn2_dhu_backward (gdn2_bwd.py:45-80).  do, dv_partial,
 * w_pseudo, qg, kg (B,H,N,64,D), gc_last (B,H,N,D), dht (B,H,D,D) or NULL.
 * dh_all (B,H,N,D,D): the gradient of the state entering each chunk (dh_all[0]
 * = dh0); dh0 (B,H,D,D); dv_all (B,H,N,64,D). */
int gdn2_bwd_dhu(void* stream, int B, int N, int H, int D, int BT, const float* dout,
                 const float* dv_partial, const float* w_pseudo, const float* qg,
                 const float* kg, const float* gc_last, float scale, const float* dht,
                 float* dh_all, float* dh0, float* dv_all, void* ws, size_t ws_bytes);

/* B2: replaces dav_backward_pallas (gdn2_bwd.py:99-122).  aqk (B,H,N,64,64),
 * taken as causal (kernel A's output); v_new, do (B,H,N,64,D).  daqk (B,H,N,64,64),
 * dv_new = aqk^T do (B,H,N,64,D). */
int gdn2_bwd_dav(void* stream, int B, int N, int H, int D, int BT, const float* aqk,
                 const float* v_new, const float* dout, float* daqk, float* dv_new, void* ws,
                 size_t ws_bytes);

/* B3: replaces wy_dqkg_backward_pallas (gdn2_bwd.py:213-244).  q, k, b, w, v,
 * gc (the in-chunk cumsum of g), v_new_all, do, dv (B,H,N,64,D); a (B,H,N,64,64);
 * h_pre_all, dh_next_all (B,H,N,D,D).  dq, dk, db, dw, dv_raw, dgc (B,H,N,64,D),
 * dakk (B,H,N,64,64). */
int gdn2_bwd_wy_dqkg(void* stream, int B, int N, int H, int D, int BT, const float* q,
                     const float* k, const float* b, const float* w, const float* v,
                     const float* gc, const float* a, const float* h_pre_all,
                     const float* v_new_all, const float* dout, const float* dv,
                     const float* dh_next_all, float scale, float* dq, float* dk, float* db,
                     float* dw, float* dv_raw, float* dgc, float* dakk, void* ws,
                     size_t ws_bytes);

/* B4: replaces intra_backward_pallas (gdn2_bwd.py:342-375).  daqk, dakk
 * (B,H,N,64,64); q, k, b, g (B,T,H,D) as the reference takes them.  dq, dk, db,
 * dgc (B,H,N,64,D), the sub-block pair clipping of gdn2_bwd.py:287-328 included. */
int gdn2_bwd_intra(void* stream, int B, int T, int H, int D, int BT, const float* daqk,
                   const float* dakk, const float* q, const float* k, const float* b,
                   const float* g, float scale, float* dq, float* dk, float* db, float* dgc,
                   void* ws, size_t ws_bytes);

/* B5: replaces reverse_cumsum_bwd (gdn2_bwd.py:32-41).  For `tiles` tiles of BT
 * rows by D columns: dg[i] = sanitize(sum_{j >= i} dgc[j]), row-wise. */
int gdn2_bwd_reverse_cumsum(void* stream, long long tiles, int BT, int D, const float* dgc,
                            float* dg);

/* ---- Gated linear recurrence ------------------------------------------------
 * Elementwise over the C channels of (B,T,C) tensors (heads and their channels
 * flattened):
 *   h_t = e^{g_t} h_{t-1} + b_t x_t,   out_t = h_t,   h_final = h_T.
 * No counterpart in the reference.  g is the log decay, as GDN-2's; the sums of g
 * over any run of tokens must stay below 88 (g <= 0 in use).  g_t = -inf (or below
 * -2.3e38, as a mask of the type's lowest value) starts anew: h_t = b_t x_t whatever
 * h_{t-1} holds, NaN included, and no gradient passes -- the sequences of a packed
 * batch.  b may be NULL (all ones).  Float32
 * arithmetic; in_dtype (GDN2_F32, GDN2_BF16) is x's, b's, out's and dout's and
 * that of their gradients, g_dtype (GDN2_F32, or GDN2_BF16 with bfloat16 inputs)
 * g's and dg's; states and their gradients are float32 (B,C).
 * x, g, b and dout may be strided: *_strides points to two host integers, the
 * elements from one batch entry and one token to the next (NULL: dense); the
 * channels are contiguous.  out, dx, dg, db are dense.  Pointers are aligned to
 * their elements, the workspace to 16 bytes; 4-element alignment of pointers, strides
 * and C is faster.
 * gdn2_set_launch_events does not reach the entry points from here on. */

/* Bytes of the states kept for the backward (float32, one for every 128 to 512
 * tokens) and of the workspace of the forward and of the backward (0 for short
 * axes, where a workgroup walks along the whole axis). */
size_t gdn2_gated_scan_kept_bytes(int B, int T, int C, int in_dtype);
size_t gdn2_gated_scan_workspace_bytes(int B, int T, int C, int in_dtype);

/* h0 may be NULL (zero) and equal to h_final; kept may be NULL (inference). */
int gdn2_gated_scan_fwd(void* stream, int B, int T, int C, int in_dtype, int g_dtype,
                        const void* x, const long long* x_strides, const void* g,
                        const long long* g_strides, const void* b, const long long* b_strides,
                        const float* h0, void* out, float* h_final, float* kept, void* ws,
                        size_t ws_bytes);

/* Gradients from those of out and h_final (either may be NULL: zero), the
 * forward's inputs and its kept states.  db is written where b is given, dh0
 * where it is not NULL.  T >= 1. */
int gdn2_gated_scan_bwd(void* stream, int B, int T, int C, int in_dtype, int g_dtype,
                        const void* x, const long long* x_strides, const void* g,
                        const long long* g_strides, const void* b, const long long* b_strides,
                        const void* dout, const long long* dout_strides, const float* dh_final,
                        const float* kept, void* dx, void* dg, void* db, float* dh0, void* ws,
                        size_t ws_bytes);

/* One token of n = B*C values, all dense; h_in may be NULL (zero) and equal to
 * h_out (update in place). */
int gdn2_gated_scan_step(void* stream, long long n, int in_dtype, int g_dtype, const void* x,
                         const void* g, const void* b, const float* h_in, float* h_out,
                         void* out);

/* ---- RMS norm with the residual's addition ----------------------------------
 * Over M rows of C <= 16384 values (no counterpart in the reference):
 *   h = x + residual, rounded to the residual's type;   y = h w / sqrt(mean h^2 + eps).
 * residual may be NULL: then h = x, and h (the output) may be NULL.  x_dtype is
 * x's, y's, dy's and dx's, r_dtype (x_dtype, or GDN2_F32) the residual's, h's, dh's and
 * dr's, w_dtype the weight's and dw's.  x and residual have rows of contiguous values,
 * *_stride elements apart; all else is dense.  Float32 arithmetic.  Pointers are aligned
 * to their elements (faster: 16 bytes, with row strides of 16 bytes and C % 8 == 0).
 * eps >= 0, GDN2_ERR_SHAPE otherwise. */

/* rstd (M) float32 is for the backward, or NULL. */
int gdn2_rms_norm(void* stream, int M, int C, int x_dtype, int r_dtype, int w_dtype,
                  const void* x, long long x_stride, const void* residual,
                  long long r_stride, const void* weight, float eps, void* y, void* h,
                  float* rstd);

/* Gradients from those of y and h (dy, dh: either may be NULL, zero): dx, and dr, the
 * residual's (NULL where it has x's type: it equals dx), and dw.  h is the forward's
 * (x without a residual). */
size_t gdn2_rms_norm_bwd_workspace_bytes(int M, int C);
int gdn2_rms_norm_bwd(void* stream, int M, int C, int x_dtype, int r_dtype, int w_dtype,
                      const void* h, const void* weight, const float* rstd, const void* dy,
                      const void* dh, void* dx, void* dr, void* dw, void* ws,
                      size_t ws_bytes);

/* y in 8 bits with a scale for each row: with t = h w and m = max |t|, q = round(127 t / m)
 * (ties to even; computed as t times 127 (1 / m) in float32) and
 * scale = m / (127 sqrt(mean h^2 + eps)).  A row whose m is below 1e-36
 * has q = 0 and scale 0; one that holds NaN or an infinity q = 0 and scale NaN.  q is 16-byte
 * aligned, its rows q_stride = C rounded up to a multiple of 16 bytes apart, the bytes
 * between zero. */
int gdn2_rms_norm_int8(void* stream, int M, int C, int x_dtype, int r_dtype, int w_dtype,
                       const void* x, long long x_stride, const void* residual,
                       long long r_stride, const void* weight, float eps, void* q,
                       long long q_stride, float* scale, void* h);

/* ---- Rows in 8 bits and their products --------------------------------------- */

/* Rows of x (C <= 32768) in 8 bits: as gdn2_rms_norm_int8 with t = x, scale = m / 127. */
int gdn2_quantize_int8(void* stream, int M, int C, int x_dtype, const void* x,
                       long long x_stride, void* q, long long q_stride, float* scale);

/* out = q scale, (M,C) dense; rows of q are q_stride bytes apart. */
int gdn2_dequantize_int8(void* stream, int M, int C, int out_dtype, const void* q,
                         long long q_stride, const float* scale, void* out);

/* out[m][n] = x_scale[m] w_scale[n] sum_k x[m][k] w[n][k] + bias[n] (bias float32 or
 * NULL), out (M,N) dense of out_dtype; x (M,K) and w (N,K) signed 8-bit integers, sums
 * exact in 32 bits (1 <= K <= 131071; N <= 2^26, and M N in 128 x 128 tiles at most
 * 2^23 of them).  x and w are 16-byte aligned, their rows *_stride
 * bytes apart, a multiple of 16, at least K rounded up to one and at most 2^24: the
 * bytes between K and its multiple are read and count for nothing. */
int gdn2_int8_matmul(void* stream, int M, int N, int K, int out_dtype, const void* x,
                     long long x_stride, const float* x_scale, const void* w,
                     long long w_stride, const float* w_scale, const float* bias, void* out);

/* ---- Short causal convolution --------------------------------------------------
 * Over each channel of (B,T,C) tensors (no counterpart in the reference):
 *   y_t = act(bias + sum_{k < W} w[k] x_{t - W + 1 + k}),   2 <= W <= 4,
 * act the identity (silu = 0) or v / (1 + e^{-v}) (silu = 1).  state (B,W-1,C) holds the
 * inputs before the first token, oldest first (NULL: zeros), last the W - 1 inputs up to the
 * last token; w (C,W) and bias (C, or NULL) are float32, all else is of dtype (GDN2_F32,
 * GDN2_BF16).  starts (B,T) bytes, or NULL: a token whose byte is not zero begins a sequence,
 * nothing from before it enters, and the entries of `last` before the last such token are zero.
 * x and dy may be strided as for the gated recurrence; all else is dense.  Pointers are
 * aligned to their elements (faster: to four, with strides and C % 4 == 0).  T >= 1;
 * float32 sums. */
int gdn2_short_conv_fwd(void* stream, int B, int T, int C, int W, int dtype, int silu,
                        const void* x, const long long* x_strides, const float* w,
                        const float* bias, const void* state, const unsigned char* starts,
                        void* y, void* last /* not state */);

/* Gradients from those of y and last (dy, dlast: either may be NULL, zero): dx, dw (C,W),
 * dbias (C, or NULL) and dstate (B,W-1,C, or NULL). */
size_t gdn2_short_conv_bwd_workspace_bytes(int B, int T, int C, int W);
int gdn2_short_conv_bwd(void* stream, int B, int T, int C, int W, int dtype, int silu,
                        const void* x, const long long* x_strides, const float* w,
                        const float* bias, const void* state, const unsigned char* starts,
                        const void* dy, const long long* dy_strides, const void* dlast, void* dx,
                        float* dw, float* dbias, void* dstate, void* ws, size_t ws_bytes);

/* One token, x and y (B,C); state_in may be NULL (zeros) and equal to state_out. */
int gdn2_short_conv_step(void* stream, int B, int C, int W, int dtype, int silu, const void* x,
                         const float* w, const float* bias, const void* state_in,
                         void* state_out, void* y);

/* ---- Selective state space scan --------------------------------------------------
 * Over (B,T,C) tensors with N <= 64 states a channel (no counterpart in the reference):
 *   d = dt + dt_bias, with softplus = 1 log(1 + e^d);
 *   h_t[c,n] = e^{d_t[c] A[c,n]} h_{t-1}[c,n] + d_t[c] x_t[c] Bm_t[n];
 *   y_t[c] = sum_n Cm_t[n] h_t[c,n] + D[c] x_t[c];   out_t = y_t z_t / (1 + e^{-z_t}).
 * Bm and Cm (B,T,G,N) are shared by the C / G channels of a group.  A (C,N), D (C, or NULL: 0),
 * dt_bias (C, or NULL: 0), h0, h_final and their gradients (B,C,N) are float32; x, Bm, Cm, z
 * (NULL: no gate), out, dout and their gradients are of in_dtype (GDN2_F32, GDN2_BF16), dt and
 * ddt of dt_dtype (GDN2_F32, or in_dtype).  Float32 arithmetic; the sums of d A over any run
 * of tokens must stay below 88 (d >= 0 and A <= 0 in use).  starts: as for the convolution, the
 * state before such a token is dropped and no gradient passes it.
 * ins: host array of x, dt, z, Bm, Cm; strides: NULL (dense) or ten host integers, for each of
 * them the elements from one batch entry and one token (at most 2^25) to the next; the rest of a
 * row is contiguous.  C <= 2^24, G <= 2^18.  Pointers are aligned to their elements, kept and ws to 16 bytes.  T >= 1. */

/* Bytes of what is kept for the backward (float32: the states before every 16th token, N padded to
 * 8, 16, 32 or 64, and the rows of Bm and Cm) and of the workspace of the forward or the backward. */
size_t gdn2_selective_scan_kept_bytes(int B, int T, int C, int G, int N);
size_t gdn2_selective_scan_workspace_bytes(int B, int T, int C, int G, int N, int backward);

/* h0 may be NULL (zero; not h_final); kept may be NULL (inference). */
int gdn2_selective_scan_fwd(void* stream, int B, int T, int C, int G, int N, int in_dtype,
                            int dt_dtype, int softplus, const void* const* ins,
                            const long long* strides, const float* A, const float* D,
                            const float* dt_bias, const float* h0, const unsigned char* starts,
                            void* out, float* h_final, float* kept, void* ws, size_t ws_bytes);

/* Gradients from those of out and h_final (either may be NULL: zero), the forward's inputs
 * and what it kept.  outs: host array of dx, ddt, dz (NULL without z), dBm, dCm, all dense;
 * dD, ddt_bias and dh0 are written where they are not NULL. */
int gdn2_selective_scan_bwd(void* stream, int B, int T, int C, int G, int N, int in_dtype,
                            int dt_dtype, int softplus, const void* const* ins,
                            const long long* strides, const float* A, const float* D,
                            const float* dt_bias, const unsigned char* starts, const void* dout,
                            const long long* dout_strides, const float* dh_final,
                            const float* kept, void* const* outs, float* dA, float* dD,
                            float* ddt_bias, float* dh0, void* ws, size_t ws_bytes);

/* One token: x, dt, z, out (B,C), Bm, Cm (B,G,N), all dense; h_in may be NULL (zero) and
 * equal to h_out. */
int gdn2_selective_scan_step(void* stream, int B, int C, int G, int N, int in_dtype, int dt_dtype,
                             int softplus, const void* x, const void* dt, const float* A,
                             const void* Bm, const void* Cm, const float* D, const void* z,
                             const float* dt_bias, const float* h_in, float* h_out, void* out);

/* ---- 8-bit floating point with a scale for each block of 128 -----------------------
 * Values are OCP e4m3 (no counterpart in the reference).  A block's scale is the smallest power
 * of two s >= 2^-126 with max|t| <= 448 s, q = e4m3(t / s), ties to even.  A block of zeros has scale
 * 0, one that holds NaN or an infinity scale NaN and q = 0. */

/* x (M,C), rows x_stride elements apart.  blocks = 0: q (M,C) with scale (ceil(C/128), M), a scale
 * for each 1 x 128 values of a row, and / or qt (C,M), x transposed, with scale_t
 * (ceil(M/128), C), one for each 128 values of a column.  blocks = 1: q with scale (ceil(M/128),
 * ceil(C/128)), one for each 128 x 128 values, and where it is given qt with the same transposed.
 * q or qt may be NULL (q not with blocks).  Rows of q and qt are C and M rounded up to 16 bytes
 * apart, the bytes between zero, both 16-byte aligned.  part (ceil(M/128), C), a workspace, and
 * sums (C), or both NULL: the sums of x's columns (of its values, not of what q stands for; the
 * gradient of a bias).  C <= 2^27, at most 2^23 blocks of 128 x 128. */
int gdn2_quantize_fp8(void* stream, int M, int C, int x_dtype, const void* x, long long x_stride,
                      int blocks, void* q, long long q_stride, float* scale, void* qt,
                      long long qt_stride, float* scale_t, float* part, float* sums);

/* out = q scale, (M,C) dense; the scale of row m and block k at scale[(m / row_block) *
 * scale_strides[0] + k * scale_strides[1]] (a host array), row_block 1 or 128. */
int gdn2_dequantize_fp8(void* stream, int M, int C, int out_dtype, const void* q,
                        long long q_stride, int row_block, const float* scale,
                        const long long* scale_strides, void* out);

/* out[m][n] = sum_b x_scale[b][m] s[n][b] sum_{k in block b} x[m][k] w[n][k] + bias[n] (bias float32
 * or NULL), out (M,N) dense of out_dtype; x (M,K) and w (N,K).  s[n][b] is w_scale[b][n] with
 * w_row_block 1, w_scale[n / 128][b] with 128; *_scale_stride are the elements between rows of
 * the scales (at least M; N or ceil(K/128)).  A scale may have any value as long as its product with
 * each of the other operand's is zero or a normal float32 number: the two may be multiplied
 * first.  Products of a block are
 * summed by the matrix cores, blocks in float32: exactly as float32 sums for float32 results; for
 * bfloat16 ones at the 8-bit instruction's rate, which drops what lies below 2^-13 of the largest of
 * eight neighbouring products.  Otherwise as gdn2_int8_matmul. */
int gdn2_fp8_matmul(void* stream, int M, int N, int K, int out_dtype, const void* x,
                    long long x_stride, const float* x_scale, long long x_scale_stride,
                    const void* w, long long w_stride, int w_row_block, const float* w_scale,
                    long long w_scale_stride, const float* bias, void* out);

/* A linear layer multiplied in 8 bits, y = x w^T + bias over x (M,K), w (N,K), y (M,N) dense, all
 * of dtype, bias float32 or NULL; rows of x, w and dy are *_stride elements apart.  Forward: x in
 * blocks of 1 x 128, w of 128 x 128.  Backward: dx from dy in blocks of 1 x 128 and w's, dw from dy
 * and x in blocks of 128 tokens, dbias (float32) the sums of dy's columns.  kept holds the
 * operands of the gradients that need_dx and need_dw name (NULL for neither), for the backward,
 * which is told the same (kept_dx, kept_dw) and writes those of dx, dw and dbias that are not NULL.
 * M, N, K <= 2^24; kept and ws 16-byte aligned. */
size_t gdn2_fp8_linear_kept_bytes(int M, int N, int K, int need_dx, int need_dw);
size_t gdn2_fp8_linear_workspace_bytes(int M, int N, int K, int backward);
int gdn2_fp8_linear_fwd(void* stream, int M, int N, int K, int dtype, const void* x,
                        long long x_stride, const void* w, long long w_stride, const float* bias,
                        int need_dx, int need_dw, void* y, void* kept, void* ws, size_t ws_bytes);
int gdn2_fp8_linear_bwd(void* stream, int M, int N, int K, int dtype, const void* dy,
                        long long dy_stride, const void* kept, int kept_dx, int kept_dw, void* dx,
                        void* dw, float* dbias, void* ws, size_t ws_bytes);

#ifdef __cplusplus
}
#endif

#endif /* GDN2_H_ */
