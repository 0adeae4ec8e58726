/*
 * hyena_b200.h -- C ABI of the B200 (sm_100a) Hyena-mixer kernels.
 *
 * Every entry point takes plain device pointers, element strides and sizes,
 * launches asynchronously on the caller's CUDA stream, performs no host<->device
 * synchronisation and never allocates device memory (workspace, where needed, is
 * caller-provided and sized by the matching *_workspace_size function).
 * All functions return HYENA_OK (0) or an error code; hyena_last_error() gives a
 * human-readable message for the calling thread.  Device-side range violations
 * (a state block index outside [0, num_blocks)) never trap: the offending row is
 * skipped and a bit is OR-ed into the optional caller-provided `error_flags` word.
 *
 * Paged mixer state follows the layout vLLM hands the reference mixers
 * (evo2_flash/mixers.py:6-17, 892-904, 940-949):
 *   S0  conv window over the 3H in_proj channels, bf16, (blocks, W0, 3H) in vLLM's
 *       SD layout (W0 = K_short-1 [+ num_spec]); oldest column first.
 *   S1  inner-FIR window over H channels, fp32, (blocks, 127, H); HCS uses the
 *       first 6 columns, HCM all 127.
 *   S2  LI modal state, fp32, (blocks, H, 16[+1 stamp column]).
 * Each slice is described by a hyena_state_view with explicit strides, so the
 * dim-first and the SD orientation, and vLLM's padded page strides, all work.
 */
#ifndef HYENA_B200_H
#define HYENA_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HYENA_ABI_VERSION 9

#if defined(__GNUC__)
#define HYENA_API __attribute__((visibility("default")))
#else
#define HYENA_API
#endif

#define HYENA_OK 0
#define HYENA_ERR_INVALID 1      /* bad argument (shape, alignment, null pointer) */
#define HYENA_ERR_CUDA 2         /* a CUDA runtime/driver call failed */
#define HYENA_ERR_UNSUPPORTED 3  /* a configuration the kernels do not implement */

/* Bits OR-ed into *error_flags by the kernels. */
#define HYENA_FLAG_BLOCK_RANGE 1 /* a state block index was outside [0, num_blocks) */
#define HYENA_FLAG_SEGMENT 2     /* query_start_loc was not non-decreasing / exceeded T */
#define HYENA_FLAG_STAMP 4       /* a position stamp did not match the request position */
#define HYENA_FLAG_COLLECTIVE 8  /* a cross-rank wait of a collective kernel expired */
#define HYENA_FLAG_WAIT 16       /* a shared-memory barrier wait of a kernel expired */

typedef struct hyena_state_view {
  void* data;            /* element (block 0, column 0, channel 0) */
  int64_t block_stride;  /* elements between consecutive blocks (vLLM page stride) */
  int64_t col_stride;    /* elements between window columns (time positions) */
  int64_t dim_stride;    /* elements between channels */
  int32_t cols;          /* window columns available in the slice */
  int32_t num_blocks;    /* valid block indices are [0, num_blocks) */
} hyena_state_view;

/* Mixer kinds. */
#define HYENA_KIND_FIR 0  /* HCS (K=7) and HCM (K=128) explicit depthwise FIR */
#define HYENA_KIND_IIR 1  /* HCL diagonal modal SSM of order 16 */

/* Parameters shared by prefill and decode of one Hyena layer.  Channel h of the
 * in_proj output occupies columns (3h, 3h+1, 3h+2) = (x2, x1, v) of z. */
typedef struct hyena_layer_params {
  int32_t kind;          /* HYENA_KIND_FIR / HYENA_KIND_IIR */
  int32_t H;             /* channels of this shard (multiple of 64) */
  int32_t K;             /* FIR taps (7 or 128); 16 (modal order) for IIR */
  const void* short_w;   /* (3H, 3) bf16 contiguous, cross-correlation order */
  const void* inner_w;   /* FIR: (H, K) bf16 taps, w[:, K-1] pairs with the current sample */
  int64_t inner_w_stride_h, inner_w_stride_k;
  const float* log_poles;/* IIR: (H, 16) fp32 */
  int64_t lp_stride_h, lp_stride_s;
  const float* residues; /* IIR: (H, 16) fp32 */
  int64_t res_stride_h, res_stride_s;
  const void* D;         /* (H,) bf16 skip, or NULL (HCS has none) */
} hyena_layer_params;

/* ---------------------------------------------------------------- prefill
 * Replaces, for the prefill rows of one step:
 *   HyenaMixerBase._short_conv prefill branch -> vLLM causal_conv1d_fn
 *     (evo2_flash/mixers.py:1121-1151, torch twin 350-383), the de-interleave and
 *     x1*v gate (mixers.py:1207-1208, 1293, 1356);
 *   FIR: HyenaFIRMixer._inner_prefill -> triton_prefill.fir_prefill
 *     (mixers.py:1258-1262; triton_prefill.py:391-501) and the +D*u, *x2 gate
 *     (mixers.py:1300-1302);
 *   IIR: the per-segment loop of HyenaIIRMixer._forward_impl and iir_segment,
 *     hcl_compute_filter, iir_final_state (mixers.py:144-210, 1378-1397;
 *     triton_hcl.py:88-123; triton_prefill.py:351-387).
 * Input z: (T, 3H) bf16 packed prefill rows (row 0 = first prefill token).
 * Output g: (T, H) bf16 = x2 * (inner(u) [+ D*u]) per row, the out_proj input.
 * Segment j covers rows [query_start_loc[j], query_start_loc[j+1]); it continues
 * from cached state when has_initial_state[j] != 0 and writes its final windows /
 * modal state into block state_indices[j * state_indices_stride].
 */
typedef struct hyena_prefill_args {
  const void* z; int64_t ldz;   /* bf16, row stride in elements */
  void* out; int64_t ldo;       /* bf16 */
  int32_t T;                    /* rows available in z / out */
  int32_t num_segments;
  const int32_t* query_start_loc;      /* (num_segments + 1) device */
  const uint8_t* has_initial_state;    /* (num_segments) device bool, or NULL = all fresh */
  const int32_t* state_indices; int64_t state_indices_stride;
  hyena_state_view conv_state;   /* S0 (bf16) */
  hyena_state_view inner_state;  /* FIR: S1 (fp32); IIR: S2 (fp32, cols = modes) */
  int32_t* error_flags;          /* optional device int */
} hyena_prefill_args;

HYENA_API size_t hyena_prefill_workspace_size(const hyena_layer_params* p, int32_t T,
                                    int32_t num_segments);
HYENA_API int hyena_prefill(const hyena_layer_params* p, const hyena_prefill_args* a,
                  void* workspace, size_t workspace_bytes, void* stream);

/* Prefill for callers that cannot allocate device memory.  No counterpart in
 * the reference (its Python path allocates through torch).  Same arguments and
 * result as hyena_prefill minus the workspace: the LI kind's scratch is a fixed
 * 32 MiB array inside this library, present on every GPU that loads it until the
 * process exits.  The LI kind needs one (H, 16) fp32 modal state per
 * segment, plus a few for splitting long segments (256 KiB each at H = 4096);
 * steps needing more (beyond ~120 segments at H = 4096) fail with
 * HYENA_ERR_INVALID.  The first call on a device looks up
 * the array's device address; make it before any stream capture.  That
 * address is cached per device for the process lifetime and belongs to the
 * device's primary context: do not use this entry point after a
 * cudaDeviceReset or from a non-primary context.  All calls share the array:
 * calls whose kernels overlap on the GPU race on it. */
HYENA_API int hyena_prefill_noalloc(const hyena_layer_params* p, const hyena_prefill_args* a,
                                    void* stream);

/* ---------------------------------------------------------------- channel-sharded out_proj
 * In-switch (NVLink SHARP) all-reduce of the row-parallel out_proj partial sums,
 * the "one all-reduce per block" of the channel-sharded mixer.  No counterpart in
 * the reference, which has no tensor parallelism (evo2_flash/mixers.py:38-41);
 * it stands where a NCCL all-reduce of the (T, H) bf16 partial would.
 * multicast: the multicast address of a symmetric buffer holding n_elems bf16 on
 * every rank (in place: every rank's buffer ends with the sum, accumulated in
 * fp32 and rounded once); signal_pads: device array of the `world` ranks' signal
 * pads (zero-initialised, signal_pad_bytes each, >= 8 * num_ctas * world bytes);
 * epoch: nonzero, larger than every earlier call's on these pads.  All ranks make
 * the same calls in the same order.  A cross-rank wait that expires (~1 s) sets
 * HYENA_FLAG_COLLECTIVE in *error_flags and the kernel returns. */
HYENA_API int hyena_nvls_allreduce_bf16(void* multicast, int64_t n_elems, void* const* signal_pads,
                                        int64_t signal_pad_bytes, int32_t rank, int32_t world,
                                        uint32_t epoch, int32_t num_ctas, int32_t* error_flags,
                                        void* stream);

/* ---------------------------------------------------------------- decode / verify
 * Replaces, for the decode rows of one step:
 *   ordinary decode: triton_decode.hyena_decode (triton_decode.py:56-211) and the
 *     unfused chain it stands for: vLLM causal_conv1d_update, _fir_decode_one /
 *     _iir_decode_one -> triton_verifier.fir_one / iir_one (mixers.py:555-575,
 *     1194-1205; triton_verifier.py:158-178);
 *   speculative verify: the _short_conv spec branch (mixers.py:1153-1193),
 *     _fir_decode_snapshots / _iir_decode_snapshots (mixers.py:578-663) ->
 *     triton_verifier.fir_snapshots / iir_snapshots (triton_verifier.py:47-155).
 * Request r owns tokens [token_start[r], token_start[r+1]) (NULL: token r only).
 * The short window is read from conv_in_block[r] at column offset accepted[r]-1
 * and the shifted window written to conv_out_block[r] (vLLM's spec convention).
 * The inner state is read from in_slots[r, accepted[r]-1]; after token p the
 * complete state snapshot is written to out_slots[r, p] (skipped for block 0 when
 * skip_null_writes != 0, which is vLLM's null block).  Ordinary decode is q = 1,
 * accepted = NULL (= 1) and in_slots == out_slots.  When zero_null_rows != 0 a
 * request whose conv_in_block equals null_block writes a zero output row and no
 * state (the fused-decode CUDA-graph padding rule, triton_decode.py:66-70).
 */
typedef struct hyena_decode_args {
  const void* z; int64_t ldz;   /* (tokens, 3H) bf16 */
  void* out; int64_t ldo;       /* (tokens, H) bf16 */
  int32_t num_reqs;
  int32_t q;                    /* max tokens per request (columns of in/out slots) */
  const int32_t* token_start;   /* (num_reqs + 1) or NULL */
  const int32_t* accepted;      /* (num_reqs), read clamped to [1, q] (above q also sets
                                   HYENA_FLAG_SEGMENT); or NULL (= 1) */
  const int32_t* conv_in_block; const int32_t* conv_out_block;  /* (num_reqs), strided below */
  const int32_t* in_slots; int64_t in_stride0, in_stride1;      /* (num_reqs, q) */
  const int32_t* out_slots; int64_t out_stride0, out_stride1;   /* (num_reqs, q) */
  int32_t zero_null_rows;
  int32_t skip_null_writes;
  int32_t null_block;
  hyena_state_view conv_state;
  hyena_state_view inner_state;
  int32_t* error_flags;
  int64_t conv_in_stride;       /* elements between consecutive conv_in_block entries */
  int64_t conv_out_stride;      /* ... conv_out_block entries; 0 reads as 1 (contiguous) */
} hyena_decode_args;

HYENA_API int hyena_decode(const hyena_layer_params* p, const hyena_decode_args* a, void* stream);

/* ---------------------------------------------------------------- fp8 projection
 * Static per-tensor E4M3 activation quantisation, q = e4m3_rn(clamp(x / sx, +-448)):
 * the rule of fp8_emul.quantize_input (fp8_emul.py:76-78) and of vLLM's static
 * W8A8 path the reference in_proj uses (mixers.py:740-757, 780-783).
 * x: (M, K) bf16 with row stride ldx; q: (M, K) e4m3 contiguous rows of ldq.
 * K % 8 == 0, K <= 16384.
 */
HYENA_API int hyena_quant_e4m3(const void* x, int64_t ldx, void* q, int64_t ldq, int32_t M,
                     int32_t K, const float* input_scale, void* stream);

/* out(M,N) bf16 = (A(M,K) e4m3 . B(N,K) e4m3^T) * (*scale_a) * (*scale_b):
 * the in_proj GEMM (mixers.py:1076-1092 -> vLLM Fp8 ReplicatedLinear; numerics
 * contract fp8_emul.py:81-88 with fp32 accumulation).  tcgen05 + TMA + TMEM.
 * Requires K % 128 == 0, N % 8 == 0, 16-byte aligned rows.
 * Small-M calls (decode batches) split K over the CTAs of a thread-block cluster
 * and reduce the slices in shared memory; `workspace` / `workspace_bytes` are
 * accepted for ABI stability and ignored (pass NULL, 0). */
HYENA_API int hyena_gemm_e4m3(const void* A, int64_t lda, const void* B, int64_t ldb,
                    void* out, int64_t ldo, int32_t M, int32_t N, int32_t K,
                    const float* scale_a, const float* scale_b, void* workspace,
                    size_t workspace_bytes, void* stream);

/* out(M,N) bf16 = A(M,K) bf16 . B(N,K) bf16^T [+ bias(N)]: the out_proj GEMM
 * (mixers.py:801-803, 1304, 1400 -> ReplicatedLinear with bias). tcgen05 + TMA.
 * Requires K % 64 == 0, N % 8 == 0, 16-byte aligned rows.  Workspace ignored,
 * as above. */
HYENA_API int hyena_gemm_bf16(const void* A, int64_t lda, const void* B, int64_t ldb,
                    void* out, int64_t ldo, int32_t M, int32_t N, int32_t K,
                    const void* bias, void* workspace, size_t workspace_bytes,
                    void* stream);

/* The Hopper FP8 fast-accumulation GEMM model of the FP8-surgery layers
 * (fp8_emul.py:1-24 and 45-73; the exact-model GPU path behind
 * static_fp8_linear_emulated_triton, fp8_emul_triton.py:181-191, called from
 * mixers.py:701-705, 1085-1090):
 *   out(N,M) bf16 = (fast_accum(A, B) * (*scale_a)) * (*scale_b),
 * fast_accum: groups of 32 k, alignment exponent from the operand exponents,
 * every product truncated to the group's ulp, the accumulator kept to 13
 * fraction bits (bit-exact, CUDA cores).  A (N, K) e4m3 rows of lda (the
 * activations after hyena_quant_e4m3); B (K, M) bf16 holding E4M3 values, rows
 * of ldb (the checkpoints' `in_proj_emul_weight_t`).  K % 32 == 0. */
HYENA_API int hyena_gemm_fp8_emulated(const void* A, int64_t lda, const void* B, int64_t ldb,
                                      void* out, int64_t ldo, int32_t N, int32_t M, int32_t K,
                                      const float* scale_a, const float* scale_b, void* stream);

/* Bytes of workspace the GEMMs above use at this shape: always 0 (kept so that
 * callers written against ABI version 2 keep working).  fp8 != 0 selects e4m3. */
HYENA_API size_t hyena_gemm_workspace_size(int32_t M, int32_t N, int32_t K, int32_t fp8);

/* ---------------------------------------------------------------- decoder-layer norm
 * Evo2RMSNorm (model.py:47-76; its CUDA form triton_norm.py:127-156 rms_norm)
 * with the residual add and the in_proj input quantisation fused into one pass:
 *   s = x + residual (bf16; residual NULL: s = x), stored to s_out if non-NULL
 *       (s_out may alias x or residual: vLLM's in-place fused add-norm);
 *   y = weight * bf16(s / bf16(bf16(bf16(||s||_2) * H^-0.5) + eps)), bf16,
 *       stored to y if non-NULL;
 *   q = e4m3(clamp(y / *input_scale, +-448)), stored to q if non-NULL (the rule
 *       of hyena_quant_e4m3), so a Hyena layer's in_proj input never exists in
 *       bf16.
 * x, residual, s_out, y: (M, H) bf16 rows with strides that are multiples of 8
 * elements, 16-byte aligned; q: (M, H) e4m3 rows of ldq (multiple of 8), 8-byte
 * aligned; weight (H) bf16.  H % 8 == 0, H <= 16384; at least one output.  The
 * fp32 sum of squares runs in this kernel's order, not ATen's: n may differ
 * from the reference's in its last bf16 bit on rare rows. */
HYENA_API int hyena_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr,
                             const void* weight, float eps, void* s_out, int64_t lds, void* y,
                             int64_t ldy, void* q, int64_t ldq, const float* input_scale,
                             int32_t M, int32_t H, void* stream);

/* ---------------------------------------------------------------- speculative bookkeeping
 * Position stamps: one fp32 per state block at stamps + block * stamp_stride
 * (the last column of S2's first channel, mixers.py:952-957).
 *
 * Accepted token count per request from the stamps, replacing _spec_accepted
 * (mixers.py:962-984): first = slots[r * slot_stride]; offset = computed[r] -
 * stamp(first); accepted[r] = clamp(offset, 0, num_spec) + 1 (int32).  Where the
 * reference's device assert would fire (a non-null first slot with offset
 * outside [0, num_spec]) HYENA_FLAG_STAMP is set in *error_flags instead; a
 * first slot outside [0, num_blocks) sets HYENA_FLAG_BLOCK_RANGE (accepted 1). */
HYENA_API int hyena_spec_accepted(const int32_t* slots, int64_t slot_stride, int32_t num_reqs,
                                  const int32_t* computed, const float* stamps,
                                  int64_t stamp_stride, int32_t num_blocks, int32_t num_spec,
                                  int32_t* accepted, int32_t* error_flags, void* stream);

/* Stamps of the verifier slots after a decode / verify step, replacing the
 * decode half of _record_stamps (mixers.py:1040-1062): for p < min(q, starts[r+1]
 * - starts[r]), stamp(out_slots[r * s0 + p * s1]) = computed[r] + p + 1.  Block 0
 * (the null block, whose stamp is never consulted) is not written; the
 * reference writes 0 there for inactive positions. */
HYENA_API int hyena_spec_record(const int32_t* out_slots, int64_t s0, int64_t s1, int32_t num_reqs,
                                int32_t q, const int32_t* starts, const int32_t* computed,
                                float* stamps, int64_t stamp_stride, int32_t num_blocks,
                                int32_t* error_flags, void* stream);

/* Every shared-memory barrier wait inside the GEMMs and hyena_paged_attention
 * (which also sets HYENA_FLAG_WAIT) is bounded (4 s); a wait
 * that expires is counted in a per-device counter and the kernel finishes
 * without its tile being complete, so its output must not be trusted.  This
 * copies the current device's counter into *count (a synchronous read: call it
 * between steps, never during stream capture) and zeroes it when reset != 0.
 * A non-zero count is the GEMMs' error report.  No counterpart in the reference
 * (its GEMMs are library calls). */
HYENA_API int hyena_gemm_wait_timeouts(int32_t* count, int32_t reset);

/* Prefill stamps, replacing the prefill half of _record_stamps
 * (mixers.py:1070-1074): stamp(blocks[j * block_stride]) = seq_lens[j] for
 * j < n.  A block outside [0, num_blocks) sets HYENA_FLAG_BLOCK_RANGE. */
HYENA_API int hyena_spec_record_prefill(const int32_t* blocks, int64_t block_stride, int32_t n,
                                        const int32_t* seq_lens, float* stamps,
                                        int64_t stamp_stride, int32_t num_blocks,
                                        int32_t* error_flags, void* stream);

/* One paged state slice for whole-block copies: block b occupies block_bytes
 * contiguous bytes at data + b * block_stride_bytes (16-byte aligned, sizes in
 * whole 16-byte words).  data == NULL: slice absent. */
typedef struct hyena_state_block {
  void* data;
  int64_t block_stride_bytes;
  int64_t block_bytes;
} hyena_state_block;

/* Prefix-caching repair of resumed prefill rows, replacing
 * _repair_resumed_prefill_state (mixers.py:1001-1037).  For prefill row j
 * (dst = dst_blocks[j * dst_stride], src = src_blocks[j], n = computed[j]):
 * when has_init[j] != 0, neither block is the null block 0, stamp(dst) != n
 * and stamp(src) == n, the whole state of block src (every slice given) is
 * copied over block dst.  All decisions are taken from the stamps as they are
 * before any copy (first kernel, into the caller's take[num_rows] int32
 * buffer: source block or -1), then the copies run (second kernel).  Rows
 * whose blocks lie outside [0, num_blocks) set HYENA_FLAG_BLOCK_RANGE and are
 * not copied.  Distinct rows are assumed to name distinct destination blocks,
 * none of which is another repaired row's source (live requests never share
 * a block). */
HYENA_API int hyena_state_repair(int32_t num_rows, const int32_t* dst_blocks, int64_t dst_stride,
                                 const int32_t* src_blocks, const int32_t* computed,
                                 const uint8_t* has_init, const float* stamps,
                                 int64_t stamp_stride, int32_t num_blocks,
                                 const hyena_state_block* slices, int32_t num_slices,
                                 int32_t* take, int32_t* error_flags, void* stream);

/* Caps the CTAs of the persistent (large-M) GEMMs at n (n <= 0: one per SM,
 * the default).  Process-wide.  A caller that overlaps GEMMs with collectives
 * on another stream (channel-sharded out_proj all-reduces) leaves SMs free for
 * them this way.  No counterpart in the reference, which has no tensor
 * parallelism (mixers.py:38-41). */
HYENA_API void hyena_set_gemm_max_ctas(int32_t n);

/* enable != 0 (the default): kernels are launched with programmatic dependent
 * launch, so each can be scheduled while its stream predecessor drains (every
 * kernel still waits for that predecessor before touching global memory).
 * enable == 0: plain stream order, for callers that overlap these kernels with
 * work on other streams and want SMs released between kernels.  Process-wide.
 * No counterpart in the reference. */
HYENA_API void hyena_set_launch_chaining(int32_t enable);

/* ---------------------------------------------------------------- paged attention
 * The attention layers' key/value cache.  Row `at` of page p, head h:
 * k + p * k_page_stride + at * k_token_stride + h * k_head_stride (elements;
 * head_dim contiguous bf16), v alike.  Position j of request r lies in page
 * page_table[r * page_table_stride + j / page_size], row j % page_size; requests
 * may name the same pages.  page_size is a multiple of 16, head_dim 64 or 128,
 * strides multiples of 8 elements, bases 16-byte aligned.  A page outside
 * [0, num_pages), or a position beyond the table, sets HYENA_FLAG_BLOCK_RANGE
 * and is neither read nor written. */
typedef struct hyena_paged_kv {
  void* k;
  void* v;
  int64_t k_page_stride, k_token_stride, k_head_stride;
  int64_t v_page_stride, v_token_stride, v_head_stride;
  const int32_t* page_table;
  int64_t page_table_stride;
  int32_t pages_per_request; /* columns of page_table */
  int32_t num_pages;
  int32_t page_size;
  int32_t kv_heads;
  int32_t head_dim;
} hyena_paged_kv;

/* Rotary embedding (neox halves, Evo2Attention, model.py:104-152) of a step's
 * queries and keys, the keys and values written into the paged cache on the way:
 * for token t of request r at position p = positions[t],
 *   q_out[t] = rot(q[t], p);  cache.k[p] = rot(k[t], p);  cache.v[p] = v[t],
 * rot pairs element i with i + head_dim / 2 at angle p * theta^(-2i/head_dim),
 * formed in fp64, applied in fp32, rounded once.  Request r owns tokens
 * [query_start_loc[r], query_start_loc[r+1]) (NULL: token r only); tokens that no
 * request owns and tokens with a negative position are left alone, in q_out too.
 * q may be q_out (in place); q == q_out == NULL appends only.  No two tokens of a
 * step may name the same cache row. */
typedef struct hyena_kv_append_args {
  const void* q; int64_t q_token_stride, q_head_stride;          /* (T, heads, head_dim) bf16 */
  void* q_out; int64_t q_out_token_stride, q_out_head_stride;
  const void* k; int64_t k_token_stride, k_head_stride;          /* (T, kv_heads, head_dim) bf16 */
  const void* v; int64_t v_token_stride, v_head_stride;
  const int32_t* positions;        /* (T) */
  const int32_t* query_start_loc;  /* (num_requests + 1) or NULL */
  int32_t T;
  int32_t num_requests;
  int32_t heads;
  hyena_paged_kv kv;
  double rope_theta;
  int32_t* error_flags;            /* optional device int */
} hyena_kv_append_args;

HYENA_API int hyena_kv_append(const hyena_kv_append_args* a, void* stream);

/* Causal softmax attention of a step's queries over the paged cache: query i of
 * the n of request r sits at position seq_lens[r] - n + i and sees the keys
 * j <= that position (seq_lens counts the step's own tokens, appended before; where
 * it exceeds the page table, the keys that the table has).
 * A query that sees no key (seq_lens[r] = 0: a padded request) gives zeros;
 * output rows that no request owns are left alone; keys that a query does not see
 * do not touch its result, whatever they hold.  A range of query_start_loc that runs
 * past T or backwards sets HYENA_FLAG_SEGMENT; the rows that exist keep their positions.
 * Sharing: the requests [group_start[g], group_start[g+1]) (NULL: all, one group)
 * name the same key and value rows for their first shared_lens[g] positions,
 * which are then read once for the group.  What a query sees is not changed by
 * it: a run longer than what every query of the group sees is cut.
 * heads is a multiple of kv_heads (query head h reads head h / (heads / kv_heads)).
 * out may be q (same strides).
 * Up to four kernels on the stream (a plan, the shared runs of many rows, all other
 * keys, and joining the pieces of split rows).  The lengths are read on the device,
 * so captured calls serve growing contexts; the result has the same bits on every
 * call.  The workspace holds the call's plan and pieces: calls that may run at the
 * same time (two streams, two graphs replayed side by side) need one each. */
typedef struct hyena_paged_attention_args {
  const void* q; int64_t q_token_stride, q_head_stride;          /* (T, heads, head_dim) bf16 */
  void* out; int64_t out_token_stride, out_head_stride;
  const int32_t* seq_lens;         /* (num_requests) */
  const int32_t* query_start_loc;  /* (num_requests + 1) or NULL: token r only */
  const int32_t* shared_lens;      /* (num_groups) or NULL: nothing shared */
  const int32_t* group_start;      /* (num_groups + 1) or NULL */
  int32_t T;
  int32_t num_requests;            /* with num_groups at most 2048 */
  int32_t num_groups;              /* 0 with shared_lens NULL */
  int32_t heads;
  float scale;
  hyena_paged_kv kv;
  int32_t* error_flags;
} hyena_paged_attention_args;

/* Bytes of 16-byte aligned device memory the call needs (0 for invalid arguments). */
HYENA_API size_t hyena_paged_attention_workspace_size(const hyena_paged_attention_args* a);
HYENA_API int hyena_paged_attention(const hyena_paged_attention_args* a, void* workspace,
                                    size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------- gated projections
 * out(M,N) bf16 = act(A(M,K) . B1(N,K)^T) * (A . B2(N,K)^T), all bf16 with fp32
 * accumulators and one rounding: the first half of Evo2MLP (model.py:77-101);
 * hyena_gemm_bf16 with l3 is the second.  Same requirements as hyena_gemm_bf16. */
#define HYENA_ACT_NONE 0
#define HYENA_ACT_GELU 1  /* x Phi(x), with erf */
#define HYENA_ACT_SILU 2  /* x / (1 + exp(-x)) */
HYENA_API int hyena_gemm_gated_bf16(const void* A, int64_t lda, const void* B1, int64_t ldb1,
                                    const void* B2, int64_t ldb2, void* out, int64_t ldo, int32_t M,
                                    int32_t N, int32_t K, int32_t act, void* stream);

/* ---------------------------------------------------------------- misc */
HYENA_API int hyena_abi_version(void);
HYENA_API const char* hyena_last_error(void);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif /* HYENA_B200_H */
