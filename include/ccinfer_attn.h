/*
 * ccinfer_attn.h -- C ABI of the MI355X (gfx950) paged-attention hot path.
 *
 * Drop-in for the three kernel launchers of 7QiC/ccInfer declared in
 * src/kernel/cuda_kernels.h:61-84, with the same argument meaning, the same KV-cache layout
 * ([slot][num_kv_heads][head_dim] bf16, slot = block_id * cache_block_size + offset,
 * src/cache/kv_cache_storage.cpp:75-136) and the same block-table contract (int32
 * [batch][max_blocks_per_req], -1 padding, src/worker/batch_translator.cpp:213-293).
 *
 * Plain pointers and sizes only. All pointers except `stream` are device pointers.
 * `stream` is a hipStream_t (NULL = the default stream). Every call only enqueues work on
 * `stream`: no host synchronisation and no device allocation. Split-KV partials and the
 * prefill work list live in a caller-provided workspace sized by the *_workspace_size
 * queries (the reference launchers take no workspace; the C++ drop-in wrappers in
 * ccinfer_amd/csrc/dropin supply one owned per stream). Workspace contents need no
 * initialisation and are scratch between calls.
 *
 * Return value: 0 on success, otherwise the numeric value of the reference's
 * ccinfer::ErrorCode (src/base/error_code.h:8-45) -- the same codes the reference returns
 * through Result<void>.
 *
 * Thread safety: re-entrant. The C ABI keeps no global state except the per-device scratch
 * array of ccinfer_decode_attention_noalloc (and that array's cached device address), so
 * concurrent calls on different streams need only different workspaces -- apart from that
 * entry, whose calls on one GPU share the array. The C++ drop-in layer above it
 * (ccinfer_amd/csrc/dropin) adds one more piece of global state: the reference-signature
 * launchers' workspaces, one per (device, stream), reserved explicitly by
 * reserve_launcher_workspace and kept in a map behind a mutex (launches only read it; none
 * allocates). HipBackend holds its own reserved workspace and needs no global state.
 *
 * Alignment: the reference launchers accept any bf16 (2-byte aligned) view. The MFMA paths
 * move q, output and K/V cache rows in 16-byte pieces. A bf16 decode / prefill call whose
 * q or output view is only 2-byte aligned copies q (and, for prefill, output) into the
 * workspace, runs the MFMA kernels there and copies the output rows back (same bits as an
 * aligned call). A k_cache or v_cache pointer that is not 16-byte aligned runs the decode
 * MFMA kernels with 4-byte or 2-byte loads (same bits, ~1.1x / ~1.7x the time) and the
 * any-layout prefill tile kernel (~2.2x). The fp8 calls, which have the MFMA paths only, return
 * CCINFER_ERR_INVALID_ARGUMENT for any such pointer (and for k_scale / v_scale not 16-byte
 * aligned).
 */
#ifndef CCINFER_ATTN_H
#define CCINFER_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Numeric values of ccinfer::ErrorCode (src/base/error_code.h:8-45). */
enum ccinfer_status {
    CCINFER_OK = 0,
    CCINFER_ERR_DEVICE_OUT_OF_MEMORY = 1,  /* ErrorCode::CudaOutOfMemory   */
    CCINFER_ERR_LAUNCH_FAILED = 2,         /* ErrorCode::CudaLaunchFailed  */
    CCINFER_ERR_DEVICE_INVALID_VALUE = 3,  /* ErrorCode::CudaInvalidValue  */
    CCINFER_ERR_DEVICE_RUNTIME = 4,        /* ErrorCode::CudaRuntimeError  */
    CCINFER_ERR_INVALID_ARGUMENT = 6,      /* ErrorCode::InvalidArgument   */
    CCINFER_ERR_KV_EXHAUSTED = 12,         /* ErrorCode::KVBlockExhausted  */
    CCINFER_ERR_KV_INVALID_TABLE = 14,     /* ErrorCode::KVInvalidBlockTable */
    CCINFER_ERR_UNSUPPORTED = 26,          /* ErrorCode::Unsupported       */
    CCINFER_ERR_INTERNAL = 27              /* ErrorCode::InternalError     */
};

/* Replaces launch_write_kv_cache (src/kernel/cuda_kernels.h:80-83,
 * src/kernel/attention/write_kv_cache.cu:38-50).
 * k_new/v_new: [total_tokens][n_kv_heads][head_dim] bf16; k_cache/v_cache: one layer,
 * [max_slots][n_kv_heads][head_dim] bf16; slot_mapping: [total_tokens] int32. Tokens whose
 * slot is outside [0, max_slots) are skipped. Bit-exact copy. */
int ccinfer_write_kv_cache(const void* k_new, const void* v_new, void* k_cache, void* v_cache,
                           const int32_t* slot_mapping, int total_tokens, int n_kv_heads,
                           int head_dim, int max_slots, void* stream);

/* Fused attention prologue for one layer: replaces the five launches
 * launch_split_qkv, launch_rms_norm (q), launch_rms_norm (k), launch_rope and
 * launch_write_kv_cache (src/kernel/cuda_kernels.h, called in sequence by
 * src/model/qwen3/qwen3_model.cpp:174-244).
 * qkv: [num_tokens][(num_q_heads + 2 num_kv_heads) head_dim] bf16, the packed projection;
 * q_norm_weight, k_norm_weight: [head_dim] bf16 or NULL (no norm for that side);
 * positions: [num_tokens] int32; rope_cache: [rope_cache_max_position][head_dim/2] float
 * (cos, sin) pairs (src/model/rope_cache.cpp); q_out: [num_tokens][num_q_heads][head_dim]
 * bf16; k_cache/v_cache as in ccinfer_write_kv_cache. Rotation is skipped for positions
 * outside [0, rope_cache_max_position); tokens whose slot is outside [0, max_slots) write no
 * K/V. head_dim must be even and at most 1024; eps > 0 (backend.h:84). Results match the five reference kernels
 * in sequence (bf16 rounding between steps, the same reduction order). */
int ccinfer_qkv_prologue(const void* qkv, const void* q_norm_weight, const void* k_norm_weight,
                         const int32_t* positions, const void* rope_cache,
                         const int32_t* slot_mapping, void* q_out, void* k_cache, void* v_cache,
                         int num_tokens, int num_q_heads, int num_kv_heads, int head_dim,
                         int rope_cache_max_position, int max_slots, float eps, void* stream);

/* Item flags of ccinfer_build_batch_metadata. */
#define CCINFER_ITEM_DECODE 1 /* decode item: exactly one new token, always sampled */
#define CCINFER_ITEM_SAMPLE 2 /* prefill chunk whose last token needs logits */

/* Builds one step's attention metadata on the device, replacing the host array building
 * and uploads of BatchTranslator::translate (src/worker/batch_translator.cpp:213-302,
 * 305-420) and ModelRunner's blocking copy-back validation (src/model/model_runner.h:
 * 102-171). Inputs (device, int32): per item i < batch_size the tokens already in the
 * cache (item_kv_written), the new tokens (item_new_tokens), flags (CCINFER_ITEM_*), and
 * its block list after this step's allocation, as blocks[item_block_start[i] ..
 * item_block_start[i + 1]) (total_blocks entries in all; blocks may be NULL when 0).
 * Outputs (device, int32): positions[num_tokens], slot_mapping[num_tokens],
 * block_table[batch_size][max_blocks_per_req] (-1 padded), query_start_loc[batch_size + 1],
 * context_lens[batch_size], logits_indices[batch_size] (-1 = no sample), exactly as the
 * reference's host loops write them; and status[0] = 0, or CCINFER_ERR_INVALID_ARGUMENT
 * when a check of model_runner.h fails (entries that fail are written as -1). The status
 * word is written by every call (no clearing needed) and is read by the caller when it
 * chooses -- the call itself never synchronises. */
int ccinfer_build_batch_metadata(const int32_t* item_kv_written, const int32_t* item_new_tokens,
                                 const int32_t* item_flags, const int32_t* item_block_start,
                                 const int32_t* blocks, int batch_size, int num_tokens,
                                 int total_blocks, int max_blocks_per_req, int block_size,
                                 int num_cache_blocks, int32_t* positions, int32_t* slot_mapping,
                                 int32_t* block_table, int32_t* query_start_loc,
                                 int32_t* context_lens, int32_t* logits_indices, int32_t* status,
                                 void* stream);

/* Workspace bytes ccinfer_decode_attention (and ccinfer_decode_attention_fp8) needs for this
 * batch shape; 0 for invalid shapes. The figure includes two copies of the
 * q rows, which only a call with a 2-byte-aligned q or output uses; an aligned call accepts
 * a workspace that much smaller. */
size_t ccinfer_decode_workspace_size(int batch_size, int max_blocks_per_req, int num_q_heads,
                                     int num_kv_heads, int head_dim, int cache_block_size);

/* Replaces launch_decode_attention (src/kernel/cuda_kernels.h:72-77,
 * src/kernel/attention/decode_attn.cu:515-570).
 * q, output: [batch_size][num_q_heads][head_dim] bf16; block_table: [batch_size]
 * [max_blocks_per_req] int32; context_lens: [batch_size] int32, including the current
 * token (whose K/V must already be written). cache_block_size must be 16 and head_dim one
 * of {32,64,80,96,112,120,128,192,256} (as in the reference); all of them run the MFMA
 * kernels (32, 96 and 192 in tiles of their own; 80 and 112-120 padded to 128 with
 * zeros), for any query group
 * size (groups above 16 heads run as several groups of at most 16 over the same KV head).
 * Unlike the reference, there is no
 * context-length ceiling (split-KV). Batches of at most 16 (request, q-head) rows with
 * table rows of at most 512 positions run in a single launch and need no workspace. */
int ccinfer_decode_attention(const void* q, const void* k_cache, const void* v_cache,
                             const int32_t* block_table, const int32_t* context_lens,
                             void* output, int batch_size, int max_blocks_per_req,
                             int num_q_heads, int num_kv_heads, int head_dim,
                             int cache_block_size, void* workspace, size_t workspace_bytes,
                             void* stream);

/* One decode step: ccinfer_write_kv_cache of each request's new token into the slot of its
 * last position, then ccinfer_decode_attention. No single counterpart in the reference: it
 * replaces the pair launch_write_kv_cache + launch_decode_attention
 * (src/kernel/cuda_kernels.h:61-77) as src/model/qwen3/qwen3_model.cpp:230-262 issues them
 * for a decode batch, where token b is request b's newest position. k_new, v_new:
 * [batch_size][num_kv_heads][head_dim] bf16. The slot of request b's token is derived from
 * its table row: block_table[b][(ctx_b - 1) / 16] * 16 + (ctx_b - 1) % 16; rows with ctx_b
 * outside [1, max_blocks_per_req * 16], a negative block id there or a slot >= max_slots
 * write nothing (their output follows ccinfer_decode_attention). Requirement (true of any
 * decode batch): no other request of the batch reads those slots. On the MFMA path the
 * writes happen inside the decode launch (the wavefront that reads the slot writes it
 * first); otherwise a separate launch writes them first. Workspace as
 * ccinfer_decode_workspace_size. */
int ccinfer_decode_attention_write_kv(const void* q, const void* k_new, const void* v_new,
                                      void* k_cache, void* v_cache, const int32_t* block_table,
                                      const int32_t* context_lens, void* output, int batch_size,
                                      int max_blocks_per_req, int num_q_heads, int num_kv_heads,
                                      int head_dim, int cache_block_size, int max_slots,
                                      void* workspace, size_t workspace_bytes, void* stream);

/* Workspace bytes ccinfer_decode_attention_shared_prefix needs for this batch shape. */
size_t ccinfer_decode_shared_workspace_size(int batch_size, int max_blocks_per_req,
                                            int num_q_heads, int num_kv_heads, int head_dim,
                                            int cache_block_size);

/* ccinfer_decode_attention for batches whose requests share cached prompt prefixes. No
 * single counterpart in the reference: its prefix cache hands several requests the same
 * leading block ids (KVCacheManager::lookup_prefix_cache, src/cache/kv_cache_manager.cpp:
 * 93-173, counted in BlockTable::shared_count, src/cache/block.h:85-97), and its decode
 * then reads those blocks once per request. Here the call finds, on the device, the groups
 * of requests whose table rows start with the same block ids and attends each group's
 * common prefix (whole 32-token chunks before every member's last position) once per
 * subgroup of up to 16 / (num_q_heads / num_kv_heads) requests, which fill one MFMA tile
 * together; positions after the prefix, and requests in no group, run as in
 * ccinfer_decode_attention, and the parts are combined by the log-sum-exp merge. Same
 * arguments, semantics and tolerance as ccinfer_decode_attention; a batch in which nothing
 * is shared gives the same bits. Shapes outside the fast path (query groups above 8 heads,
 * more than 2048 requests, misaligned views, non-16 blocks) run ccinfer_decode_attention
 * (the workspace size covers it). */
int ccinfer_decode_attention_shared_prefix(const void* q, const void* k_cache,
                                           const void* v_cache, const int32_t* block_table,
                                           const int32_t* context_lens, void* output,
                                           int batch_size, int max_blocks_per_req,
                                           int num_q_heads, int num_kv_heads, int head_dim,
                                           int cache_block_size, void* workspace,
                                           size_t workspace_bytes, void* stream);

/* ccinfer_decode_attention without a workspace and without any allocation. No counterpart
 * in the reference: for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc). The split-KV scratch is
 * one static 32 MiB device array per GPU, resolved on the first call on each device and
 * held until the process ends; shapes whose ccinfer_decode_workspace_size exceeds 32 MiB
 * return CCINFER_ERR_INVALID_ARGUMENT (configs of batch 64 x 4096 or 32 x 32768 tokens need
 * under 9 MiB). Calls that overlap on one GPU (concurrent streams) share the array and
 * race; otherwise identical results to ccinfer_decode_attention. */
int ccinfer_decode_attention_noalloc(const void* q, const void* k_cache, const void* v_cache,
                                     const int32_t* block_table, const int32_t* context_lens,
                                     void* output, int batch_size, int max_blocks_per_req,
                                     int num_q_heads, int num_kv_heads, int head_dim,
                                     int cache_block_size, void* stream);

/* fp8 KV cache (no counterpart in the reference, whose cache is bf16 only; its KV profile
 * list, src/base/traits.h:117-124, anticipates other element types). Same [slot][n_kv_heads]
 * [head_dim] layout and block-table contract, one OCP E4M3 byte per element, plus one fp32
 * scale per cache row in k_scale / v_scale, indexed ((slot / 16) * n_kv_heads + kv_head) * 16
 * + slot % 16 (arrays of ceil(max_slots / 16) * 16 * n_kv_heads floats). A row x is stored
 * as e4m3(clamp(x / P, +-448)) with scale P, the smallest power of two >= 2^-126 with
 * max|x| <= 448 P (round to nearest even; an all-zero row stores zeros and scale 0; what an
 * element that is a NaN stores is not defined); its value is byte * scale. The attention entries accept any fp32 scale; a power of two takes
 * the faster conversion in the fp8 prefill. Halves decode bytes.
 *
 * Replaces launch_write_kv_cache (src/kernel/cuda_kernels.h:80-83) for an fp8 cache:
 * quantises each new token's K and V rows into its slot; tokens whose slot is outside
 * [0, max_slots) are skipped. head_dim even, <= 512. */
int ccinfer_write_kv_cache_fp8(const void* k_new, const void* v_new, void* k_cache,
                               void* v_cache, float* k_scale, float* v_scale,
                               const int32_t* slot_mapping, int total_tokens, int n_kv_heads,
                               int head_dim, int max_slots, void* stream);

/* Replaces launch_decode_attention (src/kernel/cuda_kernels.h:72-77) for an fp8 cache: the
 * same semantics, plan and workspace (ccinfer_decode_workspace_size) as
 * ccinfer_decode_attention, with K/V read as byte * row scale. head_dim 64, 128 or 256
 * (CCINFER_ERR_UNSUPPORTED otherwise). */
int ccinfer_decode_attention_fp8(const void* q, const void* k_cache, const void* v_cache,
                                 const float* k_scale, const float* v_scale,
                                 const int32_t* block_table, const int32_t* context_lens,
                                 void* output, int batch_size, int max_blocks_per_req,
                                 int num_q_heads, int num_kv_heads, int head_dim,
                                 int cache_block_size, void* workspace, size_t workspace_bytes,
                                 void* stream);

/* Workspace bytes ccinfer_prefill_attention (and the fp8 / overlap variants) needs for this
 * batch shape; 0 for invalid shapes. As for decode, it includes two copies of
 * the q rows used only by a call with a 2-byte-aligned q or output. It also includes the
 * memory in which a batch that fills at most half the GPU keeps the partial rows of its query
 * tiles, whose key ranges it splits over more workgroups (head dims up to 64: 17 MB where a table
 * row holds more than 1,984 positions; up to 128: 34 MB, more than 1,088); a call given a
 * workspace that much smaller is accepted and runs its tiles whole. */
size_t ccinfer_prefill_workspace_size(int batch_size, int total_query_tokens,
                                      int max_blocks_per_req, int num_q_heads,
                                      int num_kv_heads, int head_dim, int cache_block_size);

/* Replaces launch_prefill_attention (src/kernel/cuda_kernels.h:61-66,
 * src/kernel/attention/prefill_attn.cu:246-279).
 * q, output: [total_query_tokens][num_q_heads][head_dim] bf16; query_start_loc:
 * [batch_size + 1]; context_lens[r] = prefix_r + query_len_r; query i of request r sees
 * cache positions [0, prefix_r + i]. Mixed batches (single-token decode items next to
 * prompt chunks) are accepted, as in the reference. head_dim <= 256. As in the reference,
 * neither the batch size nor the table length is bounded. The MFMA path covers every
 * query group size and head dims that are multiples of 8 up to 128 (at any size; those
 * below 64 / 128 run padded with zeros) or multiples of 16 up to 256 (up to 4096 blocks per
 * table row, counted in 16-token blocks), with cache blocks of any multiple of 16 tokens
 * (read through a 16-token table the call builds in the workspace). Other block sizes,
 * head dims up to 256 and table lengths run an MFMA tile kernel that stages rows
 * element-wise. A mixed batch's decode items run on `stream` ahead of the prompt tiles. */
int ccinfer_prefill_attention(const void* q, const void* k_cache, const void* v_cache,
                              const int32_t* block_table, const int32_t* query_start_loc,
                              const int32_t* context_lens, void* output, int batch_size,
                              int total_query_tokens, int max_blocks_per_req, int num_q_heads,
                              int num_kv_heads, int head_dim, int cache_block_size,
                              void* workspace, size_t workspace_bytes, void* stream);

/* ccinfer_prefill_attention with the decode items of a mixed batch (of at least 32
 * requests) run on the caller's side_stream (a hipStream_t) concurrently with the prompt
 * tiles on `stream`: the call records fork_event on `stream`, makes side_stream wait for
 * it, and joins back by recording join_event on side_stream and making `stream` wait for it
 * -- event records and waits only, so it can be captured into a graph. fork_event and
 * join_event are caller-owned hipEvent_t (hipEventDisableTiming is enough); side_stream
 * NULL runs as ccinfer_prefill_attention. No counterpart in the reference (one stream);
 * HipBackend owns such a side stream. Concurrent calls must not share the side stream's
 * events. */
int ccinfer_prefill_attention_overlap(const void* q, const void* k_cache, const void* v_cache,
                                      const int32_t* block_table,
                                      const int32_t* query_start_loc,
                                      const int32_t* context_lens, void* output, int batch_size,
                                      int total_query_tokens, int max_blocks_per_req,
                                      int num_q_heads, int num_kv_heads, int head_dim,
                                      int cache_block_size, void* workspace,
                                      size_t workspace_bytes, void* stream, void* side_stream,
                                      void* fork_event, void* join_event);

/* Replaces launch_prefill_attention (src/kernel/cuda_kernels.h:61-66) for an fp8 cache
 * (layout and scales as for ccinfer_write_kv_cache_fp8): the same semantics, planner and
 * workspace (ccinfer_prefill_workspace_size) as ccinfer_prefill_attention, with K/V read as
 * byte * row scale; single-token requests of a mixed batch go through the fp8 decode.
 * head_dim 64 or 128 and at most 4096 blocks per table row on the MFMA path
 * (CCINFER_ERR_UNSUPPORTED otherwise). */
int ccinfer_prefill_attention_fp8(const void* q, const void* k_cache, const void* v_cache,
                                  const float* k_scale, const float* v_scale,
                                  const int32_t* block_table, const int32_t* query_start_loc,
                                  const int32_t* context_lens, void* output, int batch_size,
                                  int total_query_tokens, int max_blocks_per_req,
                                  int num_q_heads, int num_kv_heads, int head_dim,
                                  int cache_block_size, void* workspace, size_t workspace_bytes,
                                  void* stream);

/* ccinfer_prefill_attention_fp8 with the decode items of a mixed batch on side_stream, as
 * for ccinfer_prefill_attention_overlap. */
int ccinfer_prefill_attention_fp8_overlap(
    const void* q, const void* k_cache, const void* v_cache, const float* k_scale,
    const float* v_scale, const int32_t* block_table, const int32_t* query_start_loc,
    const int32_t* context_lens, void* output, int batch_size, int total_query_tokens,
    int max_blocks_per_req, int num_q_heads, int num_kv_heads, int head_dim,
    int cache_block_size, void* workspace, size_t workspace_bytes, void* stream,
    void* side_stream, void* fork_event, void* join_event);

/* ---- rotary positions ---------------------------------------------------------------
 * How the frequencies of a table are scaled for contexts past the trained length. `params`
 * is an array on the host: [0] factor, [1] the original number of positions, [2] and [3] the
 * fast and slow bounds in turns over that length, [4] the factor m of cos and sin (0: the
 * scaling's own), and for CCINFER_ROPE_FACTORS the pairs' own divisors from [5] on. */
enum ccinfer_rope_scaling {
    CCINFER_ROPE_NONE = 0,    /* f_p = theta^(-2p / rotary_dim); params unused             */
    CCINFER_ROPE_LINEAR = 1,  /* f_p / factor                                              */
    CCINFER_ROPE_NTK = 2,     /* theta * factor^(rotary_dim / (rotary_dim - 2))            */
    CCINFER_ROPE_YARN = 3,    /* a ramp over the pairs from f_p to f_p / factor, between the
                                 pairs that make `fast` and `slow` turns; m = 0.1 ln factor + 1 */
    CCINFER_ROPE_BANDS = 4,   /* f_p where a pair makes `fast` turns or more, f_p / factor at
                                 `slow` or fewer, blended linearly in the turns between    */
    CCINFER_ROPE_FACTORS = 5  /* f_p / params[5 + p]                                       */
};

/* Frequencies of the rotary_dim / 2 pairs (radians a position) and m, on the host in double
 * precision; touches no device. rotary_dim even and at most 512, theta > 1, factor >= 1,
 * fast > slow > 0. */
int ccinfer_rope_frequencies(int rotary_dim, double theta, int scaling, const double* params,
                             double* frequencies, double* magnitude);

/* rope_cache[i][p] = m (cos, sin)((first_position + i) f_p), float [num_positions]
 * [rotary_dim / 2][2], the table that the calls below and ccinfer_qkv_prologue read (the
 * reference fills one on the host, src/model/rope/rope_cache.cpp). `frequencies` is a host
 * array that the call has read when it returns (at most 65536 radians each); angles are
 * reduced in double precision: an entry is off by 2^-22 m and 2^-51 of its angle. May be
 * captured into a graph. */
int ccinfer_build_rope_cache(const double* frequencies, int rotary_dim, double magnitude,
                             int first_position, int num_positions, void* rope_cache,
                             void* stream);

/* Rotates every head of q [num_tokens][num_q_heads][head_dim] and k (NULL with num_kv_heads
 * 0: none) bf16 by table row positions[t] (launch_rope, src/kernel/pos/rope.cu:14-43, whose
 * rotary_dim is head_dim and whose pairs are p, p + rotary_dim / 2). interleaved: the pairs
 * are 2p, 2p + 1. Elements from rotary_dim on, and rows whose position is outside
 * [0, rope_cache_max_position), are copied. inverse: the opposite angle (the gradient's
 * direction). Strides in elements; a head's elements are contiguous. q_out / k_out may be
 * q / k themselves (same pointer and strides), or memory apart from them. Float32 inside,
 * rounded once. head_dim even, at most 1024. */
int ccinfer_rotary_embedding(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                             const void* k, int64_t k_token_stride, int64_t k_head_stride,
                             const int32_t* positions, const void* rope_cache, void* q_out,
                             int64_t q_out_token_stride, int64_t q_out_head_stride, void* k_out,
                             int64_t k_out_token_stride, int64_t k_out_head_stride,
                             int num_tokens, int num_q_heads, int num_kv_heads, int head_dim,
                             int rotary_dim, int rope_cache_max_position, int interleaved,
                             int inverse, void* stream);

/* ccinfer_qkv_prologue with float32 inside and one rounding at the end, for models and caches
 * that it does not take: y = x rsqrt(mean x^2 + eps) (w + weight_offset) of each q and k head
 * (a NULL weight: no norm for that side; *_per_head: the weights are [heads][head_dim], else
 * [head_dim]; eps at least 2^-126; a row whose sum of squares passes float32's largest number
 * becomes zeros), the rotation of ccinfer_rotary_embedding, q to q_out [num_tokens]
 * [num_q_heads][head_dim], K and V to their slots of a bf16 cache, or, with k_scale and
 * v_scale, of an fp8 cache (layout and quantisation of ccinfer_write_kv_cache_fp8, straight
 * from the float32 rows; a NaN is stored as E4M3's NaN, which that call does not promise).
 * qkv rows lie qkv_token_stride elements apart; q_out and the caches lie apart from them.
 * Tokens whose slot is outside [0, max_slots) write no K/V; no two tokens may have the same
 * slot. */
int ccinfer_qkv_norm_rope(const void* qkv, int64_t qkv_token_stride, const void* q_norm_weight,
                          int q_norm_per_head, const void* k_norm_weight, int k_norm_per_head,
                          const int32_t* positions, const void* rope_cache,
                          const int32_t* slot_mapping, void* q_out, void* k_cache, void* v_cache,
                          float* k_scale, float* v_scale, int num_tokens, int num_q_heads,
                          int num_kv_heads, int head_dim, int rotary_dim,
                          int rope_cache_max_position, int max_slots, int interleaved, float eps,
                          float weight_offset, void* stream);

/* ---- pages of the cache ---------------------------------------------------------------
 * Operators on the pool of blocks of all layers at once. k_cache / v_cache: layer 0 of
 * [num_layers][num_blocks][cache_block_size][n_kv_heads][head_dim], bf16, or fp8 bytes with
 * k_scale / v_scale; layer_stride in bytes and scale_layer_stride in floats lead from one
 * layer to the next (unused for one layer). A block of one layer's K has at most 2^30 bytes;
 * an fp8 cache has cache_block_size 16. The scales of an fp8 cache start as zeros (or anything
 * finite): the attention multiplies those of a block's slots that hold no token by 0.
 *
 * ref_counts [num_blocks] says how many table rows (or other owners, a prefix cache say) hold
 * a block; 0 is free. A block that is given up more often than it was counted ends below 0:
 * it is not handed out again, and a row that still holds it gets
 * CCINFER_ERR_KV_INVALID_TABLE. CCINFER_ERR_UNSUPPORTED for more than 2^24 blocks in the calls
 * that take counts, 2^14 items of an update and 2^17 pairs of a copy. */

/* Block dst_blocks[i] becomes a copy of src_blocks[i] in every layer, K, V and scales. Pairs
 * with a block outside [0, num_blocks), and of a block with itself, are skipped. Pairs that
 * depend on an order (a destination that is another pair's destination with another source,
 * or another pair's source) are skipped too, and *status, if not NULL, is set to
 * CCINFER_ERR_INVALID_ARGUMENT; it is not written otherwise. */
int ccinfer_copy_kv_blocks(void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                           const int32_t* src_blocks, const int32_t* dst_blocks, int num_pairs,
                           int num_layers, int64_t layer_stride, int64_t scale_layer_stride,
                           int num_blocks, int n_kv_heads, int head_dim, int cache_block_size,
                           int32_t* status, void* stream);

/* Workspace bytes of ccinfer_update_block_tables (0 for an invalid shape). */
size_t ccinfer_update_tables_workspace_size(int num_items, int max_blocks_per_req,
                                            int num_blocks);

/* Changes rows of block_table [num_rows][max_blocks_per_req] (-1 padded) and context_lens
 * [num_rows], and the counts with them. Item i makes row dst_rows[i] hold the first
 * min(lengths[i], context of src_rows[i]) tokens of row src_rows[i] as it was before the call
 * (-1: of none; src_rows NULL: of the row itself), followed by blocks for the tokens up to
 * lengths[i] (-1, or lengths NULL: the source's context):
 *   fork      (child, parent, -1)         admit    (row, -1, tokens)
 *   grow      (row, row, more tokens)     truncate (row, row, fewer tokens)
 *   release   (row, -1, 0)                beams    (row, the beam it goes on from, -1)
 * Whole blocks are shared. A last block that is filled in part has one owner: where it is
 * shared, or would be, its tokens are copied to a block of the row's own. New blocks are the
 * lowest-numbered ones that were free before the call, in item order; what the call releases
 * is free after it. *status (on the device, always written): CCINFER_OK, or, with nothing
 * changed, CCINFER_ERR_INVALID_ARGUMENT (a row or length out of range, two items of one row,
 * a copy needed but neither caches nor lists given), CCINFER_ERR_KV_INVALID_TABLE (a context outside the
 * row, a block outside the pool or with a count below 1 among those held), or
 * CCINFER_ERR_KV_EXHAUSTED. copy_src / copy_dst [num_items], or both NULL: the block that item
 * i copied and its copy, -1 where it copied none or the call failed. Caches NULL with
 * num_layers 0: tables and counts alone; the copies are then the caller's, from these two
 * lists (ccinfer_copy_kv_blocks for each layer held by itself). */
int ccinfer_update_block_tables(int32_t* block_table, int32_t* context_lens, int32_t* ref_counts,
                                const int32_t* dst_rows, const int32_t* src_rows,
                                const int32_t* lengths, int num_items, int num_rows,
                                int max_blocks_per_req, void* k_cache, void* v_cache,
                                float* k_scale, float* v_scale, int num_layers,
                                int64_t layer_stride, int64_t scale_layer_stride, int num_blocks,
                                int n_kv_heads, int head_dim, int cache_block_size,
                                int32_t* copy_src, int32_t* copy_dst, int32_t* status,
                                void* workspace, size_t workspace_bytes, void* stream);

/* Workspace bytes of ccinfer_compact_kv_blocks (0 for an invalid shape). */
size_t ccinfer_compact_workspace_size(int num_blocks);

/* Moves the live blocks (count not 0) into blocks [0, *num_live): those that lie past it,
 * lowest first, to the free blocks below it, lowest first; the others stay. Writes the tables
 * with the new numbers (entries of free blocks and past the pool become -1, negative ones stay), the
 * counts, and remap [num_blocks]: each block's new number, -1 for a free one. The outputs may
 * be the inputs (block_table_out = block_table, ref_counts_out = ref_counts). num_rows 0: no
 * tables. */
int ccinfer_compact_kv_blocks(const int32_t* block_table, const int32_t* ref_counts, int num_rows,
                              int max_blocks_per_req, void* k_cache, void* v_cache,
                              float* k_scale, float* v_scale, int num_layers,
                              int64_t layer_stride, int64_t scale_layer_stride, int num_blocks,
                              int n_kv_heads, int head_dim, int cache_block_size,
                              int32_t* block_table_out, int32_t* ref_counts_out, int32_t* remap,
                              int32_t* num_live, void* workspace, size_t workspace_bytes,
                              void* stream);

/* ---- drafted tokens ---------------------------------------------------------------------
 * A step that checks several drafted tokens a request at once. Request b has n = query_start_loc
 * [b + 1] - query_start_loc[b] nodes; context_lens[b] counts them, as prefill does its new tokens:
 * node i lies at position context_lens[b] - n + i of the cache, whatever its depth in the tree.
 * parents[t] is the request's node from which node t goes on (lower than its own number), -1 for
 * one that goes on from the committed context. At most 2048 requests a call (1024 of the attention)
 * and 2048 nodes a request. The reference decodes one token a request and step (src/backend/params.h:148-211). */

/* From parents [total_tokens]: tree_mask [total_tokens][mask_words] (bit j of a row, bit j % 32 of
 * word j / 32: the node sees the request's node j; its ancestors and itself), positions
 * [total_tokens] (of rotary embeddings: committed tokens + depth) and slot_mapping [total_tokens]
 * (cache slot of each node, blocks of 16 tokens). mask_words at least max_nodes / 32, rounded up.
 * status [batch_size]: CCINFER_OK, or CCINFER_ERR_INVALID_ARGUMENT for a request with more than
 * max_nodes nodes, fewer context tokens than nodes, or nodes outside [0, total_tokens) (its rows
 * then get no mask, position -1 and slot -1), with a parent out of range (taken as -1) or without
 * a block for a node, or one whose slots pass 32 bits (slot -1). Rows of no request, before the first
 * one's nodes or behind the last one's (a padded batch), get no mask, position -1 and slot -1. */
int ccinfer_build_draft_tree(const int32_t* parents, const int32_t* query_start_loc,
                             const int32_t* context_lens, const int32_t* block_table,
                             int batch_size, int total_tokens, int max_blocks_per_req,
                             int max_nodes, int mask_words, int cache_block_size,
                             int32_t* tree_mask, int32_t* positions, int32_t* slot_mapping,
                             int32_t* status, void* stream);

/* Workspace bytes of ccinfer_tree_attention (0 for an invalid or unsupported shape). */
size_t ccinfer_tree_attention_workspace_size(int batch_size, int total_query_tokens,
                                             int max_blocks_per_req, int mask_words,
                                             int num_q_heads, int num_kv_heads, int head_dim,
                                             int cache_block_size);

/* ccinfer_prefill_attention with a mask among the new tokens in place of their order: row i of
 * request b sees the positions before its request's nodes and node j where bit j of tree_mask
 * [query_start_loc[b] + i] is set (any mask, also one without itself; a node past the mask's words
 * is seen by none). Sums are held times up to 2^8: of V from 2^119 on they may pass float32, and a
 * row of an fp8 cache that holds an infinity may make NaN of its other elements. Rows that see nothing become zeros; rows of no request, and of requests whose
 * context is shorter than their nodes, are left as they are. A node's K and V that a row does not
 * see do not reach it, infinities and NaN included. k_scale / v_scale NULL: a bf16 cache, head_dim
 * a multiple of 8 up to 256; else an fp8 cache (ccinfer_write_kv_cache_fp8), head_dim 64 or 128;
 * CCINFER_ERR_UNSUPPORTED for others, for more than 1024 requests or 64 mask words, and for batches
 * whose rows and tables together pass 2^30 units of work. q, caches, scales and output 16-byte
 * aligned; num_kv_heads * head_dim below 2^23. The workspace needs no initialisation. */
int ccinfer_tree_attention(const void* q, const void* k_cache, const void* v_cache,
                           const float* k_scale, const float* v_scale, const int32_t* block_table,
                           const int32_t* query_start_loc, const int32_t* context_lens,
                           const int32_t* tree_mask, void* output, int batch_size,
                           int total_query_tokens, int max_blocks_per_req, int mask_words,
                           int num_q_heads, int num_kv_heads, int head_dim, int cache_block_size,
                           void* workspace, size_t workspace_bytes, void* stream);

/* What the model confirms of the trees. target_tokens[t] is the token that the model says after
 * node t. The path of a request starts at node 0 (the token the last step ended with, always
 * taken) and goes on to the lowest child whose draft_tokens entry equals its parent's target.
 * accepted [batch_size]: its length; accepted_nodes [total_tokens]: its nodes, from the request's
 * first row on, -1 behind them; tokens [total_tokens]: the new tokens, target_tokens of those
 * nodes, -1 behind them (the last one is the next step's node 0); context_lens_out [batch_size]:
 * the context without the nodes that were not taken. K and V (and scales) of the k-th node of the
 * path move to the position behind the committed tokens that k counts, in every layer of the
 * caches (as in the calls on pages; caches NULL with num_layers 0: none, and a later call with the
 * same arguments for each layer moves them). Blocks that hold nodes belong to one request alone.
 * A row without a block in the pool is not moved. A request without nodes, with more than 2048,
 * with fewer context tokens than nodes or with nodes outside [0, total_tokens): accepted 0, its
 * context as it is. Rows of no request keep what accepted_nodes and tokens hold. Outputs lie apart
 * from the inputs (CCINFER_ERR_INVALID_ARGUMENT where one is an input). The plan's status is not
 * looked at: see ccinfer_accept_planned_tokens. */
int ccinfer_accept_draft_tokens(const int32_t* draft_tokens, const int32_t* target_tokens,
                                const int32_t* parents, const int32_t* query_start_loc,
                                const int32_t* context_lens, const int32_t* block_table,
                                int batch_size, int total_tokens, int max_blocks_per_req,
                                void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                                int num_layers, int64_t layer_stride, int64_t scale_layer_stride,
                                int num_blocks, int n_kv_heads, int head_dim, int cache_block_size,
                                int32_t* accepted, int32_t* accepted_nodes, int32_t* tokens,
                                int32_t* context_lens_out, void* stream);

/* ccinfer_accept_draft_tokens after ccinfer_build_draft_tree's status [batch_size] (NULL: none). Nodes
 * of a request whose status is not CCINFER_OK have no mask, slot or block, or not all of them, so that
 * what the model says after them means nothing: it accepts 0, nothing of it moves, and its context
 * loses the nodes (context_lens without them, where it has as many). */
int ccinfer_accept_planned_tokens(const int32_t* draft_tokens, const int32_t* target_tokens,
                                  const int32_t* parents, const int32_t* query_start_loc,
                                  const int32_t* context_lens, const int32_t* block_table,
                                  const int32_t* status, int batch_size, int total_tokens,
                                  int max_blocks_per_req, void* k_cache, void* v_cache,
                                  float* k_scale, float* v_scale, int num_layers,
                                  int64_t layer_stride, int64_t scale_layer_stride, int num_blocks,
                                  int n_kv_heads, int head_dim, int cache_block_size,
                                  int32_t* accepted, int32_t* accepted_nodes, int32_t* tokens,
                                  int32_t* context_lens_out, void* stream);

/* ---- decode over selected blocks of the context ----------------------------------------
 * Decode that reads the blocks in which a query's weight can lie. Beside each layer's K lie
 * key_bounds, bf16 [num_blocks][num_kv_heads][2][head_dim]: the smallest and the largest of each
 * block's keys, element by element (1/16 of a bf16 cache's bytes, about 1/8 of an fp8 one's). Blocks
 * of 16 tokens. Several query tokens of one request are rows of their own, with the same table row,
 * in all of these calls. */

/* The bounds of the blocks that hold the newest tokens of each row, query_start_loc[b + 1] -
 * query_start_loc[b] of them (query_start_loc NULL: one; no fewer than were written or moved since
 * the last call), over all their positions below context_lens[b]. A key that is NaN makes both
 * bounds of its element NaN. With k_scale: an fp8 cache; bounds are rounded to bf16 where a scale
 * is no power of two. Of rows that share a block (several query tokens of one request), the longest
 * context counts. At most 2048 rows (CCINFER_ERR_UNSUPPORTED). head_dim a multiple of 8 up to 256,
 * num_kv_heads * head_dim below 2^23. */
int ccinfer_update_key_bounds(const void* k_cache, const float* k_scale, void* key_bounds,
                              const int32_t* block_table, const int32_t* context_lens,
                              const int32_t* query_start_loc, int batch_size,
                              int max_blocks_per_req, int num_kv_heads, int head_dim,
                              int cache_block_size, void* stream);

/* scores [batch_size][num_kv_heads][max_blocks_per_req] float: for block j of the row the largest,
 * over the query heads of the kv head, of sum_d max(q_d lo_d, q_d hi_d) / sqrt(head_dim): no key
 * of the block gives a larger logit (but for float32's rounding, and that of the bounds of an fp8
 * cache). -infinity past the context, for negative table entries, and
 * for rows whose context the table does not hold; NaN where a bound or q is NaN, NaN or an
 * infinity where a bound is infinite. */
int ccinfer_score_kv_blocks(const void* q, const void* key_bounds, const int32_t* block_table,
                            const int32_t* context_lens, float* scores, int batch_size,
                            int max_blocks_per_req, int num_q_heads, int num_kv_heads,
                            int head_dim, int cache_block_size, void* stream);

/* selected [batch_size][num_kv_heads][num_selected]: the row's first `first_blocks` and last
 * `last_blocks` blocks, and of the others those with the highest scores (NaN before all, equal
 * ones by the lower number), in ascending order; all of them where they are no more than
 * num_selected; -1 behind them. num_selected at least first_blocks + last_blocks; at most 2^16
 * blocks a row (CCINFER_ERR_UNSUPPORTED). */
int ccinfer_select_kv_blocks(const float* scores, const int32_t* context_lens, int batch_size,
                             int max_blocks_per_req, int num_kv_heads, int num_selected,
                             int first_blocks, int last_blocks, int cache_block_size,
                             int32_t* selected, void* stream);

/* Workspace bytes of ccinfer_sparse_decode_attention (0: none needed, or an invalid shape). */
size_t ccinfer_sparse_decode_workspace_size(int batch_size, int num_q_heads, int num_kv_heads,
                                            int head_dim, int num_selected, int cache_block_size);

/* Decode attention of each (row, kv head) over the positions below context_lens[b] that lie in its
 * blocks selected [batch_size][num_kv_heads][num_selected] (numbers within the row; ones outside
 * the context, and of negative table entries, are passed over; one that is named twice counts
 * twice). Zeros for a row that sees nothing or whose context the table does not hold. Caches, head
 * dims, alignment and the range of V as in ccinfer_tree_attention. */
int ccinfer_sparse_decode_attention(const void* q, const void* k_cache, const void* v_cache,
                                    const float* k_scale, const float* v_scale,
                                    const int32_t* block_table, const int32_t* context_lens,
                                    const int32_t* selected, void* output, int batch_size,
                                    int max_blocks_per_req, int num_q_heads, int num_kv_heads,
                                    int head_dim, int num_selected, int cache_block_size,
                                    void* workspace, size_t workspace_bytes, void* stream);

/* Human-readable text for a status code (the reference's error_message()). */
const char* ccinfer_error_message(int code);

/* Library version, "major.minor.patch". */
const char* ccinfer_version(void);

#ifdef __cplusplus
}
#endif

#endif /* CCINFER_ATTN_H */
