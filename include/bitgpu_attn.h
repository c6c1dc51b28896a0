/* bitgpu_attn.h -- C ABI of the MI355X (gfx950) attention hot path.
 *
 * Drop-in replacement for the per-layer attention dispatch of bitgpu v0.19.1's WebGPU engine
 * (src/engine.ts). Every entry point names the reference interface it replaces (file:line,
 * relative to the reference repository root).
 *
 * Conventions
 *   - All functions return int32_t status: BG_OK (0) or a negative BG_E_* code; the message of
 *     the last failure on the calling thread is in bg_last_error_message(). Nothing throws.
 *   - Device buffers are plain device pointers (hipMalloc'd or torch-owned); host buffers are
 *     plain host pointers. No framework types cross this boundary.
 *   - `stream` is a hipStream_t passed as void* (NULL = the default stream). Work is enqueued
 *     in order on that stream; calls return before the GPU finishes unless stated otherwise.
 *   - A cache object is not re-entrant: calls on one cache must be serialized by the caller
 *     (the reference serializes every engine op through one promise chain, src/engine.ts:2877-2887),
 *     and all GPU work on one cache must be ordered on ONE stream: the layers of a cache share
 *     one split workspace and one f16 prefill copy, so two bg_attention calls on different
 *     streams could overlap on the GPU and corrupt each other's partials.
 *   - Kernels never allocate. Host-side allocations happen only in bg_kv_create, bg_kv_grow,
 *     bg_attention_reserve, lazily on the first bg_attention that needs more workspace (the
 *     decode's split partials; 33 MiB for a split-K prefill's, which runs unsplit, in several times
 *     the time, where it cannot have them, as in a capture that was not reserved for) or, for a q8 or
 *     sink-mode cache, the f16 copy a long prefill runs on, and in the snapshot transfers (16 MiB of
 *     pinned memory for the process; region by region a staging buffer kept by the cache, grown when
 *     a larger region is transferred).
 *   - The decode kernel's split merge waits a bounded time for the partials of its own grid.
 *     If a wait gives up (the GPU shared with work that keeps the grid from running at once),
 *     that launch stores NaN and raises the cache's error word; the next bg_attention on the
 *     cache, or bg_stream_sync, returns BG_E_DEVICE once and resets the workspace. Until then,
 *     outputs of later launches on the cache may be wrong (a partial that lands after its
 *     merger gave up can be taken by a later launch), not only NaN.
 *   - When the device dispatches workgroups to its XCDs round robin (probed once per device at
 *     bg_kv_create), the decode kernel exchanges the split partials of a kv head through one
 *     XCD's L2. A merger that finds itself on another XCD raises the error word as above and
 *     the library writes partials through to memory from then on.
 *
 * Storage modes mirror EngineOptions.kvCache (src/types.ts:143-154): f32, f16 (one RNE rounding
 * at write, shaders/copy_kv16.wgsl:13) and q8 (int8 codes + one f32 scale per 32 values,
 * shaders/copy_kv8.wgsl:24-40). The device layout is private (head-major, V stored in
 * 32-position transposed tiles); bg_kv_export_rows / bg_kv_import_rows convert to and from the
 * reference's snapshot byte layout (src/engine.ts:2724-2734).
 */
#ifndef BITGPU_ATTN_H
#define BITGPU_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define BG_OK 0
#define BG_E_INVALID (-1)     /* bad argument */
#define BG_E_OOM (-2)         /* device allocation failed (the reference's GpuOutOfMemoryError) */
#define BG_E_DEVICE (-3)      /* HIP runtime error */
#define BG_E_UNSUPPORTED (-4) /* shape or mode this build does not implement */
#define BG_E_STATE (-5)       /* not valid in the cache's current state */

enum { BG_KV_F32 = 0, BG_KV_F16 = 1, BG_KV_Q8 = 2 };
enum { BG_K = 0, BG_V = 1, BG_KSCALE = 2, BG_VSCALE = 3 };
enum { BG_ROPE_SLOT = 0, BG_ROPE_ABSOLUTE = 1 };

typedef struct bg_kv_cache bg_kv_cache;

/* ---- utilities ------------------------------------------------------------------------- */

/* Last failure message on this thread ("" if none). Replaces the Error('bitgpu: ...') text of
 * src/errors.ts:14-19. */
const char* bg_last_error_message(void);

/* Library version string. */
const char* bg_version(void);

/* RoPE tables f32 [positions, rot_dim/2]: f64 angles p * theta^(-2j/rot_dim), each entry
 * rounded once to f32; YaRN when yarn_factor > 1 (beta_fast 32, beta_slow 1, mscale
 * 0.1 ln(factor) + 1). Host-only. Replaces synthRope, src/engine.ts:117-147. */
int32_t bg_rope_tables(double theta, int32_t rot_dim, int32_t positions, double yarn_factor,
                       int32_t yarn_original_max_positions, float* cos_out, float* sin_out);

/* Sink-mode eviction arithmetic (host-only, no cache): evict(fill, need) of
 * src/engine.ts:1188-1212. Outputs the new fill, the dropped batch and the kept count. */
int32_t bg_evict_plan(int32_t fill, int32_t need, int32_t sinks, int32_t max_seq_len,
                      int32_t* new_fill, int32_t* batch, int32_t* keep);

/* Sink-mode ring map (host-only): the physical slot holding logical slot `logical` when the
 * ring origin is `head` (logical slots < sinks are fixed; the rest rotate through
 * max_seq_len - sinks slots). With bg_evict_plan it reproduces the reference's compaction
 * (src/engine.ts:1206-1209) as pure index arithmetic. */
int32_t bg_ring_map(int32_t sinks, int32_t max_seq_len, int32_t head, int32_t logical, int32_t* physical);

/* Synchronize a stream (NULL = device). Also reports (BG_E_DEVICE, once) a decode split merge
 * on any live cache that gave up waiting, after resetting that cache's workspace. */
int32_t bg_stream_sync(void* stream);

/* Host-only diagnostic with no counterpart in the reference (the WebGPU kernels have no
 * split-K): the plan bg_attention's split-K decode kernel uses for S query rows of H heads at
 * positions pos_base.. over a plain cache of kv_heads x head_dim (dtype BG_KV_F16 or
 * BG_KV_Q8), on num_cus CUs holding resident_per_cu of its workgroups at once. out[0..5] =
 * waves per workgroup, splits per kv head, 32-slot tiles per split, merging splits per kv
 * head (the last ones), grid size, tiles. The grid never exceeds resident_per_cu * num_cus.
 * A q8 launch of 4-wave workgroups whose waves would take two tiles at one workgroup a CU takes
 * one tile a wave when resident_per_cu >= 2 and the GPU holds that grid (bg_attention runs a
 * one-tile kernel that fits two workgroups a CU there).
 * BG_E_UNSUPPORTED when the shape goes to another kernel. */
int32_t bg_decode_plan(int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t S, int32_t H,
                       int32_t pos_base, int32_t num_cus, int32_t resident_per_cu, int32_t* out);

/* The same for the f32 prefill at head_dim 128: out[0..3] = waves of a workgroup (of four) that
 * share 32 rows (0: each its own rows, the keys shared through LDS, one part), queries per workgroup,
 * parts the key range is split into, 64-key steps per part.
 * window > 0: a sink-mode ring of that many slots with `sinks` sinks and origin `head`; partials 0:
 * a launch that has no buffer for split partials. */
int32_t bg_f32_prefill_plan(int32_t kv_heads, int32_t S, int32_t H, int32_t pos_base, int32_t window,
                            int32_t sinks, int32_t head, int32_t num_cus, int32_t partials, int32_t* out);

/* Test hook with no counterpart in the reference: the decode split merge's poll bound
 * (spin_limit polls before a merger gives up; 0 = the default, 2^20) and one split index that
 * stores no partial (-1 = none), for every later bg_attention / bg_attention_noalloc call in
 * the process. With a small bound and a withheld split the merge gives up while every kernel
 * exits normally (the error path of the bounded wait, forced from the host). Host-only. */
int32_t bg_debug_merge_hooks(int32_t spin_limit, int32_t withhold_split);

/* Measurement aid with no counterpart in the reference: the streaming-read floor the decode
 * kernels are held against. `workgroups` workgroups of 512 threads each read one contiguous
 * slice of the device buffer `buf` (`bytes`, a multiple of 16) with 16-byte loads, eight in
 * flight a lane, nontemporal (the decode tiles' policy) or plain, and fold them by XOR into
 * sink[workgroup] (device memory, `workgroups` words). The XOR of the sink words equals the XOR
 * of the buffer's 32-bit words. Asynchronous on `stream`; allocates nothing. */
int32_t bg_diag_stream_read(const void* buf, size_t bytes, int32_t workgroups, int32_t nontemporal,
                            uint32_t* sink, void* stream);

/* ---- streams and event timing -------------------------------------------------------------
 * For hosts without a GPU runtime of their own (the N-API addon): the reference runs every
 * dispatch on its one WebGPU queue and times with timestamp queries (src/engine.ts:503-506);
 * here a stream is that queue (default priority; NULL = the null stream in every call) and
 * two recorded events give the elapsed time between them (bg_event_elapsed_us waits for
 * `end`). */
int32_t bg_stream_create(void** stream);
int32_t bg_stream_destroy(void* stream);
int32_t bg_event_create(void** event);
int32_t bg_event_record(void* event, void* stream);
int32_t bg_event_elapsed_us(void* start, void* end, float* us);
int32_t bg_event_destroy(void* event);

/* ---- KV cache lifecycle ------------------------------------------------------------------
 * Replaces the Kc/Vc/Ksc/Vsc allocation of src/engine.ts:1044-1079, the kvCache/overflow/
 * sinkTokens/maxSeqLen options (src/types.ts:138-177) and the roll statics (1094-1111).
 * One kv head's K (or V) region of one layer must stay below 2^31 bytes (f32: 4 bytes a value,
 * f16 and q8 2, counting a q8 layer's f16 prefill copy): max_seq_len x head_dim x that at most
 * 2^31 - 1 after rounding up to 32 positions, e.g. at most 4,194,272 positions of f16 at head_dim
 * 256; a larger one is BG_E_UNSUPPORTED. */
int32_t bg_kv_create(int32_t n_layers, int32_t kv_heads, int32_t head_dim, int32_t dtype,
                     int32_t capacity, int32_t max_seq_len, int32_t roll, int32_t sinks,
                     int32_t rope_pos_mode, bg_kv_cache** out);
int32_t bg_kv_destroy(bg_kv_cache* cache);

/* Current capacity in positions. */
int32_t bg_kv_capacity(const bg_kv_cache* cache, int32_t* capacity);

/* ensureKvCapacity, src/engine.ts:1120-1178: grow every layer to >= min(needed, max_seq_len)
 * positions (doubling), preserving content. On allocation failure the cache keeps its old
 * buffers and BG_E_OOM is returned (the reference's rollback, 1157-1173). Synchronous. */
int32_t bg_kv_grow(bg_kv_cache* cache, int32_t needed, void* stream);

/* q8 scale block (src/types.ts:145-147: the reference quantizes per 32 values,
 * shaders/copy_kv8.wgsl:30-36): 32 (the default) or head_dim, one scale per (position, kv head)
 * row -- the row's maximum |value|, stored in each of the row's head_dim/32 scale slots, so the
 * cache layout, the attention kernels and the snapshot format are the same in both modes.
 * Applies to the writes that follow. BG_E_STATE for a cache that is not q8. */
int32_t bg_kv_set_q8_block(bg_kv_cache* cache, int32_t block);

/* Device rope tables [positions, rot_dim/2] used for the sink-mode read-time K rotation
 * (the rollCosT/rollSinT bindings of attIns, src/engine.ts:1097-1104,1395-1399). The caller
 * owns the buffers; they must cover max_seq_len positions (slot mode) or every absolute
 * position attended (absolute mode). */
int32_t bg_kv_set_rope(bg_kv_cache* cache, const float* cos_tab, const float* sin_tab,
                       int32_t positions, int32_t rot_dim);

/* ---- KV writes ---------------------------------------------------------------------------- */

/* appendKV, src/engine.ts:1385-1393 (copy.wgsl / copy_kv16.wgsl / copy_kv8.wgsl): `rows` f32
 * rows of head_dim values, row r landing at reference cache row dst_row0 + r, i.e. logical
 * position (dst_row0 + r) / kv_heads and kv head (dst_row0 + r) % kv_heads. which = BG_K|BG_V. */
int32_t bg_kv_write(bg_kv_cache* cache, int32_t layer, int32_t which, const float* src,
                    int32_t rows, int32_t dst_row0, void* stream);

/* Fused attention prologue for S positions in one launch, replacing (src/engine.ts)
 *   decode : rmsnorm_rope_sg(Q) + ROPE_K / rmsnorm_rope_sg_kv8(K into the cache) + appendKV(V)
 *            (1527-1540; shaders/rmsnorm_rope_sg*.wgsl)
 *   prefill: rms(q), rms(k), rope(q), rope(k), appendKV(K), appendKV(V) (1569-1576)
 *   hybrid : split_head(query) + rms + rope_partial (q and k) + appendKV(K, V) (1470-1485)
 * q: [S, H, q_stride] (first head_dim values of each row are the query; q_stride = 2*head_dim
 * reads the hybrid's interleaved query|gate projection), k, v: [S, KV, head_dim]. Any of q, k,
 * v may be NULL to skip that part. Q rows are RMSNormed with q_gamma, roped at pos0 + s and
 * written to q_out [S, H, head_dim]; K rows are normed with k_gamma, roped at pos0 + s (left
 * unroped in a sink-mode cache, which rotates at read) and stored at logical slot slot0 + s;
 * V rows are stored unchanged at slot0 + s. Tables cos_tab/sin_tab: [rope_positions,
 * rot_dim/2] (the engine's cos/sin caches, indexed by position instead of the per-call [S, D]
 * expansion of ropeBufs, src/engine.ts:994-1009); rot_dim <= head_dim (dims >= rot_dim pass
 * through). Every buffer is 16-byte aligned and q_stride a multiple of 4 (rows move 16 bytes a
 * lane); otherwise BG_E_INVALID. */
int32_t bg_qkv_prologue(bg_kv_cache* cache, int32_t layer, const float* q, int32_t q_stride,
                        const float* k, const float* v, int32_t S, int32_t H,
                        const float* q_gamma, const float* k_gamma, float eps,
                        const float* cos_tab, const float* sin_tab, int32_t rope_positions,
                        int32_t rot_dim, int32_t pos0, int32_t slot0, float* q_out, void* stream);

/* ---- 1-bit projections on either side of attention (decode, M = 1) -------------------------
 * Weights as the engine uploads them (src/engine.ts:814-830): row n, weight k is bit k % 32 of
 * sign[n][k / 32] (u32; set = +1, clear = -1) times scales[n][k / 128] (f32); K a multiple of
 * 128; x, sign and scales 16-byte aligned. */

/* fusedMM, matmul_split_sg.wgsl (src/engine.ts:1344-1360, e.g. the qkv and gate/up weights):
 * the N0 + N1 + N2 rows of W x, rows [0, N0) to out0, [N0, N0+N1) to out1, the rest to out2. */
int32_t bg_gemv_split(const float* x, int32_t K, const uint32_t* sign, const float* scales,
                      int32_t N0, int32_t N1, int32_t N2, float* out0, float* out1, float* out2,
                      void* stream);

/* residMM, matmul_resid_mr_sg.wgsl (src/engine.ts:1364-1380, o_proj at 1547 and down_proj):
 * y = W x + resid over N rows. */
int32_t bg_gemv_resid(const float* x, int32_t K, const uint32_t* sign, const float* scales,
                      int32_t N, const float* resid, float* y, void* stream);

/* The decode qkv projection fused with the attention prologue, replacing src/engine.ts:1526-1540
 * (matmul_split_sg into q, k, v; appendKV(V); rmsnorm_rope_sg(Q); ROPE_K / rmsnorm_rope_sg_kv8
 * writing K into the cache): one token, x = the normed hidden state [K]. The weight's rows are
 * the H query heads, then the cache's kv_heads key heads, then its value heads, head_dim rows
 * each (the fused qkv weight of src/engine.ts:850). Q heads are RMSNormed with q_gamma and roped
 * at `pos` into q_out [H, head_dim]; K heads normed with k_gamma, roped at `pos` (unroped in a
 * sink-mode cache) and stored at logical slot `slot`; V heads stored at `slot`. Tables as in
 * bg_qkv_prologue (16-byte aligned). H + 2 * kv_heads <= 1024. The arithmetic of the norm and
 * the rotation is bg_qkv_prologue's: the result equals bg_gemv_split followed by
 * bg_qkv_prologue bit for bit. */
int32_t bg_qkv_proj_prologue(bg_kv_cache* cache, int32_t layer, const float* x, int32_t K,
                             const uint32_t* sign, const float* scales, int32_t H,
                             const float* q_gamma, const float* k_gamma, float eps,
                             const float* cos_tab, const float* sin_tab, int32_t rope_positions,
                             int32_t rot_dim, int32_t pos, int32_t slot, float* q_out, void* stream);

/* ---- attention ---------------------------------------------------------------------------
 * runN(ATT, [S,H,KV,D,posBase,Ltot], attIns(qr, li), att, S*H), src/engine.ts:1543,1579-1580
 * (attention_{sg,wg}{,_kv16,_kv8}{,_roll}.wgsl) and the hybrid
 * attention_online_cache{,_kv8} + gate_sigmoid, src/engine.ts:1486-1491.
 * q: [S, H, head_dim] f32 (already normed/roped); query s sits at logical slot pos_base + s and
 * attends every resident slot <= pos_base + s. scale: the softmax scale (the dense kernels use
 * 1/sqrt(head_dim), attention_sg.wgsl:24; the hybrid passes 1/sqrt(head_dim) as a param).
 * gate (nullable): [S, H, gate_stride], out = attn / (1 + exp(-gate)) (gate_sigmoid.wgsl:13).
 * out: [S, H, head_dim] f32. Rows per kv head (S x H / KV) that fit one 16-row set run the
 * split-K decode kernel (and so does sink mode up to 48 rows at head_dim 128 and 20 at 256, and
 * q8 at head_dim 128 up to 24);
 * more run the MFMA prefill kernel, whose grid is split along the key range (a second kernel
 * merging the parts) when it holds far fewer query blocks than the GPU has CUs; f32 storage runs
 * an exact-f32 kernel. */
int32_t bg_attention(bg_kv_cache* cache, int32_t layer, const float* q, int32_t S, int32_t H,
                     int32_t pos_base, float scale, const float* gate, int32_t gate_stride,
                     float* out, void* stream);

/* Allocation-free variant of bg_attention. No counterpart in the reference (WebGPU dispatches
 * never allocate per call); it is for callers that cannot call hipMalloc: code under HIP graph
 * capture, tight serving loops, harnesses that forbid allocation. Same arguments and results as
 * bg_attention, but it allocates nothing: the split partials of the decode kernel (8 MiB per GPU)
 * and of a split-K prefill (33 MiB, as much as any plan needs) live in a file-scope device array,
 * held until the process ends, instead of the cache's workspace; a q8 or sink-mode prefill
 * dequantizes and rotates in-kernel instead of through the f16 copy (the same values: identical
 * output); an f32 cache runs the f32 matrix-core kernel for every shape, decode included
 * (agrees with bg_attention to f32 rounding). A decode
 * launch whose partials would exceed its 8 MiB is rejected with BG_E_INVALID before anything runs.
 * The first call on a device sets the array up (a fill kernel, synchronized) and must not be
 * under graph capture (BG_E_STATE). Every call on one GPU shares that GPU's array: calls that
 * overlap on the GPU (different streams, or different host threads) race and corrupt each
 * other's outputs -- order them on one stream. */
int32_t bg_attention_noalloc(bg_kv_cache* cache, int32_t layer, const float* q, int32_t S, int32_t H,
                             int32_t pos_base, float scale, const float* gate, int32_t gate_stride,
                             float* out, void* stream);

/* Pre-size the split-K workspace for up to S query rows of H heads (otherwise sized on first
 * use), and for a q8 or sink-mode cache whose prefill of S rows runs on an f16 copy of the
 * attended slots, allocate that copy; for a prefill of S rows that can split along the key range
 * (an f32 one at head_dim 128: any), the 33 MiB of its partials. Call before capturing bg_attention into a HIP graph (a launch under capture
 * cannot allocate). A later call that needs a larger workspace allocates a new one and keeps the
 * old one until bg_kv_destroy, so launches captured before stay valid. BG_E_OOM where a buffer
 * cannot be had, except the partials of an f32 cache and the copy of a sink-mode one: launches run
 * without these. */
int32_t bg_attention_reserve(bg_kv_cache* cache, int32_t S, int32_t H);

/* ---- sink-mode eviction (overflow 'sinks') ------------------------------------------------
 * evict / evictFor, src/engine.ts:1187-1214. The cache is a ring behind the sinks: eviction
 * advances the ring head by the reference's batch, so the resident set and its slot order match
 * the reference's memmove compaction without moving any bytes. */
int32_t bg_kv_evict(bg_kv_cache* cache, int32_t fill, int32_t need, int32_t* new_fill);
int32_t bg_kv_evict_for(bg_kv_cache* cache, int32_t fill, int32_t n, int32_t* new_fill);

/* Ring origin and the number of rows evicted so far (absolute position of logical slot
 * L >= sinks is L + evicted). */
int32_t bg_kv_ring_state(const bg_kv_cache* cache, int32_t* head, int64_t* evicted);

/* Put the sink-mode ring into its compacted state: origin 0, `evicted` rows evicted before
 * logical slot `sinks` (0 for a new conversation). The reference's cache is always compacted
 * (evict() moves the kept rows to slot `sinks`, src/engine.ts:1206-1209), so a v2 snapshot
 * restore (restoreCache, src/engine.ts:2807-2872) writes logical slots 0..cacheLen-1 into this
 * state, and a fresh conversation (cacheLen = 0) starts from it. Contents are not touched. */
int32_t bg_kv_ring_reset(bg_kv_cache* cache, int64_t evicted);

/* ---- snapshot wire format -----------------------------------------------------------------
 * Per-region export/import in the reference snapshot layout (src/engine.ts:2724-2734,
 * 2757-2771, 2847-2860): region BG_K / BG_V is [count, KV, head_dim] elements of the storage
 * type (f32, f16, or int8 codes = the little-endian bytes of the reference's packed u32 words),
 * BG_KSCALE / BG_VSCALE is [count, KV, head_dim/32] f32 (q8 only). Positions are logical
 * slots base .. base+count-1. host: host pointer. Synchronous. */
int32_t bg_kv_region_bytes(const bg_kv_cache* cache, int32_t region, int32_t count, size_t* bytes);
int32_t bg_kv_export_rows(bg_kv_cache* cache, int32_t layer, int32_t region, int32_t base,
                          int32_t count, void* host, void* stream);
int32_t bg_kv_import_rows(bg_kv_cache* cache, int32_t layer, int32_t region, int32_t base,
                          int32_t count, const void* host, void* stream);

/* A whole snapshot's KV bytes at once, the same layout (per layer the K, V and q8 KSCALE, VSCALE
 * regions of positions base .. base+count-1; src/engine.ts:2757-2771, 2847-2860): `bytes` must be
 * their sum over layers. Through 16 MiB of pinned staging, shared by the process's caches, kept
 * until the last one is destroyed. A transfer that finds it in use by another cache's, cannot have
 * it, or whose positions exceed a 2 MiB slot goes region by region as above. Synchronous. */
int32_t bg_kv_save(bg_kv_cache* cache, int32_t base, int32_t count, void* host, size_t bytes, void* stream);
int32_t bg_kv_load(bg_kv_cache* cache, int32_t base, int32_t count, const void* host, size_t bytes, void* stream);

/* ---- paged KV cache: many sequences in one pool ---------------------------------------------
 * No counterpart in the reference, whose engine holds one conversation: the same layers for a batch of
 * conversations. A pool holds, per layer, n_pages pages of page_size positions (32, 64, 128 or 256); a
 * sequence is a list of pages, and sequences may list the same leading pages (a common system prompt, a
 * forked conversation), whose keys and values are then stored and, by bg_paged_attention, scanned once.
 * The memory is the caller's (device, 16-byte aligned), one buffer a region for all layers:
 *   BG_K       [layer][page][kv_head][slot][head_dim]                     of the storage type
 *   BG_V       [layer][page][kv_head][slot / 32][4][head_dim][8]          of the storage type: slot
 *              16 a + 8 c + 4 b + r of a 32-slot tile (a, b, c in 0..1, r in 0..3) at [2 a + b][dim][4 c + r]
 *   BG_KSCALE, BG_VSCALE (q8) [layer][page][kv_head][slot][head_dim / 32] f32, a value code * scale / 127
 * It need not be cleared: slots that no call wrote are never used, whatever they hold. Calls are not
 * re-entrant on one batch, whose launches share a workspace and read the arrays that bg_paged_batch_set
 * uploads: a call on another stream than the batch's last one waits there for what the batch enqueued before
 * (that stream still exists, and is not being captured), and replays of a graph that holds its launches are
 * the caller's to order with its other calls. Batches of one pool may use different streams where none reads
 * a page that another writes. Every call needs the pool's device current. */
typedef struct bg_paged_kv bg_paged_kv;
typedef struct bg_paged_batch bg_paged_batch;

/* Bytes of a pool's region (BG_K, BG_V, BG_KSCALE, BG_VSCALE; the scales of f32 and f16: 0). Host-only. */
int32_t bg_paged_region_bytes(int32_t n_layers, int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t page_size,
                              int32_t n_pages, int32_t region, size_t* bytes);
/* A pool over the caller's buffers, which outlive it (scales NULL unless q8). head_dim 128 or 256;
 * n_pages * page_size below 2^31, n_layers * kv_heads up to 2^22. */
int32_t bg_paged_create(int32_t n_layers, int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t page_size,
                        int32_t n_pages, void* k, void* v, float* k_scale, float* v_scale, bg_paged_kv** out);
int32_t bg_paged_destroy(bg_paged_kv* kv);
/* As bg_kv_set_q8_block. */
int32_t bg_paged_set_q8_block(bg_paged_kv* kv, int32_t block);

/* A batch of at most max_seqs sequences with max_tokens new rows and max_pages listed pages in all, for H
 * query heads. Allocates its arrays (pinned and device); needs no pool but one of this geometry. */
int32_t bg_paged_batch_create(const bg_paged_kv* kv, int32_t H, int32_t max_seqs, int32_t max_tokens, int32_t max_pages,
                              bg_paged_batch** out);
int32_t bg_paged_batch_destroy(bg_paged_batch* batch);
/* What the next calls work on (host arrays, read before the call returns): sequence s holds lens[s]
 * positions, its last rows[s] (0 to lens[s]) new, in the pages tables[s * table_stride ..] (the first
 * ceil(lens[s] / page_size) are read). The batch's rows are numbered 0 .. sum(rows) - 1, sequence by
 * sequence. positions: the new tokens' rotary positions [axes][sum(rows)], axes 1 to 4; NULL: their
 * positions in the sequence. Checks everything (BG_E_INVALID, the batch before stays set), plans the
 * attention (runs of pages that sequences share are found here) and uploads it on `stream` (BG_E_DEVICE from
 * the upload: to be set again). May allocate the workspace of partials (BG_E_OOM, the batch before stays set);
 * not under graph capture (BG_E_STATE). Launches captured in a graph read the
 * batch at replay, so a batch may be set between replays: with at most as many new rows as were captured and,
 * where a prologue was, the same number of axes and positions inside its rope table (of q or k) and no page
 * that it may not write (of k or v), else BG_E_STATE; for as long as the batch lives, and it outlives the graph. */
int32_t bg_paged_batch_set(bg_paged_batch* batch, int32_t n_seqs, const int32_t* rows, const int32_t* lens,
                           const int32_t* tables, int32_t table_stride, const int32_t* positions, int32_t axes, void* stream);
/* Diagnostic of the batch that is set: out[0..5] = new rows, workgroups of the attention, runs of shared
 * pages, positions scanned (a shared run's once), rows that are merged from partials, partials. */
int32_t bg_paged_batch_info(const bg_paged_batch* batch, int64_t* out);
/* As bg_paged_batch_info, out[0..3] = workgroups of 128, of 32 and of 16 rows, and 1 where the last kind's pages
 * (read once, more than caches keep) pass the caches by. */
int32_t bg_paged_batch_units(const bg_paged_batch* batch, int64_t* out);

/* bg_qkv_prologue for a batch: its rows' q [rows, H, q_stride], k and v [rows, kv_heads, head_dim] (any
 * may be NULL); normed and roped q into q_out [rows, H, head_dim], normed and roped k and plain v into
 * the sequences' pages at the rows' positions, the same bits as bg_qkv_prologue's. pair_axis (host,
 * rot_dim / 2 entries, NULL where the batch has one axis): which axis of the batch's positions each rotary
 * pair (dims j and j + rot_dim / 2) takes its angle from, e.g. time, height and width for images, in
 * sections or interleaved. q_out may be q where q_stride is head_dim, and overlaps no other input. The tables
 * need rope_positions rows above every position. A page that a
 * sequence writes must not be listed, with the written positions, by another one or twice (BG_E_INVALID);
 * rows of q_out and slots beyond the batch's are left as they are. */
int32_t bg_paged_qkv_prologue(const bg_paged_kv* kv, int32_t layer, bg_paged_batch* batch, const float* q, int32_t q_stride,
                              const float* k, const float* v, const float* q_gamma, const float* k_gamma, float eps,
                              const float* cos_tab, const float* sin_tab, int32_t rope_positions, int32_t rot_dim,
                              const uint8_t* pair_axis, float* q_out, void* stream);

/* bg_attention for a batch: row i of sequence s attends positions 0 .. lens[s] - rows[s] + i of its pages
 * (what they hold by then, the batch's own rows included). q, out [rows, H, head_dim] f32 (16-byte
 * aligned), scale positive and below 2^127, gate [rows, H, gate_stride] or NULL, out = attn / (1 +
 * exp(-gate)). out may be a gate of gate_stride head_dim, and overlaps no other input. Allocates nothing. Rows
 * of out beyond the batch's are left as they are.
 * Results are f32-accurate for every storage type and do not depend on which other sequences are in the
 * batch beyond that rounding: a probability counts with 22 bits or to 2^-32 of the largest, whichever is
 * more, of its position's value (f16) or of the largest scale that its 32-dim block has in the sequence
 * (q8); f32 pages round as f32 sums do. |values| from 2^100 on may overflow in the sums. A key that
 * is not finite reaches the rows that attend it, a value those and, by its factor of zero, new rows of the
 * sequence before it. */
int32_t bg_paged_attention(const bg_paged_kv* kv, int32_t layer, bg_paged_batch* batch, const float* q, float scale,
                           const float* gate, int32_t gate_stride, float* out, void* stream);

/* ---- linear attention with a decay for each head ---------------------------------------------------------
 * The hybrid's other layers (three in four): no keys and values are kept but, per conversation and value head,
 * one matrix. For a row with key k, query q (of key head h / (v_heads / k_heads)), value v, decay g <= 0 and
 * write strength beta:
 *   S <- e^g S + k (beta (v - e^g S^T k))^T     beta NULL: S <- e^g S + k v^T        out = scale S^T q
 * A cache holds them for n_slots conversations (slots) of n_layers layers, in the caller's device memory (f32,
 * 16-byte aligned), with the last inputs of the layer's causal convolution:
 *   state  [layer][slot][v_head][v_dim][k_dim]            (a row: what a value dim has of every key dim)
 *   conv   [layer][slot][conv_width - 1][channels]        channels = q heads | k heads | v heads, oldest first
 * Slots need not be cleared. A batch names the sequences of the next calls; its calls are not re-entrant and
 * follow each other on whatever streams they are made, as the paged batch's do (above), and it may be set again
 * between replays of a graph that holds its launches, with at most as many new rows as were captured; replays
 * are the caller's to order with the batch's other calls. Batches of one cache may use different streams where
 * none reads a slot that another writes. Every call needs the cache's device current. */
typedef struct bg_linear_cache bg_linear_cache;
typedef struct bg_linear_batch bg_linear_batch;

/* k_dim, v_dim 64 or 128; v_heads a multiple of k_heads; conv_width 2 to 4, or 0 and conv NULL: no convolution. At most
 * 4096 value heads, and states of less than 2^63 bytes. */
int32_t bg_linear_create(int32_t n_layers, int32_t k_heads, int32_t v_heads, int32_t k_dim, int32_t v_dim, int32_t conv_width,
                         int32_t n_slots, float* state, float* conv, bg_linear_cache** out);
int32_t bg_linear_destroy(bg_linear_cache* cache);

/* A batch of at most max_seqs sequences with max_tokens new rows in all. Allocates (pinned and device). */
int32_t bg_linear_batch_create(const bg_linear_cache* cache, int32_t max_seqs, int32_t max_tokens, bg_linear_batch** out);
int32_t bg_linear_batch_destroy(bg_linear_batch* batch);
/* What the next calls work on (host arrays, read before the call returns): sequence s has rows[s] new rows, goes
 * on from the state in slot sources[s] (NULL: slots[s]; -1: a new conversation, zeros) and leaves it in slot
 * slots[s]. Sequences may share a source (a fork); no slot is written by two, or written by one and read by
 * another (BG_E_INVALID, the batch before stays set). A sequence without new rows touches no slot. Rows are
 * numbered sequence by sequence. Not under graph capture (BG_E_STATE). Sequences of 28 new rows and more are done in
 * chunks of 64, whose operands take a workspace of at most 384 MiB (or one chunk's): it grows here (BG_E_OOM: the batch
 * before stays set), never in a layer's call. Their scans are one launch: sequences of that length times v_heads v_dim
 * / 32 below 2^23 (BG_E_UNSUPPORTED, the batch before stays set), for a captured call any that its rows allow. */
int32_t bg_linear_batch_set(bg_linear_batch* batch, int32_t n_seqs, const int32_t* rows, const int32_t* slots,
                            const int32_t* sources, void* stream);

/* The layer's prologue for a batch: qkv [rows, channels] through the causal depthwise convolution conv_weight
 * [channels][conv_width] (the last tap on the row itself) and SiLU, then q, k [rows, k_heads, k_dim] each head over
 * sqrt(its sum of squares + 1e-6), v [rows, v_heads, v_dim] as it is; g = -exp(a_log) softplus(a + dt_bias) and beta =
 * 1 / (1 + exp(-b)) [rows, v_heads] of a, b (rows ab_stride values apart), a_log, dt_bias [v_heads]; g or beta
 * may be NULL. The slots' last inputs are read from the sequences' sources and left in their slots. qkv,
 * conv_weight, q, k, v 16-byte aligned; no output overlaps an input or another. Rows of the outputs beyond the
 * batch's are left as they are. */
int32_t bg_linear_prologue(const bg_linear_cache* cache, int32_t layer, bg_linear_batch* batch, const float* qkv,
                           const float* conv_weight, const float* a, const float* b, int32_t ab_stride, const float* a_log,
                           const float* dt_bias, float* q, float* k, float* v, float* g, float* beta, void* stream);

/* The recurrence above over every sequence's new rows, its state read and left as the batch says: q, k [rows,
 * k_heads, k_dim], v, out [rows, v_heads, v_dim], g [rows, v_heads] with rows g_stride values apart (0: [v_heads], one
 * decay a head), beta [rows, v_heads] or NULL. norm (nullable, [v_dim]): out = o / sqrt(mean o^2 + eps) * norm, and
 * with gate [rows, v_heads, v_dim] times gate / (1 + exp(-gate)). q, k, v, gate, norm, out 16-byte aligned; out
 * overlaps no input. Rows of out beyond the batch's are left as they are. A v that is not finite reaches its value dim's
 * row, later rows and state; a q its row of its heads; a k, g or beta its heads' row, later rows and states (g of minus
 * infinity is a decay to zero). Norms spread what is in a row over its head. Sums are f32 for any sizes of rows and value
 * dims beside each other; in chunks, values below 2^-109 count in steps of 2^-133. */
int32_t bg_linear_attention(const bg_linear_cache* cache, int32_t layer, bg_linear_batch* batch, const float* q, const float* k,
                            const float* v, const float* g, int32_t g_stride, const float* beta, float scale, const float* gate,
                            const float* norm, float eps, float* out, void* stream);

/* ---- 4-bit projections ------------------------------------------------------------------------------------
 * bg_gemv_split and bg_gemv_resid for 4-bit weights and up to 16 rows x [rows, K]: weight k of row n has the code
 * c = bits 4 (k % 8) .. + 3 of codes[n][k / 8] (u32) and, with the scale (and min) [n][k / group], the value
 * (c - 8) * scale, or c * scale + min where mins is not NULL. scale_type (scales and mins): BG_KV_F32 or BG_KV_F16.
 * K a multiple of 128, group 32, 64 or 128; x, codes, scales and mins 16-byte aligned. Outputs [rows, N0], [rows, N1],
 * [rows, N2]; resid, y [rows, N], y may be resid; otherwise no output overlaps an input or another. A product of two
 * values may reach 2^126 and their scales 2^90; K at most 2^24. x counts to 2^-31 of the largest of its 128 (those from a
 * multiple of 128 on), sums are f32. More than four rows need a workspace of bg_gemv4_workspace(rows, K) bytes, 16-byte aligned, that no other stream
 * uses meanwhile (four or fewer: 0 bytes, NULL). What a row gives does not depend on the rows beside it. */
int64_t bg_gemv4_workspace(int32_t rows, int32_t K);
int32_t bg_gemv4_split(const float* x, int32_t rows, int32_t K, const uint32_t* codes, const void* scales, const void* mins,
                       int32_t scale_type, int32_t group, int32_t N0, int32_t N1, int32_t N2, float* out0, float* out1, float* out2,
                       void* workspace, void* stream);
int32_t bg_gemv4_resid(const float* x, int32_t rows, int32_t K, const uint32_t* codes, const void* scales, const void* mins,
                       int32_t scale_type, int32_t group, int32_t N, const float* resid, float* y, void* workspace,
                       void* stream);

#ifdef __cplusplus
}
#endif

#endif /* BITGPU_ATTN_H */
