/*
 * C ABI of the MI355X (gfx950) shared-KV INT8 ("C8") attention and INT8 KV
 * cache writer: libsharedkv_hip.so.
 *
 * Plain pointers and sizes only.  Pointer fields hold device addresses; the
 * stream argument is a hipStream_t passed as void*.  Every entry point
 * returns a hipError_t value (0 = success; hipErrorInvalidValue = 1 for a
 * rejected argument block) and launches asynchronously on that stream.
 *
 * Reference interfaces replaced (paths relative to the reference checkout):
 *   SharedKVArgs                      csrc/kernels/c8/args.h:7-14 (200 bytes, same order)
 *   CacheWriteArgs                    csrc/kernels/cache_write.h:4-8 (same order)
 *   launch_sharedkv_c8_sparse         csrc/kernels/c8/c4.cpp:70-71
 *   launch_sharedkv_c8_dense          csrc/kernels/c8/c128.cpp:107-108
 *   launch_sharedkv_c8_sparse_small   csrc/kernels/c8/c4_small.cpp:21-22
 *   launch_cache_write                csrc/kernels/cache_write.cpp:71-80
 * The reference launchers return void; these return the launch status.
 */
#pragma once
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Attention arguments (csrc/kernels/c8/args.h:7-14).  Strides are bytes
 * between pages; tables address pages.  Fields this implementation reads:
 *   q (BF16 [tokens][heads][512], heads 1..128), ori/cmp (INT8 pages
 *   [*, 32, 1, 512]), oriScale/cmpScale (FP32 [512]), oriTable/cmpTable
 *   (INT32 [batch][width]), indices (INT32 [tokens][1][topk], ratio 4), cuQ
 *   (INT32 [batch+1]), seqLens (INT32 [batch]), sinks (FP32 [heads]), out
 *   (BF16 [tokens][heads][512]), lse (FP32 [tokens][heads] or 0), partial
 *   (FP32 [rows][splits][8][520] partition states when splits > 1; with
 *   one partition 0, or the re-plan room of sharedkv_c8_partial_bytes),
 *   splits (KV partitions), oriPages (pool size
 *   of the window cache; rows on pages past it are masked), workspace (one
 *   uint32 merge ticket per row, sharedkv_c8_workspace_bytes; zero before the
 *   first launch, and each launch leaves it zero, so launches that may
 *   overlap need their own).  A row is one query token's group of eight
 *   heads: rows = tokens * ceil(heads / 8).  Above eight heads the Q and P
 *   residual codes are off (reference.py:221-222).
 * oriIndices (INT32 [tokens][1][oriTopk], oriTopk <= 1024, or 0): explicit
 * physical original slots (page = slot / 32, row = slot % 32, no table)
 * replacing the window; entries outside [0, oriPages * 32) are masked in
 * place (reference.py:236-239, sparse_gather.h:22-78). */
typedef struct SharedKVArgs {
    uint64_t q, ori, cmp, oriScale, cmpScale, oriTable, cmpTable, indices;
    uint64_t cuQ, seqLens, sinks, out, workspace, lse;
    uint64_t oriStride, cmpStride, partial, oriIndices;
    uint32_t tokens, heads, batch, oriBlock, cmpBlock, oriTableWidth, cmpTableWidth;
    uint32_t ratio, window, topk, splits, oriTopk, oriPages;
    float softmaxScale;
} SharedKVArgs;

/* Cache-writer arguments (csrc/kernels/cache_write.h:4-8).  Strides are in
 * elements: pageStride in INT8 elements, updateStride in BF16 elements,
 * slotStride / slotColumnStride in slot elements. */
typedef struct CacheWriteArgs {
    uint64_t cache, updates, slots, inverseScale;
    uint64_t pageStride, updateStride, slotStride, slotColumnStride;
    uint32_t tokens, pages, pageSize, int64Slots, pairedSlots;
} CacheWriteArgs;

/* Tree attention arguments: a tree of drafted tokens per request over the
 * INT8 caches (no counterpart in the reference).  Request b has the query
 * tokens cuQ[b] .. cuQ[b + 1] - 1 (T of them) and seqLens[b] rows, the drafted
 * ones included: C = seqLens[b] - T committed rows, and the row of its drafted
 * token i is logical row C + i of the original cache.  parents (INT32
 * [tokens]) names each drafted token's parent by its index in the request; an
 * index that is not below the token's own makes it a root.  A token of depth d
 * (a root's is 0) sees
 *   original rows j < C with j > C + d - window,
 *   its ancestors and itself, those fewer than `window` steps above it,
 *   with a compressed cache (ratio > 1) its rows r < C / ratio, or where
 *   causalCompressed is 1 (instead of 0) r < (C + d + 1) / ratio, as
 *   SharedKVArgs' queries do at position C + d.  The rows behind C / ratio are
 *   the request's: one row for all of its nodes at the depth that completes it.
 * Rows on a page outside [0, oriPages) / [0, cmpPages), or past the block
 * table, are masked.  q, out BF16 [tokens][heads][512], heads 1..128; sinks
 * FP32 [heads]; lse FP32 [tokens][heads] or 0; ori / cmp INT8 pages of 32
 * rows of 512 bytes, page strides in bytes, multiples of 16.  Tokens of
 * requests with seqLens 0 and past cuQ[batch] are graph padding: their rows
 * of out and lse are zero-filled.  workspace and partial: the scratch that
 * sharedkv_tree_scratch names; the workspace is zero before the first launch,
 * and each launch leaves it zero, so launches that may overlap need their own. */
typedef struct TreeAttentionArgs {
    uint64_t q, ori, cmp, oriScale, cmpScale, oriTable, cmpTable, cuQ;
    uint64_t seqLens, sinks, parents, out, lse, workspace, partial;
    uint64_t oriStride, cmpStride;
    uint32_t tokens, heads, batch, oriPages, cmpPages, oriTableWidth, cmpTableWidth, ratio, window;
    float softmaxScale;
    uint32_t causalCompressed;
} TreeAttentionArgs;

/* One cache of a pool, for the entries below: page i at base + i * pageStride,
 * its row r at + r * rowStride, `bytes` bytes each (a row's for the path
 * commit, whose pages have pageRows rows; a page's for fork and compaction,
 * which read no rowStride).  Everything is a multiple of 16. */
typedef struct CacheSpan {
    uint64_t base, pageStride, rowStride, bytes;
} CacheSpan;

/* Accepted paths of drafted-token trees (no counterpart in the reference).
 * Requests as in TreeAttentionArgs (cuQ, seqLens, drafted rows behind the C
 * committed ones).  paths INT32 [batch][depth] names the accepted tokens of a
 * request by their index, rising; pathLens INT32 [batch] says how many there
 * are.  A path ends before its first entry that does not rise or is none of
 * the request's tokens.  Row C + paths[b][k] moves to row C + k in every cache,
 * and lengths[b] = C + accepted (0 for padding requests, seqLens 0).  Rows on
 * pages outside [0, pages), or past the block table, do not move.  `caches`
 * is a device array of CacheSpan; lengths must not overlap seqLens. */
typedef struct PathCommitArgs {
    uint64_t caches, table, cuQ, seqLens, paths, pathLens, lengths;
    uint32_t cacheCount, batch, depth, tokens, tableWidth, pages, pageRows, rowBytes;
} PathCommitArgs;

/* Rows of a block table that go on as other rows (no counterpart in the
 * reference): forked, reordered, grown and ended requests.  Every old row is
 * given up and row i of the new table continues old row parents[i] (outside
 * [0, rows): an empty row, length 0), with pages for length + room tokens.  A
 * page holds pageRows tokens.  Its whole pages are shared; of its other pages
 * the first of a parent's children keeps those that have no other owner
 * (refs 1), the rest are the lowest free pages (refs 0 when the call begins),
 * handed out by row, then entry.  The partly filled page is copied where it
 * was not kept.  Entries behind are -1.  Where free pages run out an entry is
 * -1, a row without its partly filled page is cut back to its whole pages, and
 * `missing` counts the entries.  Old entries outside [0, pages) are no pages.
 * newTable [children][width], newLens, newRefs may be table, seqLens, refs.
 * workspace: sharedkv_page_fork_workspace bytes, zero before the first launch
 * (each launch leaves what has to be zero so). */
typedef struct PageForkArgs {
    uint64_t caches, table, seqLens, refs, parents, newTable, newLens, newRefs, missing, workspace;
    uint32_t cacheCount, rows, children, width, pages, pageRows, room;
    uint32_t unused;
    uint64_t pageBytes;
} PageForkArgs;

/* Pool compaction (no counterpart in the reference): with L pages in use
 * (refs > 0), those from L on move, in order, to the free pages below L, in
 * order.  moved INT32 [pages]: each page's new place, -1 for free ones; the
 * table's entries and the refs follow; live INT32 [1] = L.  Entries outside
 * [0, pages) or on free pages become -1.  newTable and newRefs may be table
 * and refs.  workspace: sharedkv_page_compact_workspace bytes. */
typedef struct PageCompactArgs {
    uint64_t caches, table, refs, newTable, newRefs, moved, live, workspace;
    uint32_t cacheCount, rows, width, pages;
    uint64_t pageBytes;
} PageCompactArgs;

/* Rows appended to paged 8-bit caches, their position rotation applied on the
 * way (no counterpart in the reference).  Request b has the new rows cuQ[b] ..
 * cuQ[b + 1] - 1 of updates (BF16, token t and KV head h at updates +
 * 2 (t updateStride + h updateHeadStride) bytes, 512 values), the last of its
 * seqLens[b] rows; row r lies on page table[b][r / 32] of the cache (pages of
 * 32 rows of `heads` * 512 bytes, pageStride bytes apart).
 * rotary > 0: channels 512 - rotary on are rotated.  rotation (FP32
 * [rotationRows], rotationStride floats apart) holds rotary / 2 cosines and as
 * many sines for each position; positions (INT32, or INT64 where
 * int64Positions is 1, [tokens]; 0: the row's own index) names a row's.
 * Channels 2k and 2k + 1 of the rotated ones turn together where interleaved
 * is 1, else k and k + rotary / 2: a' = a cos - b sin, b' = a sin + b cos.
 * inverseScale (FP32 [512], one KV head, INT8): the codes of launch_cache_write,
 * of the rotated value as FP32 (NaN becomes -127 there and here).  Otherwise
 * scale FP32 [pages][heads] (scaleStride floats between pages) holds a scale for
 * each page and KV head, and codes are INT8 (codes 0, largest D = 127) or OCP e4m3 (1, D = 448):
 *   a page whose row 0 is appended gets scale = max(m / D, 1e-8), m the largest
 *   absolute value of its new rows as FP32; one that has rows keeps its scale,
 *   doubled as often as it takes to reach m / D, and where it is doubled its
 *   codes become round(code / 2^k);
 *   code = round(value / scale), to the nearest, ties to even.
 * NaN values become 0 (INT8) or NaN of either sign (e4m3) and are none of m;
 * infinities count as the largest FP32 number, so the page's other rows become
 * zeros beside one.  A scale that is no positive number counts as
 * that of a new page.  Rows on no page of the pool, past the block table,
 * below row 0 or with a position outside the table are skipped: what lies there
 * counts as rows that the page has, so a page of which every new row is skipped
 * stays as it is, and one whose row 0 is skipped keeps its scale, doubled or not;
 * padding as in TreeAttentionArgs.  No two rows of a launch may lie on the same place, and
 * no two requests append to one page. */
typedef struct CacheAppendArgs {
    uint64_t cache, updates, table, cuQ, seqLens, positions, rotation, scale, inverseScale;
    uint64_t pageStride, updateStride, updateHeadStride, scaleStride, rotationStride;
    uint32_t tokens, batch, heads, pages, tableWidth, rotary, rotationRows, interleaved, int64Positions, codes;
} CacheAppendArgs;

/* Attention over caches with a scale for each page and KV head, as
 * CacheAppendArgs fills them (no counterpart in the reference).  Request b has
 * the query tokens cuQ[b] .. cuQ[b + 1] - 1 (T of them) and seqLens[b] rows; its
 * token i stands at position P = seqLens[b] - T + i and sees
 *   original rows j <= P with j > P - window,
 *   with ratio > 1 (a power of two) compressed rows r < (P + 1) / ratio.
 * Query head h attends KV head h / (heads / kvHeads).  With v_j = code_j *
 * scale[page of j] and s_j = softmaxScale q v_j,
 *   out = sum_j e^{s_j} v_j / (e^{sink} + sum_j e^{s_j}), lse = log of the denominator.
 * q, out BF16 [tokens][heads][512], heads 1..128, a multiple of kvHeads; sinks
 * FP32 [heads]; lse FP32 [tokens][heads] or 0; ori / cmp pages of 32 rows of
 * kvHeads * 512 codes (INT8: codes 0, OCP e4m3: 1), page strides in bytes,
 * multiples of 16; oriScale / cmpScale FP32 [pages][kvHeads],
 * oriScaleStride / cmpScaleStride floats between pages, no scale negative
 * (one below 2^-80 counts as 2^-80 where it weighs values).  Rows on no page
 * of the pool or past the block table are masked, and nothing they hold, nor
 * their page's scale, reaches an output; the same holds for rows that a token
 * does not see.  Padding as in TreeAttentionArgs.  partial and units: the
 * scratch that sharedkv_block_scratch names; any contents, and launches that
 * may overlap need their own. */
typedef struct BlockAttentionArgs {
    uint64_t q, ori, cmp, oriScale, cmpScale, oriTable, cmpTable, cuQ;
    uint64_t seqLens, sinks, out, lse, partial, units;
    uint64_t oriStride, cmpStride, oriScaleStride, cmpScaleStride;
    uint32_t tokens, heads, kvHeads, batch, oriPages, cmpPages, oriTableWidth, cmpTableWidth, ratio, window, codes;
    float softmaxScale;
} BlockAttentionArgs;

/* Keys per tile of the attention kernels.  Together with SharedKVArgs.splits
 * it fixes the numerics: tile k of a query (kinds in order: original window,
 * then compressed rows) is folded into partition k % splits. */
#define SHAREDKV_C8_TILE 128

/* Optional integer dumps for parity tests (all device pointers, may be 0).
 * Layout per token t, positions P = 128 + cmpCapacity:
 *   qcodes [t][2 kinds][16][512] INT8: rows 0-7 Q head codes, 8-15 residuals
 *   alpha  [t][2][8] FP32
 *   scores [t][P][16] INT32: QK S_hi heads 0-7, S_lo 8-15 per list position
 *          (original window at 0.., compressed list at 128..)
 *   probs  [t][P][16] INT8: p8 heads 0-7, p_low 8-15
 *   values [t][tileCapacity][16][512] INT32: PV V_hi rows 0-7, V_lo 8-15 */
typedef struct SharedKVDebug {
    uint64_t qcodes, alpha, scores, probs, values;
    uint32_t cmpCapacity, tileCapacity;
} SharedKVDebug;

/* C4 attention: SWA128 window plus top-k compressed rows (topk <= 1024).
 * Replaces launch_sharedkv_c8_sparse (c4.cpp:70-71).  `blocks` is accepted
 * for ABI compatibility; 0 launches nothing.  The grid is rows * splits
 * work-groups rounded up to a multiple of 8, rows = tokens * ceil(heads / 8)
 * (plus a rows-wide merge grid in merge mode 1); a launch whose grid would
 * pass 2^31 - 8 work-groups is rejected with hipErrorInvalidValue. */
int launch_sharedkv_c8_sparse(uint32_t blocks, void *stream, const SharedKVArgs *args);

/* Small-capacity C4 entry (c4_small.cpp:21-22), for launches of fewer than
 * 24 query tokens.  The same kernels, except that they also carry the joint
 * route (reference.py:246-267 with joint_sparse) and take it when every live
 * row is short (longest live sequence / 4 <= 128), whatever the block
 * table's width, as the reference's small entry chooses its narrow route
 * from live lengths (c4_small.cpp:10-19).  Through launch_sharedkv_c8_sparse
 * only launches whose compressed block table names at most 128 rows per
 * sequence take it (compiled in, the route costs tiled launches ~1 %). */
int launch_sharedkv_c8_sparse_small(uint32_t blocks, void *stream, const SharedKVArgs *args);

/* C128 attention: SWA128 window plus every compressed row (c128.cpp:107-108).
 * Also serves ratio 1 (window only; the reference's legacy R1 plan). */
int launch_sharedkv_c8_dense(uint32_t blocks, void *stream, const SharedKVArgs *args);

/* Query-grouped attention: the reference device's paired plan (c128.cpp:17-23,
 * numerics reference.py:224-323 with query_group 2, tile_size 256), here
 * chosen by the caller (PreparedAttention(query_group=2)); the reference's
 * launcher picks it inside launch_sharedkv_c8_dense (C128), its operator
 * through launch_sharedkv_paired[_sparse] (attention.py:189-190).  Tokens
 * 2j and 2j + 1 of each request form a group sharing one window list (up to
 * 129 rows) and one compressed list (C128: rows below (p_last + 1) / 128;
 * C4: every row below (p_last + 1) / 4, each token weighing a row by its
 * multiplicity among its own valid top-k entries), each masking what it may
 * not see; 256-key tiles, tile k on partition k % splits (the reference's
 * operator runs one partition), no joint rows.  Any ratio, heads <= 8, no
 * explicit original slots (else hipErrorInvalidValue).  Scratch as for the
 * other launches at rows = tokens; graph padding rows are zero-filled and
 * the launch keeps its partition plan. */
int launch_sharedkv_c8_dense_paired(uint32_t blocks, void *stream, const SharedKVArgs *args);

/* Query-grouped attention in groups of four: the reference device's packed
 * plan (c128.cpp:24-27, numerics reference.py:224-323 with query_group 4,
 * tile_size 256; the operator's launch_sharedkv_packed[_sparse],
 * attention.py:186), chosen by the caller (PreparedAttention(query_group=4)).
 * Tokens 4j .. 4j + 3 of each request form a group sharing one window list
 * (up to 131 rows) and one compressed list; otherwise as
 * launch_sharedkv_c8_dense_paired (same limits, scratch and padding
 * behaviour). */
int launch_sharedkv_c8_dense_packed(uint32_t blocks, void *stream, const SharedKVArgs *args);

/* The same two grouped plans on 128-key tiles (reference.py:224-323 with
 * tile_size 128 and that query_group; no counterpart among the reference's
 * device entries, whose grouped plans are 256-key only), chosen by
 * PreparedAttention(query_group=2 or 4, tile_size=128).  Same limits,
 * scratch and padding behaviour. */
int launch_sharedkv_c8_dense_paired_narrow(uint32_t blocks, void *stream, const SharedKVArgs *args);
int launch_sharedkv_c8_dense_packed_narrow(uint32_t blocks, void *stream, const SharedKVArgs *args);

/* Same launch as launch_sharedkv_c8_sparse / _dense (ratio taken from
 * args->ratio; ungrouped plan), with the integer dumps written to `debug`.
 * Test entry; slower. */
int sharedkv_c8_attention_debug(void *stream, const SharedKVArgs *args, const SharedKVDebug *debug);

/* Fused INT8 quantise + slot scatter (cache_write.cpp:71-80).  `blocks` is
 * accepted for ABI compatibility; 0 launches nothing.  slotStride and
 * slotColumnStride must fit 32 bits (else hipErrorInvalidValue). */
int launch_cache_write(uint32_t blocks, void *stream, const CacheWriteArgs *args);

/* Attention of drafted-token trees (TreeAttentionArgs), and the bytes of its
 * scratch (0: none needed), a host-only query that reads everything but the
 * workspace and partial fields. */
int launch_sharedkv_tree(void *stream, const TreeAttentionArgs *args);
int sharedkv_tree_scratch(const TreeAttentionArgs *args, uint64_t *workspace, uint64_t *partial);

/* Rows appended to 8-bit caches (CacheAppendArgs); attention over caches with
 * block scales (BlockAttentionArgs), one launch or, where long contexts are
 * split, two, and the bytes of its scratch (0: none needed), a host-only query
 * that reads everything but the partial and units fields. */
int launch_sharedkv_append(void *stream, const CacheAppendArgs *args);
int launch_sharedkv_block(void *stream, const BlockAttentionArgs *args);
int sharedkv_block_scratch(const BlockAttentionArgs *args, uint64_t *partial, uint64_t *units);

/* Accepted paths, and pages of a pool (argument blocks above).  pageBytes is
 * the sum of the caches' bytes and rowBytes the largest row's.  All take up to
 * 2^24 - 1 work-groups of 256 threads (a fork one for every 64 KiB of every
 * child's page) and refuse larger calls before their first launch. */
int launch_sharedkv_path_commit(void *stream, const PathCommitArgs *args);
int launch_sharedkv_page_fork(void *stream, const PageForkArgs *args);
int launch_sharedkv_page_compact(void *stream, const PageCompactArgs *args);
uint64_t sharedkv_page_fork_workspace(uint32_t children, uint32_t width, uint32_t pages);
uint64_t sharedkv_page_compact_workspace(uint32_t pages);

/* Scratch sizes in bytes for a launch with `rows` = tokens * ceil(heads / 8)
 * rows (the query token count at eight heads).  partial_bytes(rows, 1) is
 * the partition-state room of a one-partition launch's device re-plan: when
 * such a launch (merge mode 0) supplies non-zero `workspace` and `partial`
 * of these sizes, graph padding that leaves fewer live rows than `rows`
 * re-plans the live rows into several partitions merged in the launch, as
 * launches with splits > 1 do (the reference device likewise plans splits
 * from live rows, c4_wide.h:16-41); with partial = 0 it keeps one partition
 * per row.  At most 256 row partitions: min(rows, 256) * 16640 bytes. */
uint64_t sharedkv_c8_workspace_bytes(uint32_t rows, uint32_t splits);
uint64_t sharedkv_c8_partial_bytes(uint32_t rows, uint32_t splits);

/* Allocation-free attention launch.  No counterpart in the reference: it is
 * for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc).  Same
 * launch as the entry the package routes it to: launch_sharedkv_c8_dense
 * (ratio 1 or 128), launch_sharedkv_c8_sparse_small (ratio 4, fewer than 24
 * tokens) or launch_sharedkv_c8_sparse (other ratio-4 launches);
 * args->workspace and args->partial are ignored: the merge tickets and
 * partition states live in a library-owned array of
 * sharedkv_c8_noalloc_scratch_bytes() (16 MiB) per GPU, located on the first
 * call on each device (the stream's device must be current).  The array's
 * layout is fixed: tickets in its first 4096 bytes (1024 rows), partition
 * states from byte 4096 on, so launches of any sizes in any order never
 * find another launch's states where their tickets are.  One-partition
 * launches use the regions only for their device re-plan of a padded
 * launch (at most 256 rows' tickets and states); a launch with splits > 1 whose
 * partial_bytes(rows, splits) exceeds the state region (16 MiB - 4 KiB: 504
 * rows at two partitions) is rejected with hipErrorInvalidValue.  The
 * function calls no hipMalloc or hipFree.  Every call on one GPU uses that
 * GPU's array: calls that may overlap on one GPU (other streams, other
 * threads) race on it. */
int launch_sharedkv_c8_noalloc(uint32_t blocks, void *stream, const SharedKVArgs *args);
uint64_t sharedkv_c8_noalloc_scratch_bytes(void);

/* Byte offsets of the tickets and the partition states that
 * launch_sharedkv_c8_noalloc uses for a launch of `rows` rows and `splits`
 * partitions.  Host-only query (no device call).  Returns 0, or
 * hipErrorInvalidValue when that launch would be rejected. */
int sharedkv_c8_noalloc_layout(uint32_t rows, uint32_t splits, uint64_t *tickets_offset, uint64_t *states_offset);

/* Partition merge placement for launches with splits > 1 (process-wide).
 * Mode 0 (default): fused; the last partition of a query row to finish
 * (ticket in `workspace`) folds the row inside the attention launch.
 * Mode 1: a separate merge kernel follows on the same stream.  Both give
 * identical results.  Returns 0, or hipErrorInvalidValue for other modes. */
int sharedkv_c8_set_merge_mode(int mode);

/* XCD-local partition-state exchange of the fused merge (process-wide; no
 * counterpart in the reference, whose merge runs on one core's memory).
 * Enabled (1, default): on a device where a one-time dispatch probe shows
 * that work-groups whose blockIdx agree modulo 8 run on one XCD, rows whose
 * partitions all run on one XCD pass their states through that XCD's L2;
 * other rows, and every row on other devices, use device-coherent stores
 * and loads.  The probe (first eager launch per device through the launch
 * entries above, never during stream capture or from the allocation-free
 * entry) launches one small kernel and synchronizes the stream once.
 * Disabled (0): device-coherent exchange everywhere.  Results are identical
 * either way.  Returns 0, or hipErrorInvalidValue for other values. */
int sharedkv_c8_set_xcd_local(int enable);

/* The current device's probe result: 1 XCD-local exchange in use, 0 not
 * (probe failed), -1 not probed yet. */
int sharedkv_c8_xcd_local(void);

/* sizeof the argument blocks of trees, block-scaled caches and pages. */
uint32_t sharedkv_append_args_size(void);
uint32_t sharedkv_block_args_size(void);
uint32_t sharedkv_tree_args_size(void);
uint32_t sharedkv_path_commit_args_size(void);
uint32_t sharedkv_page_fork_args_size(void);
uint32_t sharedkv_page_compact_args_size(void);

/* sizeof(SharedKVArgs), sizeof(CacheWriteArgs), library ABI version (5 since
 * CacheAppendArgs and BlockAttentionArgs). */
uint32_t sharedkv_attention_args_size(void);
uint32_t sharedkv_cache_args_size(void);
uint32_t sharedkv_abi_version(void);

#ifdef __cplusplus
}
#endif
