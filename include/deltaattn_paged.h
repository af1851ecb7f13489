/*
 * deltaattn_paged.h -- C ABI of the paged key/value cache at full width of the MI355X (gfx950)
 * DeltaAttention path: new tokens rotated and written into pages, attention of new tokens over
 * the pages of their sequences, and the same where groups of sequences share their first tokens.
 *
 * The conventions are those of deltaattn.h: device pointers, int64 element strides with a
 * contiguous head dimension, caller-provided workspaces, a hipStream_t passed as void*, DA_OK or a
 * negative DA_ERR_* with the message in da_last_error(), no allocation, no synchronisation, no
 * state between calls.  The reference has no counterpart: its dense path keeps no cache of its own
 * (modeling_llama.py:778-803).
 */
#ifndef DELTAATTN_PAGED_H
#define DELTAATTN_PAGED_H

#include "deltaattn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * The pages of one layer: k, v [num_pages, Hkv, page_size, D] of any strides that are multiples of 8
 * elements, 16-byte aligned, row strides in [D, 2^23).  page_size is a power of two from 16 on.
 */
typedef struct DaPagedKV {
  void* k;
  void* v;
  int64_t num_pages, page_size;
  int64_t sk_p, sk_h, sk_n; /* page, head, row */
  int64_t sv_p, sv_h, sv_n;
} DaPagedKV;

/*
 * The sequences of a call.  Sequence b has lengths[b] tokens in its pages (those that this call
 * brings included, and last), token j in row j % page_size of page table[b][j / page_size].  It
 * brings the tokens cu[b] .. cu[b + 1] - 1 of q, k, v [T, heads, D] (null cu: token b alone), of which
 * no sequence has more than max_seqlen (which the append does not read).  Token t is its token
 * j = lengths[b] - cu[b + 1] + t, whose position is start[b] + j (null: j).
 * Rows past cu[B] are left as they are.  What the arrays hold is clamped on the device: cu into
 * [0, T] and to max_seqlen tokens, lengths into [0, width * page_size]; a page outside
 * [0, num_pages) is never touched (its tokens' keys and values count as zeros, a token meant for
 * it is not written).  A token whose place j is not in the table (before row 0, as in a sequence that
 * is shorter than what it brings, or from width * page_size on) is not written, and attends to the
 * places before its own that are there.  Attention leaves the tokens past max_seqlen of a sequence, or of
 * a prefix's group, as they are.  With a cu that does not rise no row outside the batch is touched.
 */
typedef struct DaPagedBatch {
  const int32_t* table; /* [B, width], rows table_stride apart */
  const int32_t* lengths;
  const int32_t* cu;
  const int32_t* start;
  int64_t B, width, table_stride, max_seqlen;
} DaPagedBatch;

/*
 * New tokens into their pages: v as it is, k rotated to its position, and the rotated queries into
 * q_out (q may be null).  k, v [T, Hkv, D], q, q_out [T, Hq, D] (strides s*_t, s*_h; rows 16-byte
 * aligned), of the pages' type (bf16, fp16 or fp32).  q_out may be q.  Rotation: dims d and
 * d + rot / 2 (interleaved: 2 d and 2 d + 1), d < rot / 2, become x cos - y sin and y cos + x sin, in
 * fp32, rounded once; dims from rot on stay.  cos, sin [rows, rot / 2] fp32 or of the pages' type
 * (rot_dtype), rows s_rot apart (0: one row for all); row p is for position p, or with per_token for
 * token p (rows >= T).  A position outside the rows takes the nearest row.  rot = 0: no rotation.
 * T is less than 2^26.
 * Two tokens meant for one place (tables with a page in common) leave either of them there.
 */
int da_paged_append(const void* k, int64_t sk_t, int64_t sk_h, const void* v, int64_t sv_t, int64_t sv_h,
                    const void* q, int64_t sq_t, int64_t sq_h, void* q_out, int64_t so_t, int64_t so_h, int dtype,
                    int64_t T, int64_t Hq, int64_t Hkv, int64_t D, const void* cos, const void* sin, int rot_dtype,
                    int64_t rows, int64_t s_rot, int64_t rot, int interleaved, int per_token, const DaPagedKV* kv,
                    const DaPagedBatch* batch, void* stream);

/*
 * Attention of the new tokens, which are in their pages already: query token t of sequence b over
 * the keys 0 .. lengths[b] - cu[b + 1] + t of its sequence that its table holds.  With `prefix`, the
 * batch's tokens are cut into prefix->B groups (prefix->cu, in tokens; each sequence inside one group),
 * and every query of group g also sees all prefix->lengths[g] keys in the pages prefix->table[g], as if
 * they stood before its own (prefix->start is not read, prefix->max_seqlen is the most tokens of a group).
 * q, out [T, Hq, D] (strides *_t, *_h; rows 16-byte aligned) of the pages' type; query head h reads
 * KV head h / (Hq / Hkv).  A query that sees no key gives zeros.  A key that it does not see has
 * weight 0: an infinity or a NaN in the values of a call's own later tokens can reach earlier ones.
 * Scores, maxima, sums and partial results are fp32.  Deterministic.  T is less than 2^24.  What batch and prefix point to must not
 * change while the call runs.  workspace: da_paged_attention_workspace_size() bytes of the same
 * arguments (none, and null, where it returns 0), 256-byte aligned.
 */
int64_t da_paged_attention_workspace_size(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                          const DaPagedKV* kv, const DaPagedBatch* batch,
                                          const DaPagedBatch* prefix);
int da_paged_attention(const void* q, int64_t sq_t, int64_t sq_h, void* out, int64_t so_t, int64_t so_h, int dtype,
                       int64_t T, int64_t Hq, int64_t Hkv, int64_t D, float scale, const DaPagedKV* kv,
                       const DaPagedBatch* batch, const DaPagedBatch* prefix, void* workspace,
                       int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DELTAATTN_PAGED_H */
