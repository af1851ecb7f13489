/*
 * deltaattn_cache.h -- C ABI of the bounded decode cache of the MI355X (gfx950)
 * DeltaAttention path: the attention weight each key received, key and value rows held in
 * 4 bits, eviction by accumulated weight, and decode attention over 4-bit rows.
 *
 * The conventions are those of deltaattn.h: device pointers, int64 element strides with a
 * contiguous head dimension, caller-provided workspaces, a hipStream_t passed as void*,
 * DA_OK or a negative DA_ERR_* with the message in da_last_error(), no allocation, no
 * synchronisation, no state between calls.  The reference has no counterpart: its
 * compressed cache (deltaDecoding.py:111-233) keeps every anchor at full width.
 */
#ifndef DELTAATTN_CACHE_H
#define DELTAATTN_CACHE_H

#include "deltaattn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rows held in 4 bits, for every (sequence, KV head).  A row of D dims (a multiple of 8 up to
 * 128) is ceil(D / 32) groups of 32 dims.  A group has one exponent byte x (the power of two
 * 2^(x - 127)) and 16 bytes of codes: byte i holds dims 2 i (low half) and 2 i + 1, each a
 * sign, two exponent bits and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6) times the power.
 * Dims past D have code 0.  x = 255 marks a group that held an infinity or a NaN: it reads
 * back as NaN.
 *
 * All arrays are contiguous: codes [B, Hkv, capacity, 16 groups], exponents [B, Hkv,
 * capacity, groups], counts / timestamps / mass [B, Hkv, capacity], lengths [B, Hkv] (rows in
 * use; clamped into [0, capacity] where read).  Codes must be 16-byte aligned, exponents
 * 4-byte.  mass (the attention weight each row has received) may be null where a call does not
 * use it.  At most 2^26 rows a head and 65535 (sequence, head) pairs.
 */
typedef struct DaKv4 {
  uint8_t* k_codes;
  uint8_t* k_scales;
  uint8_t* v_codes;
  uint8_t* v_scales;
  int32_t* counts;
  int32_t* timestamps;
  int32_t* lengths;
  float* mass;
  int64_t capacity;
} DaKv4;

/*
 * Rows into 4 bits: row m of (b, h) of `out` becomes row m (or row index[b, h, m] where index
 * is not null) of k, v [B, Hkv, N, D] (bf16, fp16 or fp32; strides s*_b, s*_h, s*_n; rows
 * 16-byte aligned), for m < M (M = N without an index).  A group's power is the smallest for
 * which no element exceeds 6 (exponents -125 .. 125); elements round to nearest, ties to the
 * even code.  counts, timestamps and mass ([B, Hkv, N], contiguous; null: 1, the row's
 * number, 0) are taken along; out->mass may be null.  Rows at or past lengths[b, h] (int32
 * [B, Hkv]; null: M), and rows whose index lies outside [0, N), are zero with count 0; rows
 * from M on are not written.  out->lengths receives min(lengths, M).  M <= out->capacity.
 */
int da_kv4_quantize(const void* k, const void* v, int dtype, int64_t B, int64_t Hkv, int64_t N, int64_t D,
                    int64_t sk_b, int64_t sk_h, int64_t sk_n, int64_t sv_b, int64_t sv_h, int64_t sv_n,
                    const int32_t* counts, const int32_t* timestamps, const float* mass, const int32_t* lengths,
                    const int32_t* index, int64_t M, const DaKv4* out, void* stream);

/*
 * The values of 4-bit rows: k, v [B, Hkv, N, D] contiguous, bf16, fp16 or fp32, for the first
 * N <= capacity rows; rows at or past a head's length are zero.  Exact in bf16 and fp32.
 */
int da_kv4_dequantize(const DaKv4* kv, int64_t B, int64_t Hkv, int64_t N, int64_t D, void* k, void* v, int dtype,
                      void* stream);

/*
 * The rows of `kv` that a budget leaves, in their order, moved to `out` (other memory).  A
 * head with at most `budget` rows keeps all.  A longer one keeps its first `sinks` rows, its
 * last `recent` rows, and of those between the budget - sinks - recent with the largest mass
 * (compared as numbers, -0 = 0, a NaN of either sign as the largest; ties go to the lower row).
 * sinks + recent <= budget <= out->capacity.  Rows [kept, budget) of `out` are zero, rows from
 * budget on are not written; out->lengths receives the rows kept.  kv->mass and out->mass are
 * needed.  index, if not null ([B, Hkv, budget] int32), receives the rows kept, -1 past them.
 * workspace: da_kv4_evict_workspace_size() bytes (none, and null, for a small budget).
 */
int64_t da_kv4_evict_workspace_size(int64_t B, int64_t Hkv, int64_t capacity, int64_t budget);
int da_kv4_evict(const DaKv4* kv, int64_t B, int64_t Hkv, int64_t D, int64_t budget, int64_t sinks, int64_t recent,
                 const DaKv4* out, int32_t* index, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * One decode token, as da_decode_update over 16-bit rows: where the ring [B, Hkv, W, D] is full
 * (exact_seq_len >= window) the token in slot exact_seq_len % window leaves it and merges into the
 * last row (count + 1) if it is close enough to that row's key as it was, k_last [B, Hkv, D]
 * (contiguous; Euclidean dist^2 <= threshold, cosine >= threshold), or else becomes a new row
 * (count 1, timestamp total_seq_len - window, mass 0) and the new k_last; with the capacity used up
 * it is dropped.  The new token takes the slot.  new_k, new_v [B, Hkv, 1, D] (strides sn_b, sn_h),
 * ring and k_last share one type; even strides, rows 4-byte aligned (fp32: 8-byte).
 */
int da_kv4_update(const void* new_k, const void* new_v, int dtype, int64_t B, int64_t Hkv, int64_t D, int64_t sn_b,
                  int64_t sn_h, void* k_exact, void* v_exact, int64_t sx_b, int64_t sx_h, int64_t sx_s,
                  const DaKv4* kv, void* k_last, int64_t exact_seq_len, int64_t total_seq_len, int64_t window,
                  float threshold, int use_cosine, void* stream);

/*
 * Row choice alone: mass [B, Hkv, N] fp32 contiguous, lengths [B, Hkv] (null: N) -> index
 * [B, Hkv, budget] int32 (rows kept, ascending; -1 past them) and kept [B, Hkv] int32, by the
 * rule of da_kv4_evict.  workspace as there (capacity = N).
 */
int da_heavy_rows(const float* mass, const int32_t* lengths, int64_t B, int64_t Hkv, int64_t N, int64_t budget,
                  int64_t sinks, int64_t recent, int32_t* index, int32_t* kept, void* workspace,
                  int64_t workspace_bytes, void* stream);

/*
 * q_len = 1 attention over 4-bit rows and a ring of exact rows, as da_decode_attention over
 * 16-bit ones: scores over rows [0, length) get + log(count) (a count <= 0 gives no weight),
 * then the ring slots [0, exact_len) of k_exact, v_exact [B, Hkv, W, D] (strides sx_*; may be
 * null with exact_len = 0).  q [B, Hq, D], out [B, Hq, D] and the ring share one type (bf16,
 * fp16 or fp32); q and ring rows are 16-byte aligned.  A head with no key at all gives zeros.
 * The rows' values enter as they are (bf16 holds them exactly), q and the weights in two or
 * three 16-bit parts, sums in fp32.  accumulate: kv->mass[b, g, j] += the softmax weight of
 * row j, summed over the query heads of the group.  Hq / Hkv <= 64, capacity <= 2^24.
 * workspace: da_kv4_attention_workspace_size() bytes (none, and null, for a cache of up to 768
 * rows a head, or 1024 of many heads, that one workgroup a head takes).
 */
int64_t da_kv4_attention_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t capacity, int accumulate);
int da_kv4_attention(const void* q, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t sq_b,
                     int64_t sq_h, const DaKv4* kv, const void* k_exact, const void* v_exact, int64_t sx_b,
                     int64_t sx_h, int64_t sx_s, int64_t exact_len, float scale, int accumulate, void* out,
                     int64_t so_b, int64_t so_h, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * The attention weight that every key receives from a run of queries: mass[b, g, j] = sum over
 * the query heads h of group g and the queries i of softmax_j(scale q[b, h, i] . k[b, g, j] +
 * log counts[b, g, j]) over the keys that query i sees: j < lengths[b, g] (null: Nk) and
 * timestamps[b, g, j] <= q_start + i (null timestamps: j; a count <= 0 hides the key).  Positions
 * q_start + i are taken as the nearest in [-(2^31 - 2), 2^31 - 2], so a key at 2^31 - 1 is never
 * seen.  A query that sees no key adds nothing, a key that no query sees gets 0, whatever they hold.  q [B, Hq, Nq, D], k [B, Hkv, Nk, D] of one type (bf16, fp16
 * or fp32), rows 16-byte aligned; counts, timestamps [B, Hkv, Nk] int32 contiguous or null;
 * mass [B, Hkv, Nk] fp32 contiguous, 0 from the length on.  Deterministic.  Hq / Hkv <= 64,
 * Nq * Hq / Hkv < 2^30, Nq, Nk <= 2^24, B * Hkv <= 65535, fewer than 2^32 threads a launch.
 * workspace: da_attention_mass_workspace_size() bytes.
 */
int64_t da_attention_mass_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t Nq, int64_t Nk);
int da_attention_mass(const void* q, const void* k, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Nq,
                      int64_t Nk, int64_t D, int64_t sq_b, int64_t sq_h, int64_t sq_n, int64_t sk_b, int64_t sk_h,
                      int64_t sk_n, const int32_t* counts, const int32_t* timestamps, const int32_t* lengths,
                      int64_t q_start, float scale, float* mass, void* workspace, int64_t workspace_bytes,
                      void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DELTAATTN_CACHE_H */
