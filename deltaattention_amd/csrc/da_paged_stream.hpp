// Paged attention of few rows: decode steps, short runs of tokens, small batches behind a prefix.
//
// Bound by memory: each key and value row is read once for all rows of its item, 4 D operations a
// row and key against 4 D bytes a key.  So the items' key tiles are one stream, cut into equal shares:
// a worker (workgroup) takes a contiguous run of tiles whatever the sequences' lengths are, which
// needs no length on the host and leaves no workgroup with more than another.  A worker's first and
// last item may be parts; their (sum, maximum, weights) go to its two slots and are joined after.
//
// A wave takes 32 of a tile's 128 keys for up to 32 rows, alone: its keys and values go from memory to
// its own 16 KiB of LDS (buffer_load ... lds), K of the next tile while it works on this one's
// scores, V while on the next one's, with exact vmcnt waits and no barrier.  Two workgroups a CU keep
// 8 waves' loads in flight, about 128 KiB a CU.  S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_32x32x16: a lane holds one row and 16 keys.  The weights enter in two 16-bit parts (the
// matrix unit is idle most of the time here), so the one rounding that matters is the output's.  In fp16
// they are 2^15 times as large, with the maximum less 15 as their reference point: fp16 ends at 2^-24,
// and thousands of keys below 2^-25 of the best would vanish.
#pragma once

#include "da_paged.hpp"
#include "da_tile.hpp"

namespace da {

constexpr int kStageLds = 16384;  // a wave's K and V tiles; its rows' sums at the end
constexpr int kStreamEntries = 256;
struct StreamShared {
  float ml[4][2][32];
  int first[kStreamEntries], tokens[kStreamEntries], keys[kStreamEntries], before[kStreamEntries];
  uint32_t waves[4];
  int entry;
  uint32_t offset;
  StreamRecord record;
};
constexpr int stream_lds(int stages) { return 4 * stages * kStageLds + (int)sizeof(StreamShared); }

// Waits for all but the wave's last N loads.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}
// The eight 16-byte reads at a ^ 32 j, waited for.
__device__ __forceinline__ void read_keys(u32x4 (&k)[8], uint32_t a) {
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
      "ds_read_b128 %4, %12\n\tds_read_b128 %5, %13\n\tds_read_b128 %6, %14\n\tds_read_b128 %7, %15\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(k[4]), "=&v"(k[5]), "=&v"(k[6]), "=&v"(k[7])
      : "v"(a), "v"(a ^ 32u), "v"(a ^ 64u), "v"(a ^ 96u), "v"(a ^ 128u), "v"(a ^ 160u), "v"(a ^ 192u), "v"(a ^ 224u)
      : "memory");
}
// The V^T fragments of 16 keys (OFF: their byte offset): four blocks of 32 dims at a ^ 64 db, two
// transposing reads each.
template <int OFF>
__device__ __forceinline__ void read_values(u32x4 (&v)[4], uint32_t a) {
  i16x4 lo[4], hi[4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
      "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
      "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2]), "=&v"(lo[3]), "=&v"(hi[3])
      : "v"(a), "v"(a ^ 64u), "v"(a ^ 128u), "v"(a ^ 192u), "i"(OFF), "i"(OFF + 2048)
      : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = __builtin_bit_cast(u32x4, __builtin_shufflevector(lo[i], hi[i], 0, 1, 2, 3, 4, 5, 6, 7));
}

// first token, tokens, keys and the first token's slot of list entry e: the prefix's groups, then the sequences
__device__ __forceinline__ void entry_of(const PagedAttnArgs& a, int e, int& first, int& tokens, int& keys, int& before) {
  const bool own = e >= a.prefix.B;
  const PageBatch s = list_of(a, own);
  const int b = own ? e - a.prefix.B : e;
  first = s.first(b);
  tokens = s.tokens(b);
  keys = s.keys(b);
  before = s.before(b);
}

// Exclusive sum over the workgroup's threads; all threads get the total too.
__device__ __forceinline__ uint32_t workgroup_sum(uint32_t x, StreamShared& sh, uint32_t& total) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  uint32_t incl = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(incl, d, 64);
    if (lane >= d) incl += o;
  }
  __syncthreads();  // the last sum has been read
  if (lane == 63) sh.waves[wid] = incl;
  __syncthreads();
  const uint32_t w0 = sh.waves[0], w1 = sh.waves[1], w2 = sh.waves[2], w3 = sh.waves[3];
  total = w0 + w1 + w2 + w3;
  return incl - x + (wid > 0 ? w0 : 0) + (wid > 1 ? w1 : 0) + (wid > 2 ? w2 : 0);
}

// A worker's run of tiles: from tile `offset` (head by head) of entry `entry` on.  Entries chunk ..
// chunk + 255 are in sh.
struct Share {
  int entry, chunk;
  uint32_t offset, tiles, per;
};

// Workgroup-uniform; false if there is nothing to do.  Where no item is split, worker w has item w (offset
// is its head, tiles 1).
__device__ __forceinline__ bool share_of(const PagedAttnArgs& a, const int worker, StreamShared& sh, Share& share) {
  const int tid = threadIdx.x, E = a.prefix.B + a.seq.B;
  int first = 0, tokens = 0, keys = 0, at = 0;
  if (a.whole) {
    const int e = worker / a.Hkv;
    entry_of(a, e, first, tokens, keys, at);
    if (stream_tiles(a, tokens, keys, e >= a.prefix.B) == 0) return false;
    if (tid == 0) sh.first[0] = first, sh.tokens[0] = tokens, sh.keys[0] = keys, sh.before[0] = at;
    __syncthreads();
    share = Share{e, e, (uint32_t)(worker - e * a.Hkv), 1, 1};
    return true;
  }
  // the entries' tiles summed in order, 256 entries at a time
  auto tiles_of = [&](int i) { return (uint32_t)stream_tiles(a, tokens, keys, i >= a.prefix.B) * (uint32_t)a.Hkv; };
  if (tid < E) entry_of(a, tid, first, tokens, keys, at);
  uint32_t mine = tiles_of(tid), sum, rest = 0;
  uint32_t before = workgroup_sum(mine, sh, sum);
  if (E > kStreamEntries) {
    const int f = first, t = tokens, k = keys, s = at;
    uint32_t x = 0;
    for (int i = tid + kStreamEntries; i < E; i += kStreamEntries) {
      entry_of(a, i, first, tokens, keys, at);
      x += tiles_of(i);
    }
    workgroup_sum(x, sh, rest);
    first = f, tokens = t, keys = k, at = s;
  }
  const uint32_t total = sum + rest;
  const uint32_t per = max((total + a.workers - 1) / a.workers, 1u);
  const uint32_t u = worker * per;
  if (worker == 0 && tid == 0) a.begin[0] = per, a.begin[1 + E] = total;
  int chunk = 0;
  for (uint32_t base = 0;;) {
    const int i = chunk + tid;
    sh.first[tid] = first, sh.tokens[tid] = tokens, sh.keys[tid] = keys, sh.before[tid] = at;
    if (worker == 0 && i < E) a.begin[1 + i] = base + before;
    if (u >= base + before && u < base + before + mine) sh.entry = i, sh.offset = u - base - before;
    base += sum;
    // worker 0 goes through all entries, for `begin`
    if ((worker != 0 && (u < base || u >= total)) || chunk + kStreamEntries >= E) break;
    chunk += kStreamEntries;
    first = tokens = keys = 0;
    if (chunk + tid < E) entry_of(a, chunk + tid, first, tokens, keys, at);
    mine = tiles_of(chunk + tid);
    before = workgroup_sum(mine, sh, sum);
  }
  if (u >= total) return false;
  if (tid == 0) {
    sh.record.others = 0;
    if (a.records) a.records[worker].others = 0;
  }
  __syncthreads();
  share = Share{__builtin_amdgcn_readfirstlane(sh.entry), chunk, (uint32_t)__builtin_amdgcn_readfirstlane(sh.offset),
                min(per, total - u), per};
  return true;
}

// The work of worker `worker`, a workgroup of 256 threads.  STAGES tiles of a wave in LDS: 1, with two
// workgroups a CU; 2 where there is no more than one workgroup a CU anyway, whose next tile's loads are
// then under way a tile earlier.
template <int DT, int STAGES>
__device__ __forceinline__ void stream_worker(const PagedAttnArgs& a, const int worker) {
  constexpr int kWaveLds = STAGES * kStageLds;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  StreamShared& sh = *(StreamShared*)(smem + 4 * kWaveLds);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane >> 5, ql = lane & 31;
  Share share;
  if (!share_of(a, worker, sh, share)) return;
  int e = share.entry;
  uint32_t off = share.offset, left = share.tiles;
  int part = 0;  // the segment's number

  const uint32_t kb = lds_addr(smem) + wid * kWaveLds, vb = kb + kStageLds / 2;
  char* const kl = smem + wid * kWaveLds;
  char* const vl = kl + kStageLds / 2;
  // K: rows of 256 bytes, chunk c of row r at c ^ (r & 15), the lane reads chunks 2 j + hl of row ql;
  // V: chunk c of row r at c ^ 4 (r & 3), read transposed
  const uint32_t ka = kb + ql * 256 + (((hl ^ ql) & 1) << 4) + ((ql & 14) << 4);
  const uint32_t va = vb + ((4 * ((lane >> 4) >> 1) + ((lane & 15) >> 2)) * 256 +
                            ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) << 4) + 8 * (lane & 1) + 64 * ((lane & 15) >> 2));
  // a load moves four rows, 16 bytes a lane: row 4 j + lane / 16, the chunk that the layout keeps
  // at lane % 16; chunks past the head dimension lie past every range and arrive as zeros
  const unsigned skb = (unsigned)(2 * a.pages.sk_n), svb = (unsigned)(2 * a.pages.sv_n);
  unsigned ko[4], vo;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = 4 * j + (lane >> 4), c = (lane & 15) ^ row;
    ko[j] = 8 * c < a.D ? __umul24(row, skb) + 16 * c : 1u << 30;
  }
  {
    const int row = lane >> 4, c = (lane & 15) ^ (4 * row);
    vo = 8 * c < a.D ? __umul24(row, svb) + 16 * c : 1u << 30;
  }
  const float c = a.scale_log2;
  const int shift = a.pages.shift, in_page = (1 << shift) - 1;

  while (left > 0) {
    const bool own = e >= a.prefix.B;
    if (e >= a.prefix.B + a.seq.B) return;  // lengths that changed under the call
    if ((unsigned)(e - share.chunk) >= kStreamEntries) {  // the next entries
      share.chunk = e;
      __syncthreads();
      if (e + tid < a.prefix.B + a.seq.B) entry_of(a, e + tid, sh.first[tid], sh.tokens[tid], sh.keys[tid], sh.before[tid]);
      __syncthreads();
    }
    const int f = __builtin_amdgcn_readfirstlane(sh.first[e - share.chunk]);
    const int nt = __builtin_amdgcn_readfirstlane(sh.tokens[e - share.chunk]);
    const int nk = __builtin_amdgcn_readfirstlane(sh.keys[e - share.chunk]);
    const int before = __builtin_amdgcn_readfirstlane(sh.before[e - share.chunk]);
    const int tiles = stream_tiles(a, nt, nk, own);
    if (tiles == 0) {
      ++e;
      continue;
    }
    const int h = a.whole ? off : off / tiles;
    const int t0 = a.whole ? 0 : off - h * tiles;
    const int n = a.whole ? tiles : min((uint32_t)(tiles - t0), left);
    const int rows = nt * a.G;
    // keys that row ql sees, of those that are there; row 0 sees the fewest
    const int tok = ql / a.G;
    const int seen = own ? min(nk, before + 1 + tok) : nk;
    const int least = own ? min(nk, before + 1) : nk;

    // ---- this wave's tiles: 32 keys from 128 t + 32 wid on, while there are any ----
    const int key_first = t0 * kStreamTile + 32 * wid;
    const int m = key_first >= nk ? 0 : min(n, (nk - key_first + kStreamTile - 1) / kStreamTile);
    const int32_t* table = own ? a.seq.table + (int64_t)(e - a.prefix.B) * a.seq.table_stride
                               : a.prefix.table + (int64_t)e * a.prefix.table_stride;
    const int last_row = (own ? a.seq.max_keys : a.prefix.max_keys) - 1;
    int ids = -1;
    // pages of the 16-row halves of 32 of the wave's tiles, from its tile i on: lane 2 j + half
    auto load_ids = [&](int i) {
      const int key = key_first + (i + (lane >> 1)) * kStreamTile + 16 * (lane & 1);
      const int id = table[min(key, last_row) >> shift];  // asked for before the length is known
      ids = key < nk && id >= 0 && id < a.pages.num_pages ? id : -1;
    };
    auto load_rows = [&](const bool isK, int i) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int id = __builtin_amdgcn_readlane(ids, 2 * (i & 31) + half);
        const int key = key_first + i * kStreamTile + 16 * half;
        const int64_t page = id < 0 ? 0 : id;
        const int64_t at = isK ? page * a.pages.sk_p + (key & in_page) * a.pages.sk_n + h * a.pages.sk_h
                               : page * a.pages.sv_p + (key & in_page) * a.pages.sv_n + h * a.pages.sv_h;
        const int valid = id < 0 ? 0 : clamp0_uniform(nk - key, 16);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<void*>(uniform_ptr((isK ? a.pages.k : a.pages.v) + 2 * at)), (short)0,
            valid * (int)(isK ? skb : svb), kBufferDword3);
        char* dst = (isK ? kl : vl) + (STAGES == 2 ? (i & 1) * kStageLds : 0) + 4096 * half;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(dst + 1024 * j), 16,
                                                   isK ? (int)ko[j] : (int)(vo + 4 * j * svb), 0, 0, 0);
      }
    };

    // ---- Q^T: dims 16 t + 8 hl .. + 7 of row ql ----
    u32x4 qw[8];
    {
      const bool on = ql < rows;
      const char* row = a.q + 2 * ((int64_t)(f + (on ? tok : 0)) * a.sq_t + (int64_t)(h * a.G + (on ? ql - tok * a.G : 0)) * a.sq_h);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int d = 16 * t + 8 * hl;
        qw[t] = *(const u32x4*)(row + 2 * (d < a.D ? d : 0));
        if (!on || d >= a.D) qw[t] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) asm volatile("" : "+v"(qw[t]));
    }
    f32x16 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = f32x16{};
    float mx = -INFINITY, l = 0.0f;
    if (m > 0) {
      load_ids(0);
      load_rows(true, 0);
      load_rows(false, 0);
      if (STAGES == 2 && m > 1) {
        load_rows(true, 1);
        load_rows(false, 1);
      }
    }
#pragma nounroll
    for (int i = 0; i < m; ++i) {
      // in flight, eight loads each: K and V of this tile, with two stages those of the next too
      const bool more = i + STAGES < m;
      const uint32_t stage = STAGES == 2 ? (i & 1) * kStageLds : 0;
      f32x16 x;
      {
        u32x4 k[8];
        if (STAGES == 2 && i + 1 < m) wait_loads<24>();
        else wait_loads<8>();
        read_keys(k, ka + stage);
        x = E16<DT>::mfma(k[0], qw[0], f32x16{});
#pragma unroll
        for (int j = 1; j < 8; ++j) x = E16<DT>::mfma(k[j], qw[j], x);
      }
      const int key0 = key_first + i * kStreamTile;
      // V of the tiles before has been asked for: their pages are done with
      if (more) {
        if (((i + STAGES) & 31) == 0) load_ids(i + STAGES);
        load_rows(true, i + STAGES);
      }
      if (key0 + 32 > least) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key0 + 8 * (r >> 2) + 4 * hl + (r & 3) >= seen) x[r] = -INFINITY;
      }
      float top = x[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = __builtin_fmaxf(top, x[r]);
      const float mn = __builtin_fmaxf(mx, halves_max(top) * c - (DT == DA_F16 ? 15.0f : 0.0f));
      const float ref = mn == -INFINITY ? 0.0f : mn;
      const float alpha = exp2_fast(mx - ref);
      mx = mn;
      u32x4 hi[2], lo[2];
      float ps = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = exp2_fast(__builtin_fmaf(x[r], c, -ref)), p1 = exp2_fast(__builtin_fmaf(x[r + 1], c, -ref));
        const uint32_t w = E16<DT>::pack(p0, p1);
        hi[r >> 3][(r & 7) >> 1] = w;
        lo[r >> 3][(r & 7) >> 1] = E16<DT>::pack(p0 - E16<DT>::lo(w), p1 - E16<DT>::hi(w));
        ps += p0 + p1;
      }
      if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
        l *= alpha;
      }
      l += ps;
      if (more) wait_loads<STAGES == 2 ? 24 : 8>();
      else if (STAGES == 2 && i + 1 < m) wait_loads<16>();
      else wait_loads<0>();
      u32x4 v[4];
      read_values<0>(v, va + stage);
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        o[db] = E16<DT>::mfma(v[db], hi[0], o[db]);
        o[db] = E16<DT>::mfma(v[db], lo[0], o[db]);
      }
      read_values<4096>(v, va + stage);
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        o[db] = E16<DT>::mfma(v[db], hi[1], o[db]);
        o[db] = E16<DT>::mfma(v[db], lo[1], o[db]);
      }
      if (more) load_rows(false, i + STAGES);
    }

    // ---- the four waves' results joined: each leaves its rows in its own LDS, 16-byte chunk c of row
    // r at c ^ r; thread t then adds up 16 dims of row t / 8 ----
    l = halves_sum(l);
    if (hl == 0) sh.ml[wid][0][ql] = mx, sh.ml[wid][1][ql] = l;
    if (ql < rows) {
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *(f32x4*)(kl + ql * 512 + ((8 * db + 2 * j + hl) ^ ql) * 16) =
              f32x4{o[db][4 * j], o[db][4 * j + 1], o[db][4 * j + 2], o[db][4 * j + 3]};
    }
    __syncthreads();
    const int r = tid >> 3, d0 = 16 * (tid & 7);
    if (r < rows) {
      float M = -INFINITY, L = 0.0f, fw[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) M = __builtin_fmaxf(M, sh.ml[w][0][r]);
      const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        fw[w] = exp2_fast(sh.ml[w][0][r] - ref);
        L += sh.ml[w][1][r] * fw[w];
      }
      f32x4 y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 z = *(const f32x4*)(smem + w * kWaveLds + r * 512 + (((d0 >> 2) + j) ^ r) * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[j][i] += z[i] * fw[w];
        }
      const int rt = f + r / a.G, rh = h * a.G + r % a.G;
      if (n == tiles && a.prefix.B == 0) {
        const float inv = L > 0.0f ? 1.0f / L : 0.0f;
        char* row = a.out + 2 * (rt * a.so_t + rh * a.so_h);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (d0 + 8 * j < a.D)
            *(u32x4*)(row + 2 * (d0 + 8 * j)) =
                u32x4{E16<DT>::pack(y[2 * j][0] * inv, y[2 * j][1] * inv), E16<DT>::pack(y[2 * j][2] * inv, y[2 * j][3] * inv),
                      E16<DT>::pack(y[2 * j + 1][0] * inv, y[2 * j + 1][1] * inv),
                      E16<DT>::pack(y[2 * j + 1][2] * inv, y[2 * j + 1][3] * inv)};
      } else {
        float* state = n == tiles ? a.states + (((int64_t)(own ? 1 : 0) * a.seq.T + rt) * a.Hq + rh) * kState
                                  : a.slots + ((int64_t)(2 * worker + min(part, 1)) * a.slot_rows + r) * kState;
#pragma unroll
        for (int j = 0; j < 4; ++j) *(f32x4*)(state + d0 + 4 * j) = y[j];
        if (d0 == 0) *(f32x2*)(state + 128) = f32x2{M, L};
      }
    }
    // an item that goes on in the next worker's share is joined by whoever has its first part
    if (!a.whole && a.records && tid == 0 && n < tiles) {
      if (t0 == 0) sh.record = StreamRecord{f, nt, h, (int)(2 * worker + min(part, 1)), (int)((tiles - n + share.per - 1) / share.per)};
    }
    ++part;
    const uint32_t used = a.whole ? 1 : n;
    off += used;
    left -= used;
    if (off == (uint32_t)(a.whole ? 1 : tiles) * a.Hkv) ++e, off = 0;
    if (left > 0) __syncthreads();  // the sums are read before the next tiles arrive in their place
  }
  if (!a.whole && a.records && tid == 0) a.records[worker] = sh.record;
}

}  // namespace da
