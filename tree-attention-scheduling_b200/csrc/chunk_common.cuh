// Shared by the two kernels of ta_chunk_attention: the call's parameters, and
// which rows and keys a CTA works on.
#pragma once

#include "ta_common.cuh"

namespace ta {

struct ChunkParams {
  const uint16_t* q;
  int64_t q_st, q_sh;                      // element strides: token, head
  const uint16_t *k, *v;                   // [HK, T, D]
  int64_t pool_tokens;
  const int32_t* table;                    // [B, width]
  int64_t table_stride;
  const int32_t *lens, *cu;                // [B], [B + 1]
  uint16_t* out;                           // [N, HQ, D]
  float* lse;                              // [N, HQ] or null
  float *part, *part_lse;                  // [splits, N, HQ, D], [splits, N, HQ] when splits > 1
  int32_t* status;
  float scale_log2;
  int32_t width, page_shift, num_seqs, num_tokens, hq, hk, group, causal, splits, split_keys;
  int32_t box_rows;                        // rows of the TMA boxes (0: no box maps)
  int32_t cluster;                         // the splits of a row tile are a cluster and join by themselves
};

// What a CTA works on: up to ROWS query rows of a sequence and KV head over a range of keys.
struct Work {
  int32_t seq;        // -1: nothing
  int32_t head;       // KV head
  int32_t token0;     // first token of the sequence's chunk
  int32_t row0;       // first row (token x GQA row) of the CTA within the sequence
  int32_t rows;       // its rows (1 .. ROWS)
  int32_t keys;       // kv_b (within the table)
  int32_t shift;      // keys before the first token's own: its row sees shift + 1 keys (causal)
  int32_t key0;       // first key of the split
  int32_t count;      // keys of the split that the last row sees
  int32_t pad[3];
};

// Resolve a block index, by one converged warp.  The row tiles of
// a sequence are taken from its last (most keys under the causal mask) to its
// first, KV heads fastest.
template <int ROWS>
__device__ __forceinline__ Work find_work(const ChunkParams& p, int block, int split, int lane) {
  constexpr int kSeqs = 4;                  // sequences a lane looks at per round
  Work w;
  w.seq = -1, w.rows = 0, w.count = 0;
  w.head = block % p.hk;
  const int tile = block / p.hk;
  // row tile `local` (from the last) of the `tiles` of a sequence of n tokens from `first` on
  auto resolve = [&](int seq, int first, int n, int keys, int tiles, int local) {
    w.seq = seq;
    w.token0 = first;
    w.row0 = (tiles - 1 - local) * ROWS;
    w.rows = min(ROWS, n * p.group - w.row0);
    const int64_t most = int64_t(p.width) << p.page_shift;
    if (keys < 0 || keys > most) {
      set_status(p.status, TA_ERR_BOUNDS);
      keys = keys < 0 ? 0 : int(most);
    }
    w.keys = keys;
    w.shift = p.causal ? keys - n : INT32_MAX / 2;
    // keys that the CTA's last row sees
    const int seen = max(0, min(keys, w.shift + (w.row0 + w.rows - 1) / p.group + 1));
    const int64_t start = int64_t(split) * p.split_keys;
    w.key0 = int(min(start, int64_t(seen)));
    w.count = int(min(start + int64_t(p.split_keys), int64_t(seen))) - w.key0;
  };

  if (p.num_seqs <= 32) {                   // a sequence a lane: the longest contexts first
    const int first = p.cu[min(lane, p.num_seqs)], last = p.cu[min(lane + 1, p.num_seqs)];
    const int keys = p.lens[min(lane, p.num_seqs - 1)];
    int n = last - first;                   // 0 past the last sequence
    if (first < 0 || last < first || last > p.num_tokens) {
      set_status(p.status, TA_ERR_BOUNDS);
      n = 0;
    }
    const int tiles = int((int64_t(n) * p.group + ROWS - 1) / ROWS);
    int before = 0;
    for (int j = 0; j < p.num_seqs; ++j) {
      const int theirs = __shfl_sync(0xffffffffu, keys, j), count = __shfl_sync(0xffffffffu, tiles, j);
      before += theirs > keys || (theirs == keys && j < lane) ? count : 0;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, lane < p.num_seqs && tile >= before && tile < before + tiles);
    if (hit) {
      const int src = __ffs(hit) - 1;
      resolve(src, __shfl_sync(0xffffffffu, first, src), __shfl_sync(0xffffffffu, n, src),
              __shfl_sync(0xffffffffu, keys, src), __shfl_sync(0xffffffffu, tiles, src),
              tile - __shfl_sync(0xffffffffu, before, src));
    }
    return w;
  }

  int before = 0;
  for (int b0 = 0; b0 < p.num_seqs; b0 += 32 * kSeqs) {
    int edge[kSeqs + 1], len[kSeqs];
#pragma unroll
    for (int i = 0; i <= kSeqs; ++i) edge[i] = p.cu[min(b0 + lane * kSeqs + i, p.num_seqs)];
#pragma unroll
    for (int i = 0; i < kSeqs; ++i) len[i] = p.lens[min(b0 + lane * kSeqs + i, p.num_seqs - 1)];
    int upto[kSeqs], mine = 0;              // row tiles of the lane's sequences up to i
#pragma unroll
    for (int i = 0; i < kSeqs; ++i) {
      int n = edge[i + 1] - edge[i];        // 0 past the last sequence
      if (edge[i] < 0 || edge[i + 1] < edge[i] || edge[i + 1] > p.num_tokens) {
        set_status(p.status, TA_ERR_BOUNDS);
        n = 0;
      }
      mine += int((int64_t(n) * p.group + ROWS - 1) / ROWS);
      upto[i] = mine;
    }
    int all = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, all, off);
      if (lane >= off) all += t;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, tile < before + all);
    if (hit) {
      const int src = __ffs(hit) - 1;
      int local = tile - before - (all - mine), tiles = 0, first = 0, n = 0, keys = 0, seq = 0;
      bool found = false;
#pragma unroll
      for (int i = 0; i < kSeqs; ++i) {
        const int from = i ? upto[i - 1] : 0;
        if (!found && local < upto[i]) {
          found = true;
          tiles = upto[i] - from, first = edge[i], n = edge[i + 1] - edge[i], keys = len[i];
          seq = b0 + lane * kSeqs + i;
          local -= from;
        }
      }
      resolve(__shfl_sync(0xffffffffu, seq, src), __shfl_sync(0xffffffffu, first, src),
              __shfl_sync(0xffffffffu, n, src), __shfl_sync(0xffffffffu, keys, src),
              __shfl_sync(0xffffffffu, tiles, src), __shfl_sync(0xffffffffu, local, src));
      return w;
    }
    before += __shfl_sync(0xffffffffu, all, 31);
  }
  return w;
}

// Softmax weights are carried times 2^kWeightShift: up to 2^8 above the running
// maximum, they lie in [0, 2^15] in f16, whose normal range then reaches 2^-21 of
// the maximum (2^-14 unshifted, a long context's faint keys).
template <typename T> constexpr float kWeightShift = Elem<T>::kCode == TA_DTYPE_F16 ? 7.f : 0.f;

// Rows of at most kSmallRows (token x GQA row) a sequence: chunk_rows.cu.
constexpr int kSmallRows = 16;
// Resident CTAs an SM of the small-row kernel, and the keys its splits are multiples of.
constexpr int kSmallCtas = 2, kSmallKeys = 64;
// Its splits that can join in a cluster (the portable size).
constexpr int kMaxCluster = 8;

cudaError_t launch_chunk_rows(const ChunkParams& p, int64_t tiles, int head_dim, int dtype, cudaStream_t stream);

}  // namespace ta
