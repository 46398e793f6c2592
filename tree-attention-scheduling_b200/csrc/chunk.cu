// Attention of ragged chunks of new tokens over pages of the pools, behind
// ta_chunk_attention.
//
// Row i of sequence b (n_b new tokens, kv_b keys in all) attends the keys
//   [0, min(kv_b, kv_b - n_b + i + 1))   causal, or   [0, kv_b)   otherwise,
//   out = sum_j exp(s_j - lse) v_j,   s_j = scale * q.k_j,   lse = log sum_j exp(s_j),
// a row without keys has out = 0 and lse = -inf.  Key j lies at pool position
// table[b, j / page] * page + j % page; a tree path is a table of page size 1.
//
// One CTA: up to 256 query rows (token x GQA row) of one sequence and KV head
// over a range of its keys.  Roles:
//
//   warps 0-1   load K tiles (128 keys), warps 2-3 V tiles: warp w the tiles of
//               parity w & 1 into ring slot w & 1.  Rows are gathered by
//               16-byte cp.async into the 128-byte-swizzled layout the MMAs read,
//               so any page size, order and fragmentation costs the same; keys
//               past kv_b are filled with zeros
//   warp 4      issues every tcgen05.mma (converged, one elected lane)
//   warps 8-15  softmax: warpgroup t serves stream t, one thread per query row
//
// and two streams keep the tensor pipe busy while the other's softmax runs:
//
//   more than 128 rows:  stream t = rows [128 t, 128 t + 128) over every key
//                        tile (each K/V tile feeds four 128-row MMAs)
//   up to 128 rows:      stream t = all rows over the key tiles of parity t,
//                        with its own running maximum, sum and O; the two are
//                        combined through shared memory at the end
//
// S_t and P_t share TMEM columns; O_t accumulates in TMEM and is rescaled only
// when a row's maximum grows by more than 2^8 (exact after the division).  P is
// rounded to the input type for P.V (a relative 2^-9 or 2^-12 per weight, at
// random); sums and the LSE use the unrounded f32 weights.
//
// When the (tile, KV head) pairs do not fill the GPU the keys are cut into
// splits whose normalised f32 partials chunk_merge_kernel combines by LSE.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "ta_kernels.cuh"
#include "tc_common.cuh"

namespace ta {

namespace {

constexpr int kRows = 128;                 // query rows of a tile (MMA M)
constexpr int kPairRows = 2 * kRows;       // query rows of a CTA
constexpr int kKeys = 128;                 // keys of a K/V tile
constexpr int kStages = 2;
constexpr int kLoadWarps = 4, kIssueWarp = 4, kSoftmaxWarp0 = 8;
constexpr int kThreads = 512;
// register split of the four warpgroups: 2 x 128 x 184 + 2 x 128 x 72 = 512 x 128
constexpr int kSoftmaxRegs = 184, kOtherRegs = 72;
constexpr uint32_t kTmemCols = 512, kColS = 0, kColO = 256;   // + stream * 128
constexpr float kRescaleThreshold = 8.f;   // log2 units
constexpr int kMaxSplits = 64;

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
  int32_t width, page_shift, num_seqs, num_tokens, hq, group, causal, splits, split_tiles;
};

template <int D>
struct Smem {
  static constexpr uint32_t kTile = kRows * D * 2;
  static constexpr uint32_t kBlock = D >= 64 ? kRows * 128 : kTile * 2;    // one 64-column swizzled block
  static constexpr uint32_t kSlot = D >= 64 ? kTile : kRows * 128;         // D = 32 keeps 128-byte rows
  static constexpr uint32_t off_q = 0;
  static constexpr uint32_t off_k = off_q + 2 * kSlot;
  static constexpr uint32_t off_v = off_k + kStages * kSlot;
  static constexpr uint32_t off_mz = off_v + kStages * kSlot;              // stream 1's maximum and sum per row
  static constexpr uint32_t off_bar = off_mz + kRows * 8;
  static constexpr uint32_t off_tmem = off_bar + 16 * 8;
  static constexpr uint32_t off_work = off_tmem + 16;
  static constexpr uint32_t bytes = off_work + 32;
  static constexpr uint32_t alloc = bytes + 1024;                          // slack to align the base to 1 KB
};

enum Bar { K_FULL = 0, K_EMPTY = 2, V_FULL = 4, V_EMPTY = 6, S_FULL = 8, P_FULL = 10, PV_DONE = 12, Q_FULL = 14 };

// Byte offset of 16-byte chunk c of row r in a tile of 128-byte rows (64
// columns a block) with the 128-byte swizzle.
template <int D>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  return uint32_t(c >> 3) * Smem<D>::kBlock + uint32_t(r) * 128u + uint32_t(((c & 7) ^ (r & 7)) << 4);
}

template <int R>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}

// What a CTA works on.
struct Work {
  int32_t seq;        // -1: nothing
  int32_t token0;     // first token of the sequence's chunk
  int32_t row0;       // first row (token x GQA row) of the CTA within the sequence
  int32_t rows;       // rows of the CTA (1 .. 256)
  int32_t keys;       // kv_b (within the table)
  int32_t shift;      // keys before the first token's own: its row sees shift + 1 keys (causal)
  int32_t key0;       // first key of the CTA's split
  int32_t tiles;      // key tiles of the CTA
};

// Resolve blockIdx into a Work, by one converged warp.  The tiles of a sequence
// are taken from its last (most keys under the causal mask) to its first.
__device__ __forceinline__ Work find_work(const ChunkParams& p, int tile, int split, int lane) {
  Work w;
  w.seq = -1, w.rows = 0, w.tiles = 0;
  int before = 0;
  for (int b0 = 0; b0 < p.num_seqs; b0 += 32) {
    const int b = b0 + lane;
    int first = 0, n = 0;
    if (b < p.num_seqs) {
      first = p.cu[b];
      const int last = p.cu[b + 1];
      if (first < 0 || last < first || last > p.num_tokens)
        set_status(p.status, TA_ERR_BOUNDS);
      else
        n = last - first;
    }
    const int mine = int((int64_t(n) * p.group + kPairRows - 1) / kPairRows);
    int upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += t;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, tile < before + upto);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int local = tile - before - __shfl_sync(0xffffffffu, upto - mine, src);
      const int tiles = __shfl_sync(0xffffffffu, mine, src);
      n = __shfl_sync(0xffffffffu, n, src);
      w.seq = b0 + src;
      w.token0 = __shfl_sync(0xffffffffu, first, src);
      w.row0 = (tiles - 1 - local) * kPairRows;
      w.rows = min(kPairRows, n * p.group - w.row0);
      int keys = p.lens[w.seq];
      const int64_t most = int64_t(p.width) << p.page_shift;
      if (keys < 0 || keys > most) {
        set_status(p.status, TA_ERR_BOUNDS);
        keys = keys < 0 ? 0 : int(most);
      }
      w.keys = keys;
      w.shift = p.causal ? keys - n : INT32_MAX / 2;
      // keys that the CTA's last row sees
      const int seen = max(0, min(keys, w.shift + (w.row0 + w.rows - 1) / p.group + 1));
      const int64_t start = int64_t(split) * p.split_tiles * kKeys;
      w.key0 = int(min(start, int64_t(seen)));
      const int end = int(min(start + int64_t(p.split_tiles) * kKeys, int64_t(seen)));
      w.tiles = (end - w.key0 + kKeys - 1) / kKeys;
      return w;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return w;
}

// 16 bytes of a key row per lane into a ring slot: warp-wide gather of one tile.
template <int D>
__device__ __forceinline__ void load_tile(unsigned char* slot, const uint16_t* pool, const int (&pos)[4], int lane) {
  constexpr int LPR = D / 8, RPI = 32 / LPR;     // lanes of a row, rows of an instruction
  const int c = lane % LPR, r = lane / LPR;
#pragma unroll
  for (int i = 0; i < kKeys / RPI; ++i) {
    const int row = i * RPI + r;
    const int at = __shfl_sync(0xffffffffu, pos[(i * RPI) / 32], row & 31);
    cp_async16_zfill(slot + swz<D>(row, c), pool + int64_t(max(at, 0)) * D + c * 8, at >= 0 ? 16u : 0u);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(ChunkParams p) {
  using S = Smem<D>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::off_bar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::off_tmem);
  Work* work = reinterpret_cast<Work*>(smem + S::off_work);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = blockIdx.y, split = blockIdx.z;
  const int G = p.group;

  if (warp == 0) {
    const Work w = find_work(p, blockIdx.x, split, lane);
    if (lane == 0) {
      *work = w;
      const int rows_b = max(0, w.rows - kRows);
      for (int s = 0; s < 2; ++s) {
        mbar_init(&bars[K_FULL + s], 1);
        mbar_init(&bars[K_EMPTY + s], 1);
        mbar_init(&bars[V_FULL + s], 1);
        mbar_init(&bars[V_EMPTY + s], 1);
        mbar_init(&bars[S_FULL + s], 1);
        // softmax warps with rows: those without take no part
        const int rows_t = (s == 0 || rows_b == 0) ? min(kRows, max(1, w.rows)) : rows_b;
        mbar_init(&bars[P_FULL + s], (rows_t + 31) / 32);
        mbar_init(&bars[Q_FULL + s], (rows_t + 31) / 32);
        mbar_init(&bars[PV_DONE + s], 1);
      }
      fence_barrier_init();
    }
  } else if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();                                 // the merge may be placed; it waits for this grid's end
  const uint32_t tmem = *tmem_slot;
  const Work w = *work;
  const int ntiles = w.seq < 0 ? 0 : w.tiles;
  const bool two = w.rows > kRows;               // two row tiles, else two key streams
  bool alive = true;

  if (warp < kLoadWarps) {
    regs_down<kOtherRegs>();
    // ---------------- K/V gather ----------------
    const bool is_k = warp < 2;
    const int slot = warp & 1;
    unsigned char* dst = smem + (is_k ? S::off_k : S::off_v) + slot * S::kSlot;
    const uint16_t* pool = (is_k ? p.k : p.v) + int64_t(head) * p.pool_tokens * D;
    uint64_t* full = &bars[(is_k ? K_FULL : V_FULL) + slot];
    uint64_t* empty = &bars[(is_k ? K_EMPTY : V_EMPTY) + slot];
    const int32_t* table = p.table + int64_t(max(w.seq, 0)) * p.table_stride;
    for (int j = slot; j < ntiles; j += 2) {
      int pos[4];
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = w.key0 + j * kKeys + i * 32 + lane;
        pos[i] = -1;
        if (key < w.keys) {
          const int page = 1 << p.page_shift;
          const int64_t at = int64_t(table[key >> p.page_shift]) * page + (key & (page - 1));
          if (at >= 0 && at < p.pool_tokens)
            pos[i] = int(at);
          else
            bad = true;
        }
      }
      if (bad) set_status(p.status, TA_ERR_BOUNDS);
      if (j >= kStages && !warp_wait(empty, (j / kStages + 1) & 1, p.status)) break;
      load_tile<D>(dst, pool, pos, lane);
      cp_async_wait_all();
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
    }
  } else if (warp < kSoftmaxWarp0) {
    regs_down<kOtherRegs>();
    if (warp == kIssueWarp && ntiles > 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t ab = Elem<T>::kCode == TA_DTYPE_BF16 ? 1u : 0u;
      constexpr uint32_t idesc_s = umma_idesc(ab, 0, 0, kRows, kKeys);
      constexpr uint32_t idesc_o = umma_idesc(ab, 0, 1, kRows, D);
      const uint64_t qdesc0 = smem_desc(smem_u32(smem + S::off_q), 16, 1024);
      const uint64_t kdesc0 = smem_desc(smem_u32(smem + S::off_k), 16, 1024);
      const uint64_t vdesc0 = smem_desc(smem_u32(smem + S::off_v), S::kBlock, 1024);
      // stream t's u-th key tile, and how many it has
      auto tile_of = [&](int t, int u) { return two ? u : 2 * u + t; };
      const int count[2] = {two ? ntiles : (ntiles + 1) / 2, two ? ntiles : ntiles / 2};

      auto issue_s = [&](int t, int j) {   // S_t = Q K(j)^T
        const uint64_t qd = qdesc0 + uint64_t(two ? t : 0) * (S::kSlot >> 4);
        const uint64_t kd = kdesc0 + uint64_t(j % kStages) * (S::kSlot >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t off = ((k >> 2) * S::kBlock + (k & 3) * 32) >> 4;
          umma_ss_warp(tmem + kColS + t * 128, qd + off, kd + off, idesc_s, k > 0 ? 1u : 0u);
        }
        umma_commit_warp(&bars[S_FULL + t]);
        if (!two || t == 1) umma_commit_warp(&bars[K_EMPTY + j % kStages]);
      };
      auto issue_pv = [&](int t, int u, int j) {  // O_t += P_t V(j)
        const uint64_t vd = vdesc0 + uint64_t(j % kStages) * (S::kSlot >> 4);
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          umma_ts_warp(tmem + kColO + t * 128, tmem + kColS + t * 128 + k * 8, vd + ((k * 2048) >> 4), idesc_o,
                       (u > 0 || k > 0) ? 1u : 0u);
        if (u == count[t] - 1) umma_commit_warp(&bars[PV_DONE + t]);
        if (!two || t == 1) umma_commit_warp(&bars[V_EMPTY + j % kStages]);
      };
      auto full = [&](int bar, int j) { return warp_wait(&bars[bar + j % kStages], (j / kStages) & 1, p.status); };

      for (int t = 0; t < 2 && alive; ++t) {
        if (count[t] == 0) continue;
        const int j = tile_of(t, 0);
        if (!warp_wait(&bars[Q_FULL + (two ? t : 0)], 0, p.status) || !full(K_FULL, j)) { alive = false; break; }
        tc_fence_after();
        issue_s(t, j);
      }
      for (int u = 0; u < count[0] && alive; ++u) {
        for (int t = 0; t < 2; ++t) {
          if (u >= count[t]) continue;
          const int j = tile_of(t, u), next = tile_of(t, u + 1);
          const bool more = u + 1 < count[t];
          // V(j) and the next K are normally there before P(u): wait for them
          // first, so that P's arrival is followed by MMAs only
          if (!full(V_FULL, j) || (more && !full(K_FULL, next)) ||
              !warp_wait(&bars[P_FULL + t], u & 1, p.status)) {
            alive = false;
            break;
          }
          tc_fence_after();
          issue_pv(t, u, j);
          if (more) issue_s(t, next);
        }
      }
      // the last commits must land before the CTA's shared memory is released
      if (alive)
        for (int j = max(0, ntiles - kStages); j < ntiles; ++j)
          if (!warp_wait(&bars[K_EMPTY + j % kStages], (j / kStages) & 1, p.status) ||
              !warp_wait(&bars[V_EMPTY + j % kStages], (j / kStages) & 1, p.status))
            break;
    }
  } else {
    regs_up<kSoftmaxRegs>();
    // ---------------- softmax and epilogue ----------------
    const int t = (warp - kSoftmaxWarp0) >> 2;
    const int quad = warp & 3;
    const int row = quad * 32 + lane;                       // row within the tile, its TMEM lane
    const int trow = (two ? t * kRows : 0) + row;           // row within the CTA
    const int base_row = (two ? t * kRows : 0) + quad * 32; // first row of the warp
    const bool active = w.seq >= 0 && base_row < w.rows;    // uniform in the warp
    if (active) {
      const bool mine = trow < w.rows;
      const int local = w.row0 + trow;                      // row within the sequence
      const int token = w.token0 + (mine ? local / G : 0), g = mine ? local % G : 0;
      const int hq = head * G + g;
      const int limit = mine ? min(w.keys, w.shift + local / G + 1) - w.key0 : 0;   // visible keys of the split
      const int count = two ? ntiles : (ntiles + 1 - t) / 2;
      const uint32_t lane_addr = tmem + (uint32_t(quad * 32) << 16);
      const uint32_t s_col = kColS + t * 128, o_col = kColO + t * 128;

      if (ntiles > 0 && (two || t == 0)) {
        unsigned char* qs = smem + S::off_q + (two ? t : 0) * S::kSlot;
        const uint4* src = reinterpret_cast<const uint4*>(p.q + int64_t(token) * p.q_st + int64_t(hq) * p.q_sh);
        uint4 x[D / 8];
#pragma unroll
        for (int c = 0; c < D / 8; ++c) x[c] = mine ? src[c] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(qs + swz<D>(row, c)) = x[c];
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[Q_FULL + (two ? t : 0)]);
      }

      const float scale = p.scale_log2;
      float m_run = -INFINITY, z = 0.f;
      for (int u = 0; u < count; ++u) {
        const int valid = limit - (two ? u : 2 * u + t) * kKeys;     // visible keys of this tile and after
        if (!warp_wait(&bars[S_FULL + t], u & 1, p.status)) { alive = false; break; }
        tc_fence_after();
        float s[kKeys];
        {
          uint32_t a[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(lane_addr + s_col + c * 32, a[c]);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) s[c * 32 + i] = __uint_as_float(a[c][i]);
        }
        if (__any_sync(0xffffffffu, valid < kKeys)) {
#pragma unroll
          for (int i = 0; i < kKeys; ++i) s[i] = i < valid ? s[i] : -INFINITY;
        }
        const float m_tile = max128(s) * scale;
        bool rescale = false;
        float m_new = m_run;
        if (u == 0) {
          m_new = m_tile;
        } else if (m_tile > m_run + kRescaleThreshold) {
          m_new = m_tile;
          rescale = true;
        }
        const float alpha = rescale ? fast_exp2(m_run - m_new) : 1.f;
        z *= alpha;
        m_run = m_new;
        // a row without a visible key so far: exp2(-inf - 0) = 0
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        F2 sum = splat(0.f);
        const F2 sc = splat(scale), neg_m = splat(-m_use);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t packed[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            F2 x;
            x.f = make_float2(s[32 * h + 2 * i], s[32 * h + 2 * i + 1]);
            x = ffma2(x, sc, neg_m);
            F2 e;
            e.f = make_float2(fast_exp2(x.f.x), fast_exp2(x.f.y));
            sum = fadd2(sum, e);
            packed[i] = Elem<T>::pack2(e.f.x, e.f.y);
          }
          tmem_st16(lane_addr + s_col + h * 16, packed);
        }
        z += sum.f.x + sum.f.y;
        if (__any_sync(0xffffffffu, rescale)) {
          // O_t holds the earlier tiles' P.V (S_t(u) was issued after them)
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(lane_addr + o_col + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(lane_addr + o_col + c * 32, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[P_FULL + t]);
      }
      if (count > 0 && alive && !warp_wait(&bars[PV_DONE + t], 0, p.status)) alive = false;
      tc_fence_after();
      if (!alive) z = 0.f;

      // two key streams: stream 1 hands its O, maximum and sum to stream 0
      float m = m_run, scale_a = 1.f, scale_b = 0.f;
      // its O goes where only its own MMAs read, columns halved over the second
      // query slot (not used here) and K slot 1 (the tiles of odd parity)
      auto other = [&](int chunk) {                         // 4 columns of this row
        unsigned char* half = smem + (chunk < D / 8 ? S::off_q : S::off_k) + S::kSlot;
        constexpr int kSwz = (D / 8 < 8 ? D / 8 : 8) - 1;
        return reinterpret_cast<float4*>(half) + row * (D / 8) + ((chunk % (D / 8)) ^ (row & kSwz));
      };
      float2* mz = reinterpret_cast<float2*>(smem + S::off_mz) + row;
      const bool joined = !two && ntiles > 1;
      const int warps = (w.rows + 31) / 32;                 // active warps of a stream (two key streams)
      if (joined && t == 1) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(lane_addr + o_col + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *other(c * 8 + i) =
                make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                            __uint_as_float(o[4 * i + 3]));
        }
        *mz = make_float2(m_run, z);
      }
      if (joined) named_sync(1, warps * 2 * 32);
      if (two || t == 0) {
        if (joined) {
          const float2 b = *mz;
          m = fmaxf(m_run, b.x);
          const float m_use = m == -INFINITY ? 0.f : m;
          scale_a = fast_exp2(m_run - m_use);
          scale_b = b.y > 0.f ? fast_exp2(b.x - m_use) : 0.f;
          z = z * scale_a + b.y * scale_b;
        }
        const float inv = z > 0.f ? 1.f / z : 0.f;
        scale_a = z > 0.f ? scale_a * inv : 0.f;
        scale_b *= inv;
        const int64_t index = int64_t(token) * p.hq + hq;
        const float lse = z > 0.f ? (m + fast_log2(z)) * kLn2 : -INFINITY;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          float y[32];
          if (ntiles > 0) {
            tmem_ld32(lane_addr + o_col + c * 32, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = scale_a > 0.f ? __uint_as_float(o[i]) * scale_a : 0.f;
          if (joined && scale_b > 0.f) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 b = *other(c * 8 + i);
              y[4 * i] += b.x * scale_b, y[4 * i + 1] += b.y * scale_b;
              y[4 * i + 2] += b.z * scale_b, y[4 * i + 3] += b.w * scale_b;
            }
          }
          if (!mine) continue;
          if (p.splits > 1) {
            if (!(z > 0.f)) continue;                       // no weight in the merge: not read
            float* dst = p.part + (int64_t(split) * p.num_tokens * p.hq + index) * D + c * 32;
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(dst + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
          } else {
            uint16_t* dst = p.out + index * D + c * 32;
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4*>(dst + i) =
                  make_uint4(Elem<T>::pack2(y[i], y[i + 1]), Elem<T>::pack2(y[i + 2], y[i + 3]),
                             Elem<T>::pack2(y[i + 4], y[i + 5]), Elem<T>::pack2(y[i + 6], y[i + 7]));
          }
        }
        if (mine) {
          if (p.splits > 1)
            p.part_lse[int64_t(split) * p.num_tokens * p.hq + index] = lse;
          else if (p.lse)
            p.lse[index] = lse;
        }
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kIssueWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

// Combine the splits of a row: one warp per (token, query head).
constexpr int kMergeWarps = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kMergeWarps * 32) chunk_merge_kernel(ChunkParams p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t index = int64_t(blockIdx.x) * kMergeWarps + (threadIdx.x >> 5);
  const int64_t rows = int64_t(p.num_tokens) * p.hq;
  const int first = p.cu[0], last = p.cu[p.num_seqs];        // inputs of the call
  pdl_wait();
  const int token = int(index / p.hq);
  if (index >= rows || token < first || token >= last) return;
  float l0 = lane < p.splits ? p.part_lse[lane * rows + index] : -INFINITY;
  float l1 = lane + 32 < p.splits ? p.part_lse[(lane + 32) * rows + index] : -INFINITY;
  const float m = warp_max(fmaxf(l0, l1));
  const float m_use = m == -INFINITY ? 0.f : m;
  l0 = expf(l0 - m_use);
  l1 = expf(l1 - m_use);
  const float z = warp_sum(l0 + l1);
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int s0 = 0; s0 < p.splits; s0 += 8) {
    float x[8][E];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = s0 + i;
      const float weight = s < p.splits ? __shfl_sync(0xffffffffu, s < 32 ? l0 : l1, s & 31) : 0.f;
      const float* src = p.part + (int64_t(s) * rows + index) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][e] = weight > 0.f ? src[e] * weight : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += x[i][e];
  }
  const float inv = z > 0.f ? 1.f / z : 0.f;
  uint16_t* dst = p.out + index * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[e] = Elem<T>::from_float(acc[e] * inv);
  if (lane == 0 && p.lse) p.lse[index] = z > 0.f ? m + logf(z) : -INFINITY;
}

// ---- host ---------------------------------------------------------------------
struct Split {
  int splits, tiles;
};

int sm_count() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return 148;
  }
  int sms = cached[dev].load();
  if (!sms) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
      cudaGetLastError();
      sms = 148;
    }
    cached[dev].store(sms);
  }
  return sms;
}

// Most row tiles a batch of num_tokens over num_seqs sequences can have.
int64_t tile_bound(int64_t tokens, int64_t seqs, int64_t group) {
  return tokens * group / kPairRows + std::min(tokens, seqs);
}

// Splits of the keys: the least modelled time (tenths of a microsecond) of the
// waves of CTAs, a CTA costing kFixed plus kPerTile a key tile, and the merge.
Split choose_split(int64_t tokens, int64_t seqs, int64_t group, int64_t hk, int64_t most_keys, int sms) {
  constexpr int64_t kFixed = 50, kPerTile = 10, kMerge = 35;
  const int64_t base = tile_bound(tokens, seqs, group) * hk;
  const int64_t tiles = std::max<int64_t>(1, (most_keys + kKeys - 1) / kKeys);
  Split best{1, int(std::min<int64_t>(tiles, INT32_MAX / kKeys))};
  int64_t least = INT64_MAX;
  for (int64_t s = 1; s <= std::min<int64_t>(kMaxSplits, tiles); ++s) {
    const int64_t per = (tiles + s - 1) / s;
    if (s > 1 && (tiles + per - 1) / per != s) continue;     // the same cut as a smaller s
    const int64_t waves = (base * s + sms - 1) / sms;
    const int64_t cost = waves * (kFixed + per * kPerTile) + (s > 1 ? kMerge : 0);
    if (cost < least) {
      least = cost;
      best.splits = int(s);
      best.tiles = int(per);
    }
    if (s > 1 && waves > 8) break;
  }
  return best;
}

int64_t partial_bytes(int splits, int64_t tokens, int64_t hq, int64_t dim) {
  return splits > 1 ? int64_t(splits) * tokens * hq * (dim + 1) * 4 : 0;
}

template <typename T, int D>
cudaError_t launch_typed(const ChunkParams& p, int64_t tiles, int hk, cudaStream_t stream) {
  auto kernel = chunk_kernel<T, D>;
  static std::atomic<uint64_t> configured{0};                // one bit a device
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev >= 64 || !(configured.load() >> dev & 1)) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Smem<D>::alloc));
    if (err != cudaSuccess) return err;
    if (dev < 64) configured.fetch_or(uint64_t(1) << dev);
  }
  kernel<<<dim3(unsigned(tiles), unsigned(hk), unsigned(p.splits)), kThreads, Smem<D>::alloc, stream>>>(p);
  err = cudaGetLastError();
  if (err != cudaSuccess || p.splits == 1) return err;
  const int64_t rows = int64_t(p.num_tokens) * p.hq;
  return launch_dependent(chunk_merge_kernel<T, D>, dim3(unsigned((rows + kMergeWarps - 1) / kMergeWarps)),
                          dim3(kMergeWarps * 32), 0, stream, p);
}

template <typename T>
cudaError_t launch_dim(const ChunkParams& p, int64_t tiles, int hk, int head_dim, cudaStream_t stream) {
  if (head_dim == 128) return launch_typed<T, 128>(p, tiles, hk, stream);
  if (head_dim == 64) return launch_typed<T, 64>(p, tiles, hk, stream);
  return launch_typed<T, 32>(p, tiles, hk, stream);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

}  // namespace ta

extern "C" int64_t ta_chunk_workspace_bytes(int32_t num_tokens, int32_t num_seqs, int32_t num_q_heads,
                                            int32_t num_kv_heads, int32_t head_dim, int32_t table_width,
                                            int32_t page_size) {
  using namespace ta;
  if (num_tokens <= 0 || num_seqs <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
      head_dim <= 0 || table_width < 0 || page_size <= 0)
    return 0;
  const Split s = choose_split(num_tokens, num_seqs, num_q_heads / num_kv_heads, num_kv_heads,
                               int64_t(table_width) * page_size, sm_count());
  return partial_bytes(s.splits, num_tokens, num_q_heads, head_dim);
}

extern "C" int ta_chunk_attention(const void* q, int64_t q_stride_token, int64_t q_stride_head, const void* kpool,
                                  const void* vpool, int64_t pool_tokens, const int32_t* table, int64_t table_stride,
                                  int32_t table_width, int32_t page_size, const int32_t* kv_lens, const int32_t* cu_q,
                                  int32_t num_seqs, int32_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads,
                                  int32_t head_dim, int32_t dtype, float scale, int32_t causal, void* out,
                                  float* out_lse, void* workspace, int64_t workspace_bytes, int32_t* status,
                                  void* stream) {
  using namespace ta;
  if (dtype != TA_DTYPE_BF16 && dtype != TA_DTYPE_F16) return TA_ERR_UNSUPPORTED;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) return TA_ERR_UNSUPPORTED;
  if (num_seqs < 0 || num_tokens < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
      pool_tokens < 0 || table_width < 0 || table_stride < 0)
    return TA_ERR_ARG;
  if (page_size <= 0 || (page_size & (page_size - 1))) return TA_ERR_ARG;
  if (!(scale > 0.f) || !std::isfinite(scale)) return TA_ERR_ARG;
  if (num_seqs == 0 || num_tokens == 0) return TA_OK;
  const int64_t most_keys = int64_t(table_width) * page_size;
  const int group = num_q_heads / num_kv_heads;
  if (most_keys > INT32_MAX / 4 || pool_tokens > INT32_MAX || int64_t(num_tokens) * group > INT32_MAX / 2 ||
      int64_t(num_tokens) > INT32_MAX / 4 || num_kv_heads > 65535)
    return TA_ERR_UNSUPPORTED;
  if (!q || !kpool || !vpool || !kv_lens || !cu_q || !out || (table_width > 0 && !table)) return TA_ERR_ARG;
  if (!aligned(q) || !aligned(kpool) || !aligned(vpool) || !aligned(out) || q_stride_token < 0 || q_stride_head < 0 ||
      (q_stride_token & 7) || (q_stride_head & 7))
    return TA_ERR_ARG;
  const int64_t tiles = tile_bound(num_tokens, num_seqs, group);
  const Split s = choose_split(num_tokens, num_seqs, group, num_kv_heads, most_keys, sm_count());
  const int64_t need = partial_bytes(s.splits, num_tokens, num_q_heads, head_dim);
  if (need > 0 && (!workspace || !aligned(workspace))) return TA_ERR_ARG;
  if (workspace_bytes < need) return TA_ERR_TOO_LARGE;
  ChunkParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.q_st = q_stride_token, p.q_sh = q_stride_head;
  p.k = static_cast<const uint16_t*>(kpool);
  p.v = static_cast<const uint16_t*>(vpool);
  p.pool_tokens = pool_tokens;
  p.table = table, p.table_stride = table_stride, p.width = table_width;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.lens = kv_lens, p.cu = cu_q;
  p.num_seqs = num_seqs, p.num_tokens = num_tokens;
  p.hq = num_q_heads, p.group = group;
  p.causal = causal != 0;
  p.out = static_cast<uint16_t*>(out), p.lse = out_lse;
  p.splits = s.splits, p.split_tiles = s.tiles;
  p.part = static_cast<float*>(workspace);
  p.part_lse = p.part + int64_t(s.splits) * num_tokens * num_q_heads * head_dim;
  p.status = status;
  p.scale_log2 = scale * kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t err = dtype == TA_DTYPE_BF16 ? launch_dim<__nv_bfloat16>(p, tiles, num_kv_heads, head_dim, st)
                                                 : launch_dim<__half>(p, tiles, num_kv_heads, head_dim, st);
  return err == cudaSuccess ? TA_OK : TA_ERR_LAUNCH;
}
