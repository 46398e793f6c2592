// Beam search: selection over beams x vocabulary (ta_beam_select) and the
// reordering of the beams' states (ta_beam_reorder).
//
// With x the logits of beam w, a candidate (w, t) scores
//   score[w] + x[t] - logsumexp(x),
// and a request keeps the k best of its beams x vocabulary, sorted, ties to the
// lowest w * V + t.  Two kernels, the logits read once:
//
//  1. beam_slice_kernel, one CTA per (beam row, slice of 8192 tokens).  The
//     slice stays in registers (32 values a thread).  Within a beam candidates
//     order by x alone, so the slice's k best by (x, lowest t) are all that can
//     matter; they are written with the slice's maximum and sum of exponentials.
//     The k best are found through a bound: if each of the 8 warps gives its
//     ceil(k/8)-th largest thread maximum, the least of these has at least k
//     values at or above it, and (on anything but adversarial data) not many
//     more; those are collected and ranked by counting.  Where more than
//     kMaxCand values pass (ties, most tokens at -inf), the exact k-th largest
//     thread maximum under the total order (x, -t) is the bound instead, which
//     passes at most k threads' values.
//  2. beam_merge_kernel, one CTA per request: each beam's logsumexp from its
//     slices in f64, every listed candidate's score in f64 (beams a rounding
//     apart in f32 would swap), the k-th best list head as the bound, then
//     ranking by counting.
//
// Bound: HBM for the logits (one read); small batches by the two launches'
// latency.  MUFU: one ex2 per logit, 16 a clock and SM, 0.7 of the time the
// bytes of 16-bit logits take.
#include <algorithm>

#include "ta_common.cuh"
#include "ta_kernels.cuh"

namespace ta {

namespace {

constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kPerThread = 32;                              // logits a thread holds
constexpr int kSlice = kBeamThreads * kPerThread;           // logits of a slice
constexpr int kMaxK = 32;
constexpr int kMaxCand = kMaxK * kPerThread;                // 1024: what the exact bound can pass

struct BeamEntry {     // a listed candidate of a slice
  float x;
  int32_t token;       // -1: none
};

// workspace: per (beam row, slice) the sum of exponentials (f64), the maximum
// (f32) and k entries, as three arrays
struct BeamWork {
  double* sum;
  BeamEntry* entries;
  float* top;
};

struct BeamParams {
  const void* logits;
  const float* scores;            // [R, W]
  const uint8_t* finished;        // [R, W] or null
  BeamWork work;
  float* out_scores;              // [R, k]
  int64_t *out_parents, *out_tokens;
  int64_t row_stride;             // elements between beam rows
  int32_t beams, vocab, k, slices, end_token;
};

template <int DT> struct Logit;
template <> struct Logit<TA_DTYPE_BF16> {
  static constexpr int kVec = 8;
  using Scalar = uint16_t;
  __device__ static float one(uint16_t b) { return Elem<__nv_bfloat16>::to_float(b); }
  __device__ static void unpack(const uint4& u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<__nv_bfloat16>::to_float2(w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
};
template <> struct Logit<TA_DTYPE_F16> {
  static constexpr int kVec = 8;
  using Scalar = uint16_t;
  __device__ static float one(uint16_t b) { return Elem<__half>::to_float(b); }
  __device__ static void unpack(const uint4& u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<__half>::to_float2(w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
};
template <> struct Logit<TA_DTYPE_F32> {
  static constexpr int kVec = 4;
  using Scalar = float;
  __device__ static float one(float b) { return b; }
  __device__ static void unpack(const uint4& u, float* x) {
    x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
  }
};

// Bytes [skew, skew + 16) of the 32 bytes a, b (skew even, below 16).
__device__ __forceinline__ uint4 shift_bytes(const uint4& a, const uint4& b, int skew) {
  const int bits = (skew & 3) * 8;
  uint32_t w[5];
  switch (skew >> 2) {     // the same for the whole CTA
    case 0: w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x; break;
    case 1: w[0] = a.y, w[1] = a.z, w[2] = a.w, w[3] = b.x, w[4] = b.y; break;
    case 2: w[0] = a.z, w[1] = a.w, w[2] = b.x, w[3] = b.y, w[4] = b.z; break;
    default: w[0] = a.w, w[1] = b.x, w[2] = b.y, w[3] = b.z, w[4] = b.w; break;
  }
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// Total order of a slice's candidates: larger x first, then the lower token
// (0: no candidate; -inf maps above it, and -0 equals +0).
__device__ __forceinline__ uint64_t order_key(float x, int32_t token) {
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t o = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return (uint64_t(o) << 32) | uint32_t(~token);
}

__device__ __forceinline__ int block_count(int v, int* s_warp, int warp, int lane) {
  v = __reduce_add_sync(0xffffffffu, v);
  if (lane == 0) s_warp[warp] = v;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int i = 0; i < kBeamWarps; ++i) total += s_warp[i];
  __syncthreads();
  return total;
}

template <int DT>
__global__ void __launch_bounds__(kBeamThreads, 4) beam_slice_kernel(BeamParams p) {
  using L = Logit<DT>;
  constexpr int VEC = L::kVec, NV = kPerThread / VEC;
  __shared__ uint64_t s_cand[kMaxCand];
  __shared__ uint64_t s_best[kBeamThreads];
  __shared__ float s_warp_max[kBeamWarps];
  __shared__ float s_warp_bound[kBeamWarps];
  __shared__ double s_warp_sum[kBeamWarps];
  __shared__ int s_count;
  __shared__ int s_warp_n[kBeamWarps];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int slice = blockIdx.y, k = p.k;
  const int64_t row = blockIdx.x;
  const int64_t out = row * p.slices + slice;
  BeamEntry* entries = p.work.entries + out * k;
  if (tid == 0) s_count = 0;
  pdl_trigger();                                           // the merge may be placed; it waits for this grid

  // Which tokens a thread sums goes by the token alone, not by the row's
  // address, so equal rows give equal sums wherever they lie and their
  // candidates tie exactly.  Rows that start inside a 16-byte vector (odd
  // vocabularies) are read in aligned vectors all the same: a lane's values
  // lie in its own vector and the next lane's, `skew` bytes in.
  using Scalar = typename L::Scalar;
  const Scalar* base = static_cast<const Scalar*>(p.logits) + row * p.row_stride;
  const int skew = int(reinterpret_cast<uintptr_t>(base) & 15u);
  const int back = skew / int(sizeof(Scalar));               // elements of a vector before its lane's tokens
  const int64_t first = int64_t(slice) * kSlice;
  const float score = p.scores[row];
  const bool done = p.finished && p.finished[row];
  const bool dead = !(score > -INFINITY);                  // -inf (or NaN): every candidate is at -inf
  const bool read = !done && !dead;

  auto token_of = [&](int v, int i) { return int32_t(first + (int64_t(v) * kBeamThreads + tid) * VEC + i); };
  float x[kPerThread];
  uint4 raw[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t t0 = first + (int64_t(v) * kBeamThreads + tid) * VEC - back;     // tokens of the aligned vector
    raw[v] = make_uint4(0, 0, 0, 0);
    if (read && t0 >= 0 && t0 + VEC <= p.vocab) raw[v] = *reinterpret_cast<const uint4*>(base + t0);
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t t0 = first + (int64_t(v) * kBeamThreads + tid) * VEC;
    if (back) {
      const uint4 a = raw[v];
      uint4 b = make_uint4(__shfl_down_sync(0xffffffffu, a.x, 1), __shfl_down_sync(0xffffffffu, a.y, 1),
                           __shfl_down_sync(0xffffffffu, a.z, 1), __shfl_down_sync(0xffffffffu, a.w, 1));
      const int64_t t1 = t0 - back + VEC;                   // the next warp's first vector: mostly in L1 by now
      if (lane == 31) b = read && t1 + VEC <= p.vocab ? *reinterpret_cast<const uint4*>(base + t1) : a;
      raw[v] = shift_bytes(a, b, skew);
    }
    // both vectors whole within the row
    const bool whole = read && t0 - back >= 0 && t0 - back + (back ? 2 : 1) * VEC <= p.vocab;
    if (whole) {
      L::unpack(raw[v], x + v * VEC);
    } else {
      // the row's ends, or a beam whose logits do not count: a finished beam
      // offers its end token alone, with its score unchanged
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int64_t t = t0 + i;
        float y = -INFINITY;
        if (t < p.vocab) {
          if (read)
            y = L::one(base[t]);
          else if (done && !dead && t == p.end_token)
            y = 0.f;
        }
        x[v * VEC + i] = y;
      }
    }
  }
  float mine = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) mine = fmaxf(mine, x[i]);     // fmaxf passes over NaN
  // the warp's ceil(k / 8)-th largest thread maximum, ties counted one by one
  float bound = warp_max(mine), left = mine;
  if (lane == 0) s_warp_max[warp] = bound;
  for (int j = 1; j * kBeamWarps < k; ++j) {
    const unsigned holders = __ballot_sync(0xffffffffu, left == bound);
    if (lane == __ffs(holders) - 1) left = -INFINITY;
    bound = warp_max(left);
  }
  if (lane == 0) s_warp_bound[warp] = bound;
  __syncthreads();
  float m = s_warp_max[0];
  bound = s_warp_bound[0];
#pragma unroll
  for (int i = 1; i < kBeamWarps; ++i) m = fmaxf(m, s_warp_max[i]), bound = fminf(bound, s_warp_bound[i]);

  // sum of exp(x - m): f32 over a thread's 32 values, f64 beyond.  An argument
  // of ex2 below 16 in magnitude is off by 2^-21 at most, at random, so the sum
  // over many terms keeps about 1e-8.
  float part = 0.f;
  if (m > -INFINITY) {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) part += fast_exp2((x[i] - m) * kLog2e);
  }
  // NaN counts as -inf and +inf as the largest finite value; both are rare
  // enough to be found by what they do to the sum and the maximum
  const bool odd = __syncthreads_or(!(part < INFINITY) || m == INFINITY) != 0;
  if (odd) {
    m = fminf(m, 3.402823466e38f);
    part = 0.f;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      x[i] = fminf(fmaxf(x[i], -INFINITY), 3.402823466e38f);
      part += m > -INFINITY ? fast_exp2((x[i] - m) * kLog2e) : 0.f;
    }
    bound = -INFINITY;                                     // the exact bound below
  }
  double sum = part;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane == 0) s_warp_sum[warp] = sum;

  // candidates at or above the bound
  int n = 0;
  if (bound > -INFINITY) {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) n += x[i] >= bound;
    n = block_count(n, s_warp_n, warp, lane);
  } else {
    n = kMaxCand + 1;
    __syncthreads();
  }
  if (tid == 0) {
    double total = 0;
    for (int i = 0; i < kBeamWarps; ++i) total += s_warp_sum[i];
    p.work.sum[out] = total;
    p.work.top[out] = m;
  }
  uint64_t key_bound = 1;
  if (n > kMaxCand) {
    // exact: the k-th largest of the threads' best keys
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int t = token_of(i / VEC, i % VEC);
      if (t < p.vocab) best = max(best, order_key(fmaxf(x[i], -INFINITY), t));
    }
    s_best[tid] = best;
    __syncthreads();
    int above = 0;
    for (int i = 0; i < kBeamThreads; ++i) above += s_best[i] > best;
    // keys are distinct except 0: at most one thread has exactly k - 1 above it
    __shared__ uint64_t s_bound;
    if (tid == 0) s_bound = 1;
    __syncthreads();
    if (best && above == k - 1) s_bound = best;
    __syncthreads();
    key_bound = s_bound;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int t = token_of(i / VEC, i % VEC);
      if (t < p.vocab) {
        const uint64_t key = order_key(fmaxf(x[i], -INFINITY), t);
        if (key >= key_bound) {
          const int at = atomicAdd(&s_count, 1);           // any order: ranked below
          if (at < kMaxCand) s_cand[at] = key;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (x[i] >= bound) s_cand[atomicAdd(&s_count, 1)] = order_key(x[i], token_of(i / VEC, i % VEC));
  }
  __syncthreads();
  n = min(s_count, kMaxCand);
  for (int i = tid; i < n; i += kBeamThreads) {
    const uint64_t key = s_cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s_cand[j] > key;
    if (rank < k) {
      const uint32_t o = uint32_t(key >> 32);
      entries[rank] = {__uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)), int32_t(~uint32_t(key))};
    }
  }
  for (int i = n + tid; i < k; i += kBeamThreads) entries[i] = {-INFINITY, -1};
}

struct BeamCand {
  double score;
  int64_t flat;      // beam * vocab + token
};

__device__ __forceinline__ bool better(const BeamCand& a, const BeamCand& b) {
  return a.score > b.score || (a.score == b.score && a.flat < b.flat);
}

__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(BeamParams p) {
  extern __shared__ __align__(16) unsigned char s_raw[];
  const int lists = p.beams * p.slices, k = p.k;
  BeamCand* s_head = reinterpret_cast<BeamCand*>(s_raw);                    // [lists]
  BeamCand* s_cand = s_head + lists;                                        // [k * k]
  double* s_score = reinterpret_cast<double*>(s_cand + k * k);              // [beams] score - log(sum)
  float* s_top = reinterpret_cast<float*>(s_score + p.beams);               // [beams]
  __shared__ BeamCand s_bound;
  __shared__ int s_count;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t request = blockIdx.x;
  const int64_t list0 = request * lists;
  if (tid == 0) {
    s_bound = {-INFINITY, INT64_MAX};                       // passes everything
    s_count = 0;
  }
  float score_of[4];                                        // inputs of the call: before the dependency wait
  for (int w = warp, i = 0; w < p.beams; w += kBeamWarps, ++i) score_of[i] = p.scores[request * p.beams + w];
  pdl_wait();
  for (int w = warp, i = 0; w < p.beams; w += kBeamWarps, ++i) {
    const int64_t at = list0 + int64_t(w) * p.slices;
    float m = -INFINITY;
    for (int s = lane; s < p.slices; s += 32) m = fmaxf(m, p.work.top[at + s]);
    m = warp_max(m);
    double sum = 0;
    for (int s = lane; s < p.slices; s += 32) {
      const float t = p.work.top[at + s];
      if (t > -INFINITY) sum += p.work.sum[at + s] * exp(double(t) - double(m));
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) {
      s_top[w] = m;
      s_score[w] = m > -INFINITY ? double(score_of[i]) - log(sum) : -INFINITY;
    }
  }
  __syncthreads();
  auto candidate = [&](int list, const BeamEntry& e) {
    const int w = list / p.slices;
    BeamCand c;
    c.flat = int64_t(w) * p.vocab + e.token;
    c.score = e.x > -INFINITY ? (double(e.x) - double(s_top[w])) + s_score[w] : -INFINITY;
    return c;
  };
  for (int i = tid; i < lists; i += kBeamThreads) {
    const BeamEntry e = p.work.entries[(list0 + i) * k];
    s_head[i] = e.token >= 0 ? candidate(i, e) : BeamCand{-INFINITY, INT64_MAX};
  }
  __syncthreads();
  // the k-th best head: at least k candidates are as good, in at most k lists
  for (int i = tid; i < lists; i += kBeamThreads) {
    const BeamCand c = s_head[i];
    int above = 0;
    for (int j = 0; j < lists; ++j) above += better(s_head[j], c);
    if (above == k - 1 && c.flat != INT64_MAX) s_bound = c;
  }
  __syncthreads();
  const BeamCand bound = s_bound;
  const int total = lists * k;
  for (int i = tid; i < total; i += kBeamThreads) {
    const BeamEntry e = p.work.entries[list0 * k + i];
    if (e.token < 0) continue;
    const BeamCand c = candidate(i / k, e);
    if (!better(bound, c)) {
      const int at = atomicAdd(&s_count, 1);                // any order: ranked below
      if (at < k * k) s_cand[at] = c;
    }
  }
  __syncthreads();
  const int n = min(s_count, k * k);
  for (int i = tid; i < n; i += kBeamThreads) {
    const BeamCand c = s_cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += better(s_cand[j], c);
    if (rank < k) {
      const int64_t o = request * k + rank;
      p.out_scores[o] = float(c.score);
      p.out_parents[o] = c.flat / p.vocab;
      p.out_tokens[o] = c.flat % p.vocab;
    }
  }
}

// ---- reordering ---------------------------------------------------------------
constexpr int kReorderThreads = 256, kReorderUnits = 4;

// out[r, i, :] = states[r, parents[r, i], :], in units of U bytes.
template <typename U>
__global__ void __launch_bounds__(kReorderThreads)
    beam_reorder_kernel(const U* states, int64_t stride_request, int64_t stride_beam, int beams,
                        const int64_t* parents, int64_t parent_stride, int kept, U* out, int64_t units,
                        int32_t* status) {
  const int64_t item = blockIdx.y;
  const int64_t r = item / kept, i = item % kept;
  const int64_t parent = parents[r * parent_stride + i];
  if (parent < 0 || parent >= beams) {
    if (threadIdx.x == 0 && blockIdx.x == 0) set_status(status, TA_ERR_BOUNDS);
    return;
  }
  const U* src = states + r * stride_request + parent * stride_beam;
  U* dst = out + item * units;
  const int64_t u0 = int64_t(blockIdx.x) * (kReorderThreads * kReorderUnits) + threadIdx.x;
  U v[kReorderUnits];
#pragma unroll
  for (int j = 0; j < kReorderUnits; ++j)
    if (u0 + j * kReorderThreads < units) v[j] = src[u0 + j * kReorderThreads];
#pragma unroll
  for (int j = 0; j < kReorderUnits; ++j)
    if (u0 + j * kReorderThreads < units) dst[u0 + j * kReorderThreads] = v[j];
}

template <typename U>
cudaError_t launch_reorder(const void* states, int64_t sr, int64_t sb, int requests, int beams, const int64_t* parents,
                           int64_t parent_stride, int kept, void* out, int64_t bytes, int32_t* status,
                           cudaStream_t stream) {
  const int64_t units = bytes / int64_t(sizeof(U));
  const int64_t per = kReorderThreads * kReorderUnits;
  const int64_t blocks = (units + per - 1) / per;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  // grid.y holds 65535 rows at most
  const int step = std::max(1, 65535 / kept);
  for (int r = 0; r < requests; r += step) {
    const int some = std::min(step, requests - r);
    beam_reorder_kernel<U><<<dim3(unsigned(blocks), unsigned(some * kept)), kReorderThreads, 0, stream>>>(
        static_cast<const U*>(states) + int64_t(r) * (sr / int64_t(sizeof(U))), sr / int64_t(sizeof(U)),
        sb / int64_t(sizeof(U)), beams, parents + int64_t(r) * parent_stride, parent_stride, kept,
        static_cast<U*>(out) + int64_t(r) * kept * units, units, status);
  }
  return cudaGetLastError();
}

int beam_slices(int vocab) { return int((int64_t(vocab) + kSlice - 1) / kSlice); }

}  // namespace

}  // namespace ta

extern "C" int64_t ta_beam_workspace_bytes(int32_t num_requests, int32_t num_beams, int32_t vocab, int32_t k,
                                           int32_t dtype) {
  using namespace ta;
  if (num_requests < 0 || num_beams <= 0 || vocab <= 0 || k <= 0 || k > kMaxK) return 0;
  const int64_t n = int64_t(num_requests) * num_beams * beam_slices(vocab);
  return n * (int64_t(sizeof(double)) + int64_t(sizeof(float)) + int64_t(sizeof(BeamEntry)) * k);
}

extern "C" int ta_beam_select(const void* logits, int64_t row_stride, const float* scores, const uint8_t* finished,
                              int32_t num_requests, int32_t num_beams, int32_t vocab, int32_t k, int32_t end_token,
                              int32_t dtype, float* out_scores, int64_t* out_parents, int64_t* out_tokens,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ta;
  if (dtype != TA_DTYPE_BF16 && dtype != TA_DTYPE_F16 && dtype != TA_DTYPE_F32) return TA_ERR_UNSUPPORTED;
  if (num_requests < 0 || num_beams <= 0 || vocab <= 0 || k <= 0 || row_stride < 0) return TA_ERR_ARG;
  if (num_beams > kMaxK || k > kMaxK || vocab > (1 << 30)) return TA_ERR_UNSUPPORTED;
  if (int64_t(num_beams) * vocab < k) return TA_ERR_ARG;
  if (finished && (end_token < 0 || end_token >= vocab)) return TA_ERR_ARG;
  if (num_requests == 0) return TA_OK;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens || !workspace) return TA_ERR_ARG;
  const int size = dtype == TA_DTYPE_F32 ? 4 : 2;
  const int slices = beam_slices(vocab);
  const int64_t rows = int64_t(num_requests) * num_beams;
  if (rows > INT32_MAX) return TA_ERR_UNSUPPORTED;
  const size_t smem = size_t(num_beams) * slices * sizeof(BeamCand) + size_t(k) * k * sizeof(BeamCand) +
                      size_t(num_beams) * (sizeof(double) + sizeof(float));
  if (smem > 48 * 1024) return TA_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(logits) % size) || (reinterpret_cast<uintptr_t>(workspace) & 15u)) return TA_ERR_ARG;
  if (workspace_bytes < ta_beam_workspace_bytes(num_requests, num_beams, vocab, k, dtype)) return TA_ERR_TOO_LARGE;
  BeamParams p{};
  p.logits = logits;
  p.scores = scores;
  p.finished = finished;
  p.row_stride = row_stride;
  p.beams = num_beams, p.vocab = vocab, p.k = k, p.slices = slices, p.end_token = end_token;
  p.out_scores = out_scores, p.out_parents = out_parents, p.out_tokens = out_tokens;
  const int64_t n = rows * slices;
  p.work.sum = static_cast<double*>(workspace);
  p.work.entries = reinterpret_cast<BeamEntry*>(p.work.sum + n);
  p.work.top = reinterpret_cast<float*>(p.work.entries + n * k);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid{unsigned(rows), unsigned(slices)};
  if (dtype == TA_DTYPE_BF16)
    beam_slice_kernel<TA_DTYPE_BF16><<<grid, kBeamThreads, 0, s>>>(p);
  else if (dtype == TA_DTYPE_F16)
    beam_slice_kernel<TA_DTYPE_F16><<<grid, kBeamThreads, 0, s>>>(p);
  else
    beam_slice_kernel<TA_DTYPE_F32><<<grid, kBeamThreads, 0, s>>>(p);
  cudaError_t err = cudaGetLastError();
  if (err == cudaSuccess)
    err = launch_dependent(beam_merge_kernel, dim3(unsigned(num_requests)), dim3(kBeamThreads), smem, s, p);
  return err == cudaSuccess ? TA_OK : TA_ERR_LAUNCH;
}

extern "C" int ta_beam_reorder(const void* states, int64_t stride_request, int64_t stride_beam, int32_t num_requests,
                               int32_t num_beams, int64_t row_bytes, const int64_t* parents, int64_t parent_stride,
                               int32_t kept, void* out, int32_t* status, void* stream) {
  using namespace ta;
  if (num_requests < 0 || num_beams <= 0 || kept < 0 || row_bytes < 0 || stride_request < 0 || stride_beam < 0 ||
      parent_stride < 0)
    return TA_ERR_ARG;
  if (kept > 65535) return TA_ERR_UNSUPPORTED;
  if (num_requests == 0 || kept == 0 || row_bytes == 0) return TA_OK;
  if (!states || !parents || !out) return TA_ERR_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint64_t all = reinterpret_cast<uintptr_t>(states) | reinterpret_cast<uintptr_t>(out) |
                       uint64_t(stride_request) | uint64_t(stride_beam) | uint64_t(row_bytes);
  cudaError_t err;
  if (!(all & 15u))
    err = launch_reorder<uint4>(states, stride_request, stride_beam, num_requests, num_beams, parents, parent_stride,
                                kept, out, row_bytes, status, s);
  else if (!(all & 3u))
    err = launch_reorder<uint32_t>(states, stride_request, stride_beam, num_requests, num_beams, parents,
                                   parent_stride, kept, out, row_bytes, status, s);
  else
    err = launch_reorder<uint8_t>(states, stride_request, stride_beam, num_requests, num_beams, parents,
                                  parent_stride, kept, out, row_bytes, status, s);
  return err == cudaSuccess ? TA_OK : TA_ERR_LAUNCH;
}
