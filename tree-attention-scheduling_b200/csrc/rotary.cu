// q/k RMSNorm, rotary positions and the K/V append behind ta_rotary_append.
//
// For every token and head, with x a row of q or k (f32 arithmetic throughout,
// one rounding on output):
//   y = x * rsqrt(mean(x^2) + eps) * w                (when a norm weight is given)
//   (a, b) -> s * (a cos t - b sin t, b cos t + a sin t),   t = position * inv_freq[i]
// over the pairs of the first rotary_dim elements -- (i, i + rotary_dim/2), or
// (2i, 2i + 1) when interleaved -- the rest passes through.  q rows go to
// q_out; k and v rows go straight into the pools [HK, T, D] at the token's
// target, so a prompt chunk or decode step needs one launch per layer.
//
// Angles: t reaches 1e6 rad and more in a long context, where an f32 product
// is off by 0.06 rad.  t / 2 pi is taken in f64 (a position and an f32
// frequency multiply exactly), reduced to a fraction of a turn, and only that
// fraction is rounded to f32 (2^-25 turns) for sincospif.  The rotary_dim / 2
// sines of a token are computed once per CTA and shared by all its heads.
//
// Bound: HBM.  A CTA is one token; a thread owns one 16-byte chunk of a row
// (always the same columns: its cosines stay in registers) and keeps four rows
// in flight.
#include <algorithm>

#include "ta_common.cuh"
#include "ta_kernels.cuh"

namespace ta {

namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRowsInFlight = 4;

struct RotaryParams {
  const uint16_t *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;   // element strides: token, head
  const int64_t* positions;
  const float* inv_freq;
  const uint16_t *q_weight, *k_weight;          // [D] or null
  uint16_t* q_out;                              // [N, HQ, D]
  uint16_t *kpool, *vpool;                      // [HK, T, D]
  const int64_t* targets;
  int32_t* klen;
  const int32_t* tail_jobs;
  const int64_t* count;
  int32_t* status;
  int64_t pool_tokens;
  float factor, eps;
  int num_tokens, hq, hk, half, interleaved, num_tails, offset, num_jobs;
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<T>::to_float2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kRotaryThreads) rotary_append_kernel(RotaryParams p) {
  constexpr int LPR = D / 8;                    // lanes (16-byte chunks) of a row
  __shared__ float s_cos[D / 2], s_sin[D / 2];
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t token = blockIdx.x;

  if (p.klen && token == 0) {                   // a captured decode step's first layer: the tails' lengths
    const int64_t value = *p.count + p.offset;
    for (int i = tid; i < p.num_tails; i += kRotaryThreads) {
      const int j = p.tail_jobs[i];
      if (j < 0 || j >= p.num_jobs || value < 0 || value > INT32_MAX)
        set_status(p.status, TA_ERR_BOUNDS);
      else
        p.klen[j] = int32_t(value);
    }
  }
  if (token >= p.num_tokens) return;            // a launch for the tails alone

  const int c = tid % LPR;                      // this thread's chunk of every row it handles
  const int rows = p.hq + 2 * p.hk;
  const int64_t target = p.targets[token];
  const bool stored = target >= 0 && target < p.pool_tokens;
  if (!stored && target != -1 && tid == 0) set_status(p.status, TA_ERR_BOUNDS);

  float cosv[8], sinv[8];
  bool have_angles = false;
  // lane that holds the other half of this lane's pairs, and the sign of its term
  const int hl = p.half / 8;
  const bool turns = 8 * c < 2 * p.half;
  const bool first = c < hl;
  const int partner = p.interleaved || !turns ? lane : (first ? lane + hl : lane - hl);

  for (int row0 = tid / LPR; row0 - tid / LPR < rows; row0 += kRowsInFlight * (kRotaryThreads / LPR)) {
    uint4 raw[kRowsInFlight];
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      const int row = row0 + u * (kRotaryThreads / LPR);
      raw[u] = make_uint4(0, 0, 0, 0);
      if (row < p.hq)
        raw[u] = *reinterpret_cast<const uint4*>(p.q + token * p.q_st + int64_t(row) * p.q_sh + c * 8);
      else if (row < p.hq + p.hk)
        raw[u] = *reinterpret_cast<const uint4*>(p.k + token * p.k_st + int64_t(row - p.hq) * p.k_sh + c * 8);
      else if (row < rows)
        raw[u] = *reinterpret_cast<const uint4*>(p.v + token * p.v_st + int64_t(row - p.hq - p.hk) * p.v_sh + c * 8);
    }
    if (!have_angles) {                         // behind the first loads
      have_angles = true;
      const double turn = double(p.positions[token]) * 0.15915494309189533577;   // 1 / 2 pi
      for (int i = tid; i < p.half; i += kRotaryThreads) {
        const double t = turn * double(p.inv_freq[i]);
        float s, co;
        sincospif(2.f * float(t - rint(t)), &s, &co);
        s_cos[i] = co * p.factor;
        s_sin[i] = s * p.factor;
      }
      __syncthreads();
      if (turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int pair = p.interleaved ? 4 * c + i / 2 : 8 * (first ? c : c - hl) + i;
          cosv[i] = s_cos[pair];
          // out = own * cos + other * sin', with -sin for the first element of a pair
          const bool leads = p.interleaved ? (i & 1) == 0 : first;
          sinv[i] = leads ? -s_sin[pair] : s_sin[pair];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) cosv[i] = 1.f, sinv[i] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < kRowsInFlight; ++u) {
      const int row = row0 + u * (kRotaryThreads / LPR);
      const bool is_q = row < p.hq, is_k = !is_q && row < p.hq + p.hk;
      if (!__any_sync(0xffffffffu, row < rows)) break;
      uint4 result = raw[u];
      if (__any_sync(0xffffffffu, is_q || is_k)) {
        float x[8];
        unpack8<T>(raw[u], x);
        if (p.q_weight || p.k_weight) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
#pragma unroll
          for (int off = LPR / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
          const uint16_t* w = is_q ? p.q_weight : is_k ? p.k_weight : nullptr;
          if (w) {
            const float scale = rsqrtf(sum * (1.f / D) + p.eps);
            float wf[8];
            unpack8<T>(*reinterpret_cast<const uint4*>(w + c * 8), wf);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * scale * wf[i];
          }
        }
        float y[8];
        if (p.interleaved) {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = x[i] * cosv[i] + (turns ? x[i ^ 1] * sinv[i] : 0.f);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float other = __shfl_sync(0xffffffffu, x[i], partner);
            y[i] = x[i] * cosv[i] + (turns ? other * sinv[i] : 0.f);
          }
        }
        if (is_q || is_k)
          result = make_uint4(Elem<T>::pack2(y[0], y[1]), Elem<T>::pack2(y[2], y[3]), Elem<T>::pack2(y[4], y[5]),
                              Elem<T>::pack2(y[6], y[7]));
      }
      if (is_q)
        *reinterpret_cast<uint4*>(p.q_out + (token * p.hq + row) * D + c * 8) = result;
      else if (is_k && stored)
        *reinterpret_cast<uint4*>(p.kpool + (int64_t(row - p.hq) * p.pool_tokens + target) * D + c * 8) = result;
      else if (!is_k && row < rows && stored)
        *reinterpret_cast<uint4*>(p.vpool + (int64_t(row - p.hq - p.hk) * p.pool_tokens + target) * D + c * 8) = result;
    }
  }
}

bool rows16(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && st >= 0 && sh >= 0 && (st & 7) == 0 && (sh & 7) == 0;
}

template <typename T>
void launch_rotary(const RotaryParams& p, int head_dim, cudaStream_t stream) {
  const unsigned grid = unsigned(std::max(1, p.num_tokens));
  if (head_dim == 128)
    rotary_append_kernel<T, 128><<<grid, kRotaryThreads, 0, stream>>>(p);
  else if (head_dim == 64)
    rotary_append_kernel<T, 64><<<grid, kRotaryThreads, 0, stream>>>(p);
  else
    rotary_append_kernel<T, 32><<<grid, kRotaryThreads, 0, stream>>>(p);
}

}  // namespace

}  // namespace ta

extern "C" int ta_rotary_append(const void* q, int64_t q_stride_token, int64_t q_stride_head, const void* k,
                                int64_t k_stride_token, int64_t k_stride_head, const void* v, int64_t v_stride_token,
                                int64_t v_stride_head, const int64_t* positions, const float* inv_freq,
                                int32_t rotary_dim, int32_t interleaved, float attention_factor, const void* q_weight,
                                const void* k_weight, float eps, void* q_out, void* kpool, void* vpool,
                                const int64_t* targets, int32_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads,
                                int64_t pool_tokens, int32_t head_dim, int32_t dtype, int32_t* klen,
                                const int32_t* tail_jobs, int32_t num_tails, const int64_t* count, int32_t offset,
                                int32_t num_jobs, int32_t* status, void* stream) {
  using namespace ta;
  if (dtype != TA_DTYPE_BF16 && dtype != TA_DTYPE_F16) return TA_ERR_UNSUPPORTED;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) return TA_ERR_UNSUPPORTED;
  if (num_tokens < 0 || num_q_heads < 0 || num_kv_heads < 0 || pool_tokens < 0) return TA_ERR_ARG;
  if (num_q_heads > 65536 || num_kv_heads > 65536) return TA_ERR_ARG;
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16) return TA_ERR_ARG;
  if (klen && (!tail_jobs || !count || num_tails < 0 || num_jobs < 0)) return TA_ERR_ARG;
  if (num_tokens > 0) {
    if (!positions || !targets || (rotary_dim > 0 && !inv_freq)) return TA_ERR_ARG;
    if (num_q_heads > 0 && (!q || !q_out || !rows16(q, q_stride_token, q_stride_head) || !rows16(q_out, 0, 0)))
      return TA_ERR_ARG;
    if (num_kv_heads > 0 && (!k || !v || !kpool || !vpool || !rows16(k, k_stride_token, k_stride_head) ||
                             !rows16(v, v_stride_token, v_stride_head) || !rows16(kpool, 0, 0) || !rows16(vpool, 0, 0)))
      return TA_ERR_ARG;
    if (!rows16(q_weight, 0, 0) || !rows16(k_weight, 0, 0)) return TA_ERR_ARG;
  }
  if (num_tokens == 0 && (!klen || num_tails == 0)) return TA_OK;
  RotaryParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q_st = q_stride_token, p.q_sh = q_stride_head;
  p.k_st = k_stride_token, p.k_sh = k_stride_head;
  p.v_st = v_stride_token, p.v_sh = v_stride_head;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.q_weight = static_cast<const uint16_t*>(q_weight);
  p.k_weight = static_cast<const uint16_t*>(k_weight);
  p.q_out = static_cast<uint16_t*>(q_out);
  p.kpool = static_cast<uint16_t*>(kpool);
  p.vpool = static_cast<uint16_t*>(vpool);
  p.targets = targets;
  p.klen = klen;
  p.tail_jobs = tail_jobs;
  p.count = count;
  p.status = status;
  p.pool_tokens = pool_tokens;
  p.factor = attention_factor;
  p.eps = eps;
  p.num_tokens = num_tokens;
  p.hq = num_q_heads, p.hk = num_kv_heads;
  p.half = rotary_dim / 2;
  p.interleaved = interleaved != 0;
  p.num_tails = klen ? num_tails : 0;
  p.offset = offset, p.num_jobs = num_jobs;
  if (dtype == TA_DTYPE_BF16)
    launch_rotary<__nv_bfloat16>(p, head_dim, static_cast<cudaStream_t>(stream));
  else
    launch_rotary<__half>(p, head_dim, static_cast<cudaStream_t>(stream));
  return cudaGetLastError() == cudaSuccess ? TA_OK : TA_ERR_LAUNCH;
}
