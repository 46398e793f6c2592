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
// Bound: HBM, if the instructions stay few: a thread owns the two 16-byte chunks
// of a row that hold both elements of eight pairs (so no exchange between
// lanes), always the same columns and rows: its pointers, weights and, for a
// token, sines and cosines are set up once.  A CTA walks tokens with up to 64
// rows (head_dim 128); the next token's sines are computed while the current
// one's rows are under way, one barrier a token.
#include <algorithm>

#include "ta_common.cuh"
#include "ta_kernels.cuh"

namespace ta {

namespace {

constexpr int kRotaryThreads = 128;
// Rows of a thread and resident CTAs an SM: three rows for long inputs (16384
// tokens of 32 + 8 + 8 heads: 78 us; one row 87, four rows 79); one row while
// the CTAs fit one wave, where it is latency that counts (16 tokens: 2.9 us
// against 3.8 with three rows).
template <int R> constexpr int kCtas = R == 1 ? 8 : 5;

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

template <typename T, int D, bool PAIRS, int R>  // PAIRS: (2i, 2i + 1), else (i, i + rotary_dim / 2); R rows a thread
__global__ void __launch_bounds__(kRotaryThreads, kCtas<R>) rotary_append_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int LPR = D / 16;                   // lanes of a row
  constexpr int RPP = kRotaryThreads / LPR;     // rows of a pass of the CTA
  __shared__ __align__(16) float s_cos[2][D / 2], s_sin[2][D / 2];
  const int tid = threadIdx.x;

  if (p.klen && blockIdx.x == 0 && blockIdx.y == 0) {   // a captured decode step's first layer: the tails' lengths
    const int64_t value = *p.count + p.offset;
    for (int i = tid; i < p.num_tails; i += kRotaryThreads) {
      const int j = p.tail_jobs[i];
      if (j < 0 || j >= p.num_jobs || value < 0 || value > INT32_MAX)
        set_status(p.status, TA_ERR_BOUNDS);
      else
        p.klen[j] = int32_t(value);
    }
  }
  const int rows = p.hq + 2 * p.hk;
  int token = blockIdx.x;
  if (token >= p.num_tokens || rows == 0) return;

  // this thread's pairs 8j .. 8j + 7 and the chunks they lie in
  const int j = tid % LPR, hl = p.half / 8;
  const bool turns = j < hl;
  const int c0 = PAIRS ? 2 * j : turns ? j : 2 * j, c1 = PAIRS || !turns ? c0 + 1 : j + hl;
  // its rows: q heads, then k, then v
  const uint16_t* src[R];
  uint16_t* dst[R];
  int kind[R];                      // 0 q, 1 k, 2 v, 3 none
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int row = (blockIdx.y * R + u) * RPP + tid / LPR;
    if (row < p.hq) {
      kind[u] = 0;
      src[u] = p.q + token * p.q_st + int64_t(row) * p.q_sh;
      dst[u] = p.q_out + int64_t(row) * D;
    } else if (row < p.hq + p.hk) {
      kind[u] = 1;
      src[u] = p.k + token * p.k_st + int64_t(row - p.hq) * p.k_sh;
      dst[u] = p.kpool + int64_t(row - p.hq) * p.pool_tokens * D;
    } else if (row < rows) {
      kind[u] = 2;
      src[u] = p.v + token * p.v_st + int64_t(row - p.hq - p.hk) * p.v_sh;
      dst[u] = p.vpool + int64_t(row - p.hq - p.hk) * p.pool_tokens * D;
    } else {
      kind[u] = 3;
      src[u] = nullptr;
      dst[u] = nullptr;
    }
  }
  auto sines = [&](int tok, int buffer) {
    const double turn = double(p.positions[tok]) * 0.15915494309189533577;       // 1 / 2 pi
    for (int i = tid; i < p.half; i += kRotaryThreads) {
      const double t = turn * double(p.inv_freq[i]);
      float s, co;
      sincospif(2.f * float(t - rint(t)), &s, &co);
      s_cos[buffer][i] = co * p.factor;
      s_sin[buffer][i] = s * p.factor;
    }
  };

  const bool norm = p.q_weight || p.k_weight;
  sines(token, 0);
  for (int buffer = 0;; buffer ^= 1) {
    uint4 raw[R][2];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      if (kind[u] == 3) break;                  // rows only end: later ones are none as well
      raw[u][0] = *reinterpret_cast<const uint4*>(src[u] + c0 * 8);
      raw[u][1] = *reinterpret_cast<const uint4*>(src[u] + c1 * 8);
      src[u] += (kind[u] == 0 ? p.q_st : kind[u] == 1 ? p.k_st : p.v_st) * int64_t(gridDim.x);
    }
    const int64_t target = p.targets[token];
    const bool stored = target >= 0 && target < p.pool_tokens;
    if (!stored && target != -1 && tid == 0) set_status(p.status, TA_ERR_BOUNDS);
    const int following = token + gridDim.x;
    __syncthreads();                            // this token's sines are there, the last one's are read
    float co[8], si[8];
    if (turns) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        *reinterpret_cast<float4*>(co + i) = *reinterpret_cast<const float4*>(&s_cos[buffer][8 * j + i]);
        *reinterpret_cast<float4*>(si + i) = *reinterpret_cast<const float4*>(&s_sin[buffer][8 * j + i]);
      }
    }
    if (following < p.num_tokens) sines(following, buffer ^ 1);
#pragma unroll
    for (int u = 0; u < R; ++u) {
      if (__all_sync(0xffffffffu, kind[u] == 3)) break;
      uint4 lo = raw[u][0], hi = raw[u][1];
      if (__any_sync(0xffffffffu, kind[u] < 2)) {
        float x[16];
        {
          float a[8], b[8];
          unpack8<T>(lo, a);
          unpack8<T>(hi, b);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = a[i], x[8 + i] = b[i];
        }
        if (norm) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum += x[i] * x[i];
#pragma unroll
          for (int off = LPR / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
          const uint16_t* weight = kind[u] == 0 ? p.q_weight : kind[u] == 1 ? p.k_weight : nullptr;
          if (weight) {
            const float scale = rsqrtf(sum * (1.f / D) + p.eps);
            float a[8], b[8];
            unpack8<T>(*reinterpret_cast<const uint4*>(weight + c0 * 8), a);
            unpack8<T>(*reinterpret_cast<const uint4*>(weight + c1 * 8), b);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= scale * a[i], x[8 + i] *= scale * b[i];
          }
        }
        if (turns) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float& a = x[PAIRS ? 2 * i : i];
            float& b = x[PAIRS ? 2 * i + 1 : 8 + i];
            const float ra = a * co[i] - b * si[i];
            b = b * co[i] + a * si[i];
            a = ra;
          }
        }
        if (kind[u] < 2) {
          lo = make_uint4(Elem<T>::pack2(x[0], x[1]), Elem<T>::pack2(x[2], x[3]), Elem<T>::pack2(x[4], x[5]),
                          Elem<T>::pack2(x[6], x[7]));
          hi = make_uint4(Elem<T>::pack2(x[8], x[9]), Elem<T>::pack2(x[10], x[11]), Elem<T>::pack2(x[12], x[13]),
                          Elem<T>::pack2(x[14], x[15]));
        }
      }
      if (kind[u] == 0 || (kind[u] < 3 && stored)) {
        uint16_t* out = dst[u] + (kind[u] == 0 ? int64_t(token) * p.hq : target) * D;
        *reinterpret_cast<uint4*>(out + c0 * 8) = lo;
        *reinterpret_cast<uint4*>(out + c1 * 8) = hi;
      }
    }
    token = following;
    if (token >= p.num_tokens) break;
  }
}

bool rows16(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && st >= 0 && sh >= 0 && (st & 7) == 0 && (sh & 7) == 0;
}

template <typename T, int D, int R>
void launch_rotary(const RotaryParams& p, int sms, cudaStream_t stream) {
  constexpr int kRows = kRotaryThreads / (D / 16) * R;                 // rows of a CTA
  const int batches = std::max(1, (p.hq + 2 * p.hk + kRows - 1) / kRows);
  if (R == 1 && int64_t(p.num_tokens) * batches > int64_t(sms) * kCtas<1>) return launch_rotary<T, D, 3>(p, sms, stream);
  // enough CTAs to fill the GPU, each with its share of the tokens
  const dim3 grid(std::max(1, std::min(p.num_tokens, std::max(1, sms * kCtas<R> / batches))), batches);
  if (p.interleaved)
    rotary_append_kernel<T, D, true, R><<<grid, kRotaryThreads, 0, stream>>>(p);
  else
    rotary_append_kernel<T, D, false, R><<<grid, kRotaryThreads, 0, stream>>>(p);
}

template <typename T>
void launch_rotary(const RotaryParams& p, int head_dim, int sms, cudaStream_t stream) {
  if (head_dim == 128)
    launch_rotary<T, 128, 1>(p, sms, stream);
  else if (head_dim == 64)
    launch_rotary<T, 64, 1>(p, sms, stream);
  else
    launch_rotary<T, 32, 1>(p, sms, stream);
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
    launch_rotary<__nv_bfloat16>(p, head_dim, sm_count(), static_cast<cudaStream_t>(stream));
  else
    launch_rotary<__half>(p, head_dim, sm_count(), static_cast<cudaStream_t>(stream));
  return cudaGetLastError() == cudaSuccess ? TA_OK : TA_ERR_LAUNCH;
}
