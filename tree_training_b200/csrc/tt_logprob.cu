// Log probabilities of given tokens, entropy and top alternatives of the rows
// of an LM head's logits, and their gradient.
//
//   z = x / temperature, m = max z, s = sum e^(z - m)
//   logp(v) = z_v - m - ln s
//   H       = ln s - sum (z - m) e^(z - m) / s
//   top     = the k largest x of the row, the lowest index first among equals
//
//   dx(v) = 1/temperature [ sum_j g_j (delta(v, token_j) - p_v) - g_H p_v (logp(v) + H) ]
//
// with j over the row's given tokens and, where their log probabilities carry
// gradients, its top alternatives.  Tokens outside [0, V) are ignored (log
// probability 0, no gradient).  -inf logits have probability 0; a row of
// nothing but -inf has log probabilities -inf, entropy 0 and no gradient.
//
// Forward: each thread keeps a running (reference, sum, weighted sum) in base
// 2 and the row is read once.
#include <algorithm>

#include "tt_vec.cuh"

namespace tt {
namespace logprob {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Exponents of 2 are kept from -inf, whose product with a probability of 0
// would be NaN; 2^-200 is 0 in fp32.
constexpr float kFloor = -200.f;
// The reference moves when the maximum is this far (a factor of 2^12) above it.
constexpr float kSlack = 12.f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A whole number that orders floats: NaN above all, -0 as 0, never 0 itself.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float of_order(uint32_t o) {
  if (o == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

// Larger value first, then the lower index.
__device__ __forceinline__ uint64_t key_of(uint32_t order, int64_t index) {
  return ((uint64_t)order << 32) | (uint32_t)~(uint32_t)index;
}

// Running sums of 2^t and of t 2^t, t = (x - ref) c.  The reference is
// subtracted first: logits of the type's lowest value overflow when scaled.
struct Sums {
  float ref, s, u;
};

__device__ __forceinline__ void rebase(Sums& a, float ref, float c) {
  if (a.s != 0.f) {
    const float d = max_nan((a.ref - ref) * c, kFloor), f = ex2(d);
    a.u = f * fmaf(a.s, d, a.u);
    a.s *= f;
  }
  a.ref = ref;
}

__device__ __forceinline__ Sums merged(Sums a, Sums b, float c) {
  if (b.s == 0.f) return a;
  if (a.s == 0.f) return b;
  const float ref = max_nan(a.ref, b.ref);
  rebase(a, ref, c);
  rebase(b, ref, c);
  return {ref, a.s + b.s, a.u + b.u};
}

template <int N>
__device__ __forceinline__ void accumulate(const float (&x)[N], float c, Sums& a, float& best) {
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) mx = max_nan(mx, x[i]);
  best = max_nan(best, mx);
  if ((mx - a.ref) * c > kSlack || (a.s == 0.f && mx > -INFINITY)) rebase(a, mx, c);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float t = max_nan((x[i] - a.ref) * c, kFloor);
    const float e = ex2(t);
    a.s += e;
    a.u = fmaf(t, e, a.u);
  }
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
  return __shfl_xor_sync(0xffffffffu, (unsigned long long)v, o);
}

struct Args {
  int64_t rows;
  int V, M, k;
  const void* x;
  int64_t ld;
  const int64_t* tokens;
  float temperature;
  float *logp, *ent, *top_logp;
  int64_t* top_tok;
  float* stats;              // [rows][4]: m (of x), ln s, 1 / s (0: empty row), H
};

// log probability of logit x, in the order a softmax takes its steps
__device__ __forceinline__ float logp_of(float x, float m, float ln_s, float inv_s, float temp) {
  if (inv_s == 0.f) return -INFINITY;
  return (x / temp - m / temp) - ln_s;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const Args a) {
  __shared__ Sums sums[kWarps];
  __shared__ float maxes[kWarps];
  __shared__ uint64_t keys[kWarps];
  __shared__ float st[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld;
  const float c = kLog2e / a.temperature;
  Sums acc{0.f, 0.f, 0.f};
  float best = -INFINITY;
  for (int i = threadIdx.x; i < a.V; i += kThreads) {
    const float v[1] = {to_f32(x[i])};
    accumulate<1>(v, c, acc, best);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums b{__shfl_xor_sync(0xffffffffu, acc.ref, o), __shfl_xor_sync(0xffffffffu, acc.s, o),
                 __shfl_xor_sync(0xffffffffu, acc.u, o)};
    acc = merged(acc, b, c);
    best = max_nan(best, __shfl_xor_sync(0xffffffffu, best, o));
  }
  if (lane == 0) sums[warp] = acc, maxes[warp] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) {
      acc = merged(acc, sums[w], c);
      best = max_nan(best, maxes[w]);
    }
    float ln_s = 0.f, inv_s = 0.f, H = 0.f;
    if (acc.s != 0.f) {
      rebase(acc, best, c);
      ln_s = logf(acc.s);
      inv_s = 1.f / acc.s;
      H = ln_s - kLn2 * (acc.u / acc.s);
    }
    st[0] = best, st[1] = ln_s, st[2] = inv_s, st[3] = H;
    a.ent[row] = H;
    if (a.stats) {
      float4* out = reinterpret_cast<float4*>(a.stats) + row;
      *out = make_float4(best, ln_s, inv_s, H);
    }
  }
  __syncthreads();
  const float m = st[0], ln_s = st[1], inv_s = st[2];
  for (int j = threadIdx.x; j < a.M; j += kThreads) {
    const int64_t tok = a.tokens[row * a.M + j];
    a.logp[row * a.M + j] =
        (tok < 0 || tok >= a.V) ? 0.f : logp_of(to_f32(x[tok]), m, ln_s, inv_s, a.temperature);
  }
  // the alternatives, one a pass: the largest key below the one before
  uint64_t below = ~0ull;
  for (int j = 0; j < a.k; ++j) {
    uint64_t mine = 0;
    for (int i = threadIdx.x; i < a.V; i += kThreads) {
      const uint64_t key = key_of(order_of(to_f32(x[i])), i);
      if (key < below && key > mine) mine = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = shfl_xor64(mine, o);
      mine = other > mine ? other : mine;
    }
    __syncthreads();
    if (lane == 0) keys[warp] = mine;
    __syncthreads();
    below = keys[0];
    for (int w = 1; w < kWarps; ++w) below = keys[w] > below ? keys[w] : below;
    if (threadIdx.x == 0) {
      a.top_tok[row * a.k + j] = (int64_t)(uint32_t)~(uint32_t)below;
      a.top_logp[row * a.k + j] =
          logp_of(of_order((uint32_t)(below >> 32)), m, ln_s, inv_s, a.temperature);
    }
  }
}

struct BwdArgs {
  int64_t rows;
  int V, M, k;
  const void* x;
  int64_t ld;
  const int64_t *tokens, *top_tok;
  float temperature;
  const float *g_logp, *g_ent, *g_top;   // any of them null: zero
  const float* stats;
  void* dx;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) bwd_kernel(const BwdArgs a) {
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld;
  T* dx = reinterpret_cast<T*>(a.dx) + row * a.V;
  const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
  const float m = st.x, ln_s = st.y, inv_s = st.z, H = st.w;
  const bool empty = inv_s == 0.f;
  const float c = kLog2e / a.temperature, inv_t = 1.f / a.temperature;
  const float ref = empty ? 0.f : m;
  const int n = a.M + (a.g_top ? a.k : 0);
  // entry j: a given token or an alternative
  auto token = [&](int j) {
    return j < a.M ? a.tokens[row * a.M + j] : a.top_tok[row * a.k + j - a.M];
  };
  auto grad = [&](int j) {
    return j < a.M ? (a.g_logp ? a.g_logp[row * a.M + j] : 0.f) : a.g_top[row * a.k + j - a.M];
  };
  float G = 0.f;
  if (!empty)
    for (int j = 0; j < n; ++j) {
      const int64_t tok = token(j);
      if (tok >= 0 && tok < a.V) G += grad(j);
    }
  const float gH = a.g_ent && !empty ? a.g_ent[row] : 0.f;
  auto base = [&](float v) {
    const float t = max_nan((v - ref) * c, kFloor);
    const float p = ex2(t) * inv_s;
    return -p * (G + gH * (fmaf(t, kLn2, -ln_s) + H));
  };
  for (int i = threadIdx.x; i < a.V; i += kThreads)
    dx[i] = from_f32<T>(base(to_f32(x[i])) * inv_t);
  __syncthreads();
  if (empty) return;
  for (int j = threadIdx.x; j < n; j += kThreads) {
    const int64_t tok = token(j);
    if (tok < 0 || tok >= a.V) continue;
    float g = 0.f;
    bool first = true;
    for (int i = 0; i < n; ++i) {
      if (token(i) != tok) continue;
      if (i < j) first = false;
      g += grad(i);
    }
    if (first) dx[tok] = from_f32<T>((base(to_f32(x[tok])) + g) * inv_t);
  }
}

bool bad(int64_t rows, int32_t V, int32_t M, int32_t k, const void* x, int64_t ld,
         const int64_t* tokens, float temperature) {
  return rows < 0 || rows > 0x7fffffff || V <= 0 || M < 0 || k < 0 || k > kMaxTop || k > V ||
         ld < V || !(temperature > 0.f) || (rows > 0 && (!x || (M > 0 && !tokens)));
}

}  // namespace
}  // namespace logprob
}  // namespace tt

extern "C" int tt_token_logprobs_fwd(int dtype, int64_t n_rows, int32_t vocab, const void* logits,
                                     int64_t ld, const int64_t* tokens, int32_t n_tokens,
                                     float temperature, int32_t top_k, float* logprobs,
                                     float* entropy, float* top_logprobs, int64_t* top_tokens,
                                     float* stats, void* stream) {
  using namespace tt::logprob;
  if (bad(n_rows, vocab, n_tokens, top_k, logits, ld, tokens, temperature) ||
      (n_rows > 0 && (!entropy || (n_tokens > 0 && !logprobs) ||
                      (top_k > 0 && (!top_logprobs || !top_tokens)))))
    return TT_ERR_INVALID_ARG;
  if (n_rows == 0) return TT_OK;
  Args a{n_rows, vocab, n_tokens, top_k, logits, ld, tokens, temperature,
         logprobs, entropy, top_logprobs, top_tokens, stats};
  const int rc = tt::vec::dispatch_float(dtype, [&](auto tag) -> int {
    fwd_kernel<decltype(tag)><<<(unsigned)n_rows, kThreads, 0, (cudaStream_t)stream>>>(a);
    return TT_OK;
  });
  if (rc != TT_OK) return rc;
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

extern "C" int tt_token_logprobs_bwd(int dtype, int64_t n_rows, int32_t vocab, const void* logits,
                                     int64_t ld, const int64_t* tokens, int32_t n_tokens,
                                     float temperature, int32_t top_k, const int64_t* top_tokens,
                                     const float* g_logprobs, const float* g_entropy,
                                     const float* g_top, const float* stats, void* dlogits,
                                     void* stream) {
  using namespace tt::logprob;
  if (bad(n_rows, vocab, n_tokens, top_k, logits, ld, tokens, temperature) ||
      (n_rows > 0 && (!stats || !dlogits || (g_top && top_k > 0 && !top_tokens))))
    return TT_ERR_INVALID_ARG;
  if (n_rows == 0) return TT_OK;
  BwdArgs a{n_rows, vocab, n_tokens, top_k, logits, ld, tokens, top_tokens, temperature,
            g_logprobs, g_entropy, g_top, stats, dlogits};
  const int rc = tt::vec::dispatch_float(dtype, [&](auto tag) -> int {
    bwd_kernel<decltype(tag)><<<(unsigned)n_rows, kThreads, 0, (cudaStream_t)stream>>>(a);
    return TT_OK;
  });
  if (rc != TT_OK) return rc;
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}
