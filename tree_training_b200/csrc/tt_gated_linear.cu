// The gated half of a feed-forward block and its gradients.
//
//   g = x Wg^T,  u = x Wu^T,  h = act(g) * u
//   dg = dh * u * act'(g),  du = dh * act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// 4 T H F operations forward, 8 T H F backward: bound by the tensor cores for many
// tokens, by the weights' bytes for few.
//
// Forward, 16-bit: one kernel forms both products of a tile side by side in one
// accumulator (its left half g, its right half u), so that x is read once for both
// and h leaves from registers.  For the backward g and u are kept in fp32: rounded
// to 16 bits they would put two more roundings into dg (its own is the one that the
// tensor cores' operands need), and the eight bytes an element stand against six
// that g, u and act(g) take in 16 bits.
//
// Backward: dg and du leave one elementwise pass in 16 bits, dx is one sum of two
// products in one accumulator, each weight's gradient one product.
//
// Up to kFewRows tokens (a rollout's single ones) no tensor core is needed: a warp a
// feature reads its two rows once, 16 bytes a lane, and multiplies by fma (2,560 x
// 9,728 bf16: 21 us a token, 25 two; the tensor cores take 23 to 25 for 2 to 128 tokens,
// so that two go there if the weights are large: 1,024 x 4,096 8 us and 13).
//
// fp32: the products on the CUDA cores (see tt_gemm_fp32.cu), h by a pass over g and u.
//
// Measured on a B200, bf16, 8,192 x 2,560 x 9,728, single launches: forward 537 us with g
// and u kept (495 without), dg and du 158 (7.1 TB/s), dx 501, both weights' gradients 528;
// a pass back to back 2,080 to 2,240 us, at the power limit.
#include "tt_gemm_sm100.cuh"

namespace tt {
namespace gated {
namespace {

enum Act { kSilu = 0, kGelu = 1, kGeluTanh = 2, kRelu = 3 };

constexpr float kTanhA = 0.7978845608028654f;      // sqrt(2 / pi)
constexpr float kTanhB = 0.044715f;

// 1 / (1 + exp(-g)) down to where fp32 ends, which exp(-g) leaves at -88 already.
__device__ __forceinline__ float sigmoid(float g) {
  return g < -80.f ? expf(g) : 1.f / (1.f + expf(-g));
}

template <int A>
__device__ __forceinline__ float act(float g) {
  if constexpr (A == kSilu) return g < -80.f ? g * expf(g) : g / (1.f + expf(-g));
  if constexpr (A == kGelu) return g * normcdff(g);
  if constexpr (A == kGeluTanh)
    return 0.5f * g * (1.f + tanhf(kTanhA * (g + kTanhB * g * g * g)));
  return g > 0.f ? g : (g != g ? g : 0.f);
}

// The same for results of 16 bits: the epilogue of the products has no time for the exact
// exponential and quotient.  The quick ones err by 2^-22 (3 + 0.6 |z|) of the value: 2^-16 of
// silu(-80), 2^-20 of what is above -4, beside 2^-12 or 2^-9 of the rounding that follows.
// 1 / (1 + exp(-z)) = exp(z) / (1 + exp(z)): by the exponential that is at most 1, so that
// neither leaves fp32.  ((1 + tanh y) / 2 = 1 / (1 + exp(-2 y)).)
template <int A>
__device__ __forceinline__ float act_16(float g) {
  if constexpr (A == kSilu || A == kGeluTanh) {
    const float z = A == kSilu ? g : 2.f * kTanhA * (g + kTanhB * g * g * g);
    const float e = __expf(-fabsf(z));
    return __fdividef(z < 0.f ? g * e : g, 1.f + e);
  }
  return act<A>(g);
}

// Of gelu with tanh past +-20: the slope is 1 or 0 there, and the cube's derivative would
// leave fp32 from 1e19 on (0 times infinity).  NaN stays.
__device__ __forceinline__ float near_zero(float g) {
  return g > 20.f ? 20.f : (g < -20.f ? -20.f : g);
}

// act(g) and its derivative.
template <int A>
__device__ __forceinline__ void act_grad(float g, float& a, float& d) {
  if constexpr (A == kSilu) {
    const float q = sigmoid(g);
    a = g * q;
    // (1 - q loses what little there is of it for large g: q(-g) instead)
    d = q * (1.f + g * sigmoid(-g));
  } else if constexpr (A == kGelu) {
    const float c = normcdff(g);
    a = g * c;
    d = c + g * expf(-0.5f * g * g) * 0.3989422804014327f;
  } else if constexpr (A == kGeluTanh) {
    const float c = near_zero(g), t = tanhf(kTanhA * (c + kTanhB * c * c * c));
    a = 0.5f * g * (1.f + t);
    d = 0.5f * (1.f + t) + 0.5f * c * (1.f - t * t) * kTanhA * (1.f + 3.f * kTanhB * c * c);
  } else {
    a = act<kRelu>(g);
    d = g > 0.f ? 1.f : (g != g ? g : 0.f);
  }
}

// The same for gradients of 16 bits (with exact quotients this pass is bound by their
// instructions, not by its bytes).
template <int A>
__device__ __forceinline__ void act_grad_16(float g, float& a, float& d) {
  if constexpr (A == kSilu || A == kGeluTanh) {
    // s = 1 / (1 + exp(-z)) and r = 1 - s, the smaller of them as exp(-|z|) times the other
    const float c = A == kSilu ? g : near_zero(g);
    const float z = A == kSilu ? g : 2.f * kTanhA * (c + kTanhB * c * c * c);
    const float e = __expf(-fabsf(z)), large = __fdividef(1.f, 1.f + e), small = e * large;
    const float s = z < 0.f ? small : large, r = z < 0.f ? large : small;
    const float dz = A == kSilu ? 1.f : 2.f * kTanhA * (1.f + 3.f * kTanhB * c * c);
    a = g * s;
    d = s * (1.f + c * (r * dz));
  } else {
    act_grad<A>(g, a, d);
  }
}

template <typename F>
int dispatch_act(int act, F f) {
  switch (act) {
    case kSilu: return f(std::integral_constant<int, kSilu>());
    case kGelu: return f(std::integral_constant<int, kGelu>());
    case kGeluTanh: return f(std::integral_constant<int, kGeluTanh>());
    case kRelu: return f(std::integral_constant<int, kRelu>());
    default: return TT_ERR_INVALID_ARG;
  }
}

// relu's slope jumps at 0: of a product that the tensor cores' cut-off sums leave within
// their own error of 0 (208 x 4,288 x 4,544: one of 945,000, which was 1.5e-3 of a weight's
// gradient) the sign is found again, by a sum in 64 bits.  Their error is about 2^-24 of
// the sums on the way for every 16 of k; these are as large as the row's other products
// of the block (fewer than kFewest say too little: their factors' sizes then).  The whole
// warp forms such a sum; a row with more than kMostDoubts of them in 32 is left as it is
// (columns of very different sizes: the estimate says nothing there).  It costs the
// forward 3 to 15% (64 x 2,560 x 9,728 23.1 -> 25.5 us, 4,096 x 1,536 x 4,096 67 -> 78, 8,192 x
// 2,560 x 9,728 kept 600 -> 632), a pass with gradients a quarter of that; a last tile of
// few features up to 6 us (2,048 x 2,560 x 2,567 55 -> 61, 8,192 x 2,560 x 9,729 537 -> 541),
// features without weights up to a fifth (8,192 x 2,560 x 9,728, four in 32: 514 -> 617).
constexpr int kMostDoubts = 4;
constexpr int kFewest = 8;

struct Doubts {
  const void *x, *w;
  int64_t x_ld, w_ld;
  int H;
  float share;                             // of a product's usual magnitude
};

// Eight elements of a row of d.H from the p-th on.
template <typename T>
__device__ __forceinline__ uint4 pack_at(const Doubts& d, const T* row, int64_t p) {
  return p + 8 <= d.H ? __ldg(reinterpret_cast<const uint4*>(row + p))
                      : vec::load_any_of<T>(row, p, d.H, row, row);
}

// The mean square of a row's elements, by kSampled packs of it (a lane on its own).
template <typename T>
__device__ __forceinline__ float mean_square(const Doubts& d, const T* row) {
  constexpr int kSampled = 32, kAhead = 16;
  const int whole = d.H / 8;
  float sum = 0.f;
  if (whole == 0) {
    for (int k = 0; k < d.H; ++k) sum = fmaf(to_f32(row[k]), to_f32(row[k]), sum);
    return sum / (float)d.H;
  }
  for (int k0 = 0; k0 < kSampled; k0 += kAhead) {
    uint4 raw[kAhead];                     // (loads without branches: none waits for another)
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      raw[k] = __ldg(reinterpret_cast<const uint4*>(row) + (int64_t)(k0 + k) * whole / kSampled);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      float v[8];
      vec::unpack<T, 8>(raw[k], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(v[j], v[j], sum);
    }
  }
  return sum / (8.f * kSampled);
}

// The usual magnitude of a row's products with `left` (under kFewest) features, from
// their factors: |x| |w| / sqrt(H), and kWider times that, since a part of the elements
// shows their size only so far (a few may be much larger) and sums are soon formed again.
template <typename T>
__device__ __noinline__ float usual_of_few(const Doubts& d, int row, bool live, int feature,
                                           int left) {
  constexpr float kWider = 256.f;
  const int lane = threadIdx.x & 31;
  float xx = 0.f, ww = 0.f;
  if (live) xx = mean_square(d, reinterpret_cast<const T*>(d.x) + (int64_t)row * d.x_ld);
  if (lane < left)
    ww = mean_square(d, reinterpret_cast<const T*>(d.w) + (int64_t)(feature + lane) * d.w_ld);
  __syncwarp();
  for (int o = 4; o; o >>= 1) ww += __shfl_xor_sync(0xffffffffu, ww, o);
  ww = __shfl_sync(0xffffffffu, ww, 0) / (float)left;
  return kWider * sqrtf(xx) * sqrtf(ww) * sqrtf((float)d.H);
}

// Whether a feature has a weight other than 0.
template <typename T>
__device__ __forceinline__ bool any_weight(const Doubts& d, int feature) {
  const T* w = reinterpret_cast<const T*>(d.w) + (int64_t)feature * d.w_ld;
  uint32_t bits = 0;
#pragma unroll 4
  for (int64_t p = (threadIdx.x & 31) * 8; p < d.H; p += 256) {
    const uint4 v = pack_at(d, w, p);
    bits |= v.x | v.y | v.z | v.w;
  }
  return __any_sync(0xffffffffu, (bits & 0x7fff7fffu) != 0);
}

// g: of `left` features (those behind them are not this block's)
template <typename T>
__device__ __forceinline__ void settle_signs(const Doubts& d, int row, bool live, int feature,
                                             int left, float (&g)[32]) {
  const int lane = threadIdx.x & 31;
  float sum_of[2] = {0.f, 0.f}, least[2] = {INFINITY, INFINITY}, usual;
  if (left >= 32) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      sum_of[i & 1] += fabsf(g[i]);
      least[i & 1] = fminf(least[i & 1], fabsf(g[i]));
    }
    usual = (sum_of[0] + sum_of[1]) / 32.f;
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < left) {
        sum_of[0] += fabsf(g[i]);
        least[0] = fminf(least[0], fabsf(g[i]));
      }
    usual = left >= kFewest ? sum_of[0] / (float)left
                            : usual_of_few<T>(d, row, live, feature, left);
  }
  const float doubt = usual * d.share;
  if (!__any_sync(0xffffffffu, live && fminf(least[0], least[1]) < doubt)) return;
  uint32_t mask = 0, zero = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    if (live && i < left && fabsf(g[i]) < doubt) mask |= 1u << i;
    if (g[i] == 0.f) zero |= 1u << i;
  }
  // exactly 0: cut off altogether, or a feature without weights
  const uint32_t features = __reduce_or_sync(0xffffffffu, zero & mask);
  if (__popc(features) > kMostDoubts) mask &= ~zero;
  else
    for (uint32_t f = features; f; f &= f - 1) {
      const int i = __ffs(f) - 1;
      if (!any_weight<T>(d, feature + i)) mask &= ~(1u << i);
    }
  if (__popc(mask) > kMostDoubts) mask = 0;
  for (uint32_t who; (who = __ballot_sync(0xffffffffu, mask != 0)) != 0;) {
    const int from = __ffs(who) - 1;
    const int i = __shfl_sync(0xffffffffu, __ffs(mask) - 1, from);
    const int64_t of_x = __shfl_sync(0xffffffffu, row, from);
    const T* a = reinterpret_cast<const T*>(d.x) + of_x * d.x_ld;
    const T* b = reinterpret_cast<const T*>(d.w) + (int64_t)(feature + i) * d.w_ld;
    constexpr int kAhead = 5;              // packs of a row that are fetched together
    double sum = 0.0, more = 0.0;
    for (int64_t p0 = lane * 8; p0 < d.H; p0 += 256 * kAhead) {
      uint4 ra[kAhead], rb[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t p = p0 + 256 * k;
        ra[k] = pack_at(d, a, p);
        rb[k] = pack_at(d, b, p);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        float va[8], vb[8];
        vec::unpack<T, 8>(ra[k], va);
        vec::unpack<T, 8>(rb[k], vb);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          sum = fma((double)va[j], (double)vb[j], sum);
          more = fma((double)va[j + 1], (double)vb[j + 1], more);
        }
      }
    }
    sum += more;
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == from) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (i == j) g[j] = (float)sum;
      mask &= mask - 1;
    }
  }
}

template <bool kB, int A>
struct GatedEpi {
  static constexpr bool kBf16 = kB, kChunks = false;
  struct Args {
    void* h;
    int64_t h_ld;
    float *g, *u;                          // null: not kept
    int64_t keep_ld;
    int F, wide;
    Doubts doubts;
  };
  static __device__ __forceinline__ void tile(const Args& a, const gemm::Problem& p,
                                              const gemm::TileAt& t, int row, uint32_t acc, int c0,
                                              float* block) {
    using T = typename std::conditional<kB, __nv_bfloat16, __half>::type;
    const int half = p.bn / 2, n0 = t.n * half, cols = min(half, a.F - n0);
    const bool live = row < p.M;
    for (int c = c0; c < cols; c += 64) {
      float g[32], u[32];
      __syncwarp();                          // (the loads are the whole warp's)
      sm100::tmem_ld32x2(acc + c, acc + half + c, g, u);
      const int left = cols - c;
      if constexpr (A == kRelu) settle_signs<T>(a.doubts, row, live, n0 + c, left, g);
      if (a.g) {
        const int64_t at = (int64_t)row * a.keep_ld + n0 + c;
        gemm::store_block(live ? a.g + at : nullptr, g, left, true, block);
        gemm::store_block(live ? a.u + at : nullptr, u, left, true, block);
      }
      // (not of rows past the last: what stands there may be anything, and the exact
      // division's way through NaN and infinities took 14 us of 43 for 64 tokens)
      if (live) {
#pragma unroll
        for (int i = 0; i < 32; ++i) g[i] = act_16<A>(g[i]) * u[i];
      }
      T* h = reinterpret_cast<T*>(a.h) + (int64_t)row * a.h_ld + n0 + c;
      gemm::store_block(live ? h : nullptr, g, left, a.wide, block);
    }
  }
};

// Two rows go here up to kFewWeights elements of a weight (H x F; us here and by the
// tensor cores: 1,024 x 4,096 9.4 and 14.4, 2,048 x 8,192 19.5 and 25.0, 2,560 x 9,728 25.1 and
// 24.3, 4,096 x 12,288 45.7 and 39.6; 2,560 x 8,192, past the limit, 23.0 and 33.3: tiles of
// a wave and a bit).
constexpr int kFewRows = 2;
constexpr int kFewBytes = 40960;           // of x in shared memory
constexpr int64_t kFewWeights = 1 << 24;

// A warp a feature, N rows of x.  Of a feature's two rows five packs each are fetched
// together: 10 loads a lane (us of one row with four, five and eight: 2,560 x 9,728 22.3, 21.0
// and 26.9, whose 320 packs are two rounds of five; 4,096 x 12,288 39.6, 41.6 and 41.6; 3,584 x
// 18,944 48.5, 47.7 and 51.9; 2,048 x 8,192 16.8, 17.7 and 18.2).
template <typename T, int A, int N>
__global__ void __launch_bounds__(256)
    few_rows_kernel(const T* x, int64_t x_ld, const T* wg, int64_t wg_ld, const T* wu,
                    int64_t wu_ld, int rows, int H, int F, T* h, float* g_out, float* u_out,
                    int64_t keep_ld) {
  constexpr int kAhead = 5;
  extern __shared__ uint4 xs[];            // [N][packs]
  const int packs = (H + 7) / 8, lane = threadIdx.x & 31;
  const int f = blockIdx.x * 8 + threadIdx.x / 32;
  const T* rg = wg + (int64_t)min(f, F - 1) * wg_ld;
  const T* ru = wu + (int64_t)min(f, F - 1) * wu_ld;
  // (a row's last pack may be a part of one: element by element, then)
  auto pack_of = [&](const T* row, int p) {
    return (p + 1) * 8 <= H ? __ldg(reinterpret_cast<const uint4*>(row) + p)
                            : vec::load_any_of<T>(row, p * 8, H, row, row);
  };
  uint4 a[kAhead], b[kAhead];
  auto fetch = [&](int p0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int p = p0 + j * 32 + lane;
      a[j] = b[j] = make_uint4(0, 0, 0, 0);
      if (p < packs) a[j] = pack_of(rg, p), b[j] = pack_of(ru, p);
    }
  };
  fetch(0);
  for (int i = threadIdx.x; i < N * packs; i += blockDim.x) {
    const int t = i / packs, p = i - t * packs;
    xs[i] = t < rows ? pack_of(x + t * x_ld, p) : make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  float g[N], u[N];
#pragma unroll
  for (int t = 0; t < N; ++t) g[t] = u[t] = 0.f;
  for (int p0 = 0; p0 < packs; p0 += 32 * kAhead) {
    if (p0) fetch(p0);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int p = p0 + j * 32 + lane;
      if (p >= packs) continue;
      float vg[8], vu[8];
      vec::unpack<T, 8>(a[j], vg);
      vec::unpack<T, 8>(b[j], vu);
#pragma unroll
      for (int t = 0; t < N; ++t) {
        float vx[8];
        vec::unpack<T, 8>(xs[t * packs + p], vx);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          g[t] = fmaf(vg[i], vx[i], g[t]);
          u[t] = fmaf(vu[i], vx[i], u[t]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      g[t] += __shfl_xor_sync(0xffffffffu, g[t], o);
      u[t] += __shfl_xor_sync(0xffffffffu, u[t], o);
    }
#pragma unroll
  for (int t = 0; t < N; ++t)
    if (lane == t && t < rows && f < F) {
      h[(int64_t)t * F + f] = from_f32<T>(act<A>(g[t]) * u[t]);
      if (g_out) g_out[t * keep_ld + f] = g[t], u_out[t * keep_ld + f] = u[t];
    }
}

template <typename T, int A>
int few_rows(const void* x, int64_t x_ld, const void* wg, int64_t wg_ld, const void* wu,
             int64_t wu_ld, int rows, int H, int F, void* h, float* g, float* u, int64_t keep_ld,
             cudaStream_t st) {
  auto* kernel = rows == 1 ? few_rows_kernel<T, A, 1> : few_rows_kernel<T, A, 2>;
  kernel<<<(F + 7) / 8, 256, rows * ((H + 7) / 8) * 16, st>>>(
      (const T*)x, x_ld, (const T*)wg, wg_ld, (const T*)wu, wu_ld, rows, H, F, (T*)h, g, u,
      keep_ld);
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

// h of fp32 g and u.
template <int A>
__global__ void __launch_bounds__(256)
    forward_kernel(const float* g, const float* u, int64_t ld, int64_t rows, int F, float* h) {
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
    for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < F; c += gridDim.x * blockDim.x)
      h[r * F + c] = act<A>(g[r * ld + c]) * u[r * ld + c];
}

// dg and du out of g, u (fp32) and dh, in packs of 16 bytes: g, u, dg and du have rows
// of whole packs (columns from F on are zeroed), rows of dh may begin anywhere.
template <typename T, int A>
__global__ void __launch_bounds__(256)
    backward_kernel(const float* g, const float* u, int64_t keep_ld, const T* dh, int64_t dh_ld,
                    int64_t rows, int F, T* dg, T* du, int64_t ld) {
  constexpr int V = 16 / (int)sizeof(T);
  const int packs = (F + V - 1) / V;
  const T* hi = dh + (rows - 1) * dh_ld + F;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
    for (int p = blockIdx.x * blockDim.x + threadIdx.x; p < packs; p += gridDim.x * blockDim.x) {
      const int c = p * V;
      float vg[V], vu[V], vd[V];
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(g + r * keep_ld + c + i));
        const float4 y = __ldg(reinterpret_cast<const float4*>(u + r * keep_ld + c + i));
        vg[i] = x.x, vg[i + 1] = x.y, vg[i + 2] = x.z, vg[i + 3] = x.w;
        vu[i] = y.x, vu[i + 1] = y.y, vu[i + 2] = y.z, vu[i + 3] = y.w;
      }
      vec::unpack<T, V>(vec::load_any_of<T>(dh + r * dh_ld, c, F, dh, hi), vd);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float a, d;
        if constexpr (sizeof(T) == 4) act_grad<A>(vg[i], a, d);
        else act_grad_16<A>(vg[i], a, d);
        const bool in = c + i < F;             // (what is kept past F is not written)
        vg[i] = in ? vd[i] * vu[i] * d : 0.f;
        vu[i] = in ? vd[i] * a : 0.f;
      }
      vec::store<T, V>(dg + r * ld + c, vg);
      vec::store<T, V>(du + r * ld + c, vu);
    }
}

int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }
int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

bool sizes_ok(int64_t T, int32_t H, int32_t F) {
  // (dg and du side by side, a pad and a tile past them are counted in 32 bits)
  return T >= 0 && T < ((int64_t)1 << 31) - 256 && H >= 1 && H < INT32_MAX - 256 && F >= 1 &&
         F <= (1 << 30) - 256;
}

int size_of(int dtype) { return dtype == TT_F32 ? 4 : 2; }

template <typename T, int A>
void run_backward(const float* g, const float* u, int64_t keep_ld, const void* dh, int64_t dh_ld,
                  int64_t rows, int F, void* dg, void* du, int64_t ld, cudaStream_t st) {
  const int packs = (int)((F * (int64_t)sizeof(T) + 15) / 16);
  const dim3 grid((unsigned)std::min((packs + 255) / 256, 64),
                  (unsigned)std::min<int64_t>(rows, 32768));
  backward_kernel<T, A><<<grid, 256, 0, st>>>(g, u, keep_ld, (const T*)dh, dh_ld, rows, F, (T*)dg,
                                              (T*)du, ld);
  tt_count_launches(1);
}

template <bool kB>
int forward_16(int64_t T, int H, int F, const void* x, int64_t x_ld, const void* wg,
               int64_t wg_ld, const void* wu, int64_t wu_ld, int act, void* h, float* g, float* u,
               int64_t keep_ld, int32_t* status, cudaStream_t st) {
  return dispatch_act(act, [&](auto a) -> int {
    const gemm::Factor all[3] = {{x, x_ld, false}, {wg, wg_ld, false}, {wu, wu_ld, false}};
    for (const gemm::Factor& f : all)
      if (!gemm::copyable(f)) return TT_ERR_UNSUPPORTED;
    if (T <= kFewRows && T * ((H + 7) / 8) * 16 <= kFewBytes &&
        (T == 1 || (int64_t)H * F <= kFewWeights))
      return few_rows<typename std::conditional<kB, __nv_bfloat16, __half>::type,
                      decltype(a)::value>(x, x_ld, wg, wg_ld, wu, wu_ld, (int)T, H, F, h, g, u,
                                          keep_ld, st);
    using Epi = GatedEpi<kB, decltype(a)::value>;
    const gemm::Plan plan =
        gemm::plan_product(T, F, (H + gemm::kBK - 1) / gemm::kBK, 16, true, false);
    const gemm::Factor fx{x, x_ld, false};
    const gemm::Term terms[2] = {{fx, {wg, wg_ld, false}, H}, {fx, {wu, wu_ld, false}, H}};
    gemm::Problem q;
    if (!gemm::set_up(&q, plan, kB, T, F, terms, 2, true, status)) return TT_ERR_UNSUPPORTED;
    typename Epi::Args ea{};
    ea.h = h, ea.h_ld = F, ea.g = g, ea.u = u, ea.keep_ld = keep_ld, ea.F = F;
    ea.doubts = {x, wg, x_ld, wg_ld, H, (float)(H / 16 + 4) * 0x1p-24f};
    ea.wide = F % 8 == 0 && (reinterpret_cast<uintptr_t>(h) & 15) == 0;
    return gemm::launch<false, false, Epi>(plan, q, ea, st);
  });
}

}  // namespace
}  // namespace gated
}  // namespace tt

using namespace tt;
using namespace tt::gated;

extern "C" int64_t tt_gated_linear_fwd_workspace_size(int dtype, int64_t T, int32_t H, int32_t F) {
  if (!sizes_ok(T, H, F) || dtype != TT_F32) return 0;
  return gemm::fp32_work(T, F, H, 2);
}

extern "C" int tt_gated_linear_fwd(int dtype, int64_t T, int32_t H, int32_t F, const void* x,
                                   int64_t x_ld, const void* wg, int64_t wg_ld, const void* wu,
                                   int64_t wu_ld, int act, void* h, float* g, float* u,
                                   int64_t keep_ld, void* workspace, int64_t workspace_bytes,
                                   int32_t* status, void* stream) {
  if (!sizes_ok(T, H, F) || act < kSilu || act > kRelu || x_ld < H || wg_ld < H || wu_ld < H ||
      !g != !u ||
      (g && (keep_ld < round8(F) || keep_ld % 4 ||
             ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(u)) & 15))) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15))
    return TT_ERR_INVALID_ARG;
  if (dtype < TT_F32 || dtype > TT_F16) return TT_ERR_UNSUPPORTED;
  if (T == 0) return TT_OK;
  if (!x || !wg || !wu || !h || (dtype == TT_F32 && !g)) return TT_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TT_BF16)
    return forward_16<true>(T, H, F, x, x_ld, wg, wg_ld, wu, wu_ld, act, h, g, u, keep_ld, status,
                            st);
  if (dtype == TT_F16)
    return forward_16<false>(T, H, F, x, x_ld, wg, wg_ld, wu, wu_ld, act, h, g, u, keep_ld, status,
                             st);
  if (workspace_bytes < tt_gated_linear_fwd_workspace_size(dtype, T, H, F))
    return TT_ERR_WORKSPACE;
  const gemm::Factor fx{x, x_ld, false};
  const gemm::Term terms[2] = {{fx, {wg, wg_ld, false}, H}, {fx, {wu, wu_ld, false}, H}};
  const gemm::Result r[2] = {{TT_F32, g, keep_ld, nullptr, 0, 1.f, nullptr},
                             {TT_F32, u, keep_ld, nullptr, 0, 1.f, nullptr}};
  if (const int rc = gemm::fp32_products(T, F, terms, r, workspace, workspace_bytes, st)) return rc;
  return dispatch_act(act, [&](auto a) -> int {
    const dim3 grid((unsigned)std::min((F + 255) / 256, 64),
                    (unsigned)std::min<int64_t>(T, 32768));
    forward_kernel<decltype(a)::value><<<grid, 256, 0, st>>>(g, u, keep_ld, T, F, (float*)h);
    tt_count_launches(1);
    return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
  });
}

namespace {
// dg and du side by side, du from column round8(F) on; then the parts of a split sum.
int64_t grad_bytes(int dtype, int64_t T, int32_t F) {
  return round256(T * 2 * round8(F) * size_of(dtype));
}
int64_t slices(int64_t k) { return (k + gemm::kBK - 1) / gemm::kBK; }
int64_t parts_bytes(int dtype, int64_t T, int32_t H, int32_t F) {
  const int64_t both = round8(F) + F;
  if (dtype == TT_F32)
    return std::max({gemm::fp32_work(T, H, 2 * (int64_t)F), gemm::fp32_work(F, H, T),
                     gemm::fp32_work(F, H, T, 2)});
  return std::max({gemm::tc_work(T, H, 2 * slices(F), true), gemm::tc_work(F, H, slices(T), true),
                   gemm::tc_work(both, H, slices(T), true)});
}
}  // namespace

extern "C" int64_t tt_gated_linear_bwd_workspace_size(int dtype, int64_t T, int32_t H, int32_t F) {
  if (!sizes_ok(T, H, F) || dtype < TT_F32 || dtype > TT_F16) return 0;
  return grad_bytes(dtype, T, F) + parts_bytes(dtype, T, H, F);
}

extern "C" int tt_gated_linear_bwd(int dtype, int64_t T, int32_t H, int32_t F, const void* x,
                                   int64_t x_ld, const void* wg, int64_t wg_ld, const void* wu,
                                   int64_t wu_ld, int act, const float* g, const float* u,
                                   int64_t keep_ld, const void* dh, int64_t dh_ld, void* dx,
                                   void* dwg, void* dwu, void* workspace, int64_t workspace_bytes,
                                   int32_t* status, void* stream) {
  if (!sizes_ok(T, H, F) || act < kSilu || act > kRelu || x_ld < H || wg_ld < H || wu_ld < H ||
      keep_ld < F || dh_ld < F)
    return TT_ERR_INVALID_ARG;
  if (dtype < TT_F32 || dtype > TT_F16) return TT_ERR_UNSUPPORTED;
  if (T == 0) return TT_OK;
  if (!x || !wg || !wu || !g || !u || !dh) return TT_ERR_INVALID_ARG;
  if (keep_ld < round8(F) || keep_ld % 4 ||
      ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(u) |
        reinterpret_cast<uintptr_t>(workspace)) & 15))
    return TT_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < tt_gated_linear_bwd_workspace_size(dtype, T, H, F))
    return TT_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t F8 = round8(F), ld = 2 * F8, bytes = grad_bytes(dtype, T, F);
  char* ws = (char*)workspace;
  void *dg = ws, *du = ws + F8 * size_of(dtype), *work = ws + bytes;
  const int64_t work_bytes = workspace_bytes - bytes;
  int rc = dispatch_act(act, [&](auto a) -> int {
    constexpr int A = decltype(a)::value;
    return vec::dispatch_float(dtype, [&](auto t) -> int {
      run_backward<decltype(t), A>(g, u, keep_ld, dh, dh_ld, T, F, dg, du, ld, st);
      return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
    });
  });
  if (rc != TT_OK) return rc;
  auto product = [&](int64_t M, int64_t N, const gemm::Term* terms, int n, void* c) {
    const gemm::Result r{dtype, c, N, nullptr, 0, 1.f, nullptr};
    return dtype == TT_F32
               ? gemm::fp32_product(M, N, terms, n, r, work, work_bytes, st)
               : gemm::tc_product(dtype == TT_BF16, M, N, terms, n, r, work, work_bytes, status,
                                  st);
  };
  if (dx) {
    const gemm::Term terms[2] = {{{dg, ld, false}, {wg, wg_ld, true}, F},
                                 {{du, ld, false}, {wu, wu_ld, true}, F}};
    if ((rc = product(T, H, terms, 2, dx))) return rc;
  }
  if (dwg && dwu && dtype == TT_F32) {
    const gemm::Factor fx{x, x_ld, true};
    const gemm::Term terms[2] = {{{dg, ld, true}, fx, T}, {{du, ld, true}, fx, T}};
    const gemm::Result r[2] = {{dtype, dwg, H, nullptr, 0, 1.f, nullptr},
                               {dtype, dwu, H, nullptr, 0, 1.f, nullptr}};
    return gemm::fp32_products(F, H, terms, r, work, work_bytes, st);
  }
  if (dwg && dwu) {
    // one product for both: its last wave of tiles comes once
    const gemm::Term term{{dg, ld, true}, {x, x_ld, true}, T};
    gemm::Result r{dtype, dwg, H, nullptr, 0, 1.f, nullptr};
    r.p2 = dwu, r.gap = F, r.second = F8;
    return gemm::tc_product(dtype == TT_BF16, F8 + F, H, &term, 1, r, work, work_bytes, status, st);
  }
  for (int i = 0; i < 2; ++i) {
    void* dw = i ? dwu : dwg;
    if (!dw) continue;
    const gemm::Term term{{i ? du : dg, ld, true}, {x, x_ld, true}, T};
    if ((rc = product(F, H, &term, 1, dw))) return rc;
  }
  return TT_OK;
}
