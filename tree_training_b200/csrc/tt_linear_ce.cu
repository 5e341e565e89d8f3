// The cross entropy of an LM head without its logits, and its gradients.
//
//   z = scale * x W^T                          x [T, H], W [V, H]
//   lse[t] = log sum_v exp z[t, v],  loss[t, m] = lse[t] - z[t, y[t, m]]
//   dz[t, v] = (sum_m g[t, m] + g_lse[t]) p[t, v] - sum_{m: y[t, m] = v} g[t, m]
//   dx = scale dz W,  dW = scale dz^T x
//
// (m: a token of a tree has several successors; labels outside [0, V) are ignored.)
//
// 2 T H V operations forward; backward 4 T H V, and 2 T H V again for the logits:
// bound by the tensor cores, for few tokens by W's bytes.
//
// Forward, 16-bit: the product's epilogue reduces each row of a tile of logits to its
// maximum and the sum of exp above it (8 bytes for 64 logits) and picks out the
// labels' logits; a second kernel joins the tiles in order.  Backward: by pieces of
// the vocabulary, each formed again, turned into 16-bit dz by the epilogue, and
// multiplied twice: dW's rows of the piece are complete, dx is summed up in fp32.
// The pieces are as wide as a quarter of a gigabyte of dz allows, and at least
// 4,096: every piece reads and writes dx's fp32 sum once.  Both workspaces grow with the
// rows: the forward's 8 bytes for 64 logits are T V / 8 (155 MB for 8,192 rows of 151,936
// words, 2.5 GB for 131,072; more where tiles are narrower), the backward's dz 8,192 T
// past 32,768 rows.
//
// dz is rounded to 16 bits once, as the tensor cores' operands need.  A row's label
// dominates its dz, so that over few rows that one rounding (2^-9 in bf16) would show
// in dx and dW beside their own: up to 256 rows, where W's bytes bound the products
// anyway, dz is two 16-bit terms, and each product a sum of two.  In fp16 it is
// multiplied by a power of two first that brings the largest weight of a row to
// about 2^14 (and divided out of the sums): softmax probabilities times weights of
// 1 / T lie below fp16's smallest number.
//
// Where one piece holds all logits (a quarter of a gigabyte of fp32 at most: few rows or
// a small vocabulary) the forward leaves them for the backward, whose fourth product
// would cost a third more.  (16-bit: not where k is so short that forming them again
// takes less than their 8 bytes each way.)
//
// fp32: the same steps with products on the CUDA cores and passes over the logits
// of a piece.
//
// Measured on a B200, bf16, W of 151,936 x 2,560: 8,192 rows forward and backward 19.2 to
// 20.8 ms (1,230 to 1,330 TFLOP/s with the logits formed again, at the power limit); 2,047
// rows forward 1.25 ms (1,280 TFLOP/s), 47 rows 140 us forward (5.6 TB/s) and 543 with the
// backward.
#include <cfloat>

#include "tt_gemm_sm100.cuh"

namespace tt {
namespace linear_ce {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// A row's labels inside the vocabulary, moved to the front: (label, m).
struct Labels {
  const int32_t* count;                    // [T]
  const int2* list;                        // [T][M]
  int M;
};

__global__ void __launch_bounds__(256)
    labels_kernel(const int64_t* labels, int64_t T, int M, int64_t V, int32_t* count, int2* list) {
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= T) return;
  int n = 0;
  for (int m = 0; m < M; ++m) {
    const int64_t y = labels[t * M + m];
    if (y >= 0 && y < V) list[t * M + n++] = make_int2((int)y, m);
  }
  count[t] = n;
}

// Which of a row's 32-column chunks of columns c0 .. c0 + n hold labels.
__device__ __forceinline__ uint32_t chunks_with_labels(const Labels& l, int64_t row, int count,
                                                       int c0, int n) {
  uint32_t mask = 0;
  for (int i = 0; i < count; ++i) {
    const int at = l.list[row * l.M + i].x - c0;
    if (at >= 0 && at < n) mask |= 1u << (at >> 5);
  }
  return mask;
}

// ---- forward, 16-bit ---------------------------------------------------------------

// Maximum and sum of exp above it, of one more chunk of a row.
template <int N>
__device__ __forceinline__ void take(const float (&z)[N], float& m, float& s) {
  float top = m;
#pragma unroll
  for (int i = 0; i < N; ++i) top = fmaxf(top, z[i]);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) sum += exp2f((z[i] - ref) * kLog2e);
  s = s * exp2f((m - ref) * kLog2e) + sum;
  m = top;
}

// (kKeep: a form of its own, since the stores cost the registers that the sums need)
template <bool kB, bool kKeep>
struct LseEpi {
  static constexpr bool kBf16 = kB, kChunks = true;
  struct Args {
    float2* part;                          // [tiles of n][4][T]
    Labels labels;
    float* picked;                         // [T][M]
    float scale;
    float* kept;                           // kKeep: the logits
    int64_t kept_ld;
  };
  static __device__ __forceinline__ void finish(const Args& a, const gemm::Problem& p,
                                                const gemm::TileAt& t, int row, int c0,
                                                float (&z)[64]) {
    const int n0 = t.n * p.bn + c0, cols = min(64, min(p.bn, p.N - t.n * p.bn) - c0);
    if (row >= p.M) return;
    float m = -INFINITY, s = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) z[i] = i < cols ? z[i] * a.scale : -INFINITY;
    take<64>(z, m, s);
    if constexpr (kKeep) {
      float* to = a.kept + (int64_t)row * a.kept_ld + n0;
      // (tiles are multiples of 16 wide: eights that go over the end go into the row's pad)
#pragma unroll
      for (int i = 0; i < 64; i += 8)
        if (i < cols)
          asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + i),
                       "f"(z[i]), "f"(z[i + 1]), "f"(z[i + 2]), "f"(z[i + 3]), "f"(z[i + 4]),
                       "f"(z[i + 5]), "f"(z[i + 6]), "f"(z[i + 7])
                       : "memory");
    }
    a.part[(int64_t)(4 * t.n + c0 / 64) * p.M + row] = make_float2(m, s);
    const int count = a.labels.count[row];
    for (int k = 0; k < count; ++k) {
      const int2 l = a.labels.list[(int64_t)row * a.labels.M + k];
      const int at = l.x - n0;
      if (at < 0 || at >= cols) continue;
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 64; ++i)
        if (at == i) v = z[i];
      a.picked[(int64_t)row * a.labels.M + l.y] = v;
    }
  }
};

// (m, s) of two parts of a row together.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  const float ref = m == -INFINITY ? 0.f : m;
  return make_float2(m, a.y * expf(a.x - ref) + b.y * expf(b.x - ref));
}

constexpr int kJoinThreads = 512;

// lse and losses of R rows a block (a power of two): its threads share out the parts,
// twice over: the maximum of all, then the sums above it.
__global__ void __launch_bounds__(kJoinThreads)
    finish_kernel(const float2* part, int parts, int64_t T, int R, const int64_t* labels, int M,
                  int64_t V, const float* picked, float* lse, float* losses) {
  __shared__ float sm[kJoinThreads];
  const int r = threadIdx.x % R, lanes = kJoinThreads / R, mine = threadIdx.x / R;
  const int64_t row = (int64_t)blockIdx.x * R + r;
  const float2* p = part + row;
  float m = -INFINITY;
  if (row < T) {
#pragma unroll 4
    for (int i = mine; i < parts; i += lanes) m = fmaxf(m, p[(int64_t)i * T].x);
  }
  sm[threadIdx.x] = m;
  for (int o = lanes / 2; o; o >>= 1) {
    __syncthreads();
    if (mine < o) sm[threadIdx.x] = fmaxf(sm[threadIdx.x], sm[threadIdx.x + o * R]);
  }
  __syncthreads();
  m = sm[r];
  __syncthreads();
  const float ref = m == -INFINITY ? 0.f : m;
  float s = 0.f;
  if (row < T) {
#pragma unroll 4
    for (int i = mine; i < parts; i += lanes) {
      const float2 v = p[(int64_t)i * T];
      s += v.y * expf(v.x - ref);
    }
  }
  sm[threadIdx.x] = s;
  for (int o = lanes / 2; o; o >>= 1) {
    __syncthreads();
    if (mine < o) sm[threadIdx.x] += sm[threadIdx.x + o * R];
  }
  __syncthreads();
  s = sm[r];
  if (row >= T) return;
  if (mine == 0) lse[row] = m + logf(s);
  for (int k = mine; k < M; k += lanes) {
    const int64_t i = row * M + k, y = labels[i];
    losses[i] = y >= 0 && y < V ? (m - picked[i]) + logf(s) : 0.f;
  }
}

// ---- backward ------------------------------------------------------------------------

// The weight of a row's probabilities, and (fp16) the largest weight of all, as bits.
__global__ void __launch_bounds__(256)
    weights_kernel(const Labels l, int64_t T, const float* g_loss, const float* g_lse, float scale,
                   float* weight, uint32_t* largest) {
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  float most = 0.f;
  if (t < T) {
    float w = g_lse ? g_lse[t] : 0.f;
    most = fabsf(w);
    for (int i = 0; g_loss && i < l.count[t]; ++i) {
      const float g = g_loss[t * l.M + l.list[t * l.M + i].y];
      w += g;
      most += fabsf(g);
    }
    weight[t] = w * scale;
    most *= fabsf(scale);
  }
  for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (largest && (threadIdx.x & 31) == 0 && most > 0.f) atomicMax(largest, __float_as_uint(most));
}

// The power of two that fp16's dz is multiplied by, and one over it.
__global__ void factor_kernel(const uint32_t* largest, float* factor) {
  const float most = __uint_as_float(*largest);
  int e = 0;
  if (most > 0.f && most <= FLT_MAX) frexpf(most, &e);
  const int up = max(-100, min(100, 14 - e));
  factor[0] = ldexpf(1.f, up);
  factor[1] = ldexpf(1.f, -up);
}

struct Grad {
  Labels labels;
  const float *weight, *lse, *g_loss;
  const float* factor;                     // null: 1
  float scale;
  int64_t v0;                              // of the piece
};

// dz of a chunk of a row (in place of its logits), col0: the chunk's first column in
// the vocabulary.
template <int N>
__device__ __forceinline__ void gradient(const Grad& a, int64_t row, int count, bool labels_here,
                                         float lse, float w, float f, int col0, float (&z)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) z[i] = w * exp2f((z[i] - lse) * kLog2e);
  if (!labels_here || !a.g_loss) return;
  for (int k = 0; k < count; ++k) {
    const int2 l = a.labels.list[row * a.labels.M + k];
    const int at = l.x - col0;
    if (at < 0 || at >= N) continue;
    const float g = a.g_loss[row * a.labels.M + l.y] * a.scale * f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at == i) z[i] -= g;
  }
}

template <bool kB>
struct GradEpi {
  static constexpr bool kBf16 = kB, kChunks = false;
  struct Args {
    Grad g;
    void *dz, *rest;                       // rest: what rounding took off dz, or null
    int64_t ld;
  };
  static __device__ __forceinline__ void tile(const Args& a, const gemm::Problem& p,
                                              const gemm::TileAt& t, int row, uint32_t acc, int c0,
                                              float* block) {
    using T = typename std::conditional<kB, __nv_bfloat16, __half>::type;
    const int n0 = t.n * p.bn, cols = min(p.bn, p.N - n0);
    const bool live = row < p.M;
    const int count = live ? a.g.labels.count[row] : 0;
    const int v0 = (int)a.g.v0 + n0;
    const uint32_t mask = chunks_with_labels(a.g.labels, row, count, v0, cols);
    const float lse = live ? a.g.lse[row] : 0.f;
    const float f = a.g.factor ? *a.g.factor : 1.f;
    const float w = live ? a.g.weight[row] * f : 0.f;
    for (int c = c0; c < cols; c += 64) {
      float z[32];
      __syncwarp();                          // (the load is the whole warp's)
      sm100::tmem_ld32(acc + c, z);
#pragma unroll
      for (int i = 0; i < 32; ++i) z[i] *= a.g.scale;
      gradient<32>(a.g, row, count, (mask >> (c >> 5)) & 1, lse, w, f, v0 + c, z);
      const int64_t at = (int64_t)row * a.ld + n0 + c;
      gemm::store_block(live ? reinterpret_cast<T*>(a.dz) + at : nullptr, z, cols - c, true, block);
      if (a.rest) {
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i] -= to_f32(from_f32<T>(z[i]));
        gemm::store_block(live ? reinterpret_cast<T*>(a.rest) + at : nullptr, z, cols - c, true,
                          block);
      }
    }
  }
};

// ---- fp32: passes over the logits of a piece --------------------------------------------

// (m, s) of a row's columns of a piece, by segments (blockIdx.y) of them, and its
// labels' logits.
__global__ void __launch_bounds__(256)
    lse_kernel(const float* z, int64_t T, int64_t v0, int n, int64_t ld, int segment,
               const Labels l, float2* part, float* picked) {
  __shared__ float2 sm[256];
  const int c0 = blockIdx.y * segment, c1 = min(n, c0 + segment);
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
    const float* row = z + t * ld;
    float m = -INFINITY, s = 0.f;
    for (int c = c0 + threadIdx.x; c < c1; c += blockDim.x) m = fmaxf(m, row[c]);
    const float ref = m == -INFINITY ? 0.f : m;
    for (int c = c0 + threadIdx.x; c < c1; c += blockDim.x) s += expf(row[c] - ref);
    sm[threadIdx.x] = make_float2(m, s);
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
      if (threadIdx.x < o) sm[threadIdx.x] = join(sm[threadIdx.x], sm[threadIdx.x + o]);
      __syncthreads();
    }
    if (threadIdx.x == 0) part[(int64_t)blockIdx.y * T + t] = sm[0];
    for (int i = threadIdx.x; i < l.count[t]; i += blockDim.x) {
      const int2 y = l.list[t * l.M + i];
      if (y.x >= v0 + c0 && y.x < v0 + c1) picked[t * l.M + y.y] = row[y.x - v0];
    }
    __syncthreads();
  }
}

// dz out of the logits of a piece (which it may replace).
__global__ void __launch_bounds__(256)
    grad_kernel(const float* z, int64_t z_ld, float* dz, int64_t T, int n, int64_t ld, int segment,
                const Grad g) {
  const int c0 = blockIdx.y * segment, c1 = min(n, c0 + segment);
  for (int64_t t = blockIdx.x; t < T; t += gridDim.x) {
    const int count = g.labels.count[t];
    const float w = g.weight[t], lse = g.lse[t];
    const float* from = z + t * z_ld;
    float* row = dz + t * ld;
    for (int c = c0 + threadIdx.x; c < c1; c += blockDim.x) row[c] = w * expf(from[c] - lse);
    __syncthreads();
    // (one thread: a label may be given twice)
    if (threadIdx.x == 0 && g.g_loss)
      for (int k = 0; k < count; ++k) {
        const int2 l = g.labels.list[t * g.labels.M + k];
        const int64_t at = l.x - g.v0;
        if (at >= c0 && at < c1) row[at] -= g.g_loss[t * g.labels.M + l.y] * g.scale;
      }
    __syncthreads();
  }
}

// The same to 16-bit dz (and what its rounding took off, or null), in packs of 8; rows
// of z and dz begin on 32- and 16-byte boundaries and have whole packs.
template <typename T>
__global__ void __launch_bounds__(256)
    grad_16_kernel(const float* z, int64_t z_ld, T* dz, T* rest, int64_t rows, int n, int64_t ld,
                   int segment, const Grad g) {
  const int c0 = blockIdx.y * segment, c1 = min(n, c0 + segment);
  const float f = g.factor ? *g.factor : 1.f;
  for (int64_t t = blockIdx.x; t < rows; t += gridDim.x) {
    const int count = g.g_loss ? g.labels.count[t] : 0;
    const int2* list = g.labels.list + t * g.labels.M;
    const float w = g.weight[t] * f, lse = g.lse[t];
    const float* from = z + t * z_ld;
    auto put = [&](int64_t at, float v) {
      dz[at] = from_f32<T>(v);
      if (rest) rest[at] = from_f32<T>(v - to_f32(from_f32<T>(v)));
    };
    for (int c = c0 + threadIdx.x * 8; c < c1; c += blockDim.x * 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(from + c + i);
        v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = w * exp2f((v[i] - lse) * kLog2e);
      vec::store<T, 8>(dz + t * ld + c, v);
      if (rest) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] -= to_f32(from_f32<T>(v[i]));
        vec::store<T, 8>(rest + t * ld + c, v);
      }
    }
    __syncthreads();
    // a thread a label, the first of those that are equal
    for (int k = threadIdx.x; k < count; k += blockDim.x) {
      const int at = list[k].x;
      if (at < c0 || at >= c1) continue;
      float sum = 0.f;
      bool first = true;
      for (int j = 0; j < count; ++j)
        if (list[j].x == at) {
          first &= j >= k;
          sum += g.g_loss[t * g.labels.M + list[j].y];
        }
      if (first) put(t * ld + at, w * exp2f((from[at] - lse) * kLog2e) - sum * g.scale * f);
    }
    __syncthreads();
  }
}

// Columns of a segment: four blocks an SM where there are few rows.
int segment_of(int64_t T, int64_t n) {
  const int64_t want = std::max<int64_t>(1, 4 * vec::kSMs / T);
  return (int)std::max<int64_t>(512, (n + want - 1) / want + 7) / 8 * 8;
}
int64_t segments_of(int64_t T, int64_t n) {
  return (n + segment_of(T, n) - 1) / segment_of(T, n);
}

// ---- host ------------------------------------------------------------------------------

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

bool sizes_ok(int64_t T, int32_t H, int64_t V, int64_t M) {
  return T >= 0 && T < ((int64_t)1 << 31) - 256 && H >= 1 && H < INT32_MAX - 256 && V >= 1 &&
         V < ((int64_t)1 << 31) - 256 && M >= 0 && M <= 0x7fffffff;
}

constexpr int64_t kTwoTermRows = 256;      // see the top

bool two_terms(int dtype, int64_t T) { return dtype != TT_F32 && T <= kTwoTermRows; }

constexpr int64_t kPieceBytes = (int64_t)1 << 28;

// Bytes of dz (of fp32 logits) an element.
int64_t dz_size(int dtype, int64_t T) { return dtype == TT_F32 || two_terms(dtype, T) ? 4 : 2; }

// Columns of a piece of the vocabulary: a quarter of a gigabyte of dz, at least 4,096.
int64_t most_columns(int dtype, int64_t T) {
  const int64_t wide = kPieceBytes / (dz_size(dtype, T) * std::max<int64_t>(T, 1));
  return std::max<int64_t>(4096, wide / 256 * 256);
}
int64_t piece_of(int dtype, int64_t T, int64_t V) {
  return std::min((V + 255) / 256 * 256, most_columns(dtype, T));
}

// The row stride of the logits that the forward leaves for the backward; 0: none.
int64_t kept_ld(int dtype, int64_t T, int32_t H, int64_t V) {
  const int64_t ld = (V + 7) / 8 * 8;
  // (forming them again takes 2 H operations each at 1.4e15 a second, or W's 2 H bytes
  // for T of them at 6.5e12; keeping them 8 bytes)
  const bool worth = dtype == TT_F32 || H >= 1024 || H > 4 * T;
  return worth && T > 0 && T * ld * 4 <= kPieceBytes && V <= most_columns(dtype, T) ? ld : 0;
}

int64_t labels_bytes(int64_t T, int64_t M) { return round256(4 * T) + round256(8 * T * M); }

// The forward's tiles of the vocabulary.
gemm::Plan forward_plan(int64_t T, int32_t H, int64_t V) {
  return gemm::plan_product(T, V, (H + gemm::kBK - 1) / gemm::kBK, 16, false, false);
}

struct Carve {
  char* p;
  template <typename T>
  T* take(int64_t bytes) {
    char* q = p;
    p += round256(bytes);
    return reinterpret_cast<T*>(q);
  }
};

Labels sort_labels(const int64_t* labels, int64_t T, int64_t M, int64_t V, Carve& ws,
                   cudaStream_t st) {
  int32_t* count = ws.take<int32_t>(4 * T);
  int2* list = ws.take<int2>(8 * T * M);
  labels_kernel<<<(unsigned)((T + 255) / 256), 256, 0, st>>>(labels, T, (int)M, V, count, list);
  tt_count_launches(1);
  return Labels{count, list, (int)M};
}

unsigned row_blocks(int64_t T) { return (unsigned)std::min<int64_t>(T, 16 * vec::kSMs); }

struct Shape {
  int dtype;
  int64_t T;
  int32_t H;
  int64_t V, M;
};

template <bool kB>
int forward_16(const Shape& s, const void* x, int64_t x_ld, const void* w, int64_t w_ld,
               const Labels& l, float scale, float2* part, float* picked, float* kept,
               int* parts, int32_t* status, cudaStream_t st) {
  const gemm::Plan plan = forward_plan(s.T, s.H, s.V);
  const gemm::Term term{{x, x_ld, false}, {w, w_ld, false}, s.H};
  gemm::Problem q;
  if (!gemm::set_up(&q, plan, kB, s.T, s.V, &term, 1, false, status)) return TT_ERR_UNSUPPORTED;
  *parts = 4 * q.tiles_n;
  if (kept)
    return gemm::launch<false, false, LseEpi<kB, true>>(
        plan, q, {part, l, picked, scale, kept, kept_ld(s.dtype, s.T, s.H, s.V)}, st);
  return gemm::launch<false, false, LseEpi<kB, false>>(plan, q,
                                                       {part, l, picked, scale, nullptr, 0}, st);
}

template <bool kB>
int gradient_16(const Shape& s, const void* x, int64_t x_ld, const void* w, int64_t w_ld, int64_t n,
                const Grad& g, void* dz, void* rest, int64_t ld, int32_t* status, cudaStream_t st) {
  using Epi = GradEpi<kB>;
  const gemm::Plan plan = gemm::plan_product(s.T, n, (s.H + gemm::kBK - 1) / gemm::kBK, 16, false,
                                             false);
  const gemm::Term term{{x, x_ld, false}, {w, w_ld, false}, s.H};
  gemm::Problem q;
  if (!gemm::set_up(&q, plan, kB, s.T, n, &term, 1, false, status)) return TT_ERR_UNSUPPORTED;
  typename Epi::Args ea{g, dz, rest, ld};
  return gemm::launch<false, false, Epi>(plan, q, ea, st);
}

int check(const Shape& s, const void* x, int64_t x_ld, const void* w, int64_t w_ld,
          const int64_t* labels) {
  if (!sizes_ok(s.T, s.H, s.V, s.M) || x_ld < s.H || w_ld < s.H) return TT_ERR_INVALID_ARG;
  if (s.dtype < TT_F32 || s.dtype > TT_F16) return TT_ERR_UNSUPPORTED;
  if (s.T > 0 && (!x || !w || (s.M > 0 && !labels))) return TT_ERR_INVALID_ARG;
  return TT_OK;
}

// Whether p is off a boundary of n bytes.
bool off(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

const char* row_of(const Shape& s, const void* w, int64_t w_ld, int64_t v) {
  return (const char*)w + v * w_ld * (s.dtype == TT_F32 ? 4 : 2);
}

}  // namespace
}  // namespace linear_ce
}  // namespace tt

using namespace tt;
using namespace tt::linear_ce;

extern "C" int64_t tt_linear_ce_kept_ld(int dtype, int64_t T, int32_t H, int64_t V) {
  if (!sizes_ok(T, H, V, 0) || dtype < TT_F32 || dtype > TT_F16) return 0;
  return kept_ld(dtype, T, H, V);
}

extern "C" int64_t tt_linear_ce_fwd_workspace_size(int dtype, int64_t T, int32_t H, int64_t V,
                                                   int64_t M) {
  if (!sizes_ok(T, H, V, M) || dtype < TT_F32 || dtype > TT_F16) return 0;
  const int64_t base = labels_bytes(T, M) + round256(4 * T * M);
  if (T == 0) return base;
  if (dtype == TT_F32) {
    const int64_t P = piece_of(dtype, T, V);
    return base + round256(8 * T * segments_of(T, P) * ((V + P - 1) / P)) +
           round256(4 * T * P) + gemm::fp32_work(T, P, H);
  }
  const gemm::Plan p = forward_plan(T, H, V);
  return base + round256(32 * T * ((V + p.bn - 1) / p.bn));
}

extern "C" int tt_linear_ce_fwd(int dtype, int64_t T, int32_t H, int64_t V, int64_t M,
                                const void* x, int64_t x_ld, const void* w, int64_t w_ld,
                                const int64_t* labels, float scale, float* losses, float* lse,
                                float* kept, void* workspace, int64_t workspace_bytes,
                                int32_t* status, void* stream) {
  const Shape s{dtype, T, H, V, M};
  if (const int rc = check(s, x, x_ld, w, w_ld, labels)) return rc;
  if (T == 0) return TT_OK;
  if (!lse || (M > 0 && !losses) || (kept && !kept_ld(dtype, T, H, V))) return TT_ERR_INVALID_ARG;
  if (off(kept, 32) || off(workspace, 16)) return TT_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < tt_linear_ce_fwd_workspace_size(dtype, T, H, V, M))
    return TT_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  Carve ws{(char*)workspace};
  const Labels l = sort_labels(labels, T, M, V, ws, st);
  float* picked = ws.take<float>(4 * T * M);
  int parts = 1, rc = TT_OK;
  float2* part;
  if (dtype == TT_F32) {
    const int64_t P = piece_of(dtype, T, V), segments = segments_of(T, P);
    part = ws.take<float2>(8 * T * segments * ((V + P - 1) / P));
    parts = 0;
    float* room = ws.take<float>(4 * T * P);
    float* z = kept ? kept : room;
    const int64_t ld = kept ? kept_ld(dtype, T, H, V) : P;
    for (int64_t v0 = 0; v0 < V; v0 += P) {
      const int64_t n = std::min(P, V - v0);
      const gemm::Term term{{x, x_ld, false}, {row_of(s, w, w_ld, v0), w_ld, false}, H};
      const gemm::Result r{TT_F32, z, ld, nullptr, 0, scale, nullptr};
      if ((rc = gemm::fp32_product(T, n, &term, 1, r, ws.p, gemm::fp32_work(T, P, H), st)))
        return rc;
      // (the last piece may have fewer of them)
      const int segment = segment_of(T, P), here = (int)((n + segment - 1) / segment);
      lse_kernel<<<dim3(row_blocks(T), here), 256, 0, st>>>(z, T, v0, (int)n, ld, segment, l,
                                                            part + (int64_t)parts * T, picked);
      parts += here;
      tt_count_launches(1);
    }
  } else {
    part = (float2*)ws.p;
    rc = dtype == TT_BF16 ? forward_16<true>(s, x, x_ld, w, w_ld, l, scale, part, picked, kept,
                                             &parts, status, st)
                          : forward_16<false>(s, x, x_ld, w, w_ld, l, scale, part, picked, kept,
                                              &parts, status, st);
    if (rc) return rc;
  }
  // 32 rows a block read whole lines of the parts; with few rows there are more blocks
  int R = 32;
  while (R > 1 && T / R < 2 * vec::kSMs) R /= 2;
  finish_kernel<<<(unsigned)((T + R - 1) / R), kJoinThreads, 0, st>>>(
      part, parts, T, R, labels, (int)M, V, picked, lse, losses);
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

namespace {
int64_t slices(int64_t k) { return (k + gemm::kBK - 1) / gemm::kBK; }
int terms_of(int dtype, int64_t T) { return two_terms(dtype, T) ? 2 : 1; }
int64_t product_work(int dtype, int64_t T, int32_t H, int64_t P) {
  return dtype == TT_F32 ? std::max({gemm::fp32_work(T, P, H), gemm::fp32_work(T, H, P),
                                     gemm::fp32_work(P, H, T)})
                         : std::max(gemm::tc_work(T, H, terms_of(dtype, T) * slices(P), true),
                                    gemm::tc_work(P, H, terms_of(dtype, T) * slices(T), true));
}
}  // namespace

extern "C" int64_t tt_linear_ce_bwd_workspace_size(int dtype, int64_t T, int32_t H, int64_t V,
                                                   int64_t M) {
  if (!sizes_ok(T, H, V, M) || dtype < TT_F32 || dtype > TT_F16) return 0;
  if (T == 0) return 0;
  const int64_t P = piece_of(dtype, T, V);
  return labels_bytes(T, M) + round256(4 * T) + 2 * 256 + round256(dz_size(dtype, T) * T * P) +
         (P < V ? round256(4 * T * H) : 0) + product_work(dtype, T, H, P);
}

extern "C" int tt_linear_ce_bwd(int dtype, int64_t T, int32_t H, int64_t V, int64_t M,
                                const void* x, int64_t x_ld, const void* w, int64_t w_ld,
                                const int64_t* labels, float scale, const float* lse,
                                const float* kept, const float* g_loss, const float* g_lse,
                                void* dx, void* dw, void* workspace, int64_t workspace_bytes,
                                int32_t* status, void* stream) {
  const Shape s{dtype, T, H, V, M};
  if (const int rc = check(s, x, x_ld, w, w_ld, labels)) return rc;
  if (T == 0) return TT_OK;
  if (!lse || (kept && !kept_ld(dtype, T, H, V))) return TT_ERR_INVALID_ARG;
  if (off(kept, 32) || off(workspace, 16)) return TT_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < tt_linear_ce_bwd_workspace_size(dtype, T, H, V, M))
    return TT_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  const bool f32 = dtype == TT_F32;
  const int64_t P = piece_of(dtype, T, V), size = f32 ? 4 : 2;
  Carve ws{(char*)workspace};
  Grad g{};
  g.labels = sort_labels(labels, T, M, V, ws, st);
  float* weight = ws.take<float>(4 * T);
  uint32_t* largest = ws.take<uint32_t>(4);
  float* factor = ws.take<float>(8);
  const int n_terms = terms_of(dtype, T);
  char* dz = ws.take<char>(dz_size(dtype, T) * T * P);
  char* rest = n_terms == 2 ? dz + 2 * T * P : nullptr;
  float* sum = P < V ? ws.take<float>(4 * T * H) : nullptr;
  void* work = ws.p;
  const int64_t work_bytes = product_work(dtype, T, H, P);
  const bool f16 = dtype == TT_F16;
  if (f16 && cudaMemsetAsync(largest, 0, 4, st) != cudaSuccess) return TT_ERR_CUDA;
  weights_kernel<<<(unsigned)((T + 255) / 256), 256, 0, st>>>(g.labels, T, g_loss, g_lse, scale,
                                                              weight, f16 ? largest : nullptr);
  tt_count_launches(1);
  const float* back = nullptr;
  if (f16) {
    factor_kernel<<<1, 1, 0, st>>>(largest, factor);
    tt_count_launches(1);
    g.factor = factor, back = factor + 1;
  }
  g.weight = weight, g.lse = lse, g.g_loss = g_loss, g.scale = scale;
  auto product = [&](int64_t m, int64_t n, const gemm::Term& term, const gemm::Result& r) {
    if (f32) return gemm::fp32_product(m, n, &term, 1, r, work, work_bytes, st);
    gemm::Term terms[2] = {term, term};
    terms[1].a.p = rest;
    return gemm::tc_product(dtype == TT_BF16, m, n, terms, n_terms, r, work, work_bytes, status,
                            st);
  };
  int rc = TT_OK;
  for (int64_t v0 = 0; v0 < V; v0 += P) {
    const int64_t n = std::min(P, V - v0);
    const void* wp = row_of(s, w, w_ld, v0);
    g.v0 = v0;
    if (f32) {
      const gemm::Term term{{x, x_ld, false}, {wp, w_ld, false}, H};
      if (!kept &&
          (rc = product(T, n, term, gemm::Result{TT_F32, dz, P, nullptr, 0, scale, nullptr})))
        return rc;
      const int segment = segment_of(T, P);
      grad_kernel<<<dim3(row_blocks(T), (unsigned)((n + segment - 1) / segment)), 256, 0, st>>>(
          kept ? kept : (const float*)dz, kept ? kept_ld(dtype, T, H, V) : P, (float*)dz, T,
          (int)n, P, segment, g);
      tt_count_launches(1);
    } else if (kept) {
      const int segment = segment_of(T, P);
      const dim3 grid(row_blocks(T), (unsigned)((n + segment - 1) / segment));
      const int64_t z_ld = kept_ld(dtype, T, H, V);
      if (dtype == TT_BF16)
        grad_16_kernel<<<grid, 256, 0, st>>>(kept, z_ld, (__nv_bfloat16*)dz, (__nv_bfloat16*)rest,
                                             T, (int)n, P, segment, g);
      else
        grad_16_kernel<<<grid, 256, 0, st>>>(kept, z_ld, (__half*)dz, (__half*)rest, T, (int)n, P,
                                             segment, g);
      tt_count_launches(1);
    } else {
      auto* form = dtype == TT_BF16 ? gradient_16<true> : gradient_16<false>;
      rc = form(s, x, x_ld, wp, w_ld, n, g, dz, rest, P, status, st);
      if (rc) return rc;
    }
    if (dx) {
      const bool last = v0 + P >= V;
      const gemm::Term term{{dz, P, false}, {wp, w_ld, true}, n};
      const gemm::Result r{last ? dtype : TT_F32, last ? dx : sum, H, v0 ? sum : nullptr, H, 1.f,
                           back};
      if ((rc = product(T, H, term, r))) return rc;
    }
    if (dw) {
      const gemm::Term term{{dz, P, true}, {x, x_ld, true}, T};
      const gemm::Result r{dtype, (char*)dw + v0 * H * size, H, nullptr, 0, 1.f, back};
      if ((rc = product(n, H, term, r))) return rc;
    }
  }
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}
