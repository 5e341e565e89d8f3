// The edge between two blocks of a decoder layer in one pass each way: the norm
// after a block, its gate, the residual sum and the norm before the next block.
//
//   h = x                              or  x i1 (o + w1),  i1 = rsqrt(mean x^2 + eps)
//   r = residual + scale g h           g: 1, one value a channel, a row or an element
//   y = r i2 (o + w2),                 i2 = rsqrt(mean r^2 + eps)
//
// and, given dy and dr (the gradients of y and r), with a = dr + i2 dy (o + w2)
// and c = i2^3 / D * sum dy (o + w2) r:
//
//   d  = a - c r                        gradient of the residual
//   dh = scale g d;  dg = scale h d     (summed over what g was spread over)
//   dx = i1 dh (o + w1) - x i1^3 / D * sum dh (o + w1) x     (dh without w1)
//   dw2 = sum over rows of dy r i2;  dw1 = sum over rows of dh x i1
//
// All sums over a row that the backward needs come out of one reduction: the
// sum in dx splits into sum scale g (o + w1) x a  -  c sum scale g (o + w1) x r,
// and both terms are known before c is.  r is recomputed from x and residual,
// so no rounding of the stored r enters the gradients; i1 and i2 are kept from
// the forward (8 bytes a row).
//
// A row lies in the registers of `tpr` threads, E elements each; a block of
// 256 threads or one row takes whole rows and goes on to further ones, so the
// weights, and in the backward the column sums of dw, are kept in registers.
// The columns' sums leave as one row of partials a block, which a second
// kernel adds up in a fixed order (no atomics).  Everything is fp32, rounded
// once at the store.
#include <algorithm>

#include "tt_sm100.cuh"
#include "tt_vec.cuh"

namespace tt {
namespace resnorm {
namespace {

enum Gate { kNone = 0, kChannel = 1, kRow = 2, kFull = 3 };

struct Args {
  int64_t rows;
  int D, tpr;               // threads a row
  const void *x, *res, *gate, *w2, *w1;
  int64_t x_st, res_st, gate_st;
  int gate_mode, w_f32;
  float scale, offset, eps;
  void *y, *r;
  float* stats;             // [rows][2] i1, i2
  const void *dy, *dr;
  int64_t dy_st, dr_st;
  void *dx, *dres, *dgate;
  float* part;              // [3][blocks][D]: dw2, dw1, dgate of the channels
};

// How a row lies in the threads: packs of 8 elements (rows aligned), pairs (pairs
// aligned), packs of 8 with 16-byte words shifted into place (any element, whole
// warps a row), or single elements.  Shifting takes more instructions than pairs:
// 26,298 x 1,534 gated, forward and backward, 827 us against 430; by elements,
// 8,000 x 4,095 takes 782 us against 510.
constexpr int kAligned = 8, kPairs = 2, kShifted = 0, kSingle = 1;

// Column of element e of thread t of a row.
template <int K>
__device__ __forceinline__ int column(int e, int t, int tpr) {
  constexpr int P = K == kShifted ? 8 : K;
  return (e / P * tpr + t) * P + e % P;
}

template <typename T, int K, int E>
struct Row {
  // raw words as loaded, so that a row can be fetched ahead at its own width
  // elements of a load
  static constexpr int L = K == kSingle || K == kPairs ? K : 16 / (int)sizeof(T);
  vec::Raw<T, L> raw[E / L];

  // Row `row` of `rows`, `st` apart.
  __device__ __forceinline__ void fetch(const T* base, int64_t st, int64_t row, int64_t rows,
                                        int t, int tpr, int D, bool live) {
#pragma unroll
    for (int i = 0; i < E / L; ++i) {
      const int c = column<K>(i * L, t, tpr);
      raw[i] = vec::Raw<T, L>{};
      if (!live || c >= D) continue;
      if constexpr (K == kShifted)
        raw[i] = vec::load_any_of<T>(base + row * st, c, D, base, base + (rows - 1) * st + D);
      else
        raw[i] = vec::load_raw<T, L>(base + row * st + c);
    }
  }

  __device__ __forceinline__ void get(float (&v)[E]) const {
#pragma unroll
    for (int i = 0; i < E / L; ++i) {
      float o[L];
      vec::unpack<T, L>(raw[i], o);
#pragma unroll
      for (int j = 0; j < L; ++j) v[i * L + j] = o[j];
    }
  }
};

// Stores a row.  Shifted: a thread joins the end of the pack before its own to the
// start of its own, which is a whole 16-byte word of memory; what has no neighbour
// in the warp is stored by elements.  All lanes of a warp come here together.
template <typename T, int K, int E>
__device__ __forceinline__ void put(T* row, int t, int tpr, int D, const float (&v)[E]) {
  constexpr int L = Row<T, K, E>::L;
  if constexpr (K != kShifted) {
#pragma unroll
    for (int i = 0; i < E / L; ++i) {
      const int c = column<K>(i * L, t, tpr);
      if (c < D) {
        float o[L];
#pragma unroll
        for (int j = 0; j < L; ++j) o[j] = v[i * L + j];
        vec::store<T, L>(row + c, o);
      }
    }
  } else {
    constexpr int U = 8 / L;                  // words of a pack
    const int b = (int)(reinterpret_cast<uintptr_t>(row) & 15), bs = b / (int)sizeof(T);
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int q = 0; q < E / 8; ++q) {
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float o[L];
#pragma unroll
        for (int j = 0; j < L; ++j) o[j] = v[q * 8 + u * L + j];
        w[u] = vec::pack<T, L>(o);
      }
      const int c0 = column<K>(q * 8, t, tpr);
      const uint4 z = w[U - 1];
      const uint4 up = make_uint4(
          __shfl_up_sync(0xffffffffu, z.x, 1), __shfl_up_sync(0xffffffffu, z.y, 1),
          __shfl_up_sync(0xffffffffu, z.z, 1), __shfl_up_sync(0xffffffffu, z.w, 1));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * L;
        const int n = min(max(D - c, 0), L), n_next = min(max(D - c - L, 0), L);
        const bool joint = (u > 0 || lane > 0) && n >= L - bs;
        const bool next_joint = (u + 1 < U || lane < 31) && n_next >= L - bs;
        if (b == 0) {
          vec::store_part<T>(row, c, D, w[u]);
          continue;
        }
        if (joint)
          *reinterpret_cast<uint4*>(row + c - bs) = vec::window(u > 0 ? w[u - 1] : up, w[u], 16 - b);
#pragma unroll
        for (int i = 0; i < L; ++i) {
          const bool mine = i < L - bs ? !joint : !next_joint;
          if (mine && i < n) row[c + i] = from_f32<T>(v[q * 8 + u * L + i]);
        }
      }
    }
  }
}

template <typename T, int K, int E>
__device__ __forceinline__ void weights(const void* w, int f32, float offset, int t, int tpr,
                                        int D, float (&v)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = column<K>(e, t, tpr);
    v[e] = c >= D ? 0.f
                  : offset + (f32 ? reinterpret_cast<const float*>(w)[c]
                                  : to_f32(reinterpret_cast<const T*>(w)[c]));
  }
}

// Sums of N values over the tpr threads of a row, the same in all of them.
// tpr is a power of two up to 32, or a multiple of 32 (then `red`, N floats a
// warp, is used; the caller alternates between two such areas, so that one
// barrier a call is enough).
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int tpr, float* red) {
  const int width = tpr < 32 ? tpr : 32;
  for (int o = width >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if (tpr <= 32) return;
  const int warp = threadIdx.x >> 5, nw = tpr >> 5;
  const int first = warp / nw * nw;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[warp * N + i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (int q = 0; q < nw; ++q) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += red[(first + q) * N + i];
  }
}

constexpr int kMaxWarps = 32;

template <typename T, typename R, int K, int E, int kMaxThreads, bool kFullForm>
__global__ void __launch_bounds__(kMaxThreads) fwd_kernel(const Args a) {
  __shared__ float red[2][kMaxWarps];
  const int t = threadIdx.x % a.tpr, slot = threadIdx.x / a.tpr;
  const int per = blockDim.x / a.tpr;
  const int D = a.D, tpr = a.tpr;
  const bool post = kFullForm && a.w1 != nullptr;
  const int mode = kFullForm ? a.gate_mode : kNone;
  float w2[E], w1[E], gc[E];
  weights<T, K, E>(a.w2, a.w_f32, a.offset, t, tpr, D, w2);
  if (post) weights<T, K, E>(a.w1, a.w_f32, a.offset, t, tpr, D, w1);
  if (mode == kChannel) weights<T, K, E>(a.gate, 0, 0.f, t, tpr, D, gc);
  int turn = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * per; row0 < a.rows; row0 += (int64_t)gridDim.x * per) {
    const int64_t row = row0 + slot;
    const bool live = row < a.rows;
    Row<T, K, E> rx;
    Row<R, K, E> rr;
    Row<T, K, E> rg;
    rx.fetch(reinterpret_cast<const T*>(a.x), a.x_st, row, a.rows, t, tpr, D, live);
    rr.fetch(reinterpret_cast<const R*>(a.res), a.res_st, row, a.rows, t, tpr, D, live && a.res);
    if (mode == kFull)
      rg.fetch(reinterpret_cast<const T*>(a.gate), a.gate_st, row, a.rows, t, tpr, D, live);
    float h[E], r[E];
    rx.get(h);
    rr.get(r);
    float i1 = 1.f;
    if (post) {
      float s[1] = {0.f};
#pragma unroll
      for (int e = 0; e < E; ++e) s[0] = fmaf(h[e], h[e], s[0]);
      row_sum<1>(s, tpr, red[turn]);
      turn ^= 1;
      i1 = rsqrtf(s[0] / D + a.eps);
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] *= i1 * w1[e];
    }
    float k = a.scale;
    if (mode == kRow && live)
      k *= to_f32(reinterpret_cast<const T*>(a.gate)[row * a.gate_st]);
    if (mode == kChannel) {
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] *= gc[e];
    } else if (mode == kFull) {
      float g[E];
      rg.get(g);
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] *= g[e];
    }
    float s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      r[e] = fmaf(k, h[e], r[e]);
      s[0] = fmaf(r[e], r[e], s[0]);
    }
    row_sum<1>(s, tpr, red[turn]);
    turn ^= 1;
    const float i2 = rsqrtf(s[0] / D + a.eps);
    if (live) {
      put<R, K, E>(reinterpret_cast<R*>(a.r) + row * D, t, tpr, D, r);
#pragma unroll
      for (int e = 0; e < E; ++e) r[e] *= i2 * w2[e];
      put<T, K, E>(reinterpret_cast<T*>(a.y) + row * D, t, tpr, D, r);
      if (t == 0 && a.stats) {
        a.stats[2 * row] = i1;
        a.stats[2 * row + 1] = i2;
      }
    }
  }
}

template <typename T, typename R, int K, int E, int kMaxThreads, bool kFullForm>
__global__ void __launch_bounds__(kMaxThreads) bwd_kernel(const Args a) {
  constexpr int N = kFullForm ? 3 : 1;
  __shared__ float red[2][kMaxWarps * N];
  extern __shared__ float cols[];           // [rows a block][D], where that is over one
  const int t = threadIdx.x % a.tpr, slot = threadIdx.x / a.tpr;
  const int per = blockDim.x / a.tpr;
  const int D = a.D, tpr = a.tpr;
  const bool post = kFullForm && a.w1 != nullptr;
  const int mode = kFullForm ? a.gate_mode : kNone;
  float w2[E], w1[E], gc[E], dw2[E], dw1[E], dgc[E];
  weights<T, K, E>(a.w2, a.w_f32, a.offset, t, tpr, D, w2);
  if (kFullForm) {
#pragma unroll
    for (int e = 0; e < E; ++e) w1[e] = gc[e] = 1.f;
    if (post) weights<T, K, E>(a.w1, a.w_f32, a.offset, t, tpr, D, w1);
    if (mode == kChannel) weights<T, K, E>(a.gate, 0, 0.f, t, tpr, D, gc);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) dw2[e] = dw1[e] = dgc[e] = 0.f;
  int turn = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * per; row0 < a.rows; row0 += (int64_t)gridDim.x * per) {
    const int64_t row = row0 + slot;
    const bool live = row < a.rows;
    Row<T, K, E> rx, ry, rg;
    Row<R, K, E> rr, rd;
    rx.fetch(reinterpret_cast<const T*>(a.x), a.x_st, row, a.rows, t, tpr, D, live);
    rr.fetch(reinterpret_cast<const R*>(a.res), a.res_st, row, a.rows, t, tpr, D, live && a.res);
    ry.fetch(reinterpret_cast<const T*>(a.dy), a.dy_st, row, a.rows, t, tpr, D, live && a.dy);
    rd.fetch(reinterpret_cast<const R*>(a.dr), a.dr_st, row, a.rows, t, tpr, D, live && a.dr);
    if (mode == kFull)
      rg.fetch(reinterpret_cast<const T*>(a.gate), a.gate_st, row, a.rows, t, tpr, D, live);
    // a block's rows past the last hold zeros: they add nothing to any sum
    const float i1 = live ? a.stats[2 * row] : 0.f, i2 = live ? a.stats[2 * row + 1] : 0.f;
    float k = a.scale;
    if (mode == kRow) k *= live ? to_f32(reinterpret_cast<const T*>(a.gate)[row * a.gate_st]) : 0.f;
    float x[E], u[E], r[E], d[E], dy[E];
    rx.get(x);
    rr.get(r);
    ry.get(dy);
    rd.get(d);
    if (mode == kFull) rg.get(u);
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (kFullForm) {
        u[e] = mode == kFull ? u[e] : gc[e];     // the gate without a row's own
        r[e] = fmaf(k * i1 * u[e] * w1[e], x[e], r[e]);
      } else {
        r[e] = fmaf(k, x[e], r[e]);
      }
      const float gy = dy[e] * w2[e];
      dw2[e] = fmaf(dy[e] * i2, r[e], dw2[e]);
      d[e] = fmaf(i2, gy, d[e]);                 // a
      s[0] = fmaf(gy, r[e], s[0]);
      if constexpr (kFullForm) {
        const float ux = u[e] * w1[e] * x[e];
        s[1] = fmaf(ux, d[e], s[1]);
        s[2] = fmaf(ux, r[e], s[2]);
      }
    }
    row_sum<N>(s, tpr, red[turn]);
    turn ^= 1;
    const float c = i2 * i2 * i2 * s[0] / D;
#pragma unroll
    for (int e = 0; e < E; ++e) d[e] = fmaf(-c, r[e], d[e]);
    if (live && a.dres) put<R, K, E>(reinterpret_cast<R*>(a.dres) + row * D, t, tpr, D, d);
    if constexpr (!kFullForm) {
      if (live && a.dx) {
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] *= k;
        put<T, K, E>(reinterpret_cast<T*>(a.dx) + row * D, t, tpr, D, d);
      }
    } else {
      const float dot = s[1] - c * s[2];         // sum of u w1 x d
      const float back = post ? k * i1 * i1 * i1 * dot / D : 0.f;
      if (mode == kRow && live && t == 0 && a.dgate)
        reinterpret_cast<T*>(a.dgate)[row] = from_f32<T>(a.scale * i1 * dot);
      float dx[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float xd = i1 * x[e] * d[e];
        const float dh = k * u[e] * d[e];        // gradient of h
        dw1[e] = fmaf(k * u[e], xd, dw1[e]);
        dgc[e] += xd;                            // times scale (o + w1) at the end
        dx[e] = fmaf(-back, x[e], i1 * dh * w1[e]);
        d[e] = a.scale * w1[e] * xd;             // gradient of the element's gate
      }
      if (live && a.dx) put<T, K, E>(reinterpret_cast<T*>(a.dx) + row * D, t, tpr, D, dx);
      if (mode == kFull && live && a.dgate)
        put<T, K, E>(reinterpret_cast<T*>(a.dgate) + row * D, t, tpr, D, d);
    }
  }
  // the block's column sums: its rows' slots added in order
  float* part = a.part + (int64_t)blockIdx.x * D;
  const int64_t plane = (int64_t)gridDim.x * D;
  auto leave = [&](const float (&v)[E], float* out) {
    if (per == 1) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = column<K>(e, t, tpr);
        if (c < D) out[c] = v[e];
      }
      return;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = column<K>(e, t, tpr);
      if (c < D) cols[slot * D + c] = v[e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      float sum = 0.f;
      for (int q = 0; q < per; ++q) sum += cols[q * D + c];
      out[c] = sum;
    }
  };
  leave(dw2, part);
  if constexpr (kFullForm) {
    if (post) leave(dw1, part + plane);
    if (mode == kChannel) {
#pragma unroll
      for (int e = 0; e < E; ++e) dgc[e] *= a.scale * w1[e];
      leave(dgc, part + 2 * plane);
    }
  }
}

// ---- rows through shared memory ---------------------------------------------
//
// The same for aligned rows of 520 to 8,192 elements (one a block, weights of x's
// type): thread 0
// keeps a ring of `stages` rows filled by bulk copies, so that the next rows
// arrive while this one is reduced and stored, and raw 16-bit packs instead of
// fp32 values are what stays in registers across the reduction.  A stage is
// filled again only behind a barrier that every thread reaches after it has used
// what it read.  A wait that gives up records its error and lets the block run
// on over what is in the ring, so all threads keep meeting at the same barriers.
//
// Bound by HBM.  Measured on a B200 (straight to registers; at the rate of a copy):
// 16,384 x 2,560 bf16, residual sum and norm: forward 53 us (71; 52), backward 72
// (89; 65).  8,191 x 4,096, both norms, element gate, fp32 stream: forward 85 (117;
// 73), backward 122 (191; 112).

struct Ring {
  int stages, stage_bytes;
  int32_t* status;
};

constexpr int kMaxStages = 8;

// After a wait that gave up: the copies in flight land (stage i took the issues
// i, i + S, ... of `issued`) before the block ends.
__device__ __forceinline__ void land(uint64_t* full, int S, int64_t issued) {
  for (int i = 0; i < S; ++i)
    if (issued > i) sm100::mbar_wait(&full[i], (uint32_t)((issued - 1 - i) / S) & 1, nullptr);
}

// Sums over the block's warps; red: [N][32] floats.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[i * 32 + (threadIdx.x >> 5)] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane < nw ? red[i * 32 + lane] : 0.f;
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
}

// Eight elements of a row as they lie in shared memory.
template <typename T>
struct Raw8 {
  static constexpr int P = (int)sizeof(T) / 2;
  uint4 r[P];
  __device__ __forceinline__ void read(const uint8_t* row, int t) {
#pragma unroll
    for (int p = 0; p < P; ++p) r[p] = reinterpret_cast<const uint4*>(row)[t * P + p];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int p = 0; p < P; ++p) r[p] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    constexpr int W = 16 / (int)sizeof(T);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float o[W];
      vec::unpack<T, W>(r[p], o);
#pragma unroll
      for (int j = 0; j < W; ++j) v[p * W + j] = o[j];
    }
  }
};

template <typename T>
__device__ __forceinline__ void put8(T* row, int t, const float (&v)[8]) {
  constexpr int W = 16 / (int)sizeof(T);
#pragma unroll
  for (int p = 0; p < 8 / W; ++p) {
    float o[W];
#pragma unroll
    for (int j = 0; j < W; ++j) o[j] = v[p * W + j];
    vec::store<T, W>(row + t * 8 + p * W, o);
  }
}

template <typename T, typename R, bool kFullForm, bool kByChannel>
__global__ void __launch_bounds__(1024, 1) ring_fwd(const Args a, const Ring ring) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red[2][32];
  __shared__ uint64_t full[kMaxStages];
  __shared__ int32_t abort_flag;
  const int D = a.D, t = threadIdx.x, S = ring.stages;
  const bool in = t * 8 < D;
  const bool post = kFullForm && a.w1, gated = kFullForm && a.gate_mode == kFull;
  const bool by_row = kFullForm && a.gate_mode == kRow;
  const int x_bytes = D * (int)sizeof(T), r_bytes = a.res ? D * (int)sizeof(R) : 0;
  const float inv_D = 1.f / D;
  if (t == 0) {
    for (int i = 0; i < S; ++i) sm100::mbar_init(&full[i], 1);
    abort_flag = 0;
    sm100::fence_mbar_init();
  }
  __syncthreads();
  int64_t issued = 0;
  auto issue = [&](int64_t row, int stage) {
    if (row >= a.rows || *(volatile int32_t*)&abort_flag) return;
    ++issued;
    uint8_t* to = smem + stage * ring.stage_bytes;
    sm100::mbar_arrive_expect_tx(&full[stage], ring.stage_bytes);
    sm100::bulk_load(to, reinterpret_cast<const T*>(a.x) + row * a.x_st, x_bytes, &full[stage]);
    if (a.res)
      sm100::bulk_load(to + x_bytes, reinterpret_cast<const R*>(a.res) + row * a.res_st, r_bytes,
                       &full[stage]);
    if (gated)
      sm100::bulk_load(to + x_bytes + r_bytes,
                       reinterpret_cast<const T*>(a.gate) + row * a.gate_st, x_bytes,
                       &full[stage]);
  };
  if (t == 0)
    for (int i = 0; i < S; ++i) issue(blockIdx.x + (int64_t)i * gridDim.x, i);
  Raw8<T> w2, w1, wg;
  w2.zero(), w1.zero(), wg.zero();
  if (in) {
    w2.read(reinterpret_cast<const uint8_t*>(a.w2), t);
    if (post) w1.read(reinterpret_cast<const uint8_t*>(a.w1), t);
    if (kByChannel) wg.read(reinterpret_cast<const uint8_t*>(a.gate), t);
  }
  int stage = 0;
  uint32_t phase = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (!sm100::mbar_wait(&full[stage], phase, &abort_flag)) {
      set_status(ring.status, TT_ERR_DEVICE_TIMEOUT);
      *(volatile int32_t*)&abort_flag = 1;
    }
    const uint8_t* at = smem + stage * ring.stage_bytes;
    Raw8<T> raw;
    float h[8], r[8], g[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = r[e] = g[e] = 0.f;
    if (in) {
      raw.read(at, t);
      raw.get(h);
      if (a.res) {
        Raw8<R> rr;
        rr.read(at + x_bytes, t);
        rr.get(r);
      }
      if (gated) {
        raw.read(at + x_bytes + r_bytes, t);
        raw.get(g);
      }
    }
    float k = a.scale, i1 = 1.f;
    if (by_row) k *= to_f32(reinterpret_cast<const T*>(a.gate)[row * a.gate_st]);
    if (post) {
      float s[1] = {0.f}, w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0] = fmaf(h[e], h[e], s[0]);
      block_sum<1>(s, red[0]);
      i1 = rsqrtf(fmaf(s[0], inv_D, a.eps));
      w1.get(w);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] *= i1 * (a.offset + w[e]);
    }
    if (kByChannel) wg.get(g);
    float s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (gated || kByChannel) h[e] *= g[e];
      r[e] = fmaf(k, h[e], r[e]);
      s[0] = fmaf(r[e], r[e], s[0]);
    }
    block_sum<1>(s, red[1]);
    if (t == 0) issue(row + (int64_t)S * gridDim.x, stage);
    if (++stage == S) stage = 0, phase ^= 1;
    const float i2 = rsqrtf(fmaf(s[0], inv_D, a.eps));
    if (in) {
      put8<R>(reinterpret_cast<R*>(a.r) + row * D, t, r);
      float w[8];
      w2.get(w);
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] *= i2 * (a.offset + w[e]);
      put8<T>(reinterpret_cast<T*>(a.y) + row * D, t, r);
    }
    if (t == 0 && a.stats) reinterpret_cast<float2*>(a.stats)[row] = make_float2(i1, i2);
    // without the first sum, a barrier before the second area is written again
    if (!post) __syncthreads();
  }
  if (t == 0 && *(volatile int32_t*)&abort_flag) land(full, S, issued);
}

// Q: packs of 8 elements a thread, a block's threads apart. kShared: the weights'
// sums lie behind the stages, each read and written by its own thread alone.
template <typename T, typename R, bool kFullForm, int kThreads, bool kByChannel, int Q,
          bool kShared>
__global__ void __launch_bounds__(kThreads, 1) ring_bwd(const Args a, const Ring ring) {
  constexpr int N = kFullForm ? 3 : 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red[2][N * 32];
  __shared__ uint64_t full[kMaxStages];
  __shared__ int32_t abort_flag;
  const int D = a.D, t = threadIdx.x, S = ring.stages;
  auto index = [&](int q) { return q * (int)blockDim.x + t; };       // of a pack of the row
  auto in = [&](int q) { return index(q) * 8 < D; };
  const bool post = kFullForm && a.w1, gated = kFullForm && a.gate_mode == kFull;
  const bool by_row = kFullForm && a.gate_mode == kRow;
  const int x_bytes = D * (int)sizeof(T), r_bytes = D * (int)sizeof(R);
  const int at_dy = x_bytes, at_g = at_dy + (a.dy ? x_bytes : 0);
  const int at_r = at_g + (gated ? x_bytes : 0), at_dr = at_r + (a.res ? r_bytes : 0);
  const float inv_D = 1.f / D;
  if (t == 0) {
    for (int i = 0; i < S; ++i) sm100::mbar_init(&full[i], 1);
    abort_flag = 0;
    sm100::fence_mbar_init();
  }
  __syncthreads();
  int64_t issued = 0;
  auto issue = [&](int64_t row, int stage) {
    if (row >= a.rows || *(volatile int32_t*)&abort_flag) return;
    ++issued;
    uint8_t* to = smem + stage * ring.stage_bytes;
    uint64_t* bar = &full[stage];
    sm100::mbar_arrive_expect_tx(bar, ring.stage_bytes);
    sm100::bulk_load(to, reinterpret_cast<const T*>(a.x) + row * a.x_st, x_bytes, bar);
    if (a.dy)
      sm100::bulk_load(to + at_dy, reinterpret_cast<const T*>(a.dy) + row * a.dy_st, x_bytes, bar);
    if (gated)
      sm100::bulk_load(to + at_g, reinterpret_cast<const T*>(a.gate) + row * a.gate_st, x_bytes,
                       bar);
    if (a.res)
      sm100::bulk_load(to + at_r, reinterpret_cast<const R*>(a.res) + row * a.res_st, r_bytes,
                       bar);
    if (a.dr)
      sm100::bulk_load(to + at_dr, reinterpret_cast<const R*>(a.dr) + row * a.dr_st, r_bytes, bar);
  };
  if (t == 0)
    for (int i = 0; i < S; ++i) issue(blockIdx.x + (int64_t)i * gridDim.x, i);
  Raw8<T> rw2[Q], rw1[Q], rwg[Q];
  // the weights' sums over the block's rows, in registers or behind the stages
  constexpr int kHeld = kShared ? 1 : Q;
  float dw2[kHeld][8], dw1[kHeld][8], dgc[kHeld][8];
  float4* sums = reinterpret_cast<float4*>(smem + S * ring.stage_bytes);
  auto at_sum = [&](int plane, int q, int half) {
    return sums + ((plane * Q + q) * 2 + half) * (int)blockDim.x + t;
  };
  auto held = [&](float (&v)[kHeld][8], int plane, int q) -> float (&)[8] {
    if constexpr (kShared) {
      const float4 lo = *at_sum(plane, q, 0), hi = *at_sum(plane, q, 1);
      v[0][0] = lo.x, v[0][1] = lo.y, v[0][2] = lo.z, v[0][3] = lo.w;
      v[0][4] = hi.x, v[0][5] = hi.y, v[0][6] = hi.z, v[0][7] = hi.w;
    }
    return v[kShared ? 0 : q];
  };
  auto keep = [&](float (&v)[8], int plane, int q) {
    if constexpr (kShared) {
      *at_sum(plane, q, 0) = make_float4(v[0], v[1], v[2], v[3]);
      *at_sum(plane, q, 1) = make_float4(v[4], v[5], v[6], v[7]);
    }
  };
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    rw2[q].zero(), rw1[q].zero(), rwg[q].zero();
    if (in(q)) {
      rw2[q].read(reinterpret_cast<const uint8_t*>(a.w2), index(q));
      if (post) rw1[q].read(reinterpret_cast<const uint8_t*>(a.w1), index(q));
      if (kByChannel) rwg[q].read(reinterpret_cast<const uint8_t*>(a.gate), index(q));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      dw2[kShared ? 0 : q][e] = dw1[kShared ? 0 : q][e] = dgc[kShared ? 0 : q][e] = 0.f;
    keep(dw2[kShared ? 0 : q], 0, q);
    if (post) keep(dw1[kShared ? 0 : q], 1, q);
    if (kByChannel) keep(dgc[kShared ? 0 : q], 2, q);
  }
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  // a row's own values are fetched a row ahead
  float2 next = make_float2(0.f, 0.f);
  float next_g = 1.f;
  auto fetch = [&](int64_t row) {
    if (row >= a.rows) return;
    next = reinterpret_cast<const float2*>(a.stats)[row];
    if (by_row) next_g = to_f32(reinterpret_cast<const T*>(a.gate)[row * a.gate_st]);
  };
  fetch(blockIdx.x);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float i1 = next.x, i2 = next.y, k = a.scale * next_g;
    fetch(row + gridDim.x);
    if (!sm100::mbar_wait(&full[stage], phase, &abort_flag)) {
      set_status(ring.status, TT_ERR_DEVICE_TIMEOUT);
      *(volatile int32_t*)&abort_flag = 1;
    }
    const uint8_t* at = smem + stage * ring.stage_bytes;
    Raw8<T> rx[Q], rg[Q];
    float r[Q][8], d[Q][8], s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0.f;
    const float ki = kFullForm ? k * i1 : k;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      rx[q].zero(), rg[q].zero();
#pragma unroll
      for (int e = 0; e < 8; ++e) r[q][e] = d[q][e] = 0.f;
      if (!in(q)) continue;
      rx[q].read(at, index(q));
      if (gated) rg[q].read(at + at_g, index(q));
      if (a.res) {
        Raw8<R> raw;
        raw.read(at + at_r, index(q));
        raw.get(r[q]);
      }
      if (a.dr) {
        Raw8<R> raw;
        raw.read(at + at_dr, index(q));
        raw.get(d[q]);
      }
      float x[8], u[8], w[8], dy[8];
      Raw8<T> ry;
      if (a.dy)
        ry.read(at + at_dy, index(q));
      else
        ry.zero();
      ry.get(dy);
      rx[q].get(x);
      if (kFullForm) {
        // u x: the block's output without scale, row gate and i1
        if (post) {
          rw1[q].get(u);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= a.offset + u[e];
        }
        if (gated || kByChannel) {
          (kByChannel ? rwg[q] : rg[q]).get(u);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= u[e];
        }
      }
      rw2[q].get(w);
      float (&sum2)[8] = held(dw2, 0, q);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        r[q][e] = fmaf(ki, x[e], r[q][e]);
        const float gy = dy[e] * (a.offset + w[e]);
        sum2[e] = fmaf(dy[e] * i2, r[q][e], sum2[e]);
        d[q][e] = fmaf(i2, gy, d[q][e]);               // a
        s[0] = fmaf(gy, r[q][e], s[0]);
        if constexpr (kFullForm) {
          s[1] = fmaf(x[e], d[q][e], s[1]);
          s[2] = fmaf(x[e], r[q][e], s[2]);
        }
      }
      keep(sum2, 0, q);
    }
    block_sum<N>(s, red[turn]);
    turn ^= 1;
    if (t == 0) issue(row + (int64_t)S * gridDim.x, stage);
    if (++stage == S) stage = 0, phase ^= 1;
    const float c = i2 * i2 * i2 * s[0] * inv_D;
    float dot = 0.f, back = 0.f;
    if constexpr (kFullForm) {
      dot = s[1] - c * s[2];                     // sum of u x d
      back = post ? k * i1 * i1 * i1 * dot * inv_D : 0.f;
      if (by_row && t == 0 && a.dgate)
        reinterpret_cast<T*>(a.dgate)[row] = from_f32<T>(a.scale * i1 * dot);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (!in(q)) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) d[q][e] = fmaf(-c, r[q][e], d[q][e]);
      if (a.dres) put8<R>(reinterpret_cast<R*>(a.dres) + row * D, index(q), d[q]);
      if constexpr (!kFullForm) {
        if (a.dx) {
#pragma unroll
          for (int e = 0; e < 8; ++e) d[q][e] *= k;
          put8<T>(reinterpret_cast<T*>(a.dx) + row * D, index(q), d[q]);
        }
      } else {
        float x[8], w[8], g[8];
        rx[q].get(x);
        if (post) {
          rw1[q].get(w);
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] += a.offset;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = 1.f;
        }
        if (gated || kByChannel) {
          (kByChannel ? rwg[q] : rg[q]).get(g);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = 1.f;
        }
        float (&sum1)[8] = held(dw1, post ? 1 : 0, q);
        float (&sumg)[8] = held(dgc, kByChannel ? 2 : 0, q);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float xd = i1 * x[e] * d[q][e], kg = k * g[e];
          if (post) sum1[e] = fmaf(kg, xd, sum1[e]);
          if (kByChannel) sumg[e] = fmaf(a.scale * w[e], xd, sumg[e]);
          r[q][e] = fmaf(-back, x[e], i1 * (kg * d[q][e]) * w[e]);     // dx
          d[q][e] = a.scale * w[e] * xd;                               // the element's gate
        }
        if (post) keep(sum1, 1, q);
        if (kByChannel) keep(sumg, 2, q);
        if (a.dx) put8<T>(reinterpret_cast<T*>(a.dx) + row * D, index(q), r[q]);
        if (gated && a.dgate) put8<T>(reinterpret_cast<T*>(a.dgate) + row * D, index(q), d[q]);
      }
    }
  }
  if (t == 0 && *(volatile int32_t*)&abort_flag) land(full, S, issued);
  const int64_t plane = (int64_t)gridDim.x * D;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    if (!in(q)) continue;
    float* part = a.part + (int64_t)blockIdx.x * D + index(q) * 8;
    float (&sum2)[8] = held(dw2, 0, q);
    float (&sum1)[8] = held(dw1, post ? 1 : 0, q);
    float (&sumg)[8] = held(dgc, kByChannel ? 2 : 0, q);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      part[e] = sum2[e];
      if (post) part[plane + e] = sum1[e];
      if (kByChannel) part[2 * plane + e] = sumg[e];
    }
  }
}

// out[c] = sum over the blocks' partials, in a fixed order: 32 threads a
// column, each over every 32nd block, four loads in flight.
constexpr int kSumRows = 32;

struct Out {
  void* p[3];
  int dtype[3];
};

__global__ void __launch_bounds__(32 * kSumRows)
sum_partials(int blocks, int D, const float* __restrict__ part, const Out out) {
  if (!out.p[blockIdx.y]) return;
  __shared__ float red[kSumRows][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  const float* src = part + (int64_t)blockIdx.y * blocks * D;
  float s = 0.f;
  if (c < D) {
    for (int b = threadIdx.y; b < blocks; b += 4 * kSumRows) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = b + j * kSumRows < blocks ? src[(int64_t)(b + j * kSumRows) * D + c] : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) s += v[j];
    }
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < D) {
    s = 0.f;
    for (int q = 0; q < kSumRows; ++q) s += red[q][threadIdx.x];
    void* p = out.p[blockIdx.y];
    switch (out.dtype[blockIdx.y]) {
      case TT_F32: reinterpret_cast<float*>(p)[c] = s; break;
      case TT_BF16: reinterpret_cast<__nv_bfloat16*>(p)[c] = from_f32<__nv_bfloat16>(s); break;
      default: reinterpret_cast<__half*>(p)[c] = from_f32<__half>(s); break;
    }
  }
}

// Threads of a row and rows of a block for D columns, E elements a thread.
struct Shape {
  int E, tpr, per;
};

constexpr int kMaxD = 16384;

Shape shape_of(int D) {
  Shape s;
  s.E = D <= 4096 ? 8 : 16;
  const int need = (D + s.E - 1) / s.E;
  if (need <= 32) {
    s.tpr = 1;
    while (s.tpr < need) s.tpr *= 2;
  } else {
    s.tpr = (need + 31) / 32 * 32;
  }
  s.per = std::max(1, 256 / s.tpr);
  return s;
}

// Rows of elements of `size` bytes can be read in packs of `pack`.
bool aligned(const void* p, int64_t stride, int size, int pack) {
  return reinterpret_cast<uintptr_t>(p) % std::min(16, pack * size) == 0 && stride % pack == 0;
}

template <typename T, typename R, bool kBwd>
int launch(const Args& a, int pack, bool full, Shape s, int blocks, cudaStream_t st) {
  const int threads = s.tpr * s.per;
  const size_t smem = kBwd && s.per > 1 ? sizeof(float) * s.per * a.D : 0;
  auto go = [&](auto v, auto e, auto m, auto f) {
    constexpr bool F = decltype(f)::value;
    constexpr int V = decltype(v)::value, E = decltype(e)::value, M = decltype(m)::value;
    if constexpr (kBwd)
      bwd_kernel<T, R, V, E, M, F><<<blocks, threads, smem, st>>>(a);
    else
      fwd_kernel<T, R, V, E, M, F><<<blocks, threads, smem, st>>>(a);
  };
  using Y = std::true_type;
  using N = std::false_type;
  std::integral_constant<int, 8> e8;
  std::integral_constant<int, 16> e16;
  std::integral_constant<int, 512> m512;
  std::integral_constant<int, 1024> m1024;
  std::integral_constant<int, kSingle> k1;
  std::integral_constant<int, kPairs> k2;
  std::integral_constant<int, kShifted> k0;
  std::integral_constant<int, kAligned> k8;
  if (pack == kSingle) {
    s.E == 8 ? go(k1, e8, m512, Y()) : go(k1, e16, m1024, Y());
  } else if (pack == kPairs) {
    s.E == 8 ? go(k2, e8, m512, Y()) : go(k2, e16, m1024, Y());
  } else if (pack == kShifted) {
    s.E == 8 ? go(k0, e8, m512, Y()) : go(k0, e16, m1024, Y());
  } else if (s.E == 8) {
    full ? go(k8, e8, m512, Y()) : go(k8, e8, m512, N());
  } else if (threads <= 512) {
    full ? go(k8, e16, m512, Y()) : go(k8, e16, m512, N());
  } else {
    full ? go(k8, e16, m1024, Y()) : go(k8, e16, m1024, N());
  }
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

// Threads of a block of the ring: a pack of 8 elements each, or two.
int ring_threads(int D, bool two) {
  const int packs = D / 8;
  return ((two ? (packs + 1) / 2 : packs) + 31) / 32 * 32;
}

// Whether the backward's threads take two packs each. The full form keeps 128
// registers a thread, so 512 threads an SM: above 4,096 one row needs two packs.
// The weights' sums then lie in shared memory behind the stages (in registers
// they spill, past an L1 that the stages leave no room: 8,000 x 5,120 fully
// gated 252 us forward and backward, 339 in registers). Below, 16-bit rows
// gain by it from 1,024 on (20,480 x 2,048 post weight and row gate: 194 us,
// one pack 210; 40,960 x 1,024 fully gated 226, one pack 217), others do not
// (10,240 x 4,096, 32-bit residual: 268, one pack 258; 4,000 x 2,560 in 32 bits
// 159 and 111; a gate by channel, with its third sum, at 10,240 x 4,096 227 and
// 215), unless one pack leaves an SM a single block of 5/8 of its threads or less
// and x is of 16 bits (16,384 x 2,560: gate by channel 228, one pack 253; 32-bit
// residual 259 and 291; at 2,816, 352 threads, 257 and 244 by channel).
bool two_packs(int D, bool full, bool channel, int x_size, int res_size) {
  if (!full) return false;
  const int one = ring_threads(D, false);
  return D > 4096 || (D > 1024 && x_size == 2 && res_size == 2 && !channel) ||
         (x_size == 2 && one > 256 && one <= 320);
}

// The ring's shape: as many blocks an SM as `most` threads allow (1,024 with 64
// registers each, 512 with 128) while each has two stages or more beside its
// sum_bytes; blocks 0: rows go straight to registers. The full form's backward
// spills in 64 registers: 40,960 x 1,024 fully gated 267 us with 1,024 threads.
struct RingShape {
  int blocks, stages, stage_bytes, sum_bytes;
};

constexpr int kSharedPerSM = 228 * 1024, kSharedOwn = 2048;   // kSharedOwn: static, reserved

RingShape ring_of(int64_t rows, int D, int threads, int stage_bytes, int most = 1024,
                  int sum_bytes = 0) {
  RingShape best{0, 0, stage_bytes, sum_bytes};
  for (int per = most / threads; per > 0; --per) {
    const int stages = std::min(kMaxStages, (kSharedPerSM / per - kSharedOwn - sum_bytes) / stage_bytes);
    if (stages >= 2) {
      best.blocks = (int)std::min<int64_t>(rows, (int64_t)vec::kSMs * per);
      best.stages = stages;
      break;
    }
  }
  return best;
}

bool rows_by_ring(int D, int dtype, bool vec, const Args& a) {
  return vec && D > 512 && D <= 8192 && (!a.w_f32 || dtype == TT_F32) &&
         (a.gate_mode != kChannel || reinterpret_cast<uintptr_t>(a.gate) % 16 == 0) &&
         reinterpret_cast<uintptr_t>(a.w2) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(a.w1) % 16 == 0;
}

template <typename T, typename R, bool kBwd>
int launch_ring(const Args& a, bool full, int threads, const RingShape& shape, int32_t* status,
                cudaStream_t st) {
  const Ring ring{shape.stages, shape.stage_bytes, status};
  const int smem = shape.stages * shape.stage_bytes + shape.sum_bytes;
  // (the limit belongs to the kernel, not to the call: it is the same for every
  // size, since another thread may set it between here and the launch)
  auto go = [&](auto kern) -> int {
    TT_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    kSharedPerSM - kSharedOwn));
    kern<<<shape.blocks, threads, smem, st>>>(a, ring);
    return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
  };
  if constexpr (kBwd) {
    if (!full) return go(ring_bwd<T, R, false, 1024, false, 1, false>);
    const bool channel = a.gate_mode == kChannel;
    if (shape.sum_bytes)
      return channel ? go(ring_bwd<T, R, true, 512, true, 2, true>)
                     : go(ring_bwd<T, R, true, 512, false, 2, true>);
    if (threads * 8 < a.D)
      return channel ? go(ring_bwd<T, R, true, 512, true, 2, false>)
                     : go(ring_bwd<T, R, true, 512, false, 2, false>);
    return channel ? go(ring_bwd<T, R, true, 512, true, 1, false>)
                   : go(ring_bwd<T, R, true, 512, false, 1, false>);
  } else {
    if (!full) return go(ring_fwd<T, R, false, false>);
    return a.gate_mode == kChannel ? go(ring_fwd<T, R, true, true>)
                                   : go(ring_fwd<T, R, true, false>);
  }
}

template <bool kBwd>
int dispatch_ring(int dtype, int res_dtype, const Args& a, int threads, const RingShape& shape,
                  int32_t* status, cudaStream_t st) {
  const bool full = a.w1 || a.gate_mode != kNone;
  return vec::dispatch_float(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    if (res_dtype == dtype) return launch_ring<T, T, kBwd>(a, full, threads, shape, status, st);
    if (res_dtype == TT_F32)
      return launch_ring<T, float, kBwd>(a, full, threads, shape, status, st);
    return TT_ERR_UNSUPPORTED;
  });
}

int size_of(int dtype) { return dtype == TT_F32 ? 4 : 2; }

template <bool kBwd>
int dispatch(int dtype, int res_dtype, const Args& a, int pack, Shape s, int blocks,
             cudaStream_t st) {
  const bool full = a.w1 || a.gate_mode != kNone;
  return vec::dispatch_float(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    if (res_dtype == dtype) return launch<T, T, kBwd>(a, pack, full, s, blocks, st);
    if (res_dtype == TT_F32) return launch<T, float, kBwd>(a, pack, full, s, blocks, st);
    return TT_ERR_UNSUPPORTED;
  });
}

bool bad_sizes(int64_t rows, int32_t D, int gate_mode, const void* gate) {
  return rows < 0 || D <= 0 || D > kMaxD || gate_mode < kNone || gate_mode > kFull ||
         (gate_mode != kNone && rows > 0 && !gate);
}

}  // namespace
}  // namespace resnorm
}  // namespace tt

extern "C" int tt_residual_norm_fwd(int dtype, int res_dtype, int64_t rows, int32_t D,
                                    const void* x, int64_t x_st, const void* residual,
                                    int64_t res_st, const void* weight, const void* post_weight,
                                    int weight_f32, float weight_offset, const void* gate,
                                    int64_t gate_st, int gate_mode, float scale, float eps,
                                    void* y, void* r, float* stats, int32_t* status,
                                    void* stream) {
  using namespace tt::resnorm;
  if (bad_sizes(rows, D, gate_mode, gate) || (rows > 0 && (!x || !weight || !y || !r)) ||
      reinterpret_cast<uintptr_t>(stats) % 8)
    return TT_ERR_INVALID_ARG;
  if (rows == 0) return TT_OK;
  Args a{};
  a.rows = rows, a.D = D;
  a.x = x, a.res = residual, a.gate = gate, a.w2 = weight, a.w1 = post_weight;
  a.x_st = x_st, a.res_st = res_st, a.gate_st = gate_st;
  a.gate_mode = gate_mode, a.w_f32 = weight_f32;
  a.scale = scale, a.offset = weight_offset, a.eps = eps;
  a.y = y, a.r = r, a.stats = stats;
  Shape s = shape_of(D);
  a.tpr = s.tpr;
  const int xs = size_of(dtype), rs = size_of(res_dtype);
  auto fits = [&](int k) {
    return D % k == 0 && aligned(x, x_st, xs, k) && aligned(residual, residual ? res_st : 0, rs, k) &&
           aligned(y, D, xs, k) && aligned(r, D, rs, k) &&
           (gate_mode != kFull || aligned(gate, gate_st, xs, k));
  };
  const int pack = fits(8) ? kAligned : fits(2) ? kPairs : s.tpr >= 32 ? kShifted : kSingle;
  const int64_t want = (rows + s.per - 1) / s.per;
  const int blocks = (int)std::min<int64_t>(want, tt::vec::kSMs * 16ll);
  RingShape ring{};
  if (rows_by_ring(D, dtype, pack == kAligned, a))
    ring = ring_of(rows, D, ring_threads(D, false),
                   D * (size_of(dtype) * (gate_mode == kFull ? 2 : 1) +
                        (residual ? size_of(res_dtype) : 0)));
  const int rc = ring.blocks
                     ? dispatch_ring<false>(dtype, res_dtype, a, ring_threads(D, false), ring, status,
                                            (cudaStream_t)stream)
                     : dispatch<false>(dtype, res_dtype, a, pack, s, blocks, (cudaStream_t)stream);
  if (rc == TT_OK) tt_count_launches(1);
  return rc;
}

extern "C" int tt_residual_norm_bwd_blocks(int64_t rows, int32_t D) {
  using namespace tt::resnorm;
  if (rows <= 0 || D <= 0 || D > kMaxD) return 1;
  const Shape s = shape_of(D);
  // (the ring's blocks are of one row; with two packs a thread they are no more)
  const int threads = D > 512 && D <= 8192 ? ring_threads(D, false) : s.tpr * s.per;
  return (int)std::max<int64_t>(
      1, std::min<int64_t>(rows, tt::vec::kSMs * (int64_t)std::max(1, 1024 / threads)));
}

extern "C" int tt_residual_norm_bwd(
    int dtype, int res_dtype, int64_t rows, int32_t D, const void* x, int64_t x_st,
    const void* residual, int64_t res_st, const void* weight, const void* post_weight,
    int weight_f32, float weight_offset, const void* gate, int64_t gate_st, int gate_mode,
    float scale, const float* stats, const void* dy, int64_t dy_st, const void* dr,
    int64_t dr_st, void* dx, void* dres, void* dgate, void* dweight, void* dpost, float* part,
    int32_t blocks, int32_t* status, void* stream) {
  using namespace tt::resnorm;
  if (bad_sizes(rows, D, gate_mode, gate) || blocks <= 0 ||
      (rows > 0 && (!x || !weight || !stats || !part)) || reinterpret_cast<uintptr_t>(stats) % 8)
    return TT_ERR_INVALID_ARG;
  if (rows == 0) return TT_OK;
  Args a{};
  a.rows = rows, a.D = D;
  a.x = x, a.res = residual, a.gate = gate, a.w2 = weight, a.w1 = post_weight;
  a.x_st = x_st, a.res_st = res_st, a.gate_st = gate_st;
  a.gate_mode = gate_mode, a.w_f32 = weight_f32;
  a.scale = scale, a.offset = weight_offset;
  a.stats = const_cast<float*>(stats);
  a.dy = dy, a.dr = dr, a.dy_st = dy_st, a.dr_st = dr_st;
  a.dx = dx, a.dres = dres, a.dgate = gate_mode == kChannel ? nullptr : dgate;
  a.part = part;
  Shape s = shape_of(D);
  a.tpr = s.tpr;
  const int xs = size_of(dtype), rs = size_of(res_dtype);
  auto fits = [&](int k) {
    return D % k == 0 && aligned(x, x_st, xs, k) && aligned(residual, residual ? res_st : 0, rs, k) &&
           aligned(dy, dy ? dy_st : 0, xs, k) && aligned(dr, dr ? dr_st : 0, rs, k) &&
           aligned(dx, D, xs, k) && aligned(dres, D, rs, k) &&
           (gate_mode != kFull || (aligned(gate, gate_st, xs, k) && aligned(dgate, D, xs, k)));
  };
  const int pack = fits(8) ? kAligned : fits(2) ? kPairs : s.tpr >= 32 ? kShifted : kSingle;
  cudaStream_t st = (cudaStream_t)stream;
  const bool full = post_weight || gate_mode != kNone, channel = gate_mode == kChannel;
  const bool two = two_packs(D, full, channel, xs, rs);
  const int threads = ring_threads(D, two), most = full ? 512 : 1024;
  RingShape ring{};
  if (rows_by_ring(D, dtype, pack == kAligned, a)) {
    const int stage_bytes = D * (xs * (1 + (dy ? 1 : 0) + (gate_mode == kFull ? 1 : 0)) +
                                 rs * ((residual ? 1 : 0) + (dr ? 1 : 0)));
    if (two)
      ring = ring_of(rows, D, threads, stage_bytes, most,
                     threads * 64 * (channel ? 3 : post_weight ? 2 : 1));
    if (!ring.blocks) ring = ring_of(rows, D, threads, stage_bytes, most);
  }
  if (ring.blocks)
    ring.blocks = blocks = std::min(blocks, ring.blocks);
  else
    blocks = (int)std::min<int64_t>(
        {blocks, (rows + s.per - 1) / s.per,
         tt::vec::kSMs * (int64_t)std::max(1, 1024 / (s.tpr * s.per))});
  const int rc = ring.blocks
                     ? dispatch_ring<true>(dtype, res_dtype, a, threads, ring, status, st)
                     : dispatch<true>(dtype, res_dtype, a, pack, s, blocks, st);
  if (rc != TT_OK) return rc;
  Out out{};
  out.p[0] = dweight;
  out.p[1] = post_weight ? dpost : nullptr;
  out.p[2] = gate_mode == kChannel ? dgate : nullptr;
  out.dtype[0] = out.dtype[1] = weight_f32 ? TT_F32 : dtype;
  out.dtype[2] = dtype;
  const int planes = out.p[2] ? 3 : out.p[1] ? 2 : out.p[0] ? 1 : 0;
  if (planes)
    sum_partials<<<dim3((D + 31) / 32, planes), dim3(32, kSumRows), 0, st>>>(blocks, D, part, out);
  tt_count_launches(planes ? 2 : 1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}
