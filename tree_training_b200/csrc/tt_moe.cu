// Tokens sorted by expert and back, with the router's weights, and gradients.
//
//   plan      a stable counting sort of the T K entries (token t's k-th choice
//             is entry t K + k) by expert: slots[entry] = its sorted row or -1
//             (no such expert: dropped), entries[row] = its entry or -1 (rows
//             past the last kept one), offsets[e] = first row of expert e
//   dispatch  xs[slots[t, k]] = x[t]; rows past the last kept one are zero
//   collect   dx[t] = sum_k dxs[slots[t, k]]               (dispatch's gradient)
//   combine   y[t] = sum_k w[t, k] ys[slots[t, k]]
//   spread    dys[slots[t, k]] = w[t, k] dy[t],  dw[t, k] = <dy[t], ys[slots[t, k]]>
//
// All but the plan are bound by HBM.  They go by token, not by sorted row: a
// token's row is read (or its sum written) once for its K rows, and every sum
// over k runs in the order of k in fp32 registers, so that no atomics are
// needed and results do not depend on the order of blocks.
//
// Measured on a B200, 8,191 tokens of 2,048 bf16 over 128 experts, eight a token
// (at the rate of a copy): plan 10 us, dispatch 48 (47), combine 56 (47), collect
// 50 (47), spread 91 (89).  32,768 of 2,560, four a token: dispatch 133 (131),
// combine 149 (131).
#include <algorithm>

#include "tt_vec.cuh"

namespace tt {
namespace moe {
namespace {

// ---- plan --------------------------------------------------------------------

// Two launches: blocks take runs of the entries, count them by expert and leave
// each entry's rank among its block's entries of the same expert; then each block
// adds up the counts of all blocks and of the earlier ones, and places its
// entries. One block does both in one launch where it is enough. Bound by
// latency, not by the 20 bytes an entry: many blocks of few steps each (eight
// blocks that meet in a cluster took 14.5 us for 65,528 entries).

constexpr int kPlanWarps = 8;
constexpr int kMaxExperts = 1024;
constexpr int kSteps = 8;          // of 32 entries, fetched together

__device__ __forceinline__ int expert_of(const void* ids, int ids64, int64_t i, int E) {
  const int64_t e = ids64 ? reinterpret_cast<const int64_t*>(ids)[i]
                          : reinterpret_cast<const int32_t*>(ids)[i];
  return (e >= 0 && e < E) ? (int)e : E;      // E: dropped, sorted behind the others
}

// The lanes whose e is this lane's, by one vote a bit (a match instruction takes
// several times as long over 32 different values).
__device__ __forceinline__ unsigned same_as(int e, int bits) {
  unsigned m = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const bool one = (e >> b) & 1;
    const unsigned v = __ballot_sync(0xffffffffu, one);
    m &= one ? v : ~v;
  }
  return m;
}

struct PlanArgs {
  const void* ids;
  int ids64;
  int64_t n, run;                  // entries, and those of a warp (a multiple of 32)
  int E;
  int32_t *slots, *entries, *offsets;
  int32_t* counts;                 // [blocks][E + 1]
};

// The exclusive sums over the experts of `all` (each thread's experts are
// x0 = threadIdx.x * per, ...): the first of them.
__device__ __forceinline__ int scan_experts(int sum, int* warp_sum) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int scan = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += up;
  }
  if (lane == 31) warp_sum[warp] = scan;
  __syncthreads();
  int first = scan - sum;
  for (int w = 0; w < warp; ++w) first += warp_sum[w];
  return first;
}

template <bool kSingle>
__global__ void __launch_bounds__(32 * kPlanWarps) plan_rank(const PlanArgs a) {
  extern __shared__ int sm[];
  int* hist = sm;                             // [warps][E + 1]: counts, then next ranks
  __shared__ int warp_sum[kPlanWarps];
  const int E = a.E, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t begin = min(a.n, ((int64_t)blockIdx.x * kPlanWarps + warp) * a.run);
  const int64_t end = min(a.n, begin + a.run);
  for (int i = threadIdx.x; i < kPlanWarps * (E + 1); i += blockDim.x) hist[i] = 0;
  __syncthreads();
  int* mine = hist + warp * (E + 1);
  const int bits = 32 - __clz(E + 1);
  int e[kSteps];
  unsigned same[kSteps];
  auto fetch = [&](int64_t from) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int64_t i = from + s * 32 + lane;
      e[s] = i < end ? expert_of(a.ids, a.ids64, i, E) : E + 1;
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      if (from + s * 32 < end) same[s] = same_as(e[s], bits);
  };
  for (int64_t from = begin; from < end; from += 32 * kSteps) {
    fetch(from);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      if (e[s] <= E && lane == __ffs(same[s]) - 1) atomicAdd(mine + e[s], __popc(same[s]));
  }
  __syncthreads();
  // counts become the ranks that each warp starts with
  const int per = kSingle ? (E + (int)blockDim.x) / (int)blockDim.x : 1;
  const int stride = kSingle ? 1 : (int)blockDim.x;
  int sum = 0, first = 0;
  auto warps_of = [&](int x, int at, bool write) {
    int c[kPlanWarps], all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) c[w] = hist[w * (E + 1) + x];
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) {
      if (write) hist[w * (E + 1) + x] = at + all;
      all += c[w];
    }
    return all;
  };
  if constexpr (kSingle) {
    const int x0 = threadIdx.x * per, x1 = min(x0 + per, E + 1);
    for (int x = x0; x < x1; ++x) sum += warps_of(x, 0, false);
    first = scan_experts(sum, warp_sum);
    for (int x = x0; x < x1; ++x) {
      a.offsets[x] = first;                   // offsets[E]: the rows that are kept
      first += warps_of(x, first, true);
    }
  } else {
    for (int x = threadIdx.x; x <= E; x += stride)
      a.counts[(int64_t)blockIdx.x * (E + 1) + x] = warps_of(x, 0, true);
  }
  __syncthreads();
  // The warp's counters hand out ranks in the order of its steps: each step's
  // leaders add theirs before the lanes part again for the next step's.
  const bool kept = end - begin <= 32 * kSteps;        // the ids are still in e
  for (int64_t from = begin; from < end; from += 32 * kSteps) {
    if (!kept) fetch(from);
    int base[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      base[s] = 0;
      if (e[s] <= E && lane == __ffs(same[s]) - 1)
        base[s] = atomicAdd(mine + e[s], __popc(same[s]));
      __syncwarp();
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int64_t i = from + s * 32 + lane;
      if (from + s * 32 >= end) continue;
      const int rank = __shfl_sync(0xffffffffu, base[s], __ffs(same[s]) - 1) +
                       __popc(same[s] & ((1u << lane) - 1));
      if (e[s] > E) continue;
      if constexpr (kSingle) {
        a.slots[i] = e[s] < E ? rank : -1;
        a.entries[rank] = e[s] < E ? (int32_t)i : -1;
      } else {
        a.slots[i] = rank;
      }
    }
  }
}

constexpr int kPlaceThreads = 512;

__global__ void __launch_bounds__(kPlaceThreads) plan_place(const PlanArgs a, int blocks) {
  extern __shared__ int sm[];
  int* total = sm;                            // [E + 1]
  int* first = sm + a.E + 1;                  // [E + 1]: this block's first rows
  __shared__ int warp_sum[kPlaceThreads / 32];
  const int E = a.E, b0 = blockIdx.x;
  // an expert's counts are shared out over as many threads as there are
  const int parts = max(1, (int)blockDim.x / (E + 1)), share = (blocks + parts - 1) / parts;
  for (int x = threadIdx.x; x < 2 * (E + 1); x += blockDim.x) sm[x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < parts * (E + 1); i += blockDim.x) {
    const int part = i / (E + 1), x = i - part * (E + 1);
    const int end = min(blocks, (part + 1) * share);
    int all = 0, before = 0;
    for (int b = part * share; b < end; b += 16) {
      int c[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        c[j] = b + j < end ? __ldg(a.counts + (int64_t)(b + j) * (E + 1) + x) : 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        all += c[j];
        before += b + j < b0 ? c[j] : 0;
      }
    }
    atomicAdd(total + x, all);
    atomicAdd(first + x, before);
  }
  __syncthreads();
  const int per = (E + (int)blockDim.x) / (int)blockDim.x;
  const int x0 = threadIdx.x * per, x1 = min(x0 + per, E + 1);
  int sum = 0;
  for (int x = x0; x < x1; ++x) sum += total[x];
  int at = scan_experts(sum, warp_sum);
  for (int x = x0; x < x1; ++x) {
    if (b0 == 0) a.offsets[x] = at;           // offsets[E]: the rows that are kept
    first[x] += at;
    at += total[x];
  }
  __syncthreads();
  const int64_t begin = min(a.n, (int64_t)b0 * kPlanWarps * a.run);
  const int64_t end = min(a.n, begin + kPlanWarps * a.run);
  for (int64_t i = begin + threadIdx.x; i < end; i += blockDim.x) {
    const int e = expert_of(a.ids, a.ids64, i, E);
    const int row = first[e] + a.slots[i];
    a.slots[i] = e < E ? row : -1;
    a.entries[row] = e < E ? (int32_t)i : -1;
  }
}

// Blocks of the two-launch form (each adds up `blocks` counts an expert), 1: the
// one-launch form, whose warps take up to two fetches.
int plan_blocks(int64_t n, int E) {
  if (n <= 32 * kSteps * kPlanWarps) return 1;
  const int64_t most = std::max<int64_t>(8, std::min<int64_t>(64, 32768 / (E + 1)));
  return (int)std::min<int64_t>(most, (n + 32 * kPlanWarps - 1) / (32 * kPlanWarps));
}

// ---- rows --------------------------------------------------------------------

struct Args {
  int64_t T;
  int K, H, E;
  uint32_t rows;             // sorted ones: T K
  int group;                 // threads of a token
  const int32_t *slots, *offsets;
  const void *src, *ys;      // by token (dispatch, spread) or by row (collect, combine)
  void *dst, *dw;
  const void* w;
  int w_dtype;
  int by_four;               // slots can be read four at a time
};

// Zeroes the rows past the last kept one; the blocks share them out.
template <typename T, int V>
__device__ __forceinline__ void zero_tail(const Args& a) {
  const int64_t n = a.T * a.K;
  const int64_t kept = max((int64_t)0, (int64_t)a.offsets[a.E]);
  const int packs = a.H / V;
  float z[V];
#pragma unroll
  for (int i = 0; i < V; ++i) z[i] = 0.f;
  for (int64_t r = kept + blockIdx.x; r < n; r += gridDim.x)
    for (int p = threadIdx.x; p < packs; p += blockDim.x)
      vec::store<T, V>(reinterpret_cast<T*>(a.dst) + r * a.H + p * V, z);
}

// A block's threads are groups of `group`, one token each; a token's slots and
// weights are fetched KC at a time, and so are the rows they lead to, so that
// KC loads of 16 bytes a thread are in flight.
struct Place {
  int t, slot;               // thread of its group, group of the block
  int64_t tok;
  bool live;
};

__device__ __forceinline__ Place place(const Args& a) {
  const int q = threadIdx.x / a.group;
  Place p;
  p.t = threadIdx.x - q * a.group;
  p.slot = q;
  p.tok = (int64_t)blockIdx.x * (blockDim.x / a.group) + q;
  p.live = p.tok < a.T;
  return p;
}

// Whether a slot is a sorted row; else its choice is dropped: -1, and whatever a
// plan of the caller's may hold.
__device__ __forceinline__ bool kept(const Args& a, int64_t slot) {
  return (uint32_t)slot < a.rows;
}

template <int KC>
__device__ __forceinline__ void slots_of(const Args& a, int64_t tok, int k0, int (&r)[KC]) {
  const int32_t* at = a.slots + tok * a.K + k0;
  if (KC >= 4 && a.by_four) {
#pragma unroll
    for (int k = 0; k < KC; k += 4) {
      const int4 q = k0 + k < a.K ? __ldg(reinterpret_cast<const int4*>(at + k))
                                  : make_int4(-1, -1, -1, -1);
      r[k] = q.x, r[k + 1] = q.y, r[k + 2] = q.z, r[k + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < KC; ++k) r[k] = k0 + k < a.K ? __ldg(at + k) : -1;
  }
}

__device__ __forceinline__ float weight_of(const Args& a, const Place& pl, int k) {
  if (!pl.live || k >= a.K) return 0.f;
  const int64_t i = pl.tok * a.K + k;
  switch (a.w_dtype) {
    case TT_F32: return reinterpret_cast<const float*>(a.w)[i];
    case TT_BF16: return to_f32(reinterpret_cast<const __nv_bfloat16*>(a.w)[i]);
    default: return to_f32(reinterpret_cast<const __half*>(a.w)[i]);
  }
}

constexpr int kMaxK = 64;
constexpr int kMaxTokens = 8;                      // of a block

template <typename T, int V, int KC>
__global__ void __launch_bounds__(512) dispatch_kernel(const Args a) {
  const Place pl = place(a);
  const int packs = a.H / V;
  if (pl.live) {
    const T* src = reinterpret_cast<const T*>(a.src) + pl.tok * a.H;
    for (int k0 = 0; k0 < a.K; k0 += KC) {
      int r[KC];
      slots_of<KC>(a, pl.tok, k0, r);
      for (int p = pl.t; p < packs; p += a.group) {
        const vec::Raw<T, V> v = vec::load_raw<T, V>(src + p * V);
#pragma unroll
        for (int k = 0; k < KC; ++k)
          if (kept(a, r[k]))
            *reinterpret_cast<vec::Raw<T, V>*>(reinterpret_cast<T*>(a.dst) + (int64_t)r[k] * a.H +
                                               p * V) = v;
      }
    }
  }
  zero_tail<T, V>(a);
}

// One choice after another in 32 registers, so that an SM is full of warps: the
// loads of other warps stand in for those of other choices.  With KC rows in
// flight a thread, as in collect, this took 60 us against 57 (8,191 tokens of 8 x
// 2,048) and 162 against 150 (32,768 of 4 x 2,560).
template <typename T, int V>
__global__ void __launch_bounds__(512, 4) combine_kernel(const Args a) {
  const Place pl = place(a);
  if (!pl.live) return;
  const int packs = a.H / V;
  const int32_t* slot = a.slots + pl.tok * a.K;
  for (int p = pl.t; p < packs; p += a.group) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int k = 0; k < a.K; ++k) {
      const int64_t r = __ldg(slot + k);
      if (!kept(a, r)) continue;
      const float w = weight_of(a, pl, k);
      float v[V];
      vec::load<T, V>(reinterpret_cast<const T*>(a.src) + r * a.H + p * V, v);
      vec::axpy<V>(w, v, acc);
    }
    vec::store<T, V>(reinterpret_cast<T*>(a.dst) + pl.tok * a.H + p * V, acc);
  }
}

template <typename T, int V, int KC>
__global__ void __launch_bounds__(512, 2) collect_kernel(const Args a) {
  const Place pl = place(a);
  if (!pl.live) return;
  const int packs = a.H / V;
  const T* src = reinterpret_cast<const T*>(a.src);
  int r[KC];
  slots_of<KC>(a, pl.tok, 0, r);
  for (int p = pl.t; p < packs; p += a.group) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int k0 = 0; k0 < a.K; k0 += KC) {
      if (a.K > KC) slots_of<KC>(a, pl.tok, k0, r);
      vec::Raw<T, V> raw[KC];
#pragma unroll
      for (int k = 0; k < KC; ++k)
        if (kept(a, r[k])) raw[k] = vec::load_raw<T, V>(src + (int64_t)r[k] * a.H + p * V);
#pragma unroll
      for (int k = 0; k < KC; ++k) {
        if (!kept(a, r[k])) continue;
        float v[V];
        vec::unpack<T, V>(raw[k], v);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += v[i];
      }
    }
    vec::store<T, V>(reinterpret_cast<T*>(a.dst) + pl.tok * a.H + p * V, acc);
  }
}

template <typename T, int V, int KC>
__global__ void __launch_bounds__(512, 2) spread_kernel(const Args a) {
  __shared__ float red[16][KC];
  __shared__ float sw[kMaxTokens * kMaxK];
  const Place pl = place(a);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = a.group >> 5;
  const int packs = a.H / V;
  const int64_t tok = pl.live ? pl.tok : 0;
  const float* w = sw + pl.slot * a.K;
  if (pl.t < a.K) sw[pl.slot * a.K + pl.t] = weight_of(a, pl, pl.t);
  if (pl.t + a.group < a.K)
    sw[pl.slot * a.K + pl.t + a.group] = weight_of(a, pl, pl.t + a.group);
  int r[KC];
  slots_of<KC>(a, tok, 0, r);
  __syncthreads();
  for (int k0 = 0; k0 < a.K; k0 += KC) {
    float dot[KC];
#pragma unroll
    for (int k = 0; k < KC; ++k) dot[k] = 0.f;
    if (pl.live) {
      if (k0) slots_of<KC>(a, tok, k0, r);
      for (int p = pl.t; p < packs; p += a.group) {
        constexpr int B = KC < 4 ? KC : 4;         // of them in flight
        const vec::Raw<T, V> raw_g =
            vec::load_raw<T, V>(reinterpret_cast<const T*>(a.src) + tok * a.H + p * V);
#pragma unroll
        for (int b = 0; b < KC; b += B) {
          vec::Raw<T, V> raw[B];
#pragma unroll
          for (int k = 0; k < B; ++k)
            if (kept(a, r[b + k]))
              raw[k] = vec::load_raw<T, V>(reinterpret_cast<const T*>(a.ys) +
                                           (int64_t)r[b + k] * a.H + p * V);
          float g[V];
          vec::unpack<T, V>(raw_g, g);
#pragma unroll
          for (int k = 0; k < B; ++k) {
            if (!kept(a, r[b + k])) continue;
            const float wk = w[k0 + b + k];
            float v[V], o[V];
            vec::unpack<T, V>(raw[k], v);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              dot[b + k] = fmaf(g[i], v[i], dot[b + k]);
              o[i] = wk * g[i];
            }
            vec::store<T, V>(reinterpret_cast<T*>(a.dst) + (int64_t)r[b + k] * a.H + p * V, o);
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < KC; ++k)
      for (int o = 16; o > 0; o >>= 1) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], o);
    if (k0) __syncthreads();            // the sums before have been read
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < KC; ++k) red[warp][k] = dot[k];
    }
    __syncthreads();
    if (pl.live && pl.t < min(KC, a.K - k0)) {
      float s = 0.f;
      for (int q = 0; q < nw; ++q) s += red[warp + q][pl.t];
      const int64_t i = tok * a.K + k0 + pl.t;
      switch (a.w_dtype) {
        case TT_F32: reinterpret_cast<float*>(a.dw)[i] = s; break;
        case TT_BF16: reinterpret_cast<__nv_bfloat16*>(a.dw)[i] = from_f32<__nv_bfloat16>(s); break;
        default: reinterpret_cast<__half*>(a.dw)[i] = from_f32<__half>(s); break;
      }
    }
  }
  zero_tail<T, V>(a);
}

// ---- rows at any element ---------------------------------------------------------
//
// With 16-bit rows whose width is no multiple of 8, every row starts at another
// place of a 16-byte word.  Threads go by the words of the row that is written
// (in spread: of the sorted row), and shift what they read into place.

// Elements of a row's first 16-byte word that lie before the row.
template <typename T>
__device__ __forceinline__ int lead(const T* row) {
  return (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
}

template <typename T>
__global__ void __launch_bounds__(512) dispatch_any(const Args a) {
  constexpr int N = 16 / (int)sizeof(T);
  const Place pl = place(a);
  if (pl.live) {
    const T *lo = reinterpret_cast<const T*>(a.src), *hi = lo + a.T * a.H;
    const T* src = lo + pl.tok * a.H;
    for (int k = 0; k < a.K; ++k) {
      const int64_t r = __ldg(a.slots + pl.tok * a.K + k);
      if (!kept(a, r)) continue;
      T* dst = reinterpret_cast<T*>(a.dst) + r * a.H;
      for (int64_t e = (int64_t)pl.t * N - lead(dst); e < a.H; e += a.group * N)
        vec::store_part<T>(dst, e, a.H, vec::load_any_of<T>(src, e, a.H, lo, hi));
    }
  }
  zero_tail<T, 1>(a);
}

template <typename T, bool kWeighted>
__global__ void __launch_bounds__(512) combine_any(const Args a) {
  constexpr int N = 16 / (int)sizeof(T);
  const Place pl = place(a);
  if (!pl.live) return;
  const T *lo = reinterpret_cast<const T*>(a.src), *hi = lo + a.T * a.K * a.H;
  T* dst = reinterpret_cast<T*>(a.dst) + pl.tok * a.H;
  for (int64_t e = (int64_t)pl.t * N - lead(dst); e < a.H; e += a.group * N) {
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    for (int k = 0; k < a.K; ++k) {
      const int64_t r = __ldg(a.slots + pl.tok * a.K + k);
      if (!kept(a, r)) continue;
      float v[N];
      vec::unpack<T, N>(vec::load_any_of<T>(lo + r * a.H, e, a.H, lo, hi), v);
      vec::axpy<N>(kWeighted ? weight_of(a, pl, k) : 1.f, v, acc);
    }
    vec::store_part<T>(dst, e, a.H, vec::pack<T, N>(acc));
  }
}

template <typename T>
__global__ void __launch_bounds__(512) spread_any(const Args a) {
  constexpr int N = 16 / (int)sizeof(T);
  __shared__ float red[16];
  const Place pl = place(a);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = a.group >> 5;
  const T *lo = reinterpret_cast<const T*>(a.src), *hi = lo + a.T * a.H;
  for (int k = 0; k < a.K; ++k) {
    float dot = 0.f;
    if (pl.live) {
      const int64_t r = __ldg(a.slots + pl.tok * a.K + k);
      if (kept(a, r)) {
        const float w = weight_of(a, pl, k);
        const T* ys = reinterpret_cast<const T*>(a.ys) + r * a.H;
        T* dst = reinterpret_cast<T*>(a.dst) + r * a.H;
        const T* yhi = reinterpret_cast<const T*>(a.ys) + a.T * a.K * a.H;
        for (int64_t e = (int64_t)pl.t * N - lead(dst); e < a.H; e += a.group * N) {
          float g[N], v[N], o[N];
          vec::unpack<T, N>(vec::load_any_of<T>(lo + pl.tok * a.H, e, a.H, lo, hi), g);
          vec::unpack<T, N>(vec::load_any_of<T>(ys, e, a.H, reinterpret_cast<const T*>(a.ys), yhi),
                            v);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            dot = fmaf(g[i], v[i], dot);
            o[i] = w * g[i];
          }
          vec::store_part<T>(dst, e, a.H, vec::pack<T, N>(o));
        }
      }
    }
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (k) __syncthreads();             // the sums before have been read
    if (lane == 0) red[warp] = dot;
    __syncthreads();
    if (pl.live && pl.t == 0) {
      float s = 0.f;
      for (int q = 0; q < nw; ++q) s += red[warp + q];
      const int64_t i = pl.tok * a.K + k;
      switch (a.w_dtype) {
        case TT_F32: reinterpret_cast<float*>(a.dw)[i] = s; break;
        case TT_BF16: reinterpret_cast<__nv_bfloat16*>(a.dw)[i] = from_f32<__nv_bfloat16>(s); break;
        default: reinterpret_cast<__half*>(a.dw)[i] = from_f32<__half>(s); break;
      }
    }
  }
  zero_tail<T, 1>(a);
}

enum Op { kDispatch, kCollect, kCombine, kSpread };

template <typename T>
int launch_any(Op op, Args& a, cudaStream_t st) {
  const int packs = a.H / 8 + 2;
  const int turns = (packs + 511) / 512;
  a.group = ((packs + turns - 1) / turns + 31) / 32 * 32;
  const int per = std::max(1, 256 / a.group), threads = a.group * per;
  const int64_t blocks = (a.T + per - 1) / per;
  if (blocks > 0x7fffffff) return TT_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)blocks;
  switch (op) {
    case kDispatch: dispatch_any<T><<<grid, threads, 0, st>>>(a); break;
    case kCollect: combine_any<T, false><<<grid, threads, 0, st>>>(a); break;
    case kCombine: combine_any<T, true><<<grid, threads, 0, st>>>(a); break;
    case kSpread: spread_any<T><<<grid, threads, 0, st>>>(a); break;
  }
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

template <typename T, int V, int KC>
int launch(Op op, Args& a, cudaStream_t st) {
  // a group of whole warps for a token, up to 512 threads, that its packs fill as
  // evenly as they can; short rows share a block of about 256
  const int packs = a.H / V;
  const int turns = (packs + 511) / 512;
  a.group = ((packs + turns - 1) / turns + 31) / 32 * 32;
  const int per = std::max(1, 256 / a.group), threads = a.group * per;
  const int64_t blocks = (a.T + per - 1) / per;
  if (blocks > 0x7fffffff) return TT_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)blocks;
  switch (op) {
    case kDispatch: dispatch_kernel<T, V, KC><<<grid, threads, 0, st>>>(a); break;
    case kCollect: collect_kernel<T, V, KC><<<grid, threads, 0, st>>>(a); break;
    case kCombine: combine_kernel<T, V><<<grid, threads, 0, st>>>(a); break;
    case kSpread: spread_kernel<T, V, KC><<<grid, threads, 0, st>>>(a); break;
  }
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

template <typename T, int V>
int launch_k(Op op, Args& a, cudaStream_t st) {
  a.by_four = a.K % 4 == 0 && reinterpret_cast<uintptr_t>(a.slots) % 16 == 0;
  if (a.K <= 2) return launch<T, V, 2>(op, a, st);
  if (a.K <= 4) return launch<T, V, 4>(op, a, st);
  return launch<T, V, 8>(op, a, st);
}

int run(Op op, int dtype, Args& a, void* stream) {
  if (a.T < 0 || a.K < 0 || a.K > kMaxK || a.H <= 0 || a.E <= 0 || a.T * a.K > 0x7fffffff)
    return TT_ERR_INVALID_ARG;
  if (a.T == 0) return TT_OK;
  a.rows = (uint32_t)(a.T * a.K);
  // with K = 0 there are no sorted rows: the side of them may be null
  const bool by_token = op == kDispatch || op == kSpread;      // src is
  if (!a.offsets || (a.K > 0 && !a.slots) || (!a.src && (by_token || a.K > 0)) ||
      (!a.dst && (!by_token || a.K > 0)))
    return TT_ERR_INVALID_ARG;
  if (by_token && a.K == 0) return TT_OK;
  return vec::dispatch_float(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    constexpr int V = 16 / (int)sizeof(T);
    // 16-byte packs where rows are aligned; 16-bit rows at any element by shifted
    // words; 32-bit ones in pairs or by elements
    auto fits = [&](int v) {
      auto ok = [&](const void* p) {
        return reinterpret_cast<uintptr_t>(p) % (v * sizeof(T)) == 0;
      };
      return a.H % v == 0 && ok(a.src) && ok(a.dst) && ok(a.ys);
    };
    if (fits(V)) return launch_k<T, V>(op, a, (cudaStream_t)stream);
    if constexpr (sizeof(T) == 2) {
      return launch_any<T>(op, a, (cudaStream_t)stream);
    } else {
      return fits(2) ? launch_k<T, 2>(op, a, (cudaStream_t)stream)
                     : launch_k<T, 1>(op, a, (cudaStream_t)stream);
    }
  });
}

}  // namespace
}  // namespace moe
}  // namespace tt

extern "C" int64_t tt_moe_plan_workspace_size(int64_t n_entries, int32_t n_experts) {
  if (n_entries < 0 || n_experts <= 0 || n_experts > tt::moe::kMaxExperts) return -1;
  const int blocks = tt::moe::plan_blocks(n_entries, n_experts);
  return blocks > 1 ? (int64_t)blocks * (n_experts + 1) * 4 : 0;
}

extern "C" int tt_moe_plan(const void* ids, int ids64, int64_t n_entries, int32_t n_experts,
                           int32_t* slots, int32_t* entries, int32_t* offsets, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  using namespace tt::moe;
  if (n_entries < 0 || n_entries > 0x7fffffff || n_experts <= 0 || n_experts > kMaxExperts ||
      !offsets || (n_entries > 0 && (!ids || !slots || !entries)))
    return TT_ERR_INVALID_ARG;
  const int E = n_experts, blocks = plan_blocks(n_entries, E);
  if (blocks > 1 && (!workspace || workspace_bytes < tt_moe_plan_workspace_size(n_entries, E)))
    return TT_ERR_WORKSPACE;
  const int64_t warps = (int64_t)blocks * kPlanWarps;
  const int64_t run = std::max<int64_t>(32, ((n_entries + warps - 1) / warps + 31) / 32 * 32);
  const PlanArgs a{ids, ids64, n_entries, run, E, slots, entries, offsets, (int32_t*)workspace};
  cudaStream_t st = (cudaStream_t)stream;
  const int threads = 32 * kPlanWarps;
  const size_t smem = sizeof(int) * kPlanWarps * (E + 1);
  if (blocks == 1) {
    plan_rank<true><<<1, threads, smem, st>>>(a);
  } else {
    plan_rank<false><<<blocks, threads, smem, st>>>(a);
    plan_place<<<blocks, kPlaceThreads, sizeof(int) * 2 * (E + 1), st>>>(a, blocks);
  }
  tt_count_launches(blocks > 1 ? 2 : 1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

extern "C" int tt_moe_dispatch(int dtype, int64_t n_tok, int32_t k, int32_t H, int32_t n_experts,
                               const int32_t* slots, const int32_t* offsets, const void* x,
                               void* xs, void* stream) {
  using namespace tt::moe;
  Args a{};
  a.T = n_tok, a.K = k, a.H = H, a.E = n_experts, a.slots = slots, a.offsets = offsets;
  a.src = x, a.dst = xs;
  return run(kDispatch, dtype, a, stream);
}

extern "C" int tt_moe_collect(int dtype, int64_t n_tok, int32_t k, int32_t H, int32_t n_experts,
                              const int32_t* slots, const int32_t* offsets, const void* dxs,
                              void* dx, void* stream) {
  using namespace tt::moe;
  Args a{};
  a.T = n_tok, a.K = k, a.H = H, a.E = n_experts, a.slots = slots, a.offsets = offsets;
  a.src = dxs, a.dst = dx;
  return run(kCollect, dtype, a, stream);
}

extern "C" int tt_moe_combine(int dtype, int weight_dtype, int64_t n_tok, int32_t k, int32_t H,
                              int32_t n_experts, const int32_t* slots, const int32_t* offsets,
                              const void* ys, const void* weights, void* y, void* stream) {
  using namespace tt::moe;
  if (weight_dtype < TT_F32 || weight_dtype > TT_F16) return TT_ERR_UNSUPPORTED;
  if (n_tok > 0 && k > 0 && !weights) return TT_ERR_INVALID_ARG;
  Args a{};
  a.T = n_tok, a.K = k, a.H = H, a.E = n_experts, a.slots = slots, a.offsets = offsets;
  a.src = ys, a.dst = y, a.w = weights, a.w_dtype = weight_dtype;
  return run(kCombine, dtype, a, stream);
}

extern "C" int tt_moe_spread(int dtype, int weight_dtype, int64_t n_tok, int32_t k, int32_t H,
                             int32_t n_experts, const int32_t* slots, const int32_t* offsets,
                             const void* dy, const void* ys, const void* weights, void* dys,
                             void* dweights, void* stream) {
  using namespace tt::moe;
  if (weight_dtype < TT_F32 || weight_dtype > TT_F16) return TT_ERR_UNSUPPORTED;
  if (n_tok > 0 && k > 0 && (!weights || !ys || !dweights)) return TT_ERR_INVALID_ARG;
  Args a{};
  a.T = n_tok, a.K = k, a.H = H, a.E = n_experts, a.slots = slots, a.offsets = offsets;
  a.src = dy, a.ys = ys, a.dst = dys, a.dw = dweights, a.w = weights, a.w_dtype = weight_dtype;
  return run(kSpread, dtype, a, stream);
}
