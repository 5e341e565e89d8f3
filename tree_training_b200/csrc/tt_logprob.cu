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
// Both directions are bound by HBM.  Forward: the row is read once, in 16-byte
// packs; each thread keeps running sums in base 2 (two fp32 values relative to a
// reference that moves only when the maximum is 2^12 above it) and its largest
// logit, from which the alternatives' candidates are found (block_top).  Few
// rows are split over the blocks of a cluster, which meet in shared memory.
// Backward: one pass from the four statistics a row that the forward keeps.
//
// Measured on a B200 (at the rate of a copy): 2,047 x 151,936 bf16: forward 117 us
// (97; 101 with the maximum alone), backward 202 (194); 4,096 x 151,936 with sixteen
// alternatives 283 (194): what they cost is the wait of the second look's loads
// beside a busy memory.  One row of 151,936: 5.5 us, with eight alternatives 11.
#include <cooperative_groups.h>

#include <algorithm>

#include "tt_sm100.cuh"
#include "tt_vec.cuh"

namespace cg = cooperative_groups;

namespace tt {
namespace logprob {
namespace {

// Threads of a block: 256, or 64 for short rows, of which an SM then takes more.
constexpr int kThreads = 256;
constexpr int kFewThreads = 64;
constexpr int kFewPacks = 512;    // 16-byte packs of a row that 64 threads read
constexpr int kMaxTop = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Exponents of 2 are kept from -inf, whose product with a probability of 0
// would be NaN; 2^-200 is 0 in fp32.
constexpr float kFloor = -200.f;
constexpr float kGradFloor = -300.f;    // where they are 2^100 times as large
// Between these 1 / temperature and gradients over it are far from the ends of fp32:
// an infinite or flushed factor would make NaN of a difference of 0 or of -inf.
constexpr float kMinTemperature = 1e-20f, kMaxTemperature = 1e20f;
// The reference moves when the maximum is this far (a factor of 2^12) above it.
constexpr float kSlack = 12.f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x, 0 where that is under 2^-126.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
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

__device__ __forceinline__ Sums shfl_xor(const Sums& a, int o) {
  return {__shfl_xor_sync(0xffffffffu, a.ref, o), __shfl_xor_sync(0xffffffffu, a.s, o),
          __shfl_xor_sync(0xffffffffu, a.u, o)};
}

__device__ __forceinline__ void load32(const uint4* p, uint4& a, uint4& b) {
  asm("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
      : "l"(p));
}

// A row as 16-byte packs that start on 16-byte boundaries: pack v holds the
// elements [v N - shift, (v + 1) N - shift), of which those of the row are
// loaded and the others are -inf (no probability, and no candidates: their
// index is out of range).
template <typename T>
struct Packs {
  static constexpr int N = 16 / (int)sizeof(T);
  const T* x;
  int V, shift;
  int n, whole0, whole1;        // packs; those that lie in the row as a whole

  __device__ __forceinline__ Packs(const T* row, int vocab) : x(row), V(vocab) {
    shift = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % N);
    n = (int)(((int64_t)shift + vocab + N - 1) / N);
    whole0 = shift ? 1 : 0;
    whole1 = (int)(((int64_t)shift + vocab) / N);
  }
  __device__ __forceinline__ bool whole(int v) const { return v >= whole0 && v < whole1; }
  __device__ __forceinline__ int64_t first(int v) const { return (int64_t)v * N - shift; }
  __device__ __forceinline__ uint4 raw(int v) const {
    if (whole(v)) return __ldg(reinterpret_cast<const uint4*>(x - shift) + v);
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t e = first(v) + i;
      o[i] = (e >= 0 && e < V) ? to_f32(x[e]) : -INFINITY;
    }
    return vec::pack<T, N>(o);
  }
  __device__ __forceinline__ void load(int v, float (&o)[N]) const {
    vec::unpack<T, N>(raw(v), o);
  }
  // Whether pack v lies on a 32-byte boundary.
  __device__ __forceinline__ bool wide(int v) const {
    return (reinterpret_cast<uintptr_t>(x - shift) + (uint64_t)v * 16) % 32 == 0;
  }
  // Packs v to v + G - 1, those below `end` (the others are left alone); `wide`:
  // 32 bytes a load.
  template <int G>
  __device__ __forceinline__ void some(int v, int end, bool wide, uint4 (&r)[G]) const {
    if (v >= whole0 && v + G - 1 < min(whole1, end)) {
      const uint4* p = reinterpret_cast<const uint4*>(x - shift) + v;
      if (G > 1 && wide) {
#pragma unroll
        for (int i = 0; i + 1 < G; i += 2) load32(p + i, r[i], r[i + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < G; ++i) r[i] = __ldg(p + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < G; ++i)
        if (v + i < end) r[i] = raw(v + i);
    }
  }
};

// The largest of a pack (NaN aside).
template <typename T>
__device__ __forceinline__ float pack_max(const uint4& r) {
  if constexpr (std::is_same<T, float>::value) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)),
                 fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2,
                                         __nv_bfloat162>::type;
    const T2* p = reinterpret_cast<const T2*>(&r);
    const T2 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(to_f32(m.x), to_f32(m.y));
  }
}

// A thread's sums, the even and the odd elements' apart (paired arithmetic).
struct Running {
  float ref, over;              // over: the maximum that moves ref
  float2 s, u;

  __device__ __forceinline__ Running() : ref(0.f), over(-INFINITY) {
    s = u = make_float2(0.f, 0.f);
  }
  __device__ __forceinline__ void move(float mx, float c) {
    const float d = max_nan((ref - mx) * c, kFloor), f = ex2(d);
    if (s.x != 0.f) u.x = f * fmaf(s.x, d, u.x), s.x *= f;
    if (s.y != 0.f) u.y = f * fmaf(s.y, d, u.y), s.y *= f;
    ref = mx;
    over = mx + kSlack / c;
  }
  template <typename T>
  __device__ __forceinline__ float add(const uint4& raw, float c) {
    constexpr int N = 16 / (int)sizeof(T);
    const float mx = pack_max<T>(raw);
    if (mx > over) move(mx, c);
    float x[N];
    vec::unpack<T, N>(raw, x);
    const float2 c2 = make_float2(c, c), r2 = make_float2(-ref, -ref);
    float2 ps = make_float2(0.f, 0.f), pu = ps;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      float2 t = sm100::fmul2(sm100::fadd2(make_float2(x[i], x[i + 1]), r2), c2);
      t.x = max_nan(t.x, kFloor);
      t.y = max_nan(t.y, kFloor);
      const float2 e = make_float2(ex2(t.x), ex2(t.y));
      ps = i ? sm100::fadd2(ps, e) : e;
      pu = i ? sm100::ffma2(t, e, pu) : sm100::fmul2(t, e);
    }
    s = sm100::fadd2(s, ps);
    u = sm100::fadd2(u, pu);
    return mx;
  }
  __device__ __forceinline__ Sums sums() const { return {ref, s.x + s.y, u.x + u.y}; }
};

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

// Log probability of logit x.  The maximum is subtracted before the division, as
// in the sums: the type's lowest value overflows when it is divided by a
// temperature under 1.
__device__ __forceinline__ float logp_of(float x, float m, float ln_s, float inv_s, float temp) {
  if (inv_s == 0.f) return -INFINITY;
  return (x - m) / temp - ln_s;
}

constexpr int kUnroll = 4;        // packs in flight a thread
constexpr int kMaxCluster = 8;

template <int TH>
struct TopShared {
  // (with 64 threads: all of a short row's elements up to 1,024)
  static constexpr int kCandidates = TH == kThreads ? 4096 : 1024;
  ulonglong2 keys[TH / 2];        // the threads' largest
  ulonglong2 found[kCandidates / 2];
  uint64_t list[kMaxTop];         // this block's largest, in order
  uint64_t lists[TH == kThreads ? kMaxCluster : 1][kMaxTop];   // block 0: every block's
  uint64_t bar;                   // the k-th largest of keys: a lower bound
  int n_threads, n_found, n_kept;
  int at_least[64];
  int threads[TH];
};

// How many of the first n keys (n even, or a 0 behind them) are above `mine`.
__device__ __forceinline__ int count_above(const ulonglong2* keys, int n, uint64_t mine) {
  int above = 0;
#pragma unroll 4
  for (int i = 0; i < (n + 1) / 2; ++i) {
    const ulonglong2 q = keys[i];
    above += (q.x > mine) + (q.y > mine);
  }
  return above;
}

// The k largest keys of the block's packs [begin, end) into sh.list, in order
// (0 where there are fewer).  `best` is this thread's largest logit and
// `best_pack` the first pack that has it (-1: none); `nan` is set where a sum of
// the block is NaN, as then `best` may have missed a NaN.  The k-th largest key
// of any elements is a lower bound of the k-th largest of all, so: take it from
// the threads' largest, look once more through the packs of the threads that
// reach it (about k of them), and rank what is found.  Should more than
// kCandidates elements reach the bound, or with a NaN, the list is made one pass
// an entry.
// G: how many packs in a row a thread reads, every G TH packs.
template <typename T, int TH, int G>
__device__ __forceinline__ void block_top(const Packs<T>& row, int begin, int end, int k,
                                          float best, int best_pack, bool nan,
                                          TopShared<TH>& sh) {
  constexpr int N = Packs<T>::N, W = TH / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) sh.bar = 0, sh.n_threads = 0, sh.n_found = 0, sh.n_kept = 0;
  if (threadIdx.x < 64) sh.at_least[threadIdx.x] = 0;
  // a key no larger than that of the thread's largest: its pack's last index
  const uint32_t order = order_of(best);
  const uint64_t low = best_pack < 0 ? 0 : key_of(order, row.first(best_pack) + N - 1);
  // the k-th of them: among all, or, where k is small, among the largest of each
  // warp (one row: 8 us with k = 1 and 11 with 8, against 10 and 12.5)
  uint64_t* keys = reinterpret_cast<uint64_t*>(sh.keys);
  int n_keys = TH;
  if (k <= 8 || k <= 2 * W) {
    const int each = min(k, 8);
    n_keys = W * each;
    uint32_t hi = (uint32_t)(low >> 32), lo = (uint32_t)low;
    for (int r = 0; r < each; ++r) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, hi);
      const uint32_t at = __reduce_max_sync(0xffffffffu, hi == top ? lo : 0u);
      if (lane == 0) keys[warp * each + r] = top ? ((uint64_t)top << 32) | at : 0;
      if (hi == top && lo == at) hi = 0;
    }
  } else {
    keys[threadIdx.x] = low;
  }
  __syncthreads();
  if ((int)threadIdx.x < n_keys) {
    const uint64_t mine = keys[threadIdx.x];         // keys differ unless they are 0
    if (mine && count_above(sh.keys, n_keys, mine) == k - 1) sh.bar = mine;
  }
  __syncthreads();
  const uint64_t bar = sh.bar;
  if (best_pack >= 0 && key_of(order, max((int64_t)0, row.first(best_pack))) >= bar)
    sh.threads[atomicAdd(&sh.n_threads, 1)] = threadIdx.x;
  __syncthreads();
  uint64_t* found = reinterpret_cast<uint64_t*>(sh.found);
  const int n_threads = nan ? 0 : sh.n_threads;
  const uint32_t bar_order = (uint32_t)(bar >> 32);
  // their packs, over all threads
  const int per = (end - begin + G * TH - 1) / (G * TH);
  const bool wide = row.wide(begin);
  for (int i = threadIdx.x; i < n_threads * per; i += TH) {
    const int q = i / per, v = begin + G * (sh.threads[q] + (i - q * per) * TH);
    if (v >= end) continue;
    uint4 raw[G];
    row.template some<G>(v, end, wide, raw);
#pragma unroll
    for (int u = 0; u < G; ++u) {
      if (v + u >= end || order_of(pack_max<T>(raw[u])) < bar_order) continue;
      float x[N];
      vec::unpack<T, N>(raw[u], x);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int64_t e = row.first(v + u) + j;
        const uint64_t key = key_of(order_of(x[j]), e);
        if (key >= bar && e >= 0 && e < row.V) {
          const int at = atomicAdd(&sh.n_found, 1);
          if (at < sh.kCandidates) found[at] = key;
        }
      }
    }
  }
  __syncthreads();
  const int n = sh.n_found;
  if (n <= sh.kCandidates && n > 512 && !nan) {
    // many equal logits: the k-th key, bit by bit from counts, then those from it on
    uint64_t kth = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t at = kth | (1ull << bit);
      int m = 0;
      for (int i = threadIdx.x; i < n; i += TH) m += found[i] >= at;
      m = __reduce_add_sync(0xffffffffu, m);
      if (lane == 0) atomicAdd(&sh.at_least[bit], m);
      __syncthreads();
      const int all = sh.at_least[bit];
      if (all >= k) kth = at;
      if (all == k) break;
    }
    for (int i = threadIdx.x; i < n; i += TH)
      if (found[i] >= kth) keys[atomicAdd(&sh.n_kept, 1)] = found[i];
    __syncthreads();
    if ((int)threadIdx.x < k) {
      int above = 0;
      for (int i = 0; i < k; ++i) above += keys[i] > keys[threadIdx.x];
      sh.list[above] = keys[threadIdx.x];
    }
    __syncthreads();
    return;
  }
  if (n <= sh.kCandidates && !nan) {
    if (n & 1) {
      if (threadIdx.x == 0) found[n] = 0;
      __syncthreads();
    }
    for (int c = threadIdx.x; c < max(n, k); c += TH) {
      if (c >= n) {
        sh.list[c] = 0;
        continue;
      }
      const uint64_t mine = found[c];
      const int above = count_above(sh.found, n, mine);
      if (above < k) sh.list[above] = mine;
    }
    __syncthreads();
    return;
  }
  uint64_t below = ~0ull;
  for (int j = 0; j < k; ++j) {
    uint64_t mine = 0;
    for (int v = begin + threadIdx.x; v < end; v += TH) {
      float x[N];
      row.load(v, x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t e = row.first(v) + i;
        const uint64_t key = key_of(order_of(x[i]), e);
        if (key < below && key > mine && e >= 0 && e < row.V) mine = key;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, (unsigned long long)mine, o);
      mine = other > mine ? other : mine;
    }
    __syncthreads();
    if (lane == 0) found[warp] = mine;
    __syncthreads();
    below = found[0];
    for (int w = 1; w < W; ++w) below = found[w] > below ? found[w] : below;
    if (threadIdx.x == 0) sh.list[j] = below;
  }
  __syncthreads();
}

struct Part {
  Sums sums;
  float best;
};

// One row a cluster: its blocks take equal runs of the row's packs and block 0
// brings their sums and lists together.  G is 0 without alternatives, else the
// packs in a row that a thread reads: 4 in long rows, since the second look's
// single packs would cost the memory a piece of 64 bytes or more each (4,096 x
// 151,936 with sixteen: 305 us against 277), 1 where threads have few packs
// (16,000 x 10,000: 248 against 297).
//
// (0 blocks an SM: left to the compiler, which then takes 48 registers; asked for
// 1 it takes up to 80, and the loop without alternatives 234 us instead of 218.
// With G = 4 four blocks are asked for: 277 against 281, 340 with five.)
template <typename T, int TH, int G>
__global__ void __launch_bounds__(TH, G == 4 ? 4 : 0) fwd_kernel(const Args a) {
  constexpr int W = TH / 32;
  constexpr bool kTop = G > 0;
  __shared__ Part warps[W];
  __shared__ Part parts[kMaxCluster];
  __shared__ float st[3];
  extern __shared__ ulonglong2 top_raw[];
  TopShared<TH>& sh = *reinterpret_cast<TopShared<TH>*>(top_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x / blocks;
  // block 0 must be running before another block writes into its shared memory
  if (blocks > 1) cluster.barrier_arrive();
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld;
  const Packs<T> packs(x, a.V);
  const int per = (packs.n + blocks - 1) / blocks;
  const int begin = min(packs.n, rank * per), end = min(packs.n, begin + per);
  const float c = kLog2e / a.temperature;

  // the first given tokens' logits are fetched along with the row
  int64_t tok0 = -1;
  float x0 = 0.f;
  if (rank == 0 && (int)threadIdx.x < a.M) {
    tok0 = a.tokens[row * a.M + threadIdx.x];
    if (tok0 >= 0 && tok0 < a.V) x0 = to_f32(x[tok0]);
  }

  Running run;
  float best = -INFINITY;
  int best_pack = -1;
  auto take = [&](const uint4& raw, int v) {
    const float mx = run.add<T>(raw, c);
    if (kTop && mx > best) best_pack = v;
    best = fmaxf(best, mx);
  };
  if constexpr (G <= 1) {
    int v = begin + threadIdx.x;
    if (v < end) best_pack = v;
    for (; v + (kUnroll - 1) * TH < end; v += kUnroll * TH) {
      uint4 raw[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) raw[i] = packs.raw(v + i * TH);
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) take(raw[i], v + i * TH);
    }
    for (; v < end; v += TH) take(packs.raw(v), v);
  } else {
    const bool wide = packs.wide(begin);
    int v = begin + G * (int)threadIdx.x;
    if (v < end) best_pack = v;
    for (; v + G - 1 < end; v += G * TH) {
      uint4 raw[G];
      packs.template some<G>(v, end, wide, raw);
#pragma unroll
      for (int i = 0; i < G; ++i) take(raw[i], v + i);
    }
    if (v < end)
      for (; v < end; ++v) take(packs.raw(v), v);
  }

  Sums acc = run.sums();
  const bool nan = acc.s != acc.s;
  float wb = best;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    acc = merged(acc, shfl_xor(acc, o), c);
    wb = fmaxf(wb, __shfl_xor_sync(0xffffffffu, wb, o));
  }
  if (lane == 0) warps[warp] = {acc, wb};
  if constexpr (kTop)
    block_top<T, TH, G>(packs, begin, end, a.k, best, best_pack, __syncthreads_or(nan), sh);
  else
    __syncthreads();
  if (blocks > 1) {
    cluster.barrier_wait();
    if (threadIdx.x == 0) {
      Part p = warps[0];
      for (int w = 1; w < W; ++w)
        p = {merged(p.sums, warps[w].sums, c), fmaxf(p.best, warps[w].best)};
      *cluster.map_shared_rank(&parts[rank], 0) = p;
    }
    if constexpr (kTop)
      for (int j = threadIdx.x; j < a.k; j += TH)
        *cluster.map_shared_rank(&sh.lists[rank][j], 0) = sh.list[j];
    cluster.sync();
    if (rank != 0) return;
  }
  if (threadIdx.x == 0) {
    const Part* from = blocks > 1 ? parts : warps;
    Part p = from[0];
    for (int i = 1; i < (blocks > 1 ? blocks : W); ++i)
      p = {merged(p.sums, from[i].sums, c), fmaxf(p.best, from[i].best)};
    float ln_s = 0.f, inv_s = 0.f, H = 0.f;
    if (p.sums.s != 0.f) {
      rebase(p.sums, p.best, c);
      ln_s = logf(p.sums.s);
      inv_s = 1.f / p.sums.s;
      H = ln_s - kLn2 * (p.sums.u / p.sums.s);
    }
    st[0] = p.best, st[1] = ln_s, st[2] = inv_s;
    a.ent[row] = H;
    if (a.stats) reinterpret_cast<float4*>(a.stats)[row] = make_float4(p.best, ln_s, inv_s, H);
  }
  if constexpr (kTop) {
    if (blocks > 1) {
      // of the blocks' lists, which share no element
      const int n = blocks * a.k;
      for (int i = threadIdx.x; i < n; i += TH) {
        const int q = i / a.k;
        const uint64_t mine = sh.lists[q][i - q * a.k];
        int above = i - q * a.k;
        for (int o = 0; o < blocks; ++o) {
          if (o == q) continue;
          int lo = 0, hi = a.k;               // entries of o above mine: lo..hi
          while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (sh.lists[o][mid] > mine)
              lo = mid + 1;
            else
              hi = mid;
          }
          above += lo;
        }
        if (mine && above < a.k) sh.list[above] = mine;
      }
    }
  }
  __syncthreads();
  const float m = st[0], ln_s = st[1], inv_s = st[2];
  for (int j = threadIdx.x; j < a.M; j += TH) {
    int64_t tok = tok0;
    float xt = x0;
    if (j != (int)threadIdx.x) {
      tok = a.tokens[row * a.M + j];
      if (tok >= 0 && tok < a.V) xt = to_f32(x[tok]);
    }
    a.logp[row * a.M + j] =
        (tok < 0 || tok >= a.V) ? 0.f : logp_of(xt, m, ln_s, inv_s, a.temperature);
  }
  if constexpr (kTop)
    for (int j = threadIdx.x; j < a.k; j += TH) {
      const uint64_t key = sh.list[j];
      a.top_tok[row * a.k + j] = (int64_t)(uint32_t)~(uint32_t)key;
      a.top_logp[row * a.k + j] =
          logp_of(of_order((uint32_t)(key >> 32)), m, ln_s, inv_s, a.temperature);
    }
}

// Rows of up to 32 P packs: a warp a row, which stays in its registers.  The k-th
// largest logit is built up bit by bit from counts over the warp; those above
// it and the first of those equal to it are ranked in shared memory.
template <typename T, int P, bool kTop>
__global__ void __launch_bounds__(kThreads) short_kernel(const Args a) {
  constexpr int N = Packs<T>::N;
  __shared__ uint64_t lists[kTop ? kThreads / 32 : 1][kMaxTop];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + warp;
  if (row >= a.rows) return;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld;
  const Packs<T> packs(x, a.V);
  const float c = kLog2e / a.temperature;
  uint4 raw[P];
#pragma unroll
  for (int i = 0; i < P; ++i)
    if (lane + 32 * i < packs.n) raw[i] = packs.raw(lane + 32 * i);
  int64_t tok0 = -1;
  float x0 = 0.f;
  if (lane < a.M) {
    tok0 = a.tokens[row * a.M + lane];
    if (tok0 >= 0 && tok0 < a.V) x0 = to_f32(x[tok0]);
  }
  Running run;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < P; ++i)
    if (lane + 32 * i < packs.n) m = fmaxf(m, run.add<T>(raw[i], c));
  Sums acc = run.sums();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    acc = merged(acc, shfl_xor(acc, o), c);
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  float ln_s = 0.f, inv_s = 0.f, H = 0.f;
  if (acc.s != 0.f) {
    rebase(acc, m, c);
    ln_s = logf(acc.s);
    inv_s = 1.f / acc.s;
    H = ln_s - kLn2 * (acc.u / acc.s);
  }
  if (lane == 0) {
    a.ent[row] = H;
    if (a.stats) reinterpret_cast<float4*>(a.stats)[row] = make_float4(m, ln_s, inv_s, H);
  }
  for (int j = lane; j < a.M; j += 32) {
    int64_t tok = tok0;
    float xt = x0;
    if (j != lane) {
      tok = a.tokens[row * a.M + j];
      if (tok >= 0 && tok < a.V) xt = to_f32(x[tok]);
    }
    a.logp[row * a.M + j] =
        (tok < 0 || tok >= a.V) ? 0.f : logp_of(xt, m, ln_s, inv_s, a.temperature);
  }
  if constexpr (kTop) {
    const int k = a.k;
    uint32_t ord[P * N];                 // 0: not of the row
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float f[N];
      vec::unpack<T, N>(raw[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int64_t e = packs.first(lane + 32 * i) + j;
        ord[i * N + j] =
            lane + 32 * i < packs.n && e >= 0 && e < a.V ? order_of(f[j]) : 0u;
      }
    }
    uint32_t tau = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t at = tau | (1u << bit);
      int n = 0;
#pragma unroll
      for (int i = 0; i < P * N; ++i) n += ord[i] >= at;
      n = __reduce_add_sync(0xffffffffu, n);
      if (n >= k) tau = at;
      if (n == k) break;
    }
    int over = 0;
#pragma unroll
    for (int i = 0; i < P * N; ++i) over += ord[i] > tau;
    const int need = k - __reduce_add_sync(0xffffffffu, over);    // of those equal to tau
    int base_over = 0, base_equal = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      int mine = 0;                      // above tau, and equal to it << 16
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t o = ord[i * N + j];
        mine += (o > tau) + ((o == tau && o != 0) << 16);
      }
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      const int before = upto - mine;
      int above = base_over + (before & 0xffff), equal = base_equal + (before >> 16);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t o = ord[i * N + j];
        const bool up = o > tau, eq = o == tau && o != 0;
        if (up || (eq && equal < need))
          lists[warp][above + min(equal, need)] = key_of(o, packs.first(lane + 32 * i) + j);
        above += up;
        equal += eq;
      }
      const int all = __shfl_sync(0xffffffffu, upto, 31);
      base_over += all & 0xffff;
      base_equal += all >> 16;
    }
    __syncwarp();
    for (int j = lane; j < k; j += 32) {
      const uint64_t key = lists[warp][j];
      int above = 0;
      for (int i = 0; i < k; ++i) above += lists[warp][i] > key;
      a.top_tok[row * k + above] = (int64_t)(uint32_t)~(uint32_t)key;
      a.top_logp[row * k + above] =
          logp_of(of_order((uint32_t)(key >> 32)), m, ln_s, inv_s, a.temperature);
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
  int chunks, per;                       // blocks of a row, packs of a block
};

// With t = (x - m) c (c = log2(e) / temperature), p = 2^t / s and
// logp = t ln 2 - ln s:
//   dx = 2^t (A + B t) + g / temperature at the given tokens,
//   A = -(G + g_H (H - ln s)) / (s temperature), B = -g_H ln 2 / (s temperature).
template <typename T, int TH>
__global__ void __launch_bounds__(TH) bwd_kernel(const BwdArgs a) {
  constexpr int N = Packs<T>::N;
  const int lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x / a.chunks;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld;
  T* dx = reinterpret_cast<T*>(a.dx) + row * a.V;
  const Packs<T> to(dx, a.V);              // packs by dx's alignment
  const bool same = Packs<T>(x, a.V).shift == to.shift;
  const int begin = min((int64_t)to.n, (int64_t)(blockIdx.x % a.chunks) * a.per);
  const int end = min((int64_t)to.n, (int64_t)begin + a.per);
  const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
  const bool empty = st.z == 0.f;
  const float c = kLog2e / a.temperature, inv_t = 1.f / a.temperature;
  const float ref = empty ? 0.f : st.x;
  const int n = a.M + (a.g_top ? a.k : 0);
  // entry j: a given token or an alternative
  auto token = [&](int j) {
    return j < a.M ? a.tokens[row * a.M + j] : a.top_tok[row * a.k + j - a.M];
  };
  auto grad = [&](int j) {
    return j < a.M ? (a.g_logp ? a.g_logp[row * a.M + j] : 0.f) : a.g_top[row * a.k + j - a.M];
  };
  float G = 0.f;
  for (int j = lane; j < n; j += 32) {
    const int64_t tok = token(j);
    if (tok >= 0 && tok < a.V) G += grad(j);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) G += __shfl_xor_sync(0xffffffffu, G, o);
  const float gH = a.g_ent ? a.g_ent[row] : 0.f;
  const float A = empty ? 0.f : -(G + gH * (st.w - st.y)) * st.z * inv_t;
  const float B = empty ? 0.f : -gH * kLn2 * st.z * inv_t;
  // Under 2^-126 the exponential is formed 2^100 times as large and the product
  // scaled back, so that it alone is rounded to a subnormal; the floor still
  // gives 0.
  auto base = [&](float v) {
    const float t = max_nan((v - ref) * c, kGradFloor);
    const bool low = t < -126.f;
    const float r = ex2(low ? t + 100.f : t) * fmaf(B, t, A);
    return low ? r * 0x1p-100f : r;
  };
  auto fetch = [&](int v) -> uint4 {
    if (same && to.whole(v))
      return __ldg(reinterpret_cast<const uint4*>(x - to.shift) + v);
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t e = to.first(v) + i;
      o[i] = (e >= 0 && e < a.V) ? to_f32(x[e]) : 0.f;
    }
    return vec::pack<T, N>(o);
  };
  auto leave = [&](const uint4& raw, int v) {
    float o[N];
    vec::unpack<T, N>(raw, o);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = base(o[i]);
    if (to.whole(v)) {
      vec::store<T, N>(dx + to.first(v), o);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t e = to.first(v) + i;
        if (e >= 0 && e < a.V) dx[e] = from_f32<T>(o[i]);
      }
    }
  };
  int v = begin + threadIdx.x;
  for (; v + (kUnroll - 1) * TH < end; v += kUnroll * TH) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) raw[i] = fetch(v + i * TH);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) leave(raw[i], v + i * TH);
  }
  for (; v < end; v += TH) leave(fetch(v), v);
  if (empty) return;
  __syncthreads();
  // the given tokens in this block's part: equal ones add up in order, by the first
  // of them (the others stop there: few steps where a row has many tokens)
  for (int j = threadIdx.x; j < n; j += TH) {
    const int64_t tok = token(j);
    if (tok < 0 || tok >= a.V || tok < to.first(begin) || tok >= to.first(end)) continue;
    bool first = true;
    for (int i = 0; i < j && first; ++i) first = token(i) != tok;
    if (!first) continue;
    float g = grad(j);
    for (int i = j + 1; i < n; ++i)
      if (token(i) == tok) g += grad(i);
    dx[tok] = from_f32<T>(fmaf(g, inv_t, base(to_f32(x[tok]))));
  }
}

// (statistics are stored and loaded as one 16-byte word a row)
bool bad(int64_t rows, int32_t V, int32_t M, int32_t k, const void* x, int64_t ld,
         const int64_t* tokens, float temperature, const float* stats) {
  return rows < 0 || rows > 0x7fffffff || V <= 0 || M < 0 || k < 0 || k > kMaxTop || k > V ||
         ld < V || !(temperature >= kMinTemperature && temperature <= kMaxTemperature) ||
         reinterpret_cast<uintptr_t>(stats) % 16 || (rows > 0 && (!x || (M > 0 && !tokens)));
}

// Blocks that share a row: enough that every SM has work, as long as each still
// has two packs a thread.
int cluster_of(int64_t rows, int64_t packs) {
  int c = 1;
  while (c < kMaxCluster && rows * c * 2 <= vec::kSMs * 8 && packs / (2 * c) >= 2 * kThreads)
    c *= 2;
  return c;
}

template <typename T, int TH, int G>
int launch_fwd(const Args& a, int c, cudaStream_t st) {
  if (a.rows * c > 0x7fffffff) return TT_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * c));
  cfg.blockDim = dim3(TH);
  cfg.dynamicSmemBytes = G ? sizeof(TopShared<TH>) : 0;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fwd_kernel<T, TH, G>, a) == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

template <typename T, int P>
int launch_short(const Args& a, cudaStream_t st) {
  constexpr int per = kThreads / 32;
  const int64_t blocks = (a.rows + per - 1) / per;
  if (a.k)
    short_kernel<T, P, true><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  else
    short_kernel<T, P, false><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  return TT_OK;
}

template <typename T>
int launch_fwd(const Args& a, cudaStream_t st) {
  const int64_t packs = a.V / Packs<T>::N;
  // a row may lie across two packs more than its size asks for; with alternatives,
  // a few rows are faster with more threads each (47 x 1,000 with 8: 6 us against
  // 11; 4,096 with 64: 62 against 34)
  if (a.k == 0 || a.rows >= 1024) {
    if (packs + 2 <= 32) return launch_short<T, 1>(a, st);
    if (packs + 2 <= 64) return launch_short<T, 2>(a, st);
    if (packs + 2 <= 128) return launch_short<T, 4>(a, st);
    if (packs + 2 <= 256) return launch_short<T, 8>(a, st);
  }
  // (64 threads' largest are too few to bound many alternatives well)
  if (packs <= kFewPacks && a.k <= 16)
    return a.k ? launch_fwd<T, kFewThreads, 1>(a, 1, st) : launch_fwd<T, kFewThreads, 0>(a, 1, st);
  const int c = cluster_of(a.rows, packs);
  if (a.k == 0) return launch_fwd<T, kThreads, 0>(a, c, st);
  return packs / c >= 16 * kThreads ? launch_fwd<T, kThreads, 4>(a, c, st)
                                    : launch_fwd<T, kThreads, 1>(a, c, st);
}

template <typename T, int TH>
int launch_bwd(BwdArgs& a, cudaStream_t st) {
  // a block takes 4 x kUnroll packs a thread; kUnroll where rows are few
  const int64_t packs = a.V / Packs<T>::N + 2;
  const int64_t one = (int64_t)kUnroll * TH;
  int64_t per = 4 * one;
  if (a.rows * ((packs + per - 1) / per) < vec::kSMs * 8) per = one;
  a.per = (int)per;
  a.chunks = (int)((packs + per - 1) / per);
  if (a.rows * a.chunks > 0x7fffffff) return TT_ERR_UNSUPPORTED;
  bwd_kernel<T, TH><<<(unsigned)(a.rows * a.chunks), TH, 0, st>>>(a);
  return TT_OK;
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
  if (bad(n_rows, vocab, n_tokens, top_k, logits, ld, tokens, temperature, stats) ||
      (n_rows > 0 && (!entropy || (n_tokens > 0 && !logprobs) ||
                      (top_k > 0 && (!top_logprobs || !top_tokens)))))
    return TT_ERR_INVALID_ARG;
  if (n_rows == 0) return TT_OK;
  Args a{n_rows, vocab, n_tokens, top_k, logits, ld, tokens, temperature,
         logprobs, entropy, top_logprobs, top_tokens, stats};
  const int rc = tt::vec::dispatch_float(dtype, [&](auto tag) -> int {
    return launch_fwd<decltype(tag)>(a, (cudaStream_t)stream);
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
  if (bad(n_rows, vocab, n_tokens, top_k, logits, ld, tokens, temperature, stats) ||
      (n_rows > 0 && (!stats || !dlogits || (g_top && top_k > 0 && !top_tokens))))
    return TT_ERR_INVALID_ARG;
  if (n_rows == 0) return TT_OK;
  BwdArgs a{n_rows, vocab, n_tokens, top_k, logits, ld, tokens, top_tokens, temperature,
            g_logprobs, g_entropy, g_top, stats, dlogits, 1, 0};
  const int rc = tt::vec::dispatch_float(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    return vocab / Packs<T>::N <= kFewPacks
               ? launch_bwd<T, kFewThreads>(a, (cudaStream_t)stream)
               : launch_bwd<T, kThreads>(a, (cudaStream_t)stream);
  });
  if (rc != TT_OK) return rc;
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}
