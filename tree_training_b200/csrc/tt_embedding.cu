// Rows of an embedding table, scaled, and the table's gradient.
//
//   y[t] = scale * W[id[t]]
//   dW[v] = scale * sum of dy[t] over the t with id[t] = v, in the order of t
//
// Bound by HBM.  Forward: a token's row is read and written once.  Backward: every
// row of dW is written (the words of no token as zeros), which is most of its
// traffic, and dy is read once.
//
// The gradient's sum goes by sorted tokens: stable counting sorts by up to ten bits of
// the id each, two launches a sort (as the experts' plan), so that a word's rows stand
// next to one another in the order of the tokens.  The sorted rows are cut into chunks
// of up to 32, whatever words they hold, so that a word of half the text is summed by as many
// blocks as its rows are; sums of words that reach over a chunk's end leave as fp32
// parts and are added up in order by a last launch.  The sorts are bound by latency
// (20 us for 32,768 tokens): the rows of words without tokens, which a bitmap of the
// first launch tells, are zeroed by further blocks of the launches after it.  The
// launches begin while the one before ends (so what that one writes is not read through
// the read-only path).
//
// Measured on a B200, bf16, forward and backward: 32,768 tokens of 151,936 x 2,560 259 us
// (48 forward; 1.05 GB backward: 5.0 TB/s), 32,768 of 32,000 x 1,024 about 150.
#include <algorithm>

#include "tt_vec.cuh"

namespace tt {
namespace embed {
namespace {

constexpr int kBits = 10;              // of a counting sort, at most

__device__ __forceinline__ int64_t id_at(const void* ids, int ids64, int64_t t) {
  return ids64 ? reinterpret_cast<const int64_t*>(ids)[t]
               : (int64_t) reinterpret_cast<const int32_t*>(ids)[t];
}

struct Rows {
  const void* ids;
  int ids64;
  int64_t n, V;
  int H;
  const void* w;
  int64_t ld;
  float scale;
  void* y;
  int32_t* status;
};

// A warp a row, in packs of 16 bytes of y; where rows of y or W are not on 16-byte
// boundaries, the packs of y that the row covers, its ends by elements.
template <typename T>
__global__ void __launch_bounds__(256) rows_kernel(const Rows a) {
  constexpr int V = 16 / (int)sizeof(T);
  const T* lo = reinterpret_cast<const T*>(a.w);
  const T* hi = lo + (a.V - 1) * a.ld + a.H;
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
  for (int64_t t = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; t < a.n;
       t += warps) {
    const int64_t id = id_at(a.ids, a.ids64, t);
    T* y = reinterpret_cast<T*>(a.y) + t * a.H;
    if (id < 0 || id >= a.V) {                 // no such row
      if (lane == 0) set_status(a.status, TT_ERR_INVALID_ARG);
      for (int i = lane; i < a.H; i += 32) y[i] = from_f32<T>(__int_as_float(0x7fc00000));
      continue;
    }
    const T* w = lo + id * a.ld;
    // the first element on a 16-byte boundary of y, and those before it
    const int ahead = (int)(reinterpret_cast<uintptr_t>(y) & 15) / (int)sizeof(T);
    for (int e0 = lane * V - ahead; e0 < a.H; e0 += 32 * V) {
      uint4 raw = vec::load_any_of<T>(w, e0, a.H, lo, hi);
      if (a.scale != 1.f) {
        float v[V];
        vec::unpack<T, V>(raw, v);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= a.scale;
        raw = vec::pack<T, V>(v);
      }
      vec::store_part<T>(y, e0, a.H, raw);
    }
  }
}

// ---- the gradient -------------------------------------------------------------

constexpr int kWarps = 8;              // of a sorting block
constexpr int kSteps = 8;              // of 32 entries, fetched together
constexpr int kPlaceThreads = 512;
constexpr int kMaxChunk = 32;

struct Grad {
  const void* ids;
  int ids64;
  int64_t n, V, padding;
  int H;
  const void* dy;
  int64_t ld;
  float scale;
  void* dw;
  uint32_t* used;                      // [V / 32]: words with tokens
  int32_t *slots, *counts;             // of the sorts
  float* parts;                        // [chunks][2][part_ld]
  int64_t part_ld, chunks;
  int chunk;                           // sorted rows of a group of threads
  int2* ends;                          // [chunks]: kBegins, kThrough; the word
};

enum { kBegins = 1, kThrough = 2 };    // a word begins in the chunk and goes on behind it;
                                       // fills it and goes on on both sides

// The entry's word, -1 where it has no gradient.
__device__ __forceinline__ int32_t word_of(const Grad& a, int64_t t) {
  if (t < 0) return -1;
  const int64_t id = id_at(a.ids, a.ids64, t);
  return id >= 0 && id < a.V && id != a.padding ? (int32_t)id : -1;
}

// Zeroes the rows of the words without tokens: share `part` of `parts`, by the blocks
// `block` of `blocks`, a warp a row.
template <typename T>
__device__ __forceinline__ void zero_rows(const Grad& a, int part, int parts, int block,
                                          int blocks) {
  constexpr int N = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 31, warps = blockDim.x / 32;
  const int64_t per = (a.V + parts - 1) / parts;
  const int64_t end = min(a.V, (part + 1) * per);
  for (int64_t v = part * per + (int64_t)block * warps + threadIdx.x / 32; v < end;
       v += (int64_t)blocks * warps) {
    if ((a.used[v >> 5] >> (v & 31)) & 1) continue;
    T* row = reinterpret_cast<T*>(a.dw) + v * a.H;
    const int ahead = (int)(reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T);
    for (int e0 = lane * N - ahead; e0 < a.H; e0 += 32 * N)
      vec::store_part<T>(row, e0, a.H, make_uint4(0, 0, 0, 0));
  }
}

// One counting sort of the entries (order: as the sort before left them; null: as
// they are) by the digit at `shift`; entries without a word go last.
struct Sort {
  const int32_t* order;
  int32_t* next;
  int shift, digits;                   // digits: how many; that one is "no word"
  int64_t run;                         // entries of a warp
  int blocks;                          // that sort; further ones zero rows
  int part, parts;                     // the share of rows (parts 0: none)
};

__device__ __forceinline__ int digit_of(const Sort& s, int32_t word) {
  return word < 0 ? s.digits : (word >> s.shift) & (s.digits - 1);
}

// The lanes whose e is this lane's, by one vote a bit.
__device__ __forceinline__ unsigned same_as(int e, int bits) {
  unsigned m = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const bool one = (e >> b) & 1;
    const unsigned v = __ballot_sync(0xffffffffu, one);
    m &= one ? v : ~v;
  }
  return m;
}

// Each entry's rank among its block's entries of the same digit, the blocks' counts,
// and (first sort) the bitmap of words.
template <typename T, bool kFirst>
__global__ void __launch_bounds__(32 * kWarps) rank_kernel(const Grad a, const Sort s) {
  extern __shared__ int hist[];               // [warps][digits + 1]: counts, then ranks
  vec::let_next_begin();
  if (!kFirst) vec::wait_previous();
  if ((int)blockIdx.x >= s.blocks) {
    zero_rows<T>(a, s.part, s.parts, blockIdx.x - s.blocks, gridDim.x - s.blocks);
    return;
  }
  const int E = s.digits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t begin = min(a.n, ((int64_t)blockIdx.x * kWarps + warp) * s.run);
  const int64_t end = min(a.n, begin + s.run);
  for (int i = threadIdx.x; i < kWarps * (E + 1); i += blockDim.x) hist[i] = 0;
  __syncthreads();
  int* mine = hist + warp * (E + 1);
  const int bits = 32 - __clz(E + 1);
  int e[kSteps];
  unsigned same[kSteps];
  auto fetch = [&](int64_t from, bool mark) {
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const int64_t i = from + j * 32 + lane;
      e[j] = E + 1;
      if (i < end) {
        const int32_t w = word_of(a, s.order ? s.order[i] : i);
        e[j] = digit_of(s, w);
        // (most tokens are of words that are marked already: a third of a text's, and all
        // its atomics, may be on one address)
        if (kFirst && mark && w >= 0 && !((__ldcg(a.used + (w >> 5)) >> (w & 31)) & 1))
          atomicOr(a.used + (w >> 5), 1u << (w & 31));
      }
    }
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
      if (from + j * 32 < end) same[j] = same_as(e[j], bits);
  };
  for (int64_t from = begin; from < end; from += 32 * kSteps) {
    fetch(from, true);
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
      if (e[j] <= E && lane == __ffs(same[j]) - 1) atomicAdd(mine + e[j], __popc(same[j]));
  }
  __syncthreads();
  for (int x = threadIdx.x; x <= E; x += blockDim.x) {
    int all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int c = hist[w * (E + 1) + x];
      hist[w * (E + 1) + x] = all;
      all += c;
    }
    a.counts[(int64_t)blockIdx.x * (E + 1) + x] = all;
  }
  __syncthreads();
  // (each step's leaders add theirs before the lanes part again for the next step's)
  const bool kept = end - begin <= 32 * kSteps;        // the digits are still in e
  for (int64_t from = begin; from < end; from += 32 * kSteps) {
    if (!kept) fetch(from, false);
    int base[kSteps];
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      base[j] = 0;
      if (e[j] <= E && lane == __ffs(same[j]) - 1)
        base[j] = atomicAdd(mine + e[j], __popc(same[j]));
      __syncwarp();
    }
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const int64_t i = from + j * 32 + lane;
      if (from + j * 32 >= end) continue;
      const int rank = __shfl_sync(0xffffffffu, base[j], __ffs(same[j]) - 1) +
                       __popc(same[j] & ((1u << lane) - 1));
      if (e[j] <= E) a.slots[i] = rank;
    }
  }
}

// The entries in their places: the blocks' counts added up, then the ranks.
template <typename T>
__global__ void __launch_bounds__(kPlaceThreads) place_kernel(const Grad a, const Sort s) {
  extern __shared__ int sm[];
  vec::let_next_begin();
  vec::wait_previous();
  if ((int)blockIdx.x >= s.blocks) {
    zero_rows<T>(a, s.part, s.parts, blockIdx.x - s.blocks, gridDim.x - s.blocks);
    return;
  }
  const int E = s.digits, b0 = blockIdx.x;
  int* total = sm;                            // [E + 1]
  int* first = sm + E + 1;                    // [E + 1]: this block's first rows
  __shared__ int warp_sum[kPlaceThreads / 32];
  const int parts = max(1, (int)blockDim.x / (E + 1)), share = (s.blocks + parts - 1) / parts;
  for (int x = threadIdx.x; x < 2 * (E + 1); x += blockDim.x) sm[x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < parts * (E + 1); i += blockDim.x) {
    const int part = i / (E + 1), x = i - part * (E + 1);
    const int end = min(s.blocks, (part + 1) * share);
    int all = 0, before = 0;
    for (int b = part * share; b < end; b += 16) {
      int c[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        c[j] = b + j < end ? __ldcg(a.counts + (int64_t)(b + j) * (E + 1) + x) : 0;
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
  const int x0 = min((int)threadIdx.x * per, E + 1), x1 = min(x0 + per, E + 1);
  int sum = 0;
  for (int x = x0; x < x1; ++x) sum += total[x];
  int scan = sum;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += up;
  }
  if (lane == 31) warp_sum[warp] = scan;
  __syncthreads();
  int at = scan - sum;
  for (int w = 0; w < warp; ++w) at += warp_sum[w];
  for (int x = x0; x < x1; ++x) {
    first[x] += at;
    at += total[x];
  }
  __syncthreads();
  const int64_t begin = min(a.n, (int64_t)b0 * kWarps * s.run);
  const int64_t end = min(a.n, begin + kWarps * s.run);
  for (int64_t i = begin + threadIdx.x; i < end; i += blockDim.x) {
    const int64_t t = s.order ? s.order[i] : i;
    const int32_t w = word_of(a, t);
    s.next[first[digit_of(s, w)] + a.slots[i]] = w < 0 ? -1 : (int32_t)t;
  }
}

// Adds up the sorted rows: a group of threads (whole warps) a chunk, a thread the
// elements e0 .. of its word's row, on 16-byte boundaries of dW; columns beyond the
// group's by gridDim.y.  Further blocks zero rows.
template <typename T, bool kAligned>
__global__ void __launch_bounds__(512)
    sum_kernel(const Grad a, const int32_t* order, int group, int sum_blocks, int part,
               int parts_of_rows) {
  constexpr int N = 16 / (int)sizeof(T);
  constexpr int kAhead = kAligned ? 8 : 4;    // rows fetched together
  vec::let_next_begin();
  vec::wait_previous();
  if ((int)blockIdx.x >= sum_blocks) {
    if (blockIdx.y == 0)
      zero_rows<T>(a, part, parts_of_rows, blockIdx.x - sum_blocks, gridDim.x - sum_blocks);
    return;
  }
  const int g = threadIdx.x / group, tid = threadIdx.x - g * group, lane = threadIdx.x & 31;
  const int64_t chunk = (int64_t)blockIdx.x * (blockDim.x / group) + g;
  if (chunk >= a.chunks) return;
  const int64_t r0 = chunk * a.chunk;
  const int rows = (int)min((int64_t)a.chunk, a.n - r0);
  const int32_t my_t = lane < rows ? order[r0 + lane] : -1;
  const int32_t my_w = word_of(a, my_t);
  const int32_t before = r0 > 0 ? word_of(a, order[r0 - 1]) : -1;
  const int32_t after = r0 + rows < a.n ? word_of(a, order[r0 + rows]) : -1;
  const T* dy = reinterpret_cast<const T*>(a.dy);
  const T* lo = dy;
  const T* hi = dy + (a.n - 1) * a.ld + a.H;
  const int64_t col = ((int64_t)blockIdx.y * group + tid) * N;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  // elements of dW before a row's 16-byte boundary (the packs begin there)
  auto ahead_of = [&](int32_t w) {
    return kAligned ? 0
                    : (int)(reinterpret_cast<uintptr_t>(reinterpret_cast<T*>(a.dw) +
                                                        (int64_t)w * a.H) & 15) / (int)sizeof(T);
  };
  int from = 0;                               // where the word's rows begin in the chunk
  for (int r = 0; r < rows; r += kAhead) {
    uint4 raw[kAhead];
    int32_t w[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int at = min(r + j, kMaxChunk - 1);
      const int32_t t = __shfl_sync(0xffffffffu, my_t, at);
      w[j] = r + j < rows ? __shfl_sync(0xffffffffu, my_w, at) : -1;
      raw[j] = make_uint4(0, 0, 0, 0);
      if (w[j] >= 0) {
        if constexpr (kAligned) {
          if (col < a.H) raw[j] = __ldg(reinterpret_cast<const uint4*>(dy + t * a.ld + col));
        } else {
          const int64_t e0 = col - ahead_of(w[j]);
          if (e0 < a.H) raw[j] = vec::load_any_of<T>(dy + t * a.ld, e0, a.H, lo, hi);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (w[j] < 0) continue;                 // (past the last word, too: they are sorted last)
      float v[N];
      vec::unpack<T, N>(raw[j], v);
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += v[i];
      const int here = r + j;
      const int32_t next = here + 1 < rows ? __shfl_sync(0xffffffffu, my_w, here + 1) : after;
      if (next == w[j]) continue;
      // the word's last row: whole, or the end of a sum that began before
      const bool whole = from > 0 || before != w[j];
      if (whole) {
        const int64_t e0 = col - ahead_of(w[j]);
        if (e0 < a.H) {
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] *= a.scale;
          T* row = reinterpret_cast<T*>(a.dw) + (int64_t)w[j] * a.H;
          if constexpr (kAligned) vec::store<T, N>(row + col, acc);
          else vec::store_part<T>(row, e0, a.H, vec::pack<T, N>(acc));
        }
      } else if (col < a.part_ld) {
        float* p = a.parts + (chunk * 2) * a.part_ld + col;
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = acc[i];
      }
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.f;
      from = here + 1;
    }
  }
  // a word that goes on in the next chunk (after whole chunks of it: from == 0)
  const int32_t last = __shfl_sync(0xffffffffu, my_w, rows - 1);
  const bool goes_on = last >= 0 && last == after, began = from > 0 || before != last;
  if (tid == 0 && blockIdx.y == 0)
    a.ends[chunk] = make_int2(!goes_on ? 0 : began ? kBegins : kThrough, last);
  if (goes_on && col < a.part_ld) {
    float* p = a.parts + (chunk * 2 + (began ? 1 : 0)) * a.part_ld + col;
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = acc[i];
  }
}

constexpr int kJoinWarps = 16;

constexpr int kShort = 8;              // parts that one warp adds up

// The chunk in which the word ends that begins in `chunk` and goes on behind it: the
// first that it does not go through.
__device__ __forceinline__ int64_t ends_in(const Grad& a, int64_t chunk) {
  for (int64_t last = chunk + 1;; last += 32) {
    const int64_t c = last + (threadIdx.x & 31);
    const unsigned stop = __ballot_sync(0xffffffffu, c >= a.chunks || a.ends[c].x != kThrough);
    if (stop) return last + __ffs(stop) - 1;
  }
}

// Parts begin .. end of a word's (slot 1 of the chunk it begins in, slot 0 of those
// after it), at columns col ...
template <int N>
__device__ __forceinline__ void add_parts(const Grad& a, int64_t chunk, int64_t begin, int64_t end,
                                          int64_t col, float (&acc)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  if (col >= a.part_ld) return;
#pragma unroll 8
  for (int64_t k = begin; k < end; ++k) {
    const float4* q = reinterpret_cast<const float4*>(
        a.parts + ((chunk + k) * 2 + (k == 0 ? 1 : 0)) * a.part_ld + col);
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = __ldcg(q + i / 4);
      acc[i] += x.x, acc[i + 1] += x.y, acc[i + 2] += x.z, acc[i + 3] += x.w;
    }
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_sum(const Grad& a, int32_t w, int64_t col, float (&acc)[N]) {
  T* row = reinterpret_cast<T*>(a.dw) + (int64_t)w * a.H;
  const int64_t e0 = col - (int)(reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T);
  if (col >= a.part_ld || e0 >= a.H) return;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] *= a.scale;
  vec::store_part<T>(row, e0, a.H, vec::pack<T, N>(acc));
}

// The sums that reach over chunks (blockIdx.y: columns): the chunks in which such a
// word begins are shared out over the blocks, which look for theirs first. A word of
// few parts is one warp's; of a longer one the warps add up runs of the parts, and the
// first warp the runs' sums, in order.
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const Grad a) {
  constexpr int N = 16 / (int)sizeof(T);
  constexpr int kThreads = 32 * kJoinWarps;
  __shared__ float sm[kJoinWarps][32][N + 1];
  __shared__ int64_t mine[kThreads], longer[kThreads];
  __shared__ int count, longer_count;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t col = ((int64_t)blockIdx.y * 32 + lane) * N;
  float acc[N];
  vec::wait_previous();
  for (int64_t base = blockIdx.x; base < a.chunks; base += (int64_t)kThreads * gridDim.x) {
    if (threadIdx.x == 0) count = longer_count = 0;
    __syncthreads();
    const int64_t c = base + (int64_t)threadIdx.x * gridDim.x;
    if (c < a.chunks && a.ends[c].x == kBegins) mine[atomicAdd(&count, 1)] = c;
    __syncthreads();
    for (int i = warp; i < count; i += kJoinWarps) {
      const int64_t chunk = mine[i], n = ends_in(a, chunk) - chunk + 1;
      if (n > kShort) {
        if (lane == 0) longer[atomicAdd(&longer_count, 1)] = chunk;
        continue;
      }
      add_parts<N>(a, chunk, 0, n, col, acc);
      store_sum<T, N>(a, a.ends[chunk].y, col, acc);
    }
    __syncthreads();
    for (int i = 0; i < longer_count; ++i) {
      const int64_t chunk = longer[i], n = ends_in(a, chunk) - chunk + 1;
      const int64_t run = (n + kJoinWarps - 1) / kJoinWarps;
      add_parts<N>(a, chunk, warp * run, min(n, (warp + 1) * run), col, acc);
#pragma unroll
      for (int x = 0; x < N; ++x) sm[warp][lane][x] = acc[x];
      __syncthreads();
      if (warp == 0) {
        for (int w = 1; w < kJoinWarps; ++w)
#pragma unroll
          for (int x = 0; x < N; ++x) acc[x] += sm[w][lane][x];
        store_sum<T, N>(a, a.ends[chunk].y, col, acc);
      }
      __syncthreads();
    }
  }
}

// ---- host ---------------------------------------------------------------------

// Sorts, and the bits of each one's digit.
int sorts_of(int64_t V, int* bits) {
  int all = 1;
  while (((int64_t)1 << all) < V) ++all;
  const int sorts = (all + kBits - 1) / kBits;
  *bits = (all + sorts - 1) / sorts;
  return sorts;
}

// Blocks of a sort (each adds up `blocks` counts a digit).
int sort_blocks(int64_t n, int digits) {
  const int64_t most = std::max<int64_t>(8, std::min<int64_t>(64, 32768 / (digits + 1)));
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, (n + 32 * kWarps - 1) / (32 * kWarps)));
}

int64_t round16(int64_t b) { return (b + 15) / 16 * 16; }

bool ok_sizes(int64_t n, int64_t V, int H) {
  // (the gradient's columns are shared out over the grid's second side, of 65,535 blocks)
  return n >= 0 && n <= 0x7fffffff && V >= 1 && V <= 0x7fffffff && H >= 1 && H <= (1 << 22);
}

}  // namespace
}  // namespace embed
}  // namespace tt

using namespace tt;
using namespace tt::embed;

extern "C" int tt_embedding_fwd(int dtype, int64_t n, int64_t V, int32_t H, const void* ids,
                                int ids64, const void* weight, int64_t ld, float scale, void* y,
                                int32_t* status, void* stream) {
  if (!ok_sizes(n, V, H) || ld < H) return TT_ERR_INVALID_ARG;
  if (n > 0 && (!ids || !weight || !y)) return TT_ERR_INVALID_ARG;
  return tt::vec::dispatch_float(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (n == 0) return TT_OK;
    const Rows a{ids, ids64, n, V, H, weight, ld, scale, y, status};
    const int64_t blocks = std::min<int64_t>((n + 7) / 8, 16 * tt::vec::kSMs);
    rows_kernel<T><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(a);
    tt_count_launches(1);
    return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
  });
}

namespace {

// (the packs of a row of dW that begins off a 16-byte boundary: one more)
int64_t part_ld(int32_t H) { return (H + 7) / 8 * 8 + 8; }

struct Layout {
  int64_t used, slots, order, counts, parts, ends, all;
  int chunk;
  Layout(int64_t n, int64_t V, int32_t H) {
    int bits;
    sorts_of(V, &bits);
    used = round16((V + 31) / 32 * 4);
    slots = round16(4 * n);
    order = round16(4 * n);
    counts = round16((int64_t)sort_blocks(n, 1 << bits) * ((1 << bits) + 1) * 4);
    // smaller chunks where there are few rows: about a thousand threads an SM
    chunk = kMaxChunk;
    while (chunk > 4 && n / chunk * ((H + 255) / 256 * 32) < (int64_t)1024 * vec::kSMs) chunk /= 2;
    const int64_t chunks = (n + chunk - 1) / chunk;
    parts = chunks * 2 * part_ld(H) * 4;
    ends = round16(chunks * 8);
    all = used + slots + 2 * order + counts + parts + ends;
  }
};

template <typename T>
int gradient(Grad a, int32_t* const* orders, cudaStream_t st) {
  int bits;
  const int sorts = sorts_of(a.V, &bits), digits = 1 << bits;
  const int blocks = sort_blocks(a.n, digits);
  const int64_t warps = (int64_t)blocks * kWarps;
  // every launch but the first zeroes a share of the rows
  const int shares = 2 * sorts;
  const int64_t bytes = a.V * a.H * (int64_t)sizeof(T) / shares;
  const int zero_blocks = (int)std::max<int64_t>(1, std::min<int64_t>(4 * vec::kSMs, bytes >> 13));
  Sort s{};
  s.digits = digits, s.blocks = blocks, s.parts = shares;
  s.run = std::max<int64_t>(32, ((a.n + warps - 1) / warps + 31) / 32 * 32);
  const size_t rank_smem = sizeof(int) * kWarps * (digits + 1);
  const size_t place_smem = sizeof(int) * 2 * (digits + 1);
  const int32_t* order = nullptr;
  for (int d = 0; d < sorts; ++d) {
    s.order = order, s.next = orders[d & 1], s.shift = bits * d;
    if (d == 0) {
      rank_kernel<T, true><<<blocks, 32 * kWarps, rank_smem, st>>>(a, s);
    } else {
      if (vec::launch_next(rank_kernel<T, false>, blocks + zero_blocks, 32 * kWarps, rank_smem, st,
                           a, s) != cudaSuccess)
        return TT_ERR_CUDA;
      ++s.part;
    }
    if (vec::launch_next(place_kernel<T>, blocks + zero_blocks, kPlaceThreads, place_smem, st, a,
                         s) != cudaSuccess)
      return TT_ERR_CUDA;
    ++s.part;
    tt_count_launches(2);
    order = s.next;
  }
  constexpr int N = 16 / (int)sizeof(T);
  const bool aligned = a.H % N == 0 && a.ld % N == 0 &&
                       ((reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.dw)) &
                        15) == 0;
  const int packs = (int)((a.H + N - 1) / N) + (aligned ? 0 : 1);
  const int group = std::min(512, (packs + 31) / 32 * 32);
  const int groups = std::max(1, 256 / group);
  const unsigned cols = (unsigned)((packs + group - 1) / group);
  const int64_t sum_blocks = (a.chunks + groups - 1) / groups;
  const dim3 grid((unsigned)(sum_blocks + zero_blocks), cols);
  if (vec::launch_next(aligned ? sum_kernel<T, true> : sum_kernel<T, false>, grid, group * groups,
                       0, st, a, order, group, (int)sum_blocks, s.part, shares) != cudaSuccess)
    return TT_ERR_CUDA;
  tt_count_launches(1);
  if (a.chunks > 1) {
    const int64_t cols = (a.part_ld / N + 31) / 32;
    const int64_t blocks = std::max<int64_t>(1, std::min(a.chunks, 4 * vec::kSMs / cols));
    if (vec::launch_next(join_kernel<T>, dim3((unsigned)blocks, (unsigned)cols), 32 * kJoinWarps, 0,
                         st, a) != cudaSuccess)
      return TT_ERR_CUDA;
    tt_count_launches(1);
  }
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

}  // namespace

extern "C" int64_t tt_embedding_bwd_workspace_size(int64_t n, int64_t V, int32_t H) {
  if (!ok_sizes(n, V, H)) return 0;
  return Layout(n, V, H).all;
}

extern "C" int tt_embedding_bwd(int dtype, int64_t n, int64_t V, int32_t H, const void* ids,
                                int ids64, const void* dy, int64_t dy_ld, float scale,
                                int64_t padding_idx, void* dweight, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  if (!ok_sizes(n, V, H) || (n > 1 && dy_ld < H)) return TT_ERR_INVALID_ARG;
  if (!dweight || (n > 0 && (!ids || !dy)) || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return TT_ERR_INVALID_ARG;
  if (dtype < TT_F32 || dtype > TT_F16) return TT_ERR_UNSUPPORTED;
  const Layout l(n, V, H);
  if (workspace_bytes < l.all || !workspace) return TT_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  char* p = (char*)workspace;
  Grad a{ids, ids64, n, V, padding_idx, H, dy, dy_ld, scale, dweight};
  a.used = (uint32_t*)p, p += l.used;
  a.slots = (int32_t*)p, p += l.slots;
  int32_t* orders[2] = {(int32_t*)p, (int32_t*)(p + l.order)};
  p += 2 * l.order;
  a.counts = (int32_t*)p, p += l.counts;
  a.ends = (int2*)p, p += l.ends;
  a.parts = (float*)p, a.part_ld = part_ld(H);
  a.chunk = l.chunk, a.chunks = (n + l.chunk - 1) / l.chunk;
  if (cudaMemsetAsync(a.used, 0, l.used, st) != cudaSuccess) return TT_ERR_CUDA;
  return tt::vec::dispatch_float(dtype, [&](auto t) -> int {
    return gradient<decltype(t)>(a, orders, st);
  });
}
