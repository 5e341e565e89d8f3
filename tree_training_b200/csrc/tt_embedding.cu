// Rows of an embedding table, scaled, and the table's gradient.
//
//   y[t] = scale * W[id[t]]
//   dW[v] = scale * sum of dy[t] over the t with id[t] = v, in the order of t
//
// Bound by HBM.  Forward: a token's row is read and written once.  Backward: every
// row of dW is written (the words of no token as zeros), which is most of its
// traffic, and dy is read once.  The sum goes by sorted tokens: two or three stable
// counting sorts by ten bits of the id each (the sort of the experts' plan), so
// that a word's rows stand next to one another in the order of the tokens.
#include <algorithm>

#include "tt_vec.cuh"

namespace tt {
namespace embed {
namespace {

constexpr int kDigits = 1024;          // of a counting sort
constexpr int kBits = 10;

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

// The digit of each entry's id in the order given (null: as they are); -1 for an
// entry without a row.
__global__ void __launch_bounds__(256)
    digits_kernel(const void* ids, int ids64, int64_t n, int64_t V, int64_t padding,
                  const int32_t* order, int shift, int32_t* digits) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t t = order ? order[i] : i;
  int32_t d = -1;
  if (t >= 0) {
    const int64_t id = id_at(ids, ids64, t);
    if (id >= 0 && id < V && id != padding) d = (int32_t)((id >> shift) & (kDigits - 1));
  }
  digits[i] = d;
}

// The entries sorted by one more digit.
__global__ void __launch_bounds__(256)
    follow_kernel(const int32_t* order, const int32_t* entries, int64_t n, int32_t* next) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int32_t e = entries[i];
  next[i] = e < 0 ? -1 : order[e];
}

// Where each word's entries begin in the sorted order; -1 (as cleared) for others.
__global__ void __launch_bounds__(256)
    heads_kernel(const void* ids, int ids64, int64_t n, const int32_t* order, int32_t* first) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n || order[i] < 0) return;
  const int64_t id = id_at(ids, ids64, order[i]);
  if (i == 0 || id_at(ids, ids64, order[i - 1]) != id) first[id] = (int32_t)i;
}

struct Sum {
  const void* ids;
  int ids64;
  int64_t n, V;
  int H;
  const int32_t *order, *first;
  const void* dy;
  int64_t ld;
  float scale;
  void* dw;
};

// A block a word.
template <typename T>
__global__ void __launch_bounds__(128) sum_kernel(const Sum a) {
  for (int64_t v = blockIdx.x; v < a.V; v += gridDim.x) {
    const int32_t first = a.first[v];
    for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
      float s = 0.f;
      if (first >= 0)
        for (int64_t i = first; i < a.n && a.order[i] >= 0; ++i) {
          const int64_t t = a.order[i];
          if (id_at(a.ids, a.ids64, t) != v) break;
          s += to_f32(reinterpret_cast<const T*>(a.dy)[t * a.ld + c]);
        }
      reinterpret_cast<T*>(a.dw)[v * a.H + c] = from_f32<T>(s * a.scale);
    }
  }
}

int digits_of(int64_t V) {
  int d = 1;
  while (d < 4 && ((int64_t)1 << (kBits * d)) < V) ++d;
  return d;
}

int64_t round16(int64_t b) { return (b + 15) / 16 * 16; }

bool ok_sizes(int64_t n, int64_t V, int H) {
  return n >= 0 && n <= 0x7fffffff && V >= 1 && V <= 0x7fffffff && H >= 1;
}

}  // namespace
}  // namespace embed
}  // namespace tt

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

extern "C" int64_t tt_embedding_bwd_workspace_size(int64_t n, int64_t V) {
  if (!ok_sizes(n, V, 1)) return 0;
  // digits, slots, entries, two orders; first rows; the sort's offsets and counts
  return 5 * round16(4 * n) + round16(4 * V) + round16(4 * (kDigits + 1)) +
         round16(tt_moe_plan_workspace_size(n, kDigits));
}

extern "C" int tt_embedding_bwd(int dtype, int64_t n, int64_t V, int32_t H, const void* ids,
                                int ids64, const void* dy, int64_t dy_ld, float scale,
                                int64_t padding_idx, void* dweight, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  if (!ok_sizes(n, V, H) || (n > 1 && dy_ld < H)) return TT_ERR_INVALID_ARG;
  if (!dweight || (n > 0 && (!ids || !dy))) return TT_ERR_INVALID_ARG;
  if (workspace_bytes < tt_embedding_bwd_workspace_size(n, V) || !workspace)
    return TT_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  char* p = (char*)workspace;
  auto take = [&](int64_t bytes) {
    char* q = p;
    p += round16(bytes);
    return q;
  };
  int32_t* digits = (int32_t*)take(4 * n);
  int32_t* slots = (int32_t*)take(4 * n);
  int32_t* entries = (int32_t*)take(4 * n);
  int32_t* orders[2] = {(int32_t*)take(4 * n), (int32_t*)take(4 * n)};
  int32_t* first = (int32_t*)take(4 * V);
  int32_t* offsets = (int32_t*)take(4 * (kDigits + 1));
  const int64_t plan_bytes = tt_moe_plan_workspace_size(n, kDigits);
  return tt::vec::dispatch_float(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const unsigned blocks = (unsigned)((n + 255) / 256);
    const int32_t* order = nullptr;
    if (cudaMemsetAsync(first, 0xff, 4 * V, st) != cudaSuccess) return TT_ERR_CUDA;
    if (n > 0) {
      for (int d = 0; d < digits_of(V); ++d) {
        digits_kernel<<<blocks, 256, 0, st>>>(ids, ids64, n, V, padding_idx, order, kBits * d,
                                              digits);
        int32_t* next = orders[d & 1];
        int32_t* to = d == 0 ? next : entries;
        if (const int rc = tt_moe_plan(digits, 0, n, kDigits, slots, to, offsets, p, plan_bytes,
                                       st))
          return rc;
        if (d > 0) follow_kernel<<<blocks, 256, 0, st>>>(order, entries, n, next);
        order = next;
        tt_count_launches(d > 0 ? 2 : 1);
      }
      heads_kernel<<<blocks, 256, 0, st>>>(ids, ids64, n, order, first);
      tt_count_launches(1);
    }
    const Sum a{ids, ids64, n, V, H, order, first, dy, dy_ld, scale, dweight};
    sum_kernel<T><<<(unsigned)std::min<int64_t>(V, 16 * tt::vec::kSMs), 128, 0, st>>>(a);
    tt_count_launches(1);
    return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
  });
}
