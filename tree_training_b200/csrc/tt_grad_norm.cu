// The norm of many tensors together, and the tensors scaled to a largest norm.
//
//   |g|_2 = sqrt(sum g^2),  |g|_1 = sum |g|,  |g|_inf = max |g|
//   out = g * min(1, max_norm / (|g| + eps))
//
// Bound by HBM: the norm reads every element, the scaling reads it again and
// writes it (3 n b bytes for what could do with 2 if it all stayed on the chip).
// The tensors' addresses and sizes travel in the launch's parameters, a table of
// up to kMaxTensors of them a launch; a chunk of them is a block's unit of work,
// found in the table by bisection: of 32 KB, or of 128 KB where there are enough of
// those for every block.
//
// Sums.  A pack's 16 bytes are added up in fp32 and the packs in fp64, so that
// neither the number of elements nor their size matters: a pack whose sum of
// squares leaves [2^-100, 2^120] is added up again in fp64.  Each block adds its
// chunks in order, and each launch after it adds the blocks' sums in order: the
// result does not depend on timing.
//
// Measured on a B200: 1.2e9 bf16 gradients in 74 tensors 1,140 us (norm 367, 6.5 TB/s;
// scaling 772, 6.2), 9.6e6 fp32 ones in 20 tensors 25 us.
#include <algorithm>
#include <cmath>

#include "tt_vec.cuh"

namespace tt {
namespace gradnorm {
namespace {

constexpr int kMaxTensors = 512;       // of a launch: a table of 14.9 KB
constexpr int kThreads = 512;
constexpr int64_t kChunkBytes = 32768, kLargeChunkBytes = 131072;
constexpr int kBlocks = 2 * vec::kSMs; // at most, of a launch: all that are resident
constexpr int kAhead = 4;              // packs of a thread that are fetched together

struct Table {
  const void* src[kMaxTensors];
  void* dst[kMaxTensors];
  int64_t n[kMaxTensors];              // elements
  int32_t first[kMaxTensors + 1];      // first chunk
  int8_t dtype[kMaxTensors];
  int32_t count, chunk_bytes;
};

enum Kind { kTwo = 0, kOne = 1, kInf = 2 };

template <typename T>
constexpr int pack_of() { return 16 / (int)sizeof(T); }

__device__ __forceinline__ double join(double a, double b, int kind) {
  if (kind != kInf) return a + b;
  return (a != a || b != b) ? a + b : fmax(a, b);   // (a maximum that keeps NaN)
}

// What a pack's V values add to the sum (the maximum).
template <int kind, int V>
__device__ __forceinline__ double pack_sum(const float (&v)[V]) {
  float s = 0.f;
  if constexpr (kind == kTwo) {
#pragma unroll
    for (int i = 0; i < V; ++i) s = fmaf(v[i], v[i], s);
    if (s >= 0x1p-100f && s <= 0x1p120f) return (double)s;
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) m = fmaxf(m, fabsf(v[i]));
    if (s == 0.f && m == 0.f) return 0.0;         // (rows of a table that had no token)
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) d = fma((double)v[i], (double)v[i], d);
    return d;
  }
  if constexpr (kind == kOne) {
#pragma unroll
    for (int i = 0; i < V; ++i) s += fabsf(v[i]);
    if (s <= 0x1p120f) return (double)s;
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) d += fabs((double)v[i]);
    return d;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) s = (v[i] != v[i] || s != s) ? s + v[i] : fmaxf(s, fabsf(v[i]));
  return (double)s;
}

__device__ __forceinline__ int tensor_of(const Table& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// The chunk's sum over this thread's elements.
template <int kind, typename T>
__device__ __forceinline__ double chunk_sum(const T* p, int64_t n) {
  constexpr int V = pack_of<T>();
  double sum = 0.0;
  // elements before the first 16-byte boundary, whole packs, the rest
  const int64_t lead =
      min(n, (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T));
  const int64_t packs = (n - lead) / V;
  auto one = [&](int64_t i) {
    const float v[1] = {to_f32(p[i])};
    sum = join(sum, pack_sum<kind, 1>(v), kind);
  };
  if ((int64_t)threadIdx.x < lead) one(threadIdx.x);
  const T* body = p + lead;
  for (int64_t i = threadIdx.x; i < packs; i += kThreads * kAhead) {
    vec::Raw<T, V> raw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j * kThreads < packs) raw[j] = vec::load_raw<T, V>(body + (i + j * kThreads) * V);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j * kThreads < packs) {
        float v[V];
        vec::unpack<T, V>(raw[j], v);
        sum = join(sum, pack_sum<kind, V>(v), kind);
      }
  }
  const int64_t at = lead + packs * V + threadIdx.x;
  if (at < n) one(at);
  return sum;
}

__device__ __forceinline__ double block_join(double v, int kind, double* sm) {
  for (int o = 16; o; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o), kind);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = sm[0];
    for (int w = 1; w < (int)blockDim.x / 32; ++w) all = join(all, sm[w], kind);
    sm[0] = all;
  }
  __syncthreads();
  return sm[0];
}

template <int kind>
__global__ void __launch_bounds__(kThreads, 2)
    norm_kernel(const __grid_constant__ Table t, double* part) {
  __shared__ double sm[kThreads / 32];
  vec::let_next_begin();
  double sum = 0.0;
  for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int i = tensor_of(t, c);
    const int64_t at = c - t.first[i];
    switch (t.dtype[i]) {
      case TT_F32: {
        const int64_t e = t.chunk_bytes / 4, n = min(e, t.n[i] - at * e);
        sum = join(sum, chunk_sum<kind>(reinterpret_cast<const float*>(t.src[i]) + at * e, n),
                   kind);
        break;
      }
      case TT_BF16: {
        const int64_t e = t.chunk_bytes / 2, n = min(e, t.n[i] - at * e);
        sum = join(
            sum, chunk_sum<kind>(reinterpret_cast<const __nv_bfloat16*>(t.src[i]) + at * e, n), kind);
        break;
      }
      default: {
        const int64_t e = t.chunk_bytes / 2, n = min(e, t.n[i] - at * e);
        sum = join(sum, chunk_sum<kind>(reinterpret_cast<const __half*>(t.src[i]) + at * e, n),
                   kind);
      }
    }
  }
  sum = block_join(sum, kind, sm);
  if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

// The norm of n blocks' sums, the same in every block that asks.
__device__ __forceinline__ double norm_of(const double* part, int n, int kind, double* sm) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) v = join(v, part[i], kind);
  v = block_join(v, kind, sm);
  return kind == kTwo ? sqrt(v) : v;
}

__global__ void __launch_bounds__(kThreads) finish_kernel(const double* part, int n, int kind,
                                                           float* norm) {
  __shared__ double sm[kThreads / 32];
  vec::wait_previous();
  const double v = norm_of(part, n, kind, sm);
  if (threadIdx.x == 0) *norm = (float)v;
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const T* p, T* q, int64_t n, float c) {
  constexpr int V = pack_of<T>();
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  if ((a & 15) != (b & 15)) {              // no pack is on a boundary of both
    for (int64_t i = threadIdx.x; i < n; i += kThreads) q[i] = from_f32<T>(to_f32(p[i]) * c);
    return;
  }
  const int64_t lead = min(n, (int64_t)((16 - (a & 15)) & 15) / (int)sizeof(T));
  const int64_t packs = (n - lead) / V;
  auto one = [&](int64_t i) { q[i] = from_f32<T>(to_f32(p[i]) * c); };
  if ((int64_t)threadIdx.x < lead) one(threadIdx.x);
  for (int64_t i = threadIdx.x; i < packs; i += kThreads * kAhead) {
    // (p and q may be one array: no read-only loads)
    uint4 raw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j * kThreads < packs)
        raw[j] = *reinterpret_cast<const uint4*>(p + lead + (i + j * kThreads) * V);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j * kThreads < packs) {
        float v[V];
        vec::unpack<T, V>(raw[j], v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] *= c;
        vec::store<T, V>(q + lead + (i + j * kThreads) * V, v);
      }
  }
  const int64_t at = lead + packs * V + threadIdx.x;
  if (at < n) one(at);
}

// Chunks from the last to the first: the norm's pass ends there, and what it
// read last is still in L2.
__global__ void __launch_bounds__(kThreads, 2)
    scale_kernel(const __grid_constant__ Table t, const double* part, int parts, int kind,
                 const float* given, float max_norm, float eps, float* norm, int in_place) {
  __shared__ double sm[kThreads / 32];
  vec::wait_previous();
  const float v = given ? *given : (float)norm_of(part, parts, kind, sm);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
  const float q = max_norm / (v + eps);
  const float c = q > 1.f ? 1.f : q;          // (NaN stays)
  if (in_place && c == 1.f) return;           // nothing would change
  for (int k = t.first[t.count] - 1 - (int)blockIdx.x; k >= 0; k -= gridDim.x) {
    const int i = tensor_of(t, k);
    const int64_t at = k - t.first[i];
    switch (t.dtype[i]) {
      case TT_F32: {
        const int64_t e = t.chunk_bytes / 4, n = min(e, t.n[i] - at * e);
        scale_chunk(reinterpret_cast<const float*>(t.src[i]) + at * e,
                    reinterpret_cast<float*>(t.dst[i]) + at * e, n, c);
        break;
      }
      case TT_BF16: {
        const int64_t e = t.chunk_bytes / 2, n = min(e, t.n[i] - at * e);
        scale_chunk(reinterpret_cast<const __nv_bfloat16*>(t.src[i]) + at * e,
                    reinterpret_cast<__nv_bfloat16*>(t.dst[i]) + at * e, n, c);
        break;
      }
      default: {
        const int64_t e = t.chunk_bytes / 2, n = min(e, t.n[i] - at * e);
        scale_chunk(reinterpret_cast<const __half*>(t.src[i]) + at * e,
                    reinterpret_cast<__half*>(t.dst[i]) + at * e, n, c);
      }
    }
  }
}

int size_of(int dtype) { return dtype == TT_F32 ? 4 : 2; }

int64_t chunk_bytes_of(int32_t count, const int32_t* dtypes, const int64_t* sizes) {
  int64_t all = 0;
  for (int32_t i = 0; i < count; ++i) all += sizes[i] * size_of(dtypes[i]);
  return all >= 8 * kBlocks * kLargeChunkBytes ? kLargeChunkBytes : kChunkBytes;
}

// Fills the table with tensors from `at` on, as many as fit: the next one.
int32_t fill(Table* t, int32_t at, int32_t count, const int32_t* dtypes, const int64_t* sizes,
             const void* const* src, void* const* dst, int64_t chunk_bytes) {
  t->count = 0;
  t->chunk_bytes = (int32_t)chunk_bytes;
  int64_t chunks = 0;
  for (; at < count && t->count < kMaxTensors; ++at) {
    if (sizes[at] == 0) continue;
    const int64_t e = chunk_bytes / size_of(dtypes[at]), c = (sizes[at] + e - 1) / e;
    if (chunks + c > 0x7fffffff) break;
    t->src[t->count] = src[at];
    t->dst[t->count] = dst ? dst[at] : nullptr;
    t->n[t->count] = sizes[at];
    t->dtype[t->count] = (int8_t)dtypes[at];
    t->first[t->count++] = (int32_t)chunks;
    chunks += c;
  }
  t->first[t->count] = (int32_t)chunks;
  return at;
}

int blocks_of(const Table& t) { return std::min<int64_t>(kBlocks, t.first[t.count]); }

int check(int32_t count, const int32_t* dtypes, const int64_t* sizes, const void* const* src) {
  if (count < 0 || (count > 0 && (!dtypes || !sizes || !src))) return TT_ERR_INVALID_ARG;
  for (int32_t i = 0; i < count; ++i) {
    if (dtypes[i] < TT_F32 || dtypes[i] > TT_F16) return TT_ERR_UNSUPPORTED;
    // (a tensor's chunks, and a launch's past its last, are counted in 32 bits)
    if (sizes[i] < 0 || sizes[i] > ((int64_t)1 << 43) || (sizes[i] > 0 && !src[i]))
      return TT_ERR_INVALID_ARG;
    const uintptr_t b = dtypes[i] == TT_F32 ? 3 : 1;
    if (reinterpret_cast<uintptr_t>(src[i]) & b) return TT_ERR_INVALID_ARG;
  }
  return TT_OK;
}

int kind_of(double p) {
  if (p == 2.0) return kTwo;
  if (p == 1.0) return kOne;
  return std::isinf(p) && p > 0 ? kInf : -1;
}

// Launches the norm's passes; *parts: how many blocks' sums there are.
int norm_passes(int32_t count, const int32_t* dtypes, const int64_t* sizes, const void* const* src,
                int kind, double* part, int64_t room, int* parts, cudaStream_t st) {
  Table t;
  const int64_t chunk = chunk_bytes_of(count, dtypes, sizes);
  *parts = 0;
  for (int32_t at = 0; at < count;) {
    at = fill(&t, at, count, dtypes, sizes, src, nullptr, chunk);
    if (t.count == 0) continue;
    const int blocks = blocks_of(t);
    if (*parts + blocks > room) return TT_ERR_WORKSPACE;
    if (kind == kTwo) norm_kernel<kTwo><<<blocks, kThreads, 0, st>>>(t, part + *parts);
    else if (kind == kOne) norm_kernel<kOne><<<blocks, kThreads, 0, st>>>(t, part + *parts);
    else norm_kernel<kInf><<<blocks, kThreads, 0, st>>>(t, part + *parts);
    tt_count_launches(1);
    *parts += blocks;
  }
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

}  // namespace
}  // namespace gradnorm
}  // namespace tt

using namespace tt::gradnorm;

extern "C" int64_t tt_grad_norm_workspace_size(int32_t count) {
  if (count < 0) return 0;
  return ((int64_t)count / kMaxTensors + 1) * kBlocks * (int64_t)sizeof(double);
}

extern "C" int tt_grad_norm(int32_t count, const int32_t* dtypes, const int64_t* sizes,
                            const void* const* tensors, double norm_type, float* norm,
                            void* workspace, int64_t workspace_bytes, void* stream) {
  const int kind = kind_of(norm_type);
  if (kind < 0 || !norm || (reinterpret_cast<uintptr_t>(workspace) & 7)) return TT_ERR_INVALID_ARG;
  if (const int rc = check(count, dtypes, sizes, tensors)) return rc;
  if (!workspace || workspace_bytes < tt_grad_norm_workspace_size(count)) return TT_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  int parts = 0;
  double* part = (double*)workspace;
  if (const int rc = norm_passes(count, dtypes, sizes, tensors, kind, part, workspace_bytes / 8,
                                 &parts, st))
    return rc;
  if (tt::vec::launch_next(finish_kernel, 1, kThreads, 0, st, part, parts, kind, norm) !=
      cudaSuccess)
    return TT_ERR_CUDA;
  tt_count_launches(1);
  return TT_OK;
}

extern "C" int tt_clip_grad_norm(int32_t count, const int32_t* dtypes, const int64_t* sizes,
                                 const void* const* tensors, void* const* outs, double norm_type,
                                 const float* given_norm, float max_norm, float eps, float* norm,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  const int kind = kind_of(norm_type);
  if (kind < 0 || !norm || (reinterpret_cast<uintptr_t>(workspace) & 7)) return TT_ERR_INVALID_ARG;
  if (const int rc = check(count, dtypes, sizes, tensors)) return rc;
  if (const int rc = check(count, dtypes, sizes, outs)) return rc;
  if (!workspace || workspace_bytes < tt_grad_norm_workspace_size(count)) return TT_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  int parts = 0;
  double* part = (double*)workspace;
  if (!given_norm)
    if (const int rc = norm_passes(count, dtypes, sizes, tensors, kind, part, workspace_bytes / 8,
                                   &parts, st))
      return rc;
  int in_place = 1;
  for (int32_t i = 0; i < count; ++i) in_place &= tensors[i] == outs[i];
  Table t;
  const int64_t chunk = kChunkBytes;
  bool first = true;
  int32_t at = 0;
  do {
    at = fill(&t, at, count, dtypes, sizes, tensors, outs, chunk);
    if (t.count == 0 && !first) break;
    if (tt::vec::launch_next(scale_kernel, std::max(1, blocks_of(t)), kThreads, 0, st, t, part,
                             parts, kind, given_norm, max_norm, eps, first ? norm : nullptr,
                             in_place) != cudaSuccess)
      return TT_ERR_CUDA;
    tt_count_launches(1);
    first = false;
  } while (at < count);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}
