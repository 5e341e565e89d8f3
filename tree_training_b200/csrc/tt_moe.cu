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
#include <algorithm>

#include "tt_vec.cuh"

namespace tt {
namespace moe {
namespace {

// ---- plan --------------------------------------------------------------------

constexpr int kPlanWarps = 8;
constexpr int kMaxExperts = 1024;
constexpr int kChunk = 2048;       // entries of a block, at least

__device__ __forceinline__ int expert_of(const void* ids, int ids64, int64_t i, int E) {
  const int64_t e = ids64 ? reinterpret_cast<const int64_t*>(ids)[i]
                          : reinterpret_cast<const int32_t*>(ids)[i];
  return (e >= 0 && e < E) ? (int)e : E;      // E: dropped, sorted behind the others
}

// Entries [begin, end) of a warp: hist[e] += their number of each expert.
__device__ __forceinline__ void warp_count(const void* ids, int ids64, int64_t begin, int64_t end,
                                           int E, int* hist) {
  const int lane = threadIdx.x & 31;
  for (int64_t i0 = begin; i0 < end; i0 += 32) {
    const int64_t i = i0 + lane;
    const int e = i < end ? expert_of(ids, ids64, i, E) : E + 1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e <= E && lane == __ffs(same) - 1) hist[e] += __popc(same);
    __syncwarp();
  }
}

// Block b's entries are [b chunk, (b + 1) chunk), warp w's the w-th eighth.
__device__ __forceinline__ void warp_range(int64_t n, int64_t chunk, int64_t* begin, int64_t* end) {
  const int64_t part = chunk / kPlanWarps;
  const int64_t b = blockIdx.x * chunk + (threadIdx.x >> 5) * part;
  *begin = min(b, n);
  *end = min(b + part, n);
}

__global__ void __launch_bounds__(32 * kPlanWarps)
plan_count(const void* ids, int ids64, int64_t n, int64_t chunk, int E, int* __restrict__ counts) {
  extern __shared__ int hist[];              // [warps][E + 1]
  for (int i = threadIdx.x; i < kPlanWarps * (E + 1); i += blockDim.x) hist[i] = 0;
  __syncthreads();
  int64_t begin, end;
  warp_range(n, chunk, &begin, &end);
  warp_count(ids, ids64, begin, end, E, hist + (threadIdx.x >> 5) * (E + 1));
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += blockDim.x) {
    int s = 0;
    for (int w = 0; w < kPlanWarps; ++w) s += hist[w * (E + 1) + e];
    counts[(int64_t)blockIdx.x * (E + 1) + e] = s;
  }
}

// counts: [blocks][E + 1] of plan_count, or null with a single block (which
// then counts for itself).
__global__ void __launch_bounds__(32 * kPlanWarps)
plan_place(const void* ids, int ids64, int64_t n, int64_t chunk, int E,
           const int* __restrict__ counts, int32_t* __restrict__ slots,
           int32_t* __restrict__ entries, int32_t* __restrict__ offsets) {
  extern __shared__ int sm[];
  int* hist = sm;                            // [warps][E + 1], then first rows
  int* total = sm + kPlanWarps * (E + 1);    // [E + 1]
  int* before = total + (E + 1);             // [E + 1]: in earlier blocks
  __shared__ int warp_sum[kPlanWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kPlanWarps * (E + 1); i += blockDim.x) hist[i] = 0;
  __syncthreads();
  int64_t begin, end;
  warp_range(n, chunk, &begin, &end);
  int* mine = hist + warp * (E + 1);
  warp_count(ids, ids64, begin, end, E, mine);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += blockDim.x) {
    int all = 0, pre = 0;
    if (counts) {
      for (int b = 0; b < (int)gridDim.x; ++b) {
        const int c = counts[(int64_t)b * (E + 1) + e];
        if (b < (int)blockIdx.x) pre += c;
        all += c;
      }
    } else {
      for (int w = 0; w < kPlanWarps; ++w) all += hist[w * (E + 1) + e];
    }
    total[e] = all;
    before[e] = pre;
  }
  __syncthreads();
  // exclusive sum of total over the experts: each thread a run of them
  const int per = (E + 1 + (int)blockDim.x - 1) / (int)blockDim.x;
  const int e0 = min((int)threadIdx.x * per, E + 1), e1 = min(e0 + per, E + 1);
  int run = 0;
  for (int e = e0; e < e1; ++e) run += total[e];
  int scan = run;
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += up;
  }
  if (lane == 31) warp_sum[warp] = scan;
  __syncthreads();
  int first = scan - run;
  for (int w = 0; w < warp; ++w) first += warp_sum[w];
  for (int e = e0; e < e1; ++e) {
    const int c = total[e];
    if (blockIdx.x == 0) offsets[e] = first;   // offsets[E]: the rows that are kept
    int at = first + before[e];
    for (int w = 0; w < kPlanWarps; ++w) {
      const int h = hist[w * (E + 1) + e];
      hist[w * (E + 1) + e] = at;
      at += h;
    }
    first += c;
  }
  __syncthreads();
  for (int64_t i0 = begin; i0 < end; i0 += 32) {
    const int64_t i = i0 + lane;
    const int e = i < end ? expert_of(ids, ids64, i, E) : E + 1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int base = e <= E ? mine[e] : 0;
    __syncwarp();
    if (e <= E) {
      const int row = base + __popc(same & ((1u << lane) - 1));
      slots[i] = e < E ? row : -1;
      entries[row] = e < E ? (int32_t)i : -1;
      if (lane == __ffs(same) - 1) mine[e] = base + __popc(same);
    }
    __syncwarp();
  }
}

// ---- rows --------------------------------------------------------------------

struct Args {
  int64_t T;
  int K, H, E;
  int group;                 // threads of a token
  const int32_t *slots, *offsets;
  const void *src, *ys;      // by token (dispatch, spread) or by row (collect, combine)
  void *dst, *dw;
  const void* w;
  int w_dtype;
};

__device__ __forceinline__ float weight_of(const void* w, int dtype, int64_t i) {
  switch (dtype) {
    case TT_F32: return reinterpret_cast<const float*>(w)[i];
    case TT_BF16: return to_f32(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
    default: return to_f32(reinterpret_cast<const __half*>(w)[i]);
  }
}

// Zeroes the rows past the last kept one; the blocks share them out.
template <typename T, int V>
__device__ __forceinline__ void zero_tail(const Args& a) {
  const int64_t n = a.T * a.K;
  const int64_t kept = a.offsets[a.E];
  const int packs = a.H / V;
  float z[V];
#pragma unroll
  for (int i = 0; i < V; ++i) z[i] = 0.f;
  for (int64_t r = kept + blockIdx.x; r < n; r += gridDim.x)
    for (int p = threadIdx.x; p < packs; p += blockDim.x)
      vec::store<T, V>(reinterpret_cast<T*>(a.dst) + r * a.H + p * V, z);
}

template <typename T, int V>
__global__ void __launch_bounds__(256) dispatch_kernel(const Args a) {
  const int t = threadIdx.x % a.group;
  const int64_t tok = (int64_t)blockIdx.x * (blockDim.x / a.group) + threadIdx.x / a.group;
  const int packs = a.H / V;
  if (tok < a.T) {
    const T* src = reinterpret_cast<const T*>(a.src) + tok * a.H;
    const int32_t* slot = a.slots + tok * a.K;
    for (int p = t; p < packs; p += a.group) {
      const vec::Raw<T, V> v = vec::load_raw<T, V>(src + p * V);
      for (int k = 0; k < a.K; ++k) {
        const int64_t r = __ldg(slot + k);
        if (r >= 0)
          *reinterpret_cast<vec::Raw<T, V>*>(reinterpret_cast<T*>(a.dst) + r * a.H + p * V) = v;
      }
    }
  }
  zero_tail<T, V>(a);
}

// kWeighted: combine, else collect.
template <typename T, int V, bool kWeighted>
__global__ void __launch_bounds__(256) combine_kernel(const Args a) {
  const int t = threadIdx.x % a.group;
  const int64_t tok = (int64_t)blockIdx.x * (blockDim.x / a.group) + threadIdx.x / a.group;
  if (tok >= a.T) return;
  const int packs = a.H / V;
  const int32_t* slot = a.slots + tok * a.K;
  for (int p = t; p < packs; p += a.group) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int k = 0; k < a.K; ++k) {
      const int64_t r = __ldg(slot + k);
      if (r < 0) continue;
      const float w = kWeighted ? weight_of(a.w, a.w_dtype, tok * a.K + k) : 1.f;
      float v[V];
      vec::load<T, V>(reinterpret_cast<const T*>(a.src) + r * a.H + p * V, v);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = fmaf(w, v[i], acc[i]);
    }
    vec::store<T, V>(reinterpret_cast<T*>(a.dst) + tok * a.H + p * V, acc);
  }
}

constexpr int kDots = 8;     // dw terms summed at a time

template <typename T, int V>
__global__ void __launch_bounds__(256) spread_kernel(const Args a) {
  __shared__ float red[8][kDots];
  const int t = threadIdx.x % a.group, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t tok = (int64_t)blockIdx.x * (blockDim.x / a.group) + threadIdx.x / a.group;
  const bool live = tok < a.T;
  const int packs = a.H / V;
  const int32_t* slot = a.slots + (live ? tok : 0) * a.K;
  for (int k0 = 0; k0 < a.K; k0 += kDots) {
    const int nk = min(kDots, a.K - k0);
    float dot[kDots];
#pragma unroll
    for (int k = 0; k < kDots; ++k) dot[k] = 0.f;
    if (live) {
      for (int p = t; p < packs; p += a.group) {
        float g[V];
        vec::load<T, V>(reinterpret_cast<const T*>(a.src) + tok * a.H + p * V, g);
#pragma unroll
        for (int k = 0; k < kDots; ++k) {
          if (k >= nk) continue;
          const int64_t r = __ldg(slot + k0 + k);
          if (r < 0) continue;
          const float w = weight_of(a.w, a.w_dtype, tok * a.K + k0 + k);
          float v[V], o[V];
          vec::load<T, V>(reinterpret_cast<const T*>(a.ys) + r * a.H + p * V, v);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            dot[k] = fmaf(g[i], v[i], dot[k]);
            o[i] = w * g[i];
          }
          vec::store<T, V>(reinterpret_cast<T*>(a.dst) + r * a.H + p * V, o);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kDots; ++k)
      for (int o = 16; o > 0; o >>= 1) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], o);
    __syncthreads();
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < kDots; ++k) red[warp][k] = dot[k];
    }
    __syncthreads();
    if (live && t < nk) {
      const int nw = a.group >> 5;
      float s = 0.f;
      for (int q = 0; q < nw; ++q) s += red[warp + q][t];
      const int64_t i = tok * a.K + k0 + t;
      switch (a.w_dtype) {
        case TT_F32: reinterpret_cast<float*>(a.dw)[i] = s; break;
        case TT_BF16: reinterpret_cast<__nv_bfloat16*>(a.dw)[i] = from_f32<__nv_bfloat16>(s); break;
        default: reinterpret_cast<__half*>(a.dw)[i] = from_f32<__half>(s); break;
      }
    }
  }
  zero_tail<T, V>(a);
}

enum Op { kDispatch, kCollect, kCombine, kSpread };

template <typename T, int V>
int launch(Op op, Args& a, cudaStream_t st) {
  // a group of whole warps, 8 warps a block: as many as the row has packs for
  const int packs = a.H / V;
  a.group = 32;
  while (a.group < 256 && a.group < packs) a.group *= 2;
  const int per = 256 / a.group;
  const int64_t blocks = (a.T + per - 1) / per;
  if (blocks > 0x7fffffff) return TT_ERR_UNSUPPORTED;
  switch (op) {
    case kDispatch: dispatch_kernel<T, V><<<(unsigned)blocks, 256, 0, st>>>(a); break;
    case kCollect: combine_kernel<T, V, false><<<(unsigned)blocks, 256, 0, st>>>(a); break;
    case kCombine: combine_kernel<T, V, true><<<(unsigned)blocks, 256, 0, st>>>(a); break;
    case kSpread: spread_kernel<T, V><<<(unsigned)blocks, 256, 0, st>>>(a); break;
  }
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

int run(Op op, int dtype, Args& a, void* stream) {
  if (a.T < 0 || a.K < 0 || a.H <= 0 || a.E <= 0 || a.T * a.K > 0x7fffffff)
    return TT_ERR_INVALID_ARG;
  if (a.T == 0) return TT_OK;
  // with K = 0 there are no sorted rows: the side of them may be null
  const bool by_token = op == kDispatch || op == kSpread;      // src is
  if (!a.offsets || (a.K > 0 && !a.slots) || (!a.src && (by_token || a.K > 0)) ||
      (!a.dst && (!by_token || a.K > 0)))
    return TT_ERR_INVALID_ARG;
  if (by_token && a.K == 0) return TT_OK;
  return vec::dispatch_float(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    constexpr int V = 16 / (int)sizeof(T);
    auto ok = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    if (a.H % V == 0 && ok(a.src) && ok(a.dst) && ok(a.ys))
      return launch<T, V>(op, a, (cudaStream_t)stream);
    return launch<T, 1>(op, a, (cudaStream_t)stream);
  });
}

int plan_blocks(int64_t n) {
  return (int)std::max<int64_t>(1, std::min<int64_t>((n + kChunk - 1) / kChunk, vec::kSMs));
}

}  // namespace
}  // namespace moe
}  // namespace tt

extern "C" int64_t tt_moe_plan_workspace_size(int64_t n_entries, int32_t n_experts) {
  if (n_entries < 0 || n_experts <= 0 || n_experts > tt::moe::kMaxExperts) return -1;
  return (int64_t)tt::moe::plan_blocks(n_entries) * (n_experts + 1) * 4;
}

extern "C" int tt_moe_plan(const void* ids, int ids64, int64_t n_entries, int32_t n_experts,
                           int32_t* slots, int32_t* entries, int32_t* offsets, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  using namespace tt::moe;
  if (n_entries < 0 || n_entries > 0x7fffffff || n_experts <= 0 || n_experts > kMaxExperts ||
      !offsets || (n_entries > 0 && (!ids || !slots || !entries)))
    return TT_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const int blocks = plan_blocks(n_entries);
  // a warp's share is a whole number of 32-entry steps
  const int64_t step = 32 * kPlanWarps;
  const int64_t chunk = std::max<int64_t>(
      step, ((n_entries + blocks - 1) / blocks + step - 1) / step * step);
  const int E = n_experts;
  if (blocks > 1 && (!workspace || workspace_bytes < tt_moe_plan_workspace_size(n_entries, E)))
    return TT_ERR_WORKSPACE;
  int* counts = blocks > 1 ? (int*)workspace : nullptr;
  if (counts)
    plan_count<<<blocks, 32 * kPlanWarps, sizeof(int) * kPlanWarps * (E + 1), st>>>(
        ids, ids64, n_entries, chunk, E, counts);
  plan_place<<<blocks, 32 * kPlanWarps, sizeof(int) * (kPlanWarps + 2) * (E + 1), st>>>(
      ids, ids64, n_entries, chunk, E, counts, slots, entries, offsets);
  tt_count_launches(counts ? 2 : 1);
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
