// Rotary positions for q and k in one pass: pairs (a, b) of the first R dims of
// every head turn by the angle of the token's position,
//   a' = a cos - b sin,   b' = b cos + a sin,
// the other D - R dims are copied.  A pair is (i, i + R/2) in the half layout
// and (2i, 2i + 1) in the interleaved one.  The gradient is the same turn with
// -sin.  cos and sin come from a table [positions, R] (R/2 cosines, R/2 sines)
// in fp32, whose rows carry any scaling for long contexts; the arithmetic is
// fp32 with one rounding at the store.
//
// A unit is V pairs of one head (two V-element packs, 16 bytes each where the
// sizes allow).  A thread holds the V cosines and sines of its (token, unit)
// in registers and walks over the heads, so the table is read once per token
// and head group.  Bound by HBM.  Measured on a B200, each way: 32,768 tokens, 32 +
// 8 heads of 128, bf16: 115 us (5.8 TB/s; at the rate of a copy 107); 8,191 tokens,
// 16 + 2 heads of 256 of which 64 dims turn, interleaved, views of a packed
// projection: 28 us (24); 47 tokens: 2.2 us.
#include <algorithm>

#include "tt_vec.cuh"

namespace tt {
namespace rotary {
namespace {

constexpr int kThreads = 256;

struct Args {
  int64_t n_tok, n_pos;
  int hq, hk, D, R;
  int units_rot, units;       // units of the turned part, all units of a head
  int tok_per_block, heads_per_group;
  const void *q, *k;
  int64_t q_st, q_sh, k_st, k_sh;
  const void* pos;
  int pos64;
  const float* table;
  float sin_sign;
  void *q_out, *k_out;
  int32_t* status;
};

// One product rounded, the other fused: the same bits in every variant.
__device__ __forceinline__ void turn_pair(float a, float b, float c, float s, float& x, float& y) {
  x = fmaf(a, c, -__fmul_rn(b, s));
  y = fmaf(b, c, __fmul_rn(a, s));
}

template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Args a) {
  const int half = a.R / 2;
  const int heads = a.hq + a.hk;
  const int h0 = blockIdx.y * a.heads_per_group;
  const int h1 = min(heads, h0 + a.heads_per_group);
  const int64_t t0 = (int64_t)blockIdx.x * a.tok_per_block;
  const int n = (int)min((int64_t)a.tok_per_block, a.n_tok - t0) * a.units;
  for (int idx = threadIdx.x; idx < n; idx += kThreads) {
    const int64_t tok = t0 + idx / a.units;
    const int u = idx % a.units;
    const bool turn = u < a.units_rot;
    // the two packs of this unit, as element offsets within a head
    int o0, o1;
    bool two = true;
    float c[V], s[V];
    if (turn) {
      o0 = kInterleaved ? 2 * u * V : u * V;
      o1 = kInterleaved ? o0 + V : half + u * V;
      const int64_t p = a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[tok]
                                : reinterpret_cast<const int32_t*>(a.pos)[tok];
      if (p >= 0 && p < a.n_pos) {
        const float* row = a.table + p * a.R + u * V;
        constexpr int W = V < 4 ? V : 4;
#pragma unroll
        for (int i = 0; i < V; i += W) {
          float cw[W], sw[W];
          vec::load<float, W>(row + i, cw);
          vec::load<float, W>(row + half + i, sw);
#pragma unroll
          for (int j = 0; j < W; ++j) {
            c[i + j] = cw[j];
            s[i + j] = a.sin_sign * sw[j];
          }
        }
      } else {
        // no such row: the turned dims become NaN and the host is told
        if (h0 == 0 && u == 0) set_status(a.status, TT_ERR_INVALID_ARG);
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
      }
    } else {
      o0 = a.R + (u - a.units_rot) * 2 * V;
      o1 = o0 + V;
      two = o1 < a.D;
      if (!two) o1 = o0;
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = 1.f, s[i] = 0.f;
    }
    for (int h = h0; h < h1; ++h) {
      const bool is_q = h < a.hq;
      const int hh = is_q ? h : h - a.hq;
      const T* src = is_q ? reinterpret_cast<const T*>(a.q) + tok * a.q_st + hh * a.q_sh
                          : reinterpret_cast<const T*>(a.k) + tok * a.k_st + hh * a.k_sh;
      T* dst = is_q ? reinterpret_cast<T*>(a.q_out) + (tok * a.hq + hh) * a.D
                    : reinterpret_cast<T*>(a.k_out) + (tok * a.hk + hh) * a.D;
      const vec::Raw<T, V> r0 = vec::load_raw<T, V>(src + o0);
      const vec::Raw<T, V> r1 = vec::load_raw<T, V>(src + o1);
      if (!turn) {
        *reinterpret_cast<vec::Raw<T, V>*>(dst + o0) = r0;
        if (two) *reinterpret_cast<vec::Raw<T, V>*>(dst + o1) = r1;
        continue;
      }
      float x0[V], x1[V], y0[V], y1[V];
      vec::unpack<T, V>(r0, x0);
      vec::unpack<T, V>(r1, x1);
      if constexpr (!kInterleaved || V == 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) turn_pair(x0[i], x1[i], c[i], s[i], y0[i], y1[i]);
      } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          turn_pair(x0[i], x0[i + 1], c[i / 2], s[i / 2], y0[i], y0[i + 1]);
          turn_pair(x1[i], x1[i + 1], c[(V + i) / 2], s[(V + i) / 2], y1[i], y1[i + 1]);
        }
      }
      vec::store<T, V>(dst + o0, y0);
      vec::store<T, V>(dst + o1, y1);
    }
  }
}

template <typename T, int V>
int launch(Args& a, bool interleaved, cudaStream_t st) {
  a.units_rot = a.R / 2 / V;
  a.units = a.units_rot + (a.D - a.R + 2 * V - 1) / (2 * V);
  a.tok_per_block = std::max(1, kThreads / a.units);
  const int64_t blocks = (a.n_tok + a.tok_per_block - 1) / a.tok_per_block;
  if (blocks > 0x7fffffff) return TT_ERR_UNSUPPORTED;
  const int heads = a.hq + a.hk;
  // few tokens: the heads are shared out over more blocks
  const int64_t want = std::max<int64_t>(1, 8ll * vec::kSMs / blocks);
  const int groups = (int)std::min<int64_t>(heads, want);
  a.heads_per_group = (heads + groups - 1) / groups;
  dim3 grid((unsigned)blocks, (unsigned)((heads + a.heads_per_group - 1) / a.heads_per_group));
  if (interleaved)
    rotary_kernel<T, V, true><<<grid, kThreads, 0, st>>>(a);
  else
    rotary_kernel<T, V, false><<<grid, kThreads, 0, st>>>(a);
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

}  // namespace
}  // namespace rotary
}  // namespace tt

extern "C" int tt_rotary(int dtype, int64_t n_tok, int32_t hq, int32_t hk, int32_t D, int32_t R,
                         int interleaved, int inverse, const void* q, int64_t q_st, int64_t q_sh,
                         const void* k, int64_t k_st, int64_t k_sh, const void* positions,
                         int positions64, const float* table, int64_t n_positions, void* q_out,
                         void* k_out, int32_t* status, void* stream) {
  using namespace tt::rotary;
  // 65,535: the most head groups a grid takes; 65,536: offsets within a head stay small
  if (n_tok < 0 || hq < 0 || hk < 0 || hq + (int64_t)hk <= 0 || hq + (int64_t)hk > 65535 ||
      D <= 0 || D > 65536 || R < 2 || R > D || (R & 1) || n_positions < 0)
    return TT_ERR_INVALID_ARG;
  if (n_tok == 0) return TT_OK;
  if (!positions || !table || (hq > 0 && (!q || !q_out)) || (hk > 0 && (!k || !k_out)))
    return TT_ERR_INVALID_ARG;
  Args a{};
  a.n_tok = n_tok, a.n_pos = n_positions;
  a.hq = hq, a.hk = hk, a.D = D, a.R = R;
  a.q = q, a.k = k, a.q_st = q_st, a.q_sh = q_sh, a.k_st = k_st, a.k_sh = k_sh;
  a.pos = positions, a.pos64 = positions64, a.table = table;
  a.sin_sign = inverse ? -1.f : 1.f;
  a.q_out = q_out, a.k_out = k_out, a.status = status;
  cudaStream_t st = (cudaStream_t)stream;
  return tt::vec::dispatch_float(dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    // the widest pack that divides every size and stride and that every base
    // address is a multiple of
    auto fits = [&](int v) {
      const int64_t bytes = v * (int64_t)sizeof(T);
      auto ok = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
      return (R / 2) % v == 0 && (D - R) % v == 0 && D % v == 0 && q_st % v == 0 &&
             q_sh % v == 0 && k_st % v == 0 && k_sh % v == 0 && ok(q) && ok(k) && ok(q_out) &&
             ok(k_out) && reinterpret_cast<uintptr_t>(table) % (4 * std::min(v, 4)) == 0;
    };
    if constexpr (sizeof(T) == 2)
      if (fits(8)) return launch<T, 8>(a, interleaved, st);
    if (fits(4)) return launch<T, 4>(a, interleaved, st);
    if (fits(2)) return launch<T, 2>(a, interleaved, st);
    return launch<T, 1>(a, interleaved, st);
  });
}
