// Matrix products of 16-bit factors into C, 16-bit or fp32.
#include "tt_gemm_sm100.cuh"

namespace tt {
namespace gemm {
namespace {

template <bool kB>
struct StoreEpi {
  static constexpr bool kBf16 = kB;
  struct Args {
    void* c;
    int64_t ld, part;                      // part: elements from one part to the next
    const float* cin;
    int64_t cin_ld;
    float alpha;
    const float* alpha_dev;
    int f32, wide, cin_wide;
  };
  static __device__ __forceinline__ void tile(const Args& a, const Problem& p, const TileAt& t,
                                              int row, uint32_t acc) {
    using T = typename std::conditional<kB, __nv_bfloat16, __half>::type;
    const float alpha = a.alpha * (a.alpha_dev ? __ldg(a.alpha_dev) : 1.f);
    const int n0 = t.n * p.bn, cols = min(p.bn, p.N - n0);
    const bool live = row < p.M;
    for (int c = 0; c < cols; c += 32) {
      float v[32];
      __syncwarp();                          // (the load is the whole warp's)
      tmem_ld32(acc + c, v);
      if (!live) continue;
      const int left = cols - c;
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= alpha;
      if (a.cin) {
        const float* q = a.cin + (int64_t)row * a.cin_ld + n0 + c;
        if (a.cin_wide && left >= 32) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(q + i);
            v[i] += x.x, v[i + 1] += x.y, v[i + 2] += x.z, v[i + 3] += x.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i < left) v[i] += q[i];
        }
      }
      const int64_t at = t.part * a.part + (int64_t)row * a.ld + n0 + c;
      if (a.f32) store_row32(reinterpret_cast<float*>(a.c) + at, v, left, a.wide);
      else store_row32(reinterpret_cast<T*>(a.c) + at, v, left, a.wide);
    }
  }
};

template <bool kB>
int product(int64_t M, int64_t N, const Term* terms, int n_terms, const Result& r, void* work,
            int64_t work_bytes, int32_t* status, cudaStream_t st) {
  using Epi = StoreEpi<kB>;
  int64_t steps = 0;
  for (int i = 0; i < n_terms; ++i) steps += (terms[i].k + kBK - 1) / kBK;
  const bool amn = terms[0].a.mn, bmn = terms[0].b.mn;
  Plan plan = plan_product(M, N, steps, bmn ? 64 : 16, false, work != nullptr);
  while (plan.parts > 1 && plan.parts * M * N * 4 > work_bytes) --plan.parts;
  Problem q;
  if (!set_up(&q, plan, kB, M, N, terms, n_terms, false, status)) return TT_ERR_UNSUPPORTED;
  typename Epi::Args a{};
  a.alpha = r.alpha, a.alpha_dev = r.alpha_dev;
  if (q.parts > 1) {
    a.c = work, a.ld = N, a.part = M * N, a.f32 = 1;
  } else {
    a.c = r.p, a.ld = r.ld, a.cin = r.cin, a.cin_ld = r.cin_ld, a.f32 = r.dtype == TT_F32;
  }
  const int size = a.f32 ? 4 : 2;
  a.wide = (reinterpret_cast<uintptr_t>(a.c) & 15) == 0 && a.ld * size % 16 == 0 &&
           a.part * size % 16 == 0;
  a.cin_wide = (reinterpret_cast<uintptr_t>(a.cin) & 15) == 0 && a.cin_ld % 4 == 0;
  int rc;
  if (amn && bmn) rc = launch<true, true, Epi>(plan, q, a, st);
  else if (!amn && bmn) rc = launch<false, true, Epi>(plan, q, a, st);
  else return TT_ERR_INVALID_ARG;          // (no operator has this form)
  if (rc != TT_OK || q.parts == 1) return rc;
  return join_parts((const float*)work, q.parts, M, N, r, st);
}

}  // namespace

int64_t tc_work(int64_t M, int64_t N, int64_t k, bool b_mn) {
  if (M <= 0 || N <= 0) return 0;
  const Plan p = plan_product(M, N, (k + kBK - 1) / kBK, b_mn ? 64 : 16, false, true);
  return p.parts > 1 ? p.parts * M * N * 4 : 0;
}

int tc_product(bool bf16, int64_t M, int64_t N, const Term* terms, int n_terms, const Result& r,
               void* work, int64_t work_bytes, int32_t* status, cudaStream_t st) {
  if (M <= 0 || N <= 0) return TT_OK;
  if (n_terms < 1 || n_terms > 2 || (r.dtype != TT_F32 && r.dtype != (bf16 ? TT_BF16 : TT_F16)))
    return TT_ERR_INVALID_ARG;
  return bf16 ? product<true>(M, N, terms, n_terms, r, work, work_bytes, status, st)
              : product<false>(M, N, terms, n_terms, r, work, work_bytes, status, st);
}

}  // namespace gemm
}  // namespace tt
