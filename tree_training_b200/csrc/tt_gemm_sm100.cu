// Matrix products of 16-bit factors into C, 16-bit or fp32.
#include "tt_gemm_sm100.cuh"

namespace tt {
namespace gemm {
namespace {

template <bool kB>
struct StoreEpi {
  static constexpr bool kBf16 = kB, kChunks = false;
  struct Args {
    void *c, *c2;
    int64_t ld;
    int gap, second;                       // c2's rows (see Result)
    float* parts;                          // [units][128 CG][bn]
    const float* cin;
    int64_t cin_ld;
    float alpha;
    const float* alpha_dev;
    int f32, wide, cin_wide;
  };
  static __device__ __forceinline__ void tile(const Args& a, const Problem& p, const TileAt& t,
                                              int row, uint32_t acc, int c0, float* block) {
    using T = typename std::conditional<kB, __nv_bfloat16, __half>::type;
    const float alpha = a.alpha * (a.alpha_dev ? __ldg(a.alpha_dev) : 1.f);
    const int n0 = t.n * p.bn, cols = min(p.bn, p.N - n0);
    const bool live = row < p.M;
    if (t.unit >= 0) {                     // a part of a sum: the tile as it is
      // (a warp's rows of the tile, whichever CTA of the pair it is in)
      const int64_t tile_rows = p.tile_rows;
      float* q = a.parts + ((int64_t)t.unit * tile_rows + (row - t.m * tile_rows)) * p.bn;
      for (int c = c0; c < cols; c += 64) {
        float v[32];
        __syncwarp();
        tmem_ld32(acc + c, v);
        store_block(live ? q + c : nullptr, v, p.bn - c, true, block);
      }
      return;
    }
    for (int c = c0; c < cols; c += 64) {
      float v[32];
      __syncwarp();                          // (the load is the whole warp's)
      tmem_ld32(acc + c, v);
      const int left = cols - c;
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= alpha;
      if (a.cin && live) {
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
      const bool none = !live || (row >= a.gap && row < a.second);
      const bool two = a.second && row >= a.second;
      void* base = two ? a.c2 : a.c;
      const int64_t at = (int64_t)(two ? row - a.second : row) * a.ld + n0 + c;
      if (a.f32)
        store_block(none ? nullptr : reinterpret_cast<float*>(base) + at, v, left, a.wide, block);
      else
        store_block(none ? nullptr : reinterpret_cast<T*>(base) + at, v, left, a.wide, block);
    }
  }
};

// The tiles that were summed in parts, into C.
template <typename T>
__global__ void __launch_bounds__(256)
    join_tiles_kernel(const __grid_constant__ Problem p, const float* parts, T* c, T* c2,
                      int gap, int second, int64_t ld, const float* cin, int64_t cin_ld,
                      float alpha, const float* alpha_dev) {
  const TileAt t = tile_at(p, p.whole + blockIdx.x * p.parts);
  const int64_t size = (int64_t)p.tile_rows * p.bn;
  const float* q = parts + (int64_t)t.unit * size;
  const int cols = min(p.bn, p.N - t.n * p.bn);
  if (alpha_dev) alpha *= *alpha_dev;
  // a thread four columns; rows by the others (bn is a multiple of 16)
  const int quads = p.bn / 4, rows = blockDim.x / quads;
  const int col = (int)(threadIdx.x % quads) * 4;
  if ((int)threadIdx.x >= quads * rows || col >= cols) return;
  for (int r = blockIdx.y * rows + threadIdx.x / quads; r < p.tile_rows; r += gridDim.y * rows) {
    const int64_t row = (int64_t)t.m * p.tile_rows + r;
    if (row >= p.M) break;
    if (row >= gap && row < second) continue;
    const float* at = q + (int64_t)r * p.bn + col;
    float4 s = __ldg(reinterpret_cast<const float4*>(at));
#pragma unroll 4
    for (int k = 1; k < p.parts; ++k) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(at + k * size));
      s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
    }
    const float v[4] = {s.x * alpha, s.y * alpha, s.z * alpha, s.w * alpha};
    const int64_t n = (int64_t)t.n * p.bn + col;
    T* to = (second && row >= second ? c2 + (row - second) * ld : c + row * ld) + n;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < cols) to[j] = from_f32<T>(cin ? v[j] + cin[row * cin_ld + n + j] : v[j]);
  }
}

template <bool kB>
int product(int64_t M, int64_t N, const Term* terms, int n_terms, const Result& r, void* work,
            int64_t work_bytes, int32_t* status, cudaStream_t st) {
  using Epi = StoreEpi<kB>;
  int64_t steps = 0;
  for (int i = 0; i < n_terms; ++i) steps += (terms[i].k + kBK - 1) / kBK;
  const bool amn = terms[0].a.mn, bmn = terms[0].b.mn;
  Plan plan = plan_product(M, N, steps, bmn ? 64 : 16, false, true);
  if (plan.work > work_bytes || !work)
    plan = plan_product(M, N, steps, bmn ? 64 : 16, false, false);
  Problem q;
  if (!set_up(&q, plan, kB, M, N, terms, n_terms, false, status)) return TT_ERR_UNSUPPORTED;
  typename Epi::Args a{};
  a.alpha = r.alpha, a.alpha_dev = r.alpha_dev, a.parts = (float*)work;
  a.c = r.p, a.c2 = r.p2, a.gap = (int)r.gap, a.second = (int)r.second, a.ld = r.ld;
  a.cin = r.cin, a.cin_ld = r.cin_ld, a.f32 = r.dtype == TT_F32;
  a.wide = ((reinterpret_cast<uintptr_t>(a.c) | reinterpret_cast<uintptr_t>(a.c2)) & 15) == 0 &&
           a.ld * (a.f32 ? 4 : 2) % 16 == 0;
  a.cin_wide = (reinterpret_cast<uintptr_t>(a.cin) & 15) == 0 && a.cin_ld % 4 == 0;
  int rc;
  if (amn && bmn) rc = launch<true, true, Epi>(plan, q, a, st);
  else if (!amn && bmn) rc = launch<false, true, Epi>(plan, q, a, st);
  else return TT_ERR_INVALID_ARG;          // (no operator has this form)
  const int64_t split = (int64_t)q.tiles_m * q.tiles_n - q.whole;
  if (rc != TT_OK || split == 0) return rc;
  return vec::dispatch_float(r.dtype, [&](auto t) -> int {
    using T = decltype(t);
    const int64_t rows = std::min<int64_t>(64, std::max<int64_t>(1, 8 * vec::kSMs / split));
    const dim3 grid((unsigned)split, (unsigned)rows);
    join_tiles_kernel<T><<<grid, 256, 0, st>>>(q, a.parts, (T*)r.p, (T*)r.p2, a.gap, a.second, r.ld,
                                               r.cin, r.cin_ld, r.alpha, r.alpha_dev);
    tt_count_launches(1);
    return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
  });
}

// 16-bit rows of up to kMaxAligned arrays onto 16-byte boundaries, in packs of 8; columns
// past the last are zero.  A block a row, or 128 packs of a longer one.
constexpr int kMaxAligned = 4, kAlignThreads = 128;

struct Aligned {
  const __nv_bfloat16* src[kMaxAligned];
  __nv_bfloat16* dst[kMaxAligned];
  int64_t ld[kMaxAligned], dst_ld[kMaxAligned], rows[kMaxAligned], cols[kMaxAligned];
  int64_t pieces[kMaxAligned];             // of a row
  int64_t first[kMaxAligned + 1];          // piece of an array
};

__global__ void __launch_bounds__(kAlignThreads)
    align_rows_kernel(const __grid_constant__ Aligned a) {
  for (int64_t i = blockIdx.x; i < a.first[kMaxAligned]; i += gridDim.x) {
    int t = 0;
#pragma unroll
    for (int k = 1; k < kMaxAligned; ++k) t = i >= a.first[k] ? k : t;
    const int64_t at = i - a.first[t], n = a.pieces[t];
    const int64_t r = n == 1 ? at : at / n, p = (at - r * n) * kAlignThreads + threadIdx.x;
    if (p * 8 >= a.cols[t]) continue;
    const __nv_bfloat16* src = a.src[t];
    *reinterpret_cast<uint4*>(a.dst[t] + r * a.dst_ld[t] + p * 8) = vec::load_any_of<__nv_bfloat16>(
        src + r * a.ld[t], p * 8, a.cols[t], src, src + (a.rows[t] - 1) * a.ld[t] + a.cols[t]);
  }
}

}  // namespace

int64_t tc_work(int64_t M, int64_t N, int64_t steps, bool b_mn) {
  if (M <= 0 || N <= 0) return 0;
  return plan_product(M, N, steps, b_mn ? 64 : 16, false, true).work;
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

extern "C" int tt_align_rows_of(int32_t count, const int64_t* rows, const int64_t* cols,
                                const void* const* src, const int64_t* ld, void* const* dst,
                                const int64_t* dst_ld, void* stream) {
  using namespace tt::gemm;
  if (count < 0 || count > kMaxAligned ||
      (count > 0 && (!rows || !cols || !src || !ld || !dst || !dst_ld)))
    return TT_ERR_INVALID_ARG;
  Aligned a{};
  for (int i = 0; i < kMaxAligned; ++i) {
    a.first[i + 1] = a.first[i];
    if (i >= count) continue;
    if (rows[i] < 0 || cols[i] < 1 || (rows[i] > 1 && ld[i] < cols[i]) || dst_ld[i] < cols[i] ||
        dst_ld[i] % 8 != 0)
      return TT_ERR_INVALID_ARG;
    if (rows[i] == 0) continue;
    if (!src[i] || !dst[i] || (reinterpret_cast<uintptr_t>(dst[i]) & 15) ||
        (reinterpret_cast<uintptr_t>(src[i]) & 1))
      return TT_ERR_INVALID_ARG;
    a.src[i] = (const __nv_bfloat16*)src[i], a.dst[i] = (__nv_bfloat16*)dst[i];
    a.ld[i] = ld[i], a.dst_ld[i] = dst_ld[i], a.rows[i] = rows[i], a.cols[i] = cols[i];
    a.pieces[i] = (cols[i] + 8 * kAlignThreads - 1) / (8 * kAlignThreads);
    a.first[i + 1] += rows[i] * a.pieces[i];
  }
  const int64_t pieces = a.first[kMaxAligned];
  if (pieces == 0) return TT_OK;
  align_rows_kernel<<<(unsigned)std::min<int64_t>(pieces, 16 * tt::vec::kSMs), kAlignThreads, 0,
                      (cudaStream_t)stream>>>(a);
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

// (for callers of the C ABI with one array: the bindings copy all of a call at once)
extern "C" int tt_align_rows(int64_t rows, int64_t cols, const void* src, int64_t ld, void* dst,
                             int64_t dst_ld, void* stream) {
  return tt_align_rows_of(1, &rows, &cols, &src, &ld, &dst, &dst_ld, stream);
}
