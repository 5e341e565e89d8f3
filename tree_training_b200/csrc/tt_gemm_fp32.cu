// Matrix products of fp32 factors, summed in fp32 on the CUDA cores.
//
// The tensor cores' sums cut off what falls below their accumulator's last bit at
// every step, which over a few thousand steps costs ten times what fp32 rounding
// does; fp32 inputs are given for their exactness, so they are summed by fma.
//
// A block forms a 128 x 128 tile of C with 256 threads of 8 x 8 elements; slices of
// 16 of k are loaded into registers while the slice before is multiplied out of
// shared memory.  Bound by the fma rate.  Where there are few tiles the sum over k
// is split over blocks, whose parts are added up in order by a second kernel.
#include <algorithm>

#include "tt_gemm.cuh"
#include "tt_vec.cuh"

namespace tt {
namespace gemm {
namespace {

constexpr int kTile = 128, kK = 16, kThreads = 256;
constexpr int kRow = kTile + 4;            // of a slice in shared memory: k by 128 (+ pad)

struct Args {
  const float *a[2], *b[2];
  int64_t a_ld[2], b_ld[2], k[2];
  int M, N, terms;
  int vec_a, vec_b;                        // 16-byte loads allowed
  int64_t k_part;                          // of k, a block's share (all: the sum of k)
  float* c;
  int64_t c_ld, c_part;                    // c_part: from one part to the next
  const float* cin;
  int64_t cin_ld;
  float alpha;
  const float* alpha_dev;
};

// A slice's 128 x 16 elements of a factor: 8 a thread.
template <bool kMN>
__device__ __forceinline__ void fetch(const float* p, int64_t ld, int rows, int64_t i0, int64_t k0,
                                      int64_t k_end, int vec, float (&v)[8]) {
  const int t = threadIdx.x;
  if constexpr (kMN) {                     // 16 rows of k, 128 contiguous elements
    const int64_t k = k0 + t / 16, i = i0 + (t % 16) * 8;
    const float* q = p + k * ld + i;
    if (k < k_end && vec && i + 8 <= rows) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(q));
      const float4 y = __ldg(reinterpret_cast<const float4*>(q + 4));
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
      v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k < k_end && i + j < rows ? __ldg(q + j) : 0.f;
    }
  } else {                                 // 128 rows, 16 contiguous elements of k
    const int64_t i = i0 + t / 2, k = k0 + (t % 2) * 8;
    const float* q = p + i * ld + k;
    if (i < rows && vec && k + 8 <= k_end) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(q));
      const float4 y = __ldg(reinterpret_cast<const float4*>(q + 4));
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
      v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i < rows && k + j < k_end ? __ldg(q + j) : 0.f;
    }
  }
}

template <bool kMN>
__device__ __forceinline__ void put(float* s, const float (&v)[8]) {
  const int t = threadIdx.x;
  if constexpr (kMN) {
    float* q = s + (t / 16) * kRow + (t % 16) * 8;
    *reinterpret_cast<float4*>(q) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(q + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) s[((t % 2) * 8 + j) * kRow + t / 2] = v[j];
  }
}

template <bool kAMN, bool kBMN>
__global__ void __launch_bounds__(kThreads, 2) product_kernel(const Args a) {
  __shared__ __align__(16) float sa[2][kK * kRow];
  __shared__ __align__(16) float sb[2][kK * kRow];
  const int64_t i0 = (int64_t)blockIdx.y * kTile, j0 = (int64_t)blockIdx.x * kTile;
  const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
  float2 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = make_float2(0.f, 0.f);
  // this part's range of k, over the terms one after another
  int64_t from = blockIdx.z * a.k_part, to = from + a.k_part;
  for (int term = 0; term < a.terms; ++term) {
    const int64_t k_all = a.k[term];
    const int64_t kb = min(max(from, (int64_t)0), k_all), ke = min(max(to, (int64_t)0), k_all);
    from -= k_all, to -= k_all;
    if (kb >= ke) continue;
    // (a part may begin in a term at a k that is no multiple of four)
    const int vec_a = a.vec_a && (kAMN || kb % 4 == 0), vec_b = a.vec_b && (kBMN || kb % 4 == 0);
    float ra[8], rb[8];
    fetch<kAMN>(a.a[term], a.a_ld[term], a.M, i0, kb, ke, vec_a, ra);
    fetch<kBMN>(a.b[term], a.b_ld[term], a.N, j0, kb, ke, vec_b, rb);
    int buf = 0;
    for (int64_t k = kb; k < ke; k += kK, buf ^= 1) {
      put<kAMN>(sa[buf], ra);
      put<kBMN>(sb[buf], rb);
      __syncthreads();
      if (k + kK < ke) {
        fetch<kAMN>(a.a[term], a.a_ld[term], a.M, i0, k + kK, ke, vec_a, ra);
        fetch<kBMN>(a.b[term], a.b_ld[term], a.N, j0, k + kK, ke, vec_b, rb);
      }
#pragma unroll
      for (int kk = 0; kk < kK; ++kk) {
        float x[8];
        float2 y[4];
        const float4 x0 = *reinterpret_cast<const float4*>(&sa[buf][kk * kRow + ti * 4]);
        const float4 x1 = *reinterpret_cast<const float4*>(&sa[buf][kk * kRow + 64 + ti * 4]);
        const float4 y0 = *reinterpret_cast<const float4*>(&sb[buf][kk * kRow + tj * 4]);
        const float4 y1 = *reinterpret_cast<const float4*>(&sb[buf][kk * kRow + 64 + tj * 4]);
        x[0] = x0.x, x[1] = x0.y, x[2] = x0.z, x[3] = x0.w;
        x[4] = x1.x, x[5] = x1.y, x[6] = x1.z, x[7] = x1.w;
        y[0] = make_float2(y0.x, y0.y), y[1] = make_float2(y0.z, y0.w);
        y[2] = make_float2(y1.x, y1.y), y[3] = make_float2(y1.z, y1.w);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[i][j] = vec::fma2(make_float2(x[i], x[i]), y[j], acc[i][j]);
      }
    }
    __syncthreads();                       // the next term's slices go into these buffers
  }
  const float alpha = a.alpha * (a.alpha_dev ? *a.alpha_dev : 1.f);
  float* c = a.c + blockIdx.z * a.c_part;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = i0 + (i / 4) * 64 + ti * 4 + i % 4;
    if (row >= a.M) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t col = j0 + (j / 4) * 64 + tj * 4 + j % 4;
      if (col >= a.N) continue;
      float v = alpha * ((j & 1) ? acc[i][j / 2].y : acc[i][j / 2].x);
      if (a.cin) v += a.cin[row * a.cin_ld + col];
      c[row * a.c_ld + col] = v;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
    join_kernel(const float* parts, int n_parts, int64_t M, int64_t N, T* c, int64_t c_ld,
                const float* cin, int64_t cin_ld) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < M * N;
       i += (int64_t)gridDim.x * blockDim.x) {
    float s = parts[i];
    for (int p = 1; p < n_parts; ++p) s += parts[p * M * N + i];
    const int64_t row = i / N, col = i - row * N;
    if (cin) s += cin[row * cin_ld + col];
    c[row * c_ld + col] = from_f32<T>(s);
  }
}

int64_t tiles_of(int64_t M, int64_t N) {
  return ((M + kTile - 1) / kTile) * ((N + kTile - 1) / kTile);
}

// Parts of the sum over k: enough blocks to fill the SMs twice over, none shorter
// than 128 of k.
int64_t parts_of(int64_t M, int64_t N, int64_t k) {
  const int64_t most = std::max<int64_t>(1, k / 128);
  return std::max<int64_t>(1, std::min(most, 2 * vec::kSMs / tiles_of(M, N)));
}

}  // namespace

int64_t fp32_work(int64_t M, int64_t N, int64_t k) {
  const int64_t p = parts_of(M, N, k);
  return p > 1 ? p * M * N * 4 : 0;
}

int fp32_product(int64_t M, int64_t N, const Term* terms, int n_terms, const Result& r, void* work,
                 int64_t work_bytes, cudaStream_t st) {
  if (M <= 0 || N <= 0) return TT_OK;
  if (n_terms < 1 || n_terms > 2 || r.dtype != TT_F32) return TT_ERR_INVALID_ARG;
  if (M > (int64_t)65535 * kTile) return TT_ERR_UNSUPPORTED;
  Args a{};
  a.M = (int)M, a.N = (int)N, a.terms = n_terms, a.vec_a = a.vec_b = 1;
  int64_t k = 0;
  auto aligned = [](const Factor& f) {
    return (reinterpret_cast<uintptr_t>(f.p) & 15) == 0 && f.ld % 4 == 0;
  };
  for (int i = 0; i < n_terms; ++i) {
    a.a[i] = (const float*)terms[i].a.p, a.b[i] = (const float*)terms[i].b.p;
    a.a_ld[i] = terms[i].a.ld, a.b_ld[i] = terms[i].b.ld, a.k[i] = terms[i].k;
    a.vec_a &= aligned(terms[i].a), a.vec_b &= aligned(terms[i].b);
    if (terms[i].a.mn != terms[0].a.mn || terms[i].b.mn != terms[0].b.mn)
      return TT_ERR_INVALID_ARG;
    k += terms[i].k;
  }
  int64_t parts = parts_of(M, N, k);
  while (parts > 1 && (!work || parts * M * N * 4 > work_bytes)) --parts;
  // (whole slices a part: 16-byte loads stay on their boundaries)
  a.k_part = parts > 1 ? ((k + parts - 1) / parts + kK - 1) / kK * kK : std::max<int64_t>(k, 1);
  parts = (k + a.k_part - 1) / a.k_part;
  parts = std::max<int64_t>(parts, 1);
  a.alpha = r.alpha, a.alpha_dev = r.alpha_dev;
  if (parts > 1) {
    a.c = (float*)work, a.c_ld = N, a.c_part = M * N;
  } else {
    a.c = (float*)r.p, a.c_ld = r.ld, a.cin = r.cin, a.cin_ld = r.cin_ld;
  }
  const dim3 grid((unsigned)((N + kTile - 1) / kTile), (unsigned)((M + kTile - 1) / kTile),
                  (unsigned)parts);
  const bool amn = terms[0].a.mn, bmn = terms[0].b.mn;
  if (amn && bmn) product_kernel<true, true><<<grid, kThreads, 0, st>>>(a);
  else if (amn) return TT_ERR_INVALID_ARG;
  else if (bmn) product_kernel<false, true><<<grid, kThreads, 0, st>>>(a);
  else product_kernel<false, false><<<grid, kThreads, 0, st>>>(a);
  tt_count_launches(1);
  if (cudaGetLastError() != cudaSuccess) return TT_ERR_CUDA;
  return parts > 1 ? join_parts((const float*)work, (int)parts, M, N, r, st) : TT_OK;
}

int join_parts(const float* parts, int n_parts, int64_t M, int64_t N, const Result& r,
               cudaStream_t st) {
  return vec::dispatch_float(r.dtype, [&](auto t) -> int {
    using T = decltype(t);
    const int64_t blocks = std::min<int64_t>((M * N + 255) / 256, 8 * vec::kSMs);
    join_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(parts, n_parts, M, N, (T*)r.p, r.ld, r.cin,
                                                     r.cin_ld);
    tt_count_launches(1);
    return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
  });
}

}  // namespace gemm
}  // namespace tt
