// Matrix products of fp32 factors, summed in fp32 on the CUDA cores.
//
// The tensor cores' sums cut off what falls below their accumulator's last bit at
// every step, which over a few thousand steps costs ten times what fp32 rounding
// does; fp32 inputs are given for their exactness, so they are summed by fma.
//
// A block forms a 128 x 128 tile of C with 256 threads of 8 x 8 elements (64 x 128 or 64 x
// 64 where there are few rows or tiles, which would leave SMs idle); slices of 16 of k
// are loaded into registers while the slice before is multiplied out of shared memory.
// Bound by the fma rate (measured on a B200 at 4,096 a side: 51 to 58 TFLOP/s of 74; the
// library's 57).  Up to eight rows have kernels of their own.  Where there are few tiles the
// sum over k is split over blocks, whose parts are added up in order by a second kernel.
#include <algorithm>

#include "tt_gemm.cuh"
#include "tt_vec.cuh"

namespace tt {
namespace gemm {
namespace {

constexpr int kK = 16, kThreads = 256;

struct Args {
  const float *a[2], *b[2];
  int64_t a_ld[2], b_ld[2], k[2];
  int M, N, terms;                         // terms of one sum, or (batch) of one each
  int batch;
  uint32_t tiles_n;
  int vec_a, vec_b, vec_c;                 // 16-byte loads and stores allowed
  int parts;
  int64_t k_part;                          // of k, a block's share (all: the sum of k)
  float* c[2];
  int64_t c_ld, c_part;                    // c_part: from one part to the next
  const float* cin;
  int64_t cin_ld;
  float alpha;
  const float* alpha_dev;
};

// A slice's S x 16 elements of a factor: S / 16 a thread.
template <int S, bool kMN>
__device__ __forceinline__ void fetch(const float* p, int64_t ld, int rows, int64_t i0, int64_t k0,
                                      int64_t k_end, int vec, float (&v)[S / 16]) {
  constexpr int E = S / 16;
  const int t = threadIdx.x;
  int64_t i, k, left;
  const float* q;
  bool live;
  if constexpr (kMN) {                     // 16 rows of k, S contiguous elements
    k = k0 + t / 16, i = i0 + (t % 16) * E;
    q = p + k * ld + i;
    live = k < k_end, left = rows - i;
  } else {                                 // S rows, 16 contiguous elements of k
    i = i0 + t / (16 / E), k = k0 + (t % (16 / E)) * E;
    q = p + i * ld + k;
    live = i < rows, left = k_end - k;
  }
  if (live && vec && left >= E) {
#pragma unroll
    for (int j = 0; j < E; j += 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(q + j));
      v[j] = x.x, v[j + 1] = x.y, v[j + 2] = x.z, v[j + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = live && j < left ? __ldg(q + j) : 0.f;
  }
}

// The slice in shared memory: k by S (and 4 floats of padding).
template <int S, bool kMN>
__device__ __forceinline__ void put(float* s, const float (&v)[S / 16]) {
  constexpr int E = S / 16;
  const int t = threadIdx.x;
  if constexpr (kMN) {
    float* q = s + (t / 16) * (S + 4) + (t % 16) * E;
#pragma unroll
    for (int j = 0; j < E; j += 4)
      *reinterpret_cast<float4*>(q + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      s[((t % (16 / E)) * E + j) * (S + 4) + t / (16 / E)] = v[j];
  }
}

// Thread (ti, tj) of 16 x 16 has rows 64 x + 4 ti .. + 3 of the tile, columns likewise.
template <int SM, int SN, bool kAMN, bool kBMN>
__global__ void __launch_bounds__(kThreads, 2) product_kernel(const Args a) {
  constexpr int EM = SM / 16, EN = SN / 16, RA = SM + 4, RB = SN + 4;
  __shared__ __align__(16) float sa[2][kK * RA];
  __shared__ __align__(16) float sb[2][kK * RB];
  const int64_t i0 = (int64_t)(blockIdx.x / a.tiles_n) * SM;
  const int64_t j0 = (int64_t)(blockIdx.x % a.tiles_n) * SN;
  const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
  const int part = blockIdx.y % a.parts, which = blockIdx.y / a.parts;
  float2 acc[EM][EN / 2];
#pragma unroll
  for (int i = 0; i < EM; ++i)
#pragma unroll
    for (int j = 0; j < EN / 2; ++j) acc[i][j] = make_float2(0.f, 0.f);
  // this part's range of k, over the terms one after another
  int64_t from = part * a.k_part, to = from + a.k_part;
  const int last = a.batch > 1 ? which + 1 : a.terms;
  for (int term = which; term < last; ++term) {
    const int64_t k_all = a.k[term];
    const int64_t kb = min(max(from, (int64_t)0), k_all), ke = min(max(to, (int64_t)0), k_all);
    from -= k_all, to -= k_all;
    if (kb >= ke) continue;
    // (a part may begin in a term at a k that is no multiple of four)
    const int vec_a = a.vec_a && (kAMN || kb % 4 == 0), vec_b = a.vec_b && (kBMN || kb % 4 == 0);
    float ra[EM], rb[EN];
    fetch<SM, kAMN>(a.a[term], a.a_ld[term], a.M, i0, kb, ke, vec_a, ra);
    fetch<SN, kBMN>(a.b[term], a.b_ld[term], a.N, j0, kb, ke, vec_b, rb);
    int buf = 0;
    for (int64_t k = kb; k < ke; k += kK, buf ^= 1) {
      put<SM, kAMN>(sa[buf], ra);
      put<SN, kBMN>(sb[buf], rb);
      __syncthreads();
      if (k + kK < ke) {
        fetch<SM, kAMN>(a.a[term], a.a_ld[term], a.M, i0, k + kK, ke, vec_a, ra);
        fetch<SN, kBMN>(a.b[term], a.b_ld[term], a.N, j0, k + kK, ke, vec_b, rb);
      }
#pragma unroll
      for (int kk = 0; kk < kK; ++kk) {
        float x[EM];
        float2 y[EN / 2];
#pragma unroll
        for (int h = 0; h < EM / 4; ++h) {
          const float4 p = *reinterpret_cast<const float4*>(&sa[buf][kk * RA + h * 64 + ti * 4]);
          x[4 * h] = p.x, x[4 * h + 1] = p.y, x[4 * h + 2] = p.z, x[4 * h + 3] = p.w;
        }
#pragma unroll
        for (int h = 0; h < EN / 4; ++h) {
          const float4 q = *reinterpret_cast<const float4*>(&sb[buf][kk * RB + h * 64 + tj * 4]);
          y[2 * h] = make_float2(q.x, q.y), y[2 * h + 1] = make_float2(q.z, q.w);
        }
#pragma unroll
        for (int i = 0; i < EM; ++i)
#pragma unroll
          for (int j = 0; j < EN / 2; ++j)
            acc[i][j] = vec::fma2(make_float2(x[i], x[i]), y[j], acc[i][j]);
      }
    }
    __syncthreads();                       // the next term's slices go into these buffers
  }
  const float alpha = a.alpha * (a.alpha_dev ? *a.alpha_dev : 1.f);
  float* c = a.c[which] + part * a.c_part;
#pragma unroll
  for (int i = 0; i < EM; ++i) {
    const int64_t row = i0 + (i / 4) * 64 + ti * 4 + i % 4;
    if (row >= a.M) continue;
#pragma unroll
    for (int h = 0; h < EN / 4; ++h) {
      const int64_t col = j0 + h * 64 + tj * 4;
      float v[4] = {acc[i][2 * h].x, acc[i][2 * h].y, acc[i][2 * h + 1].x, acc[i][2 * h + 1].y};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] *= alpha;
        if (a.cin && col + j < a.N) v[j] += a.cin[row * a.cin_ld + col + j];
      }
      float* to = c + row * a.c_ld + col;
      if (a.vec_c && col + 4 <= a.N) {
        *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + j < a.N) to[j] = v[j];
      }
    }
  }
}

// ---- few rows ---------------------------------------------------------------------
//
// Up to kFewRows rows of A: bound by B's bytes; a tile of 64 rows would spend its time on
// rows that are not there.  Both products of 2,560 x 9,728 (200 MB): 40 us one row, 41
// two, 55 four, 91 eight, where tiles take 214 to 220; A comes out of L1, whose loads bound
// it from four rows on (two rows of B a warp and two steps ahead; four of either: 62 to 67
// and 117 to 127).  For 16 it would be 180 to 400, tiles 225.

constexpr int kFewRows = 8;

// Four elements at p, of which `left` are there.
__device__ __forceinline__ float4 load4(const float* p, int64_t left) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (left > 0) v.x = __ldg(p);
  if (left > 1) v.y = __ldg(p + 1);
  if (left > 2) v.z = __ldg(p + 2);
  if (left > 3) v.w = __ldg(p + 3);
  return v;
}

// Rows of B contiguous in k: a warp R rows of B, its lanes over k, R x MR sums a lane.
template <int MR, int R>
__global__ void __launch_bounds__(kThreads) few_rows_kernel(const Args a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, which = blockIdx.y;
  const int64_t n0 = ((int64_t)blockIdx.x * (kThreads / 32) + warp) * R;
  if (n0 >= a.N) return;
  float acc[MR][R];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[m][r] = 0.f;
  const int last = a.batch > 1 ? which + 1 : a.terms;
  for (int term = which; term < last; ++term) {
    const float* rows[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      rows[r] = a.b[term] + min(n0 + r, (int64_t)a.N - 1) * a.b_ld[term];
    const int64_t K = a.k[term];
    auto step = [&](int64_t k, auto load) {
      float4 b[R];
#pragma unroll
      for (int r = 0; r < R; ++r) b[r] = load(rows[r] + k);
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const float4 x = load(a.a[term] + (int64_t)min(m, a.M - 1) * a.a_ld[term] + k);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          acc[m][r] = fmaf(x.x, b[r].x, acc[m][r]);
          acc[m][r] = fmaf(x.y, b[r].y, acc[m][r]);
          acc[m][r] = fmaf(x.z, b[r].z, acc[m][r]);
          acc[m][r] = fmaf(x.w, b[r].w, acc[m][r]);
        }
      }
    };
    // (a loop without branches: its loads wait for none)
    const int64_t whole = a.vec_a && a.vec_b ? K / 4 * 4 : 0;
#pragma unroll 2
    for (int64_t k = lane * 4; k < whole; k += 128)
      step(k, [](const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); });
    for (int64_t k = whole + lane * 4; k < K; k += 128)
      step(k, [&](const float* p) { return load4(p, K - k); });
  }
  const float alpha = a.alpha * (a.alpha_dev ? *a.alpha_dev : 1.f);
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v = acc[m][r];
#pragma unroll
      for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == (m * R + r) % 32 && m < a.M && n0 + r < a.N) {
        v *= alpha;
        if (a.cin) v += a.cin[m * a.cin_ld + n0 + r];
        a.c[which][m * a.c_ld + n0 + r] = v;
      }
    }
}

// Columns of B contiguous: a thread four columns and all rows, over a part of k, of which
// A's elements stand in shared memory.
constexpr int kFewThreads = 128, kFewK = 64;

template <int MR>
__global__ void __launch_bounds__(kFewThreads) few_columns_kernel(const Args a) {
  constexpr int kAhead = 8;                // rows of B fetched together
  __shared__ float sa[kFewK][MR];
  const int part = blockIdx.y % a.parts, which = blockIdx.y / a.parts;
  const int64_t col = ((int64_t)blockIdx.x * kFewThreads + threadIdx.x) * 4, left = a.N - col;
  float4 acc[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) acc[m] = make_float4(0.f, 0.f, 0.f, 0.f);
  int64_t from = part * a.k_part, to = from + a.k_part;
  const int last = a.batch > 1 ? which + 1 : a.terms;
  for (int term = which; term < last; ++term) {
    const int64_t k_all = a.k[term];
    const int64_t kb = min(max(from, (int64_t)0), k_all), ke = min(max(to, (int64_t)0), k_all);
    from -= k_all, to -= k_all;
    for (int64_t k0 = kb; k0 < ke; k0 += kFewK) {
      const int n = (int)min((int64_t)kFewK, ke - k0);
      __syncthreads();                     // (the rows before are multiplied)
      for (int i = threadIdx.x; i < kFewK * MR; i += kFewThreads) {
        const int m = i / kFewK, kk = i % kFewK;
        sa[kk][m] = m < a.M && kk < n ? __ldg(a.a[term] + m * a.a_ld[term] + k0 + kk) : 0.f;
      }
      __syncthreads();
      const float* b = a.b[term] + k0 * a.b_ld[term] + col;
      for (int k = 0; k < n; k += kAhead) {
        float4 y[kAhead];
        if (a.vec_b && left >= 4 && k + kAhead <= n) {
#pragma unroll
          for (int j = 0; j < kAhead; ++j)
            y[j] = __ldg(reinterpret_cast<const float4*>(b + (k + j) * a.b_ld[term]));
        } else {
#pragma unroll
          for (int j = 0; j < kAhead; ++j)
            y[j] = load4(b + (k + j) * a.b_ld[term], k + j < n ? left : 0);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
          for (int m = 0; m < MR; ++m) {
            const float x = sa[k + j][m];
            acc[m].x = fmaf(x, y[j].x, acc[m].x), acc[m].y = fmaf(x, y[j].y, acc[m].y);
            acc[m].z = fmaf(x, y[j].z, acc[m].z), acc[m].w = fmaf(x, y[j].w, acc[m].w);
          }
      }
    }
  }
  const float alpha = a.alpha * (a.alpha_dev ? *a.alpha_dev : 1.f);
  float* c = a.c[which] + part * a.c_part;
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    if (m >= a.M) continue;
    const float v[4] = {acc[m].x, acc[m].y, acc[m].z, acc[m].w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left)
        c[m * a.c_ld + col + j] = v[j] * alpha + (a.cin ? a.cin[m * a.cin_ld + col + j] : 0.f);
  }
}

// C = the parts, added up in order, + cin; blockIdx.y: of a batch.  A block 32 elements
// at a time, each warp a run of the parts.
__global__ void __launch_bounds__(256)
    join_kernel(const float* parts_, int n_parts, int64_t M, int64_t N, float* c0, float* c1,
                int64_t c_ld, const float* cin, int64_t cin_ld) {
  __shared__ float sm[8][32];
  const float* parts = parts_ + (int64_t)blockIdx.y * n_parts * M * N;
  float* c = blockIdx.y ? c1 : c0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int run = (n_parts + 7) / 8;
  for (int64_t i0 = (int64_t)blockIdx.x * 32; i0 < M * N; i0 += (int64_t)gridDim.x * 32) {
    const int64_t i = i0 + lane;
    float s = 0.f;
    if (i < M * N) {
#pragma unroll 8
      for (int p = warp * run; p < min(n_parts, (warp + 1) * run); ++p) s += parts[p * M * N + i];
    }
    sm[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && i < M * N) {
      for (int w = 1; w < 8; ++w) s += sm[w][lane];
      const int64_t row = i / N, col = i - row * N;
      if (cin) s += cin[row * cin_ld + col];
      c[row * c_ld + col] = s;
    }
    __syncthreads();
  }
}

struct Form {
  int rows, cols;                          // of a tile
  int64_t parts;
};

// The cheapest form: tiles of 128 x 128 take 2,048 clocks of fma a slice and SM, 64 x
// 128 half of that and some, 64 x 64 a quarter and some (their operands are read from
// shared memory more often); parts have at least 64 of k, and cost a launch and their
// way through L2.  From five blocks an SM on the rate counts more than how the last of
// them come out, and the smaller tiles' clocks are a quarter more (2,000 x 1,500 x 2,500
// 2,355 us by 64 x 128, 2,106 by 128 x 128; 700 x 512 x 3,000, of 3.6 an SM, 369 and 395).
Form form_of(int64_t M, int64_t N, int64_t k, int batch, bool split) {
  constexpr int kForms[3][3] = {{128, 128, 2048}, {64, 128, 1100}, {64, 64, 650}};
  Form best{128, 128, 1};
  double least = 1e300;
  for (const auto& f : kForms) {
    const int64_t tiles = ((M + f[0] - 1) / f[0]) * ((N + f[1] - 1) / f[1]) * batch;
    const int64_t most =
        split ? std::max<int64_t>(1, std::min<int64_t>(k / 64, 4 * vec::kSMs / tiles)) : 1;
    for (int64_t parts = 1; parts <= most; parts = next_parts(parts, most)) {
      const double slices = (double)((k + parts - 1) / parts + kK - 1) / kK;
      const bool full = f[0] * f[1] < 128 * 128 && tiles * parts >= 5 * vec::kSMs;
      double t = (double)((tiles * parts + vec::kSMs - 1) / vec::kSMs) * slices * f[2] *
                     (full ? 1.25 : 1.0) + 1500;
      if (parts > 1) t += 5000 + (double)(parts + 1) * batch * M * N * 4 / 1500;
      if (t < least * 0.99) least = t, best = Form{f[0], f[1], parts};
    }
  }
  return best;
}

// Parts of a sum whose B has contiguous columns, for few rows: eight blocks an SM, parts
// of 32 of k at least, and no more bytes of parts, there and back, than half of B's.
int64_t few_parts(int64_t M, int64_t N, int64_t k, int batch) {
  const int64_t blocks = (N + 4 * kFewThreads - 1) / (4 * kFewThreads) * batch;
  return std::max<int64_t>(1, std::min({8 * vec::kSMs / blocks, k / 32, k / (4 * M)}));
}

template <int MR>
void launch_few(const Args& a, bool bmn, cudaStream_t st) {
  if (bmn) {
    const dim3 grid((unsigned)((a.N + 4ll * kFewThreads - 1) / (4 * kFewThreads)),
                    (unsigned)(a.parts * a.batch));
    few_columns_kernel<MR><<<grid, kFewThreads, 0, st>>>(a);
    return;
  }
  // (two rows of B share the loads of A, where that leaves eight warps an SM)
  constexpr int R = 2, W = kThreads / 32;
  if ((int64_t)a.N * a.batch >= (int64_t)R * W * vec::kSMs)
    few_rows_kernel<MR, R><<<dim3((unsigned)((a.N + R * W - 1) / (R * W)), a.batch), kThreads, 0,
                             st>>>(a);
  else
    few_rows_kernel<MR, 1><<<dim3((unsigned)((a.N + W - 1) / W), a.batch), kThreads, 0, st>>>(a);
}

int launch_few(const Args& a, bool bmn, cudaStream_t st) {
  if (a.M == 1) launch_few<1>(a, bmn, st);
  else if (a.M == 2) launch_few<2>(a, bmn, st);
  else if (a.M <= 4) launch_few<4>(a, bmn, st);
  else launch_few<8>(a, bmn, st);
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

template <int SM, int SN>
int launch_product(const Args& a, const dim3& grid, bool amn, bool bmn, cudaStream_t st) {
  if (amn && bmn) product_kernel<SM, SN, true, true><<<grid, kThreads, 0, st>>>(a);
  else if (amn) return TT_ERR_INVALID_ARG;       // (no operator has this form)
  else if (bmn) product_kernel<SM, SN, false, true><<<grid, kThreads, 0, st>>>(a);
  else product_kernel<SM, SN, false, false><<<grid, kThreads, 0, st>>>(a);
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

int run(int64_t M, int64_t N, const Term* terms, int n_terms, const Result* r, int batch,
        void* work, int64_t work_bytes, cudaStream_t st) {
  if (M <= 0 || N <= 0) return TT_OK;
  if (n_terms < 1 || n_terms > 2 || batch < 1 || batch > 2 || (batch > 1 && n_terms != batch))
    return TT_ERR_INVALID_ARG;
  Args a{};
  a.M = (int)M, a.N = (int)N, a.terms = n_terms, a.batch = batch, a.vec_a = a.vec_b = 1;
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
    k = batch > 1 ? terms[i].k : k + terms[i].k;
  }
  const bool amn = terms[0].a.mn, bmn = terms[0].b.mn, few = M <= kFewRows && !amn;
  Form f = few ? Form{kFewRows, 4, bmn ? few_parts(M, N, k, batch) : 1}
               : form_of(M, N, k, batch, true);
  if (few && f.parts * batch * M * N * 4 > (work ? work_bytes : 0)) f.parts = 1;
  if (!few && f.parts > 1 && (!work || f.parts * batch * M * N * 4 > work_bytes))
    f = form_of(M, N, k, batch, false);
  // (whole slices a part: 16-byte loads stay on their boundaries)
  a.k_part = f.parts > 1 ? ((k + f.parts - 1) / f.parts + kK - 1) / kK * kK
                         : std::max<int64_t>(k, 1);
  a.parts = (int)std::max<int64_t>((k + a.k_part - 1) / a.k_part, 1);
  a.alpha = r[0].alpha, a.alpha_dev = r[0].alpha_dev;
  for (int i = 0; i < batch; ++i)
    a.c[i] = a.parts > 1 ? (float*)work + i * a.parts * M * N : (float*)r[i].p;
  if (a.parts > 1) a.c_ld = N, a.c_part = M * N;
  else a.c_ld = r[0].ld, a.cin = r[0].cin, a.cin_ld = r[0].cin_ld;
  a.vec_c = a.c_ld % 4 == 0 && a.c_part % 4 == 0;
  for (int i = 0; i < batch; ++i) a.vec_c &= (reinterpret_cast<uintptr_t>(a.c[i]) & 15) == 0;
  const int64_t rows = (M + f.rows - 1) / f.rows, cols = (N + f.cols - 1) / f.cols;
  if (rows * cols > 0x7fffffff) return TT_ERR_UNSUPPORTED;
  a.tiles_n = (uint32_t)cols;
  const dim3 grid((unsigned)(rows * cols), (unsigned)(a.parts * batch));
  const int rc = few             ? launch_few(a, bmn, st)
                 : f.rows == 128 ? launch_product<128, 128>(a, grid, amn, bmn, st)
                 : f.cols == 128 ? launch_product<64, 128>(a, grid, amn, bmn, st)
                                 : launch_product<64, 64>(a, grid, amn, bmn, st);
  if (rc != TT_OK || a.parts == 1) return rc;
  const int64_t blocks = std::min<int64_t>((M * N + 31) / 32, 64 * vec::kSMs);
  join_kernel<<<dim3((unsigned)blocks, (unsigned)batch), 256, 0, st>>>(
      (const float*)work, a.parts, M, N, (float*)r[0].p, (float*)r[batch - 1].p, r[0].ld, r[0].cin,
      r[0].cin_ld);
  tt_count_launches(1);
  return cudaGetLastError() == cudaSuccess ? TT_OK : TT_ERR_CUDA;
}

}  // namespace

int64_t fp32_work(int64_t M, int64_t N, int64_t k, int batch) {
  if (M <= 0 || N <= 0) return 0;
  const int64_t parts = std::max(form_of(M, N, k, batch, true).parts,
                                 M <= kFewRows ? few_parts(M, N, k, batch) : 1);
  return parts > 1 ? parts * batch * M * N * 4 : 0;
}

int fp32_product(int64_t M, int64_t N, const Term* terms, int n_terms, const Result& r, void* work,
                 int64_t work_bytes, cudaStream_t st) {
  return run(M, N, terms, n_terms, &r, 1, work, work_bytes, st);
}

int fp32_products(int64_t M, int64_t N, const Term* terms, const Result* r, void* work,
                  int64_t work_bytes, cudaStream_t st) {
  return run(M, N, terms, 2, r, 2, work, work_bytes, st);
}

}  // namespace gemm
}  // namespace tt
