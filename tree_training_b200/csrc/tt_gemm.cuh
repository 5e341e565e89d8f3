// Matrix products shared by the feed-forward block and the LM head's loss.
#pragma once

#include "tt_common.cuh"

namespace tt {
namespace gemm {

// A factor: element (i, k) at p[i * ld + k], or with `mn` at p[k * ld + i].
struct Factor {
  const void* p;
  int64_t ld;
  bool mn;
};

// The next number of parts of a sum that a plan tries: a quarter more each, and the
// most (trying all took the host 20 us a call).
inline int64_t next_parts(int64_t parts, int64_t most) {
  const int64_t next = parts + (parts + 3) / 4;
  return parts < most && next > most ? most : next;
}

// One term of a sum of products: A [M, k] times B [N, k], transposed.
struct Term {
  Factor a, b;
  int64_t k;
};

// C [M, N] = alpha * sum of the terms (+ cin): C of `dtype`, cin fp32 with the
// row stride `cin_ld` (it may be C itself).  alpha is multiplied by *alpha_dev
// where that is given.
struct Result {
  int dtype;
  void* p;
  int64_t ld;
  const float* cin;
  int64_t cin_ld;
  float alpha;
  const float* alpha_dev;
  // (tensor cores) rows from `second` on are those of another array, from its first
  // row; rows from `gap` to there are none.  0: no such rows.
  void* p2 = nullptr;
  int64_t gap = 0, second = 0;
};

// fp32 products on the CUDA cores: sums in fp32, in the order of k.  Up to two
// terms.  `work` holds the parts of a sum that is split over k (fp32_work bytes
// make room for any split; with less the sum is split less).
int fp32_product(int64_t M, int64_t N, const Term* terms, int n_terms, const Result& r, void* work,
                 int64_t work_bytes, cudaStream_t st);
int64_t fp32_work(int64_t M, int64_t N, int64_t k, int batch = 1);

// Two products of the same shape in one launch, a term and a result each.
int fp32_products(int64_t M, int64_t N, const Term* terms, const Result* r, void* work,
                  int64_t work_bytes, cudaStream_t st);

}  // namespace gemm
}  // namespace tt
