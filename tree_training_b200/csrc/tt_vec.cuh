// Packs of V elements moved as one load or store of V * sizeof(T) bytes (2 to
// 16), converted to and from fp32 registers.  A pack's address must be a
// multiple of its size.
#pragma once

#include <type_traits>

#include "tt_common.cuh"

namespace tt {
namespace vec {

constexpr int kSMs = 148;   // of a B200: grids are sized by it

template <int Bytes>
struct RawOf;
template <>
struct RawOf<16> { using type = uint4; };
template <>
struct RawOf<8> { using type = uint2; };
template <>
struct RawOf<4> { using type = uint32_t; };
template <>
struct RawOf<2> { using type = uint16_t; };

template <typename T, int V>
using Raw = typename RawOf<(int)sizeof(T) * V>::type;

// Data that no kernel writes while it is read (through L1).
template <typename R>
__device__ __forceinline__ R ld_stream(const void* p) {
  return __ldg(reinterpret_cast<const R*>(p));
}

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p) {
  return ld_stream<Raw<T, V>>(p);
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float (&v)[V]) {
  union {
    Raw<T, V> raw;
    uint32_t w[(sizeof(T) * V + 3) / 4];
    uint16_t h[(sizeof(T) * V + 1) / 2];
  } u;
  u.raw = r;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      v[i] = __uint_as_float(u.w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      if constexpr (V == 1)
        v[i] = __uint_as_float((uint32_t)u.h[0] << 16);
      else
        v[i] = __uint_as_float((i & 1) ? (u.w[i / 2] & 0xffff0000u) : (u.w[i / 2] << 16));
    } else {
      v[i] = __half2float(__ushort_as_half(u.h[i]));
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&v)[V]) {
  unpack<T, V>(load_raw<T, V>(p), v);
}

// (Pairs are converted by one instruction.)
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> pack(const float (&v)[V]) {
  union U {
    Raw<T, V> raw;
    T e[V];
    __nv_bfloat162 b2[(V + 1) / 2];
    __half2 h2[(V + 1) / 2];
    __device__ U() {}
  } u;
  if constexpr (V == 1 || sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) u.e[i] = from_f32<T>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value)
        u.b2[i / 2] = __floats2bfloat162_rn(v[i], v[i + 1]);
      else
        u.h2[i / 2] = __floats2half2_rn(v[i], v[i + 1]);
    }
  }
  return u.raw;
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&v)[V]) {
  *reinterpret_cast<Raw<T, V>*>(p) = pack<T, V>(v);
}

// a * b + c on two fp32 values in one instruction (subnormals kept).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// acc += w v over V elements
template <int V>
__device__ __forceinline__ void axpy(float w, const float (&v)[V], float (&acc)[V]) {
  if constexpr (V == 1) {
    acc[0] = fmaf(w, v[0], acc[0]);
  } else {
    const float2 w2 = make_float2(w, w);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = fma2(w2, make_float2(v[i], v[i + 1]), make_float2(acc[i], acc[i + 1]));
      acc[i] = r.x, acc[i + 1] = r.y;
    }
  }
}

// ---- 16 bytes at any element --------------------------------------------------

// Bytes b .. b + 15 of the 32 bytes (a, c), b < 16.
__device__ __forceinline__ uint4 window(const uint4& a, const uint4& c, int b) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
  if (b & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (b & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  const int bits = 8 * (b & 3);
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// 16 bytes at p, a multiple of T's size: out of the one or two aligned 16-byte
// words that hold them, where these lie in [lo, hi); element by element at the
// ends of a buffer.
template <typename T>
__device__ __forceinline__ uint4 load_any(const T* p, const T* lo, const T* hi) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  const int b = (int)(at & 15);
  const uint4* w = reinterpret_cast<const uint4*>(at - b);
  if (b == 0) return __ldg(w);
  if (reinterpret_cast<const T*>(w) >= lo && reinterpret_cast<const T*>(w + 2) <= hi)
    return window(__ldg(w), __ldg(w + 1), b);
  union U {
    uint4 raw;
    T e[16 / sizeof(T)];
    __device__ U() {}
  } u;
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i) u.e[i] = p[i];
  return u.raw;
}

// The same of the elements e0 .. of a row of n elements; those outside it are 0.
template <typename T>
__device__ __forceinline__ uint4 load_any_of(const T* row, int64_t e0, int64_t n, const T* lo,
                                             const T* hi) {
  constexpr int N = 16 / (int)sizeof(T);
  if (e0 >= 0 && e0 + N <= n) return load_any<T>(row + e0, lo, hi);
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = e0 + i >= 0 && e0 + i < n ? to_f32(row[e0 + i]) : 0.f;
  return pack<T, N>(v);
}

// Stores what lies of a pack at elements e0 .. in a row of n elements; row + e0
// is on a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void store_part(T* row, int64_t e0, int64_t n, const uint4& raw) {
  constexpr int N = 16 / (int)sizeof(T);
  if (e0 >= 0 && e0 + N <= n) {
    *reinterpret_cast<uint4*>(row + e0) = raw;
    return;
  }
  float v[N];
  unpack<T, N>(raw, v);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (e0 + i >= 0 && e0 + i < n) row[e0 + i] = from_f32<T>(v[i]);
}

// ---- launches that follow one another closely ------------------------------------

// A kernel launched by launch_next may begin while the one before it in its stream
// ends: it waits here, before it touches memory, until that one has finished.
__device__ __forceinline__ void wait_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// Lets the next kernel begin as soon as every block of this one has come here (or
// ended).
__device__ __forceinline__ void let_next_begin() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Launches a kernel that calls wait_previous first.
template <typename... P, typename... A>
cudaError_t launch_next(void (*kernel)(P...), dim3 grid, int threads, size_t smem,
                        cudaStream_t st, A... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = dim3((unsigned)threads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = attr;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, P(args)...);
}

// Calls f with a value of the C++ type of a TT_* floating dtype.
template <typename F>
int dispatch_float(int dtype, F f) {
  switch (dtype) {
    case TT_BF16: return f(__nv_bfloat16());
    case TT_F16: return f(__half());
    case TT_F32: return f(float());
    default: return TT_ERR_UNSUPPORTED;
  }
}

}  // namespace vec
}  // namespace tt
