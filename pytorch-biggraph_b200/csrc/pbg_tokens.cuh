// Shared by the token operators (lookup, log probabilities over scores, log probabilities over a table): element types, 16-byte
// vectors of them, and the exponential they all use.
//
// These entry points take no context: the caller hands over the stream and the workspace, nothing here allocates or
// synchronises, and a bad id is skipped and reported through the caller's error word.
#pragma once
#include <cuda_fp16.h>

#include "pbg_common.cuh"

#define TOK_LOG2E 1.4426950408889634f
#define TOK_LN2 0.6931471805599453f
#define TOK_ERR_ID 1                       // bits of the caller's error word
#define TOK_ERR_TIMEOUT 2
#define TOK_ERR_LSE 4

// ex2 takes z to 2^z within 2 ulp, results below 2^-126 to 0.
__device__ __forceinline__ float tok_ex2(float z) { float e; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z)); return e; }
// the smaller, the larger; NaN if either is one
__device__ __forceinline__ float tok_min_nan(float a, float b) { float m; asm("min.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b)); return m; }
__device__ __forceinline__ float tok_max_nan(float a, float b) { float m; asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b)); return m; }

// two fp32 numbers to an instruction
__device__ __forceinline__ unsigned long long f32x2(float a, float b) { unsigned long long p; asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b)); return p; }
__device__ __forceinline__ float2 f32x2_parts(unsigned long long p) { float2 f; asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p)); return f; }
__device__ __forceinline__ unsigned long long f32x2_fma(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long f32x2_add(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Element types: storage type, elements of a 16-byte vector, conversions.  Results are rounded to nearest, once.
template <class T> struct Tok;
template <> struct Tok<float> {
  static constexpr int VEC = 4;
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct Tok<__nv_bfloat16> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Tok<__half> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};

// two 16-bit elements at a time
template <class T> struct TokPair;
template <> struct TokPair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ type down(float a, float b) { return __floats2bfloat162_rn(a, b); }
  static __device__ __forceinline__ float2 up(type e) { return __bfloat1622float2(e); }
};
template <> struct TokPair<__half> {
  using type = __half2;
  static __device__ __forceinline__ type down(float a, float b) { return __floats2half2_rn(a, b); }
  static __device__ __forceinline__ float2 up(type e) { return __half22float2(e); }
};

template <class T>
__device__ __forceinline__ void tok_unpack(const uint4 &v, float (&x)[Tok<T>::VEC]) {
  const T *p = reinterpret_cast<const T *>(&v);
#pragma unroll
  for (int i = 0; i < Tok<T>::VEC; ++i) x[i] = Tok<T>::up(p[i]);
}
template <class T>
__device__ __forceinline__ uint4 tok_pack(const float (&x)[Tok<T>::VEC]) {
  uint4 v;
  T *p = reinterpret_cast<T *>(&v);
#pragma unroll
  for (int i = 0; i < Tok<T>::VEC; ++i) p[i] = Tok<T>::down(x[i]);
  return v;
}

// Sums in base 2 against reference r: S = sum 2^((x - r) c), T = sum (x - r) c 2^((x - r) c).  m: the largest x; r is m, or 0 where m
// is -inf (then S = T = 0).
struct Soft { float m, r, S, T; };
__device__ __forceinline__ float soft_reference(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ void soft_rebase(Soft &a, float r, float c) {
  // (r is not below a.r but where nothing has been added yet; bounded, because 0 * inf has no place in S and T)
  const float d = fminf(fmaxf((a.r - r) * c, -1e30f), 0.f), f = tok_ex2(d);
  a.T = (a.T + d * a.S) * f;
  a.S *= f;
  a.r = r;
}
__device__ __forceinline__ void soft_join(Soft &a, Soft b, float c) {
  a.m = fmaxf(a.m, b.m);
  const float r = soft_reference(a.m);
  soft_rebase(a, r, c);
  soft_rebase(b, r, c);
  a.S += b.S;
  a.T += b.T;
}
__device__ __forceinline__ Soft soft_shfl(const Soft &a, int o) {
  return Soft{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.r, o), __shfl_xor_sync(0xffffffffu, a.S, o), __shfl_xor_sync(0xffffffffu, a.T, o)};
}

inline size_t tok_size(int dtype) { return dtype == PBG_F32 ? 4 : 2; }
inline bool tok_type(int dtype) { return dtype == PBG_F32 || dtype == PBG_BF16 || dtype == PBG_F16; }
inline bool tok_scale(float s) { return s >= 1e-20f && s <= 1e20f; }    // (false for NaN; beyond, products of powers of two would leave fp32)
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// CALL<element type>(...) by the run-time type
#define TOK_DISPATCH(DTYPE, CALL, ...)                                 \
  do {                                                                 \
    if ((DTYPE) == PBG_F32) CALL<float>(__VA_ARGS__);                  \
    else if ((DTYPE) == PBG_BF16) CALL<__nv_bfloat16>(__VA_ARGS__);    \
    else CALL<__half>(__VA_ARGS__);                                    \
  } while (0)

// The first failed launch of a call, as its status.
inline int tok_status() { return pbg_take_launch_error() == cudaSuccess ? PBG_OK : PBG_ERR_CUDA; }
inline int64_t tok_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
