// Shared device helpers of the losses over a set of classes (vsl_vocab.hip, vsl_linear_ce.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/vsloss.h"

namespace vsl_err {
int fail(int code, const std::string& msg);  // defined in vsl_loss.hip
}

namespace vsl_vocab {

using vsl_err::fail;

constexpr float kLog2e = 1.44269504088896340736f;  // and what a float leaves of it
constexpr float kLog2eLow = (float)(1.4426950408889634 - (double)1.44269504088896340736f);
constexpr float kLn2 = 0.693147180559945309417f;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float ninf() { return __uint_as_float(0xFF800000u); }
__device__ __forceinline__ float qnan() { return __uint_as_float(0x7FC00000u); }

template <typename T>
struct Vec {
  static constexpr int E = 16 / (int)sizeof(T);  // elements of a 16-byte vector
};

__device__ __forceinline__ void unpack(u32x4 r, float (&x)[8], const __bf16*) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(r[i] << 16);
    x[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack(u32x4 r, float (&x)[8], const _Float16*) {
  const half8 h = __builtin_bit_cast(half8, r);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
}
__device__ __forceinline__ void unpack(u32x4 r, float (&x)[4], const float*) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ u32x4 pack(const float (&x)[8], const __bf16*) {
  bf16x8 h;
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (__bf16)x[i];
  return __builtin_bit_cast(u32x4, h);
}
__device__ __forceinline__ u32x4 pack(const float (&x)[8], const _Float16*) {
  half8 h;
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (_Float16)x[i];
  return __builtin_bit_cast(u32x4, h);
}
__device__ __forceinline__ u32x4 pack(const float (&x)[4], const float*) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(x[i]);
  return r;
}

// 16-byte accesses that only assume the element's own alignment: rows of an odd vocabulary start anywhere, and the
// memory pipeline splits such an access by itself.
typedef u32x4 u32x4_any2 __attribute__((aligned(2)));
typedef u32x4 u32x4_any4 __attribute__((aligned(4)));
__device__ __forceinline__ u32x4 load16(const float* p) { return *(const u32x4_any4*)p; }
__device__ __forceinline__ u32x4 load16(const __bf16* p) { return *(const u32x4_any2*)p; }
__device__ __forceinline__ u32x4 load16(const _Float16* p) { return *(const u32x4_any2*)p; }
__device__ __forceinline__ void store16(float* p, u32x4 v) { *(u32x4_any4*)p = v; }
__device__ __forceinline__ void store16(__bf16* p, u32x4 v) { *(u32x4_any2*)p = v; }
__device__ __forceinline__ void store16(_Float16* p, u32x4 v) { *(u32x4_any2*)p = v; }

// Elements [i, i + E) of a row that ends at `end`, kept in their own type; what lies behind the end reads as -infinity.
template <typename T>
__device__ __forceinline__ unsigned ninf_word() {  // all elements of a 32-bit word -infinity
  return sizeof(T) == 4 ? 0xFF800000u : __is_same(T, __bf16) ? 0xFF80FF80u : 0xFC00FC00u;
}
template <typename T>
__device__ __forceinline__ u32x4 load_row(const T* row, int i, int end) {
  if (i + Vec<T>::E <= end) return load16(row + i);
  const unsigned none = ninf_word<T>();
  if (i >= end) return u32x4{none, none, none, none};
  float x[Vec<T>::E];
#pragma unroll
  for (int e = 0; e < Vec<T>::E; ++e) x[e] = i + e < end ? (float)row[i + e] : ninf();
  return pack(x, (const T*)nullptr);
}

// ---- reductions over groups of 16 lanes by data-parallel primitives (no LDS), wider ones by shuffles
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ unsigned long long dpp(unsigned long long v) {
  return ((unsigned long long)dpp<CTRL>((unsigned)(v >> 32)) << 32) | dpp<CTRL>((unsigned)v);
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kMirror4 = 0x1B, kMirror8 = 0x141, kMirror16 = 0x140;
// the value of lane ^ X, X a power of two or one less (a mirror)
template <int X, typename V>
__device__ __forceinline__ V lane_xor(V v) {
  if (X == 1) return dpp<kXor1>(v);
  if (X == 2) return dpp<kXor2>(v);
  if (X == 3) return dpp<kMirror4>(v);
  if (X == 4) return dpp<kMirror8>(dpp<kMirror4>(v));
  if (X == 7) return dpp<kMirror8>(v);
  if (X == 8) return dpp<kMirror16>(dpp<kMirror8>(v));
  if (X == 15) return dpp<kMirror16>(v);
  return (V)__shfl_xor(v, X, 64);
}

// all L lanes of a group (L = 8, 16 or 64, aligned) get op over the group
template <int L, typename V, typename Op>
__device__ __forceinline__ V group_all(V v, Op op) {
  v = op(v, dpp<kXor1>(v));
  v = op(v, dpp<kXor2>(v));
  v = op(v, dpp<kMirror8>(v));
  if (L > 8) v = op(v, dpp<kMirror16>(v));
  if (L > 16) {
    v = op(v, (V)__shfl_xor(v, 16, 64));
    v = op(v, (V)__shfl_xor(v, 32, 64));
  }
  return v;
}
struct AddF {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
// maximum that hands a NaN on
struct MaxF {
  __device__ __forceinline__ float operator()(float a, float b) const { return __builtin_elementwise_maximum(a, b); }
};
struct MaxU {
  template <typename K>
  __device__ __forceinline__ K operator()(K a, K b) const { return a > b ? a : b; }
};

// ---- running maximum m and sum s of 2^((x - m) c); nothing seen: (-inf, 0).  The maximum stays in the logits' own scale
// and apart from the logarithm of the sum: times c, or with the logarithm added, it would overflow or swallow it in a row
// of the type's lowest values, which masks are made of.
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ float exp_ref(float m) { return m == ninf() ? 0.0f : m; }  // keeps -inf - -inf out of exponents
__device__ __forceinline__ float exp_of(float x, float ref, float c) { return __builtin_amdgcn_exp2f((x - ref) * c); }
// The same for many x <= ref as one multiply-add and one exponential each: 2^(x c - round(ref c)), which is 2^((x - ref) c) times
// a factor that all terms of one ref share, 2^rest, rest = ref c - round(ref c).  Half a step of ref c is little beside 1 only
// while the logits are small (a relative error of 4e-5 at 1000, and at -1e9, which masks are made of, 2^64), so whoever uses
// the terms multiplies by factor(): once a row, a thread or a tile; the multiply-add that gives `rest` is exact.  From 2^31 on
// ref c would leave float's range or `rest` the range of the exponential; there floats are so far apart that every other x
// gives 0 (next * c is at least 2^7 away), as it also does with c a power of two that puts them 2^8 apart; with it ref c is
// exact and `rest` 0.  The instruction gives 0 for results below 2^-126, beside a largest term of 2^rest: no sum feels them, a
// gradient loses at most 2^-62 of its factor at rest = -64, 2^-125 in ordinary rows.
struct Exponent {
  float c, shift, rest;
  __device__ __forceinline__ Exponent(float ref, float scale) {
    const unsigned far = (286u - (__float_as_uint(ref) >> 23 & 255u)) << 23;  // 2^(32 - exponent of ref)
    c = fabsf(ref * scale) < 0x1p31f ? scale : __uint_as_float(far);
    shift = -(ref * c);
    rest = fmaf(ref, c, shift);
  }
  __device__ __forceinline__ float operator()(float x) const { return __builtin_amdgcn_exp2f(fmaf(x, c, shift)); }
  __device__ __forceinline__ float factor(float log2_divisor = 0.0f) const { return __builtin_amdgcn_exp2f(-(rest + log2_divisor)); }
};
// A thread's running sum: of terms as an Exponent of its maximum gives them, times 2^-rest only at the end.
struct RunSum {
  float m = ninf(), s = 0.0f, rest = 0.0f;
  __device__ __forceinline__ Exponent move(float to, float c) {  // to >= m; the terms that follow are those of the result
    const Exponent ex(exp_ref(to), c);
    s *= __builtin_amdgcn_exp2f(fmaf(m, ex.c, ex.shift) - rest);  // 1 where the maximum stays
    m = to;
    rest = ex.rest;
    return ex;
  }
  __device__ __forceinline__ MaxSum get() const { return {m, s * __builtin_amdgcn_exp2f(-rest)}; }
};
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c) {
  const float m = __builtin_elementwise_maximum(a.m, b.m), r = exp_ref(m);
  return {m, a.s * exp_of(a.m, r, c) + b.s * exp_of(b.m, r, c)};
}

template <int L>
__device__ __forceinline__ MaxSum group_join(MaxSum a, float c) {
  const float m = group_all<L>(a.m, MaxF());
  return {m, group_all<L>(a.s * exp_of(a.m, exp_ref(m), c), AddF())};
}
// all threads of the block get the join of all; red: 2 * WAVES floats of LDS, free again after the call's last barrier
template <int WAVES>
__device__ __forceinline__ MaxSum block_join(MaxSum a, float* red, float c) {
  a = group_join<64>(a, c);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    red[2 * (threadIdx.x >> 6)] = a.m;
    red[2 * (threadIdx.x >> 6) + 1] = a.s;
  }
  __syncthreads();
  MaxSum t{red[0], red[1]};
#pragma unroll
  for (int w = 1; w < WAVES; ++w) t = join(t, {red[2 * w], red[2 * w + 1]}, c);
  return t;
}
// log2 of the sum above the maximum, for 2^((x - m) c - log2_sum); nothing seen: the maximum itself says so
__device__ __forceinline__ float log2_sum(MaxSum a) { return __builtin_amdgcn_logf(a.s); }
// natural logarithm of the whole sum, for the outputs
__device__ __forceinline__ float log_sum(MaxSum a, float inv_temperature) {
  return a.m == ninf() ? ninf() : fmaf(log2_sum(a), kLn2, a.m * inv_temperature);
}
template <int WAVES>
__device__ __forceinline__ float block_add(float v, float* red) {
  v = group_all<64>(v, AddF());
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = red[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) t += red[w];
  return t;
}

// ---- reduced loss
__device__ __forceinline__ void finish_sum(double total, double count, int reduction, float* loss, float* divisor) {
  *loss = (float)(reduction == VSL_REDUCE_MEAN ? (count == 0.0 ? 0.0 : total / count) : total);
  *divisor = (float)count;
}

// ---- host side
inline int launch_status(const char* what) {
  if (hipError_t e = hipGetLastError(); e != hipSuccess)
    return fail(VSL_ERR_LAUNCH_FAILED, std::string(what) + ": kernel launch failed: " + hipGetErrorString(e));
  return VSL_OK;
}
inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Reduced loss of `rows` row losses in a fixed order (float64 sums): *loss = sum or mean, *divisor = what the mean is
// divided by: the sum of `weights`, or the number of rows.  partial: sum_workspace_bytes(rows) bytes.
size_t sum_workspace_bytes(int64_t rows);
void launch_sum(const float* row_loss, const float* weights, int64_t rows, int reduction, void* partial, float* loss,
                float* divisor, hipStream_t s);
// The same from n (sum, count) pairs of float64 that blocks of a kernel have left.
void launch_sum_pairs(const double* pairs, int64_t n, int reduction, float* loss, float* divisor, hipStream_t s);

}  // namespace vsl_vocab
