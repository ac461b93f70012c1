// What the tiled products (ccq_linear.hip, ccq_fp8.hip) share: activations, values of a row at any element's address, and
// direct loads into LDS that a buffer resource bounds.
#pragma once

#include "ccq_block_args.h"
#include "ccq_oper.h"
#include "ccq_rows.h"

namespace ccq {

// An instruction that reads the accumulators behind products written in assembly, whose passes the compiler does not know.
__device__ __forceinline__ void acc_settled() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// ---------------------------------------------------------------------------
// activations, in fp32
// ---------------------------------------------------------------------------
constexpr int kActOther = -1;  // (of a kernel: any but none and swiglu)
constexpr float kTanhA = 0.7978845608028654f, kTanhB = 0.044715f;  // gelu_tanh: tanh(a (z + b z^3))

__device__ __forceinline__ float exp_(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + exp_(-z)); }

// erfc(x) = t e^(P(t) - x^2), t = 1 / (1 + x / 2), for x >= 0, and 2 - erfc(-x): the form of Numerical Recipes (section
// 6.2), its P of degree 9 fitted anew, the polynomial nearest to log(erfc(x) e^(x^2) / t) over t in (0, 1] in the largest
// error (1.0e-7; at 400 Chebyshev nodes with weights that even the errors out).  In fp32 within 4e-7.
__device__ __forceinline__ float erfc_(float x) {
  const float a = fabsf(x), t = __builtin_amdgcn_rcpf(1.f + 0.5f * a);
  float p = 0.168761006f;
  p = p * t - 0.813325556f;
  p = p * t + 1.47325527f;
  p = p * t - 1.12109976f;
  p = p * t + 0.271351518f;
  p = p * t - 0.183966161f;
  p = p * t + 0.0963881326f;
  p = p * t + 0.374125038f;
  p = p * t + 1.00002265f;
  p = p * t - 1.26551222f;
  const float e = t * exp_(p - a * a);
  return x < 0.f ? 2.f - e : e;
}

// the activation of C values (one switch for all: the functions are small, their selection is not)
template <int C>
__device__ __forceinline__ void act_values(int act, float (&v)[C]) {
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];  // (NaN stays)
      break;
    case kActSilu:
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] *= sigmoid(v[i]);
      break;
    case kActGelu:
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] *= 0.5f * erfc_(v[i] * -0.7071067811865476f);
      break;
    case kActGeluTanh:
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] *= sigmoid(2.f * kTanhA * (v[i] + kTanhB * v[i] * v[i] * v[i]));
      break;
    default: break;
  }
}

__device__ __forceinline__ float bias_at(const void* b, int bdtype, long i) {
  if (bdtype == kF32) return *gmem((const float*)b + i);
  if (bdtype == kBf16) return (float)*gmem((const bf16*)b + i);
  return (float)*gmem((const f16*)b + i);
}

// C consecutive values of a row of N from column n on, at any element's address
template <typename T, int C>
__device__ __forceinline__ void store_row(T* row, long n, long N, const float (&v)[C]) {
  typedef T vec __attribute__((ext_vector_type(C)));
  typedef vec any __attribute__((aligned(sizeof(T))));
  vec o;
#pragma unroll
  for (int i = 0; i < C; ++i) o[i] = (T)v[i];
  if (n + C <= N) {
    *gmem((any*)(row + n)) = o;
    return;
  }
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (n + i < N) *gmem(row + n + i) = o[i];
}
template <typename T, int C>
__device__ __forceinline__ void add_row(const T* row, long n, long N, float (&v)[C]) {
  typedef T vec __attribute__((ext_vector_type(C)));
  typedef vec any __attribute__((aligned(sizeof(T))));
  if (n + C <= N) {
    const vec r = *gmem((const any*)(row + n));
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] += (float)r[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (n + i < N) v[i] += (float)*gmem(row + n + i);
}

// C consecutive values of a row of T, at any element's address; zeros behind N
template <typename T, int C>
struct RowPiece {
  typedef T vec __attribute__((ext_vector_type(C)));
  typedef vec any __attribute__((aligned(sizeof(T))));
  vec v;
  __device__ void load(const T* row, long n, long N) {
    if (n + C <= N) {
      v = *gmem((const any*)(row + n));
      return;
    }
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = n + i < N ? *gmem(row + n + i) : (T)0.f;
  }
};

// A buffer resource bounds every load by the tile's end (along the rows: of its last row; down them: of the step's last
// row's columns); what lies behind comes as zeros.
__device__ __forceinline__ u32x4 resource(size_t base, unsigned bytes) {
  // (uniform all of it; whatever the compiler left in the vector unit all the same is brought back, and settled is called
  // before the resource is used)
  return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((int)base), (unsigned)__builtin_amdgcn_readfirstlane((int)(base >> 32)),
               (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}
// A scalar register that the vector unit wrote may be read by a memory instruction five wait states later; the compiler
// does not look into the instructions below.
__device__ __forceinline__ void settled(u32x4& r) { asm volatile("s_nop 4" : "+s"(r)); }
// A direct load of 64 pieces in two instructions, since M0 is read one wait state after it is written: between them
// stands a product, or a wait.
__device__ __forceinline__ void load_to(unsigned lds, int i) { asm volatile("s_add_u32 m0, %0, %1" ::"s"(lds), "i"(i * 1024) : "m0", "scc"); }
__device__ __forceinline__ void load_from(const u32x4& r, unsigned off) {
  asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(r) : "memory");
}
constexpr unsigned kNowhere = 0x80000000u;  // behind every resource's end

typedef __attribute__((address_space(3))) const s16x8 lds_s8;
__device__ __forceinline__ s16x8 read16(unsigned at) { return *(lds_s8*)(size_t)at; }

}  // namespace ccq
