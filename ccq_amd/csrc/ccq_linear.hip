// Linear map with an epilogue, y = act(x W^T + b) + r, for any number of rows, and its backward:
//
//   z = x W^T + b,  y = act(z) + r    act: none, relu, silu, gelu (erf), gelu (tanh), swiglu (z = [gate | up],
//                                     silu(gate) up)
//   dz = act'(z) dy,  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// All three products run on one tiled kernel: bf16 or fp16 operands, fp32 accumulation on the matrix cores
// (16x16x32), tiles staged in LDS by direct loads.  Its operands are stored with the contraction along the rows
// (x and W forward; dz in dx) or down them (W in dx; dz and x in dW); the second kind is read out of LDS by
// transposing reads, so nothing is transposed in memory.
#include <algorithm>
#include <type_traits>

#include "ccq_block_args.h"
#include "ccq_oper.h"
#include "ccq_rows.h"

namespace ccq {

namespace {

// c += a b on the matrix cores, the accumulator kept where it is: left to itself the register allocator moves the 256
// accumulator registers of a wave about between the products.  What the compiler does not know of an instruction
// written like this -- that its result may be read by others only after its passes -- is waited for by acc_settled.
template <typename T>
__device__ __forceinline__ void product16(const s16x8& a, const s16x8& b, f32x4& c) {
  if constexpr (__is_same(T, bf16)) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
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
// d = d act'(z)
template <int C, typename Z>
__device__ __forceinline__ void act_slopes(int act, const Z& z, float (&d)[C]) {
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int i = 0; i < C; ++i) d[i] *= z[i] > 0.f ? 1.f : z[i] <= 0.f ? 0.f : z[i];
      break;
    case kActSilu:
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const float g = sigmoid(z[i]);
        d[i] *= g * (1.f + z[i] * (1.f - g));
      }
      break;
    case kActGelu:
#pragma unroll
      for (int i = 0; i < C; ++i)
        d[i] *= 0.5f * erfc_(z[i] * -0.7071067811865476f) + z[i] * 0.3989422804014327f * exp_(-0.5f * z[i] * z[i]);
      break;
    case kActGeluTanh:
#pragma unroll
      for (int i = 0; i < C; ++i) {
        // (the slope is 0 or 1 long before 16; the square of a far z would overflow)
        const float x = z[i] != z[i] ? z[i] : fminf(fmaxf(z[i], -16.f), 16.f);
        const float g = sigmoid(2.f * kTanhA * (x + kTanhB * x * x * x));
        d[i] *= g + x * 2.f * g * (1.f - g) * kTanhA * (1.f + 3.f * kTanhB * x * x);
      }
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

// The values before the activation are kept for the backward in 24 bits, fp32 rounded to its upper three bytes: 16 bits of
// them would be the largest error of dx and dW (swiglu, bf16: 1.76 times the one rounding of the result; so 1.42, the
// other being that of dz), and 32 cost 8 bytes of traffic an element for 6.  A plane of 16 bits, then one of 8, both
// [M, ldz], written and read past the caches: they are used once, and late (16384 x 2816 swiglu over 1024, forward and
// backward: 668 -> 651 us).
constexpr float kMostKept = 0x1.ffffp127f;  // rounds to infinity, as all above
template <int C>
__device__ __forceinline__ void keep_z(void* z, long rows, long ld, long m, long n, long end, const float (&v)[C]) {
  unsigned short* hi = (unsigned short*)z + m * ld;
  unsigned char* lo = (unsigned char*)z + rows * ld * 2 + m * ld;
  typedef unsigned short hvec __attribute__((ext_vector_type(C)));
  typedef unsigned char lvec __attribute__((ext_vector_type(C)));
  typedef hvec hany __attribute__((aligned(2)));
  typedef lvec lany __attribute__((aligned(1)));
  hvec h;
  lvec b;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    // To the nearest (forward of 16384 x 2816 swiglu over 1024 cut off 206 us, rounded 208); what would round past the
    // largest number, infinities and NaN as they are (a sum's NaN is a quiet one, which the upper bits hold).
    unsigned u = __float_as_uint(v[i]);
    u += __builtin_fabsf(v[i]) < kMostKept ? 0x80u : 0u;
    h[i] = (unsigned short)(u >> 16);
    b[i] = (unsigned char)(u >> 8);
  }
  if (n + C <= end) {
    __builtin_nontemporal_store((hany)h, gmem((hany*)(hi + n)));
    __builtin_nontemporal_store((lany)b, gmem((lany*)(lo + n)));
    return;
  }
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (n + i < end) {
      *gmem(hi + n + i) = h[i];
      *gmem(lo + n + i) = b[i];
    }
}
template <int C>
struct KeptZ {
  typedef unsigned short hvec __attribute__((ext_vector_type(C)));
  typedef unsigned char lvec __attribute__((ext_vector_type(C)));
  typedef hvec hany __attribute__((aligned(2)));
  typedef lvec lany __attribute__((aligned(1)));
  hvec h;
  lvec b;
  __device__ void load(const void* z, long rows, long ld, long m, long n, long end) {
    const unsigned short* hi = (const unsigned short*)z + m * ld;
    const unsigned char* lo = (const unsigned char*)z + rows * ld * 2 + m * ld;
    if (n + C <= end) {
      h = __builtin_nontemporal_load(gmem((const hany*)(hi + n)));
      b = __builtin_nontemporal_load(gmem((const lany*)(lo + n)));
      return;
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      h[i] = n + i < end ? *gmem(hi + n + i) : (unsigned short)0;
      b[i] = n + i < end ? *gmem(lo + n + i) : (unsigned char)0;
    }
  }
  __device__ float operator[](int i) const { return __uint_as_float((unsigned)h[i] << 16 | (unsigned)b[i] << 8); }
};

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

// What the epilogue of C columns from n on needs of them whatever the row: the bias (swiglu: of both halves).
template <int C, bool glu>
struct ColumnBias {
  float v[C], up[glu ? C : 1];
  __device__ void load(const ProductArgs& p, long n) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      v[i] = p.bias && n + i < p.N ? bias_at(p.bias, p.bdtype, n + i) : 0.f;
      if (glu) up[glu ? i : 0] = p.bias && n + i < p.N ? bias_at(p.bias, p.bdtype, p.N + n + i) : 0.f;
    }
  }
};

// The epilogue of C consecutive columns n .. of row m (swiglu: v the gates, up the other half).  ACT: none, swiglu, or
// any other (p.act), kept apart since the code of all of them takes up the instruction cache of those that need none.
template <typename T, int C, int ACT, bool with_res, bool glu = ACT == kActSwiglu>
__device__ __forceinline__ void finish(const ProductArgs& p, long m, long n, float (&v)[C], float (&up)[C],
                                       const ColumnBias<C, glu>& bias, const RowPiece<T, C>& res) {
#pragma unroll
  for (int i = 0; i < C; ++i) {
    v[i] += bias.v[i];
    if (glu) up[i] += bias.up[glu ? i : 0];
  }
  if (p.z) {
    keep_z<C>(p.z, p.M, p.ldz, m, n, p.N, v);
    if (glu) keep_z<C>(p.z, p.M, p.ldz, m, p.N + n, 2 * p.N, up);
  }
  if (glu) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = v[i] * sigmoid(v[i]) * up[i];
  } else if (ACT != kActNone) {
    act_values<C>(p.act, v);
  }
  if (with_res)
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] += (float)res.v[i];
  store_row<T, C>((T*)p.out + m * p.ldo, n, p.N, v);
}

// ---------------------------------------------------------------------------
// the tiled product
// ---------------------------------------------------------------------------
constexpr int kStep = 64;  // contraction elements a step

// One operand's tile of a step in LDS: R rows of the product by 64 contraction elements.
//   along the rows (DOWN = false): R rows of 128 bytes, 16-byte piece s of row r at piece s ^ swz(r)
//   down the rows  (DOWN = true):  64 rows of 2 R bytes, piece s of row k at piece s ^ swz(k)
// so that the sixteen pieces that a fragment read takes at once lie in different banks.  Direct loads write 1 KiB
// (64 pieces) each, in LDS order: the swizzle is in the address that a lane reads.
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
// The whole steps of a workgroup's contraction, from step `turn` on and round to it again; behind the last one the
// resource is empty.  Few scalar instructions and no branch: it runs between two products.
template <bool DOWN>
struct StepStream {
  size_t base;           // of the step to come
  long step, back;       // bytes to the next step, from the last to the first
  unsigned bytes, last;  // along: to the tile's end, bytes of a round; down: of a step, of the last one
  int ahead, until;      // steps not yet asked for, steps to the end of the whole ones
  __device__ StepStream(size_t first, long step, int whole, int turn, unsigned bytes, unsigned last)
      : base(first + turn * step), step(step), back(-(whole - 1) * step), bytes(DOWN ? bytes : bytes - turn * 128),
        last(DOWN ? last : (whole - 1) * 128), ahead(whole), until(whole - turn) {}
  __device__ u32x4 next() {
    const bool end = until == 1;
    const u32x4 r = resource(base, ahead <= 0 ? 0u : DOWN && end ? last : bytes);
    base += end ? back : step;
    if (!DOWN) bytes += end ? last : -128u;
    --ahead;
    --until;
    return r;
  }
};
constexpr unsigned kNowhere = 0x80000000u;  // behind every resource's end

// swizzle of product row r of an operand read in consecutive rows (A), or in the order of column pairs (B)
__device__ __forceinline__ int swz_a(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int swz_b(int n) { return ((n >> 1) & 1) | (((n >> 3) & 3) << 1); }
// of contraction row k of an operand stored down the rows, R columns a row
template <int R>
__device__ __forceinline__ int swz_down(int k) { return ((k & 3) | (((k >> 3) & 1) << 2)) << 1 & (R / 8 - 1); }

// Loads of a tile: wave w of NW takes instructions w * PER .. (consecutive pieces of LDS).
template <int R, bool DOWN, bool B, int NW>
struct TileLoad {
  static constexpr int PER = R * kStep * 2 / 1024 / NW;
  static_assert(PER >= 1 && R * kStep * 2 % (1024 * NW) == 0, "whole instructions a wave");
  unsigned off[PER];  // byte offset of this lane's piece from the tile's base
  unsigned lds;       // LDS byte address of this wave's first piece, in stage 0
  __device__ void init(unsigned lds_base, int wave, int l, long ld) {
    lds = lds_base + wave * PER * 1024;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int q = (wave * PER + i) * 64 + l;  // piece of the tile in LDS order
      if (DOWN) {
        const int k = q / (R / 8), s = q % (R / 8);
        off[i] = (unsigned)(k * ld * 2) + ((s ^ swz_down<R>(k)) << 4);
      } else {
        const int r = q >> 3, s = q & 7;
        off[i] = (unsigned)(r * ld * 2) + ((s ^ (B ? swz_b(r) : swz_a(r))) << 4);
      }
    }
  }
  // all of a step at `stage` (bytes); contraction elements at and behind `limit` < 64 of an along operand as zeros
  __device__ void issue(const u32x4& r, unsigned stage, int limit, int wave, int l) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      unsigned f = off[i];
      if (!DOWN && limit < kStep) {
        const int q = (wave * PER + i) * 64 + l, row = q >> 3;
        if ((((q & 7) ^ (B ? swz_b(row) : swz_a(row))) << 3) >= limit) f = kNowhere;
      }
      load_to(lds + stage, i);
      asm volatile("s_nop 0");
      load_from(r, f);
    }
  }
};

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) const s16x8 lds_s8;
__device__ __forceinline__ s16x8 read16(unsigned at) { return *(lds_s8*)(size_t)at; }
__device__ __forceinline__ s16x4_t read_tr4(unsigned at) {
  typedef __attribute__((address_space(3))) s16x4_t lds_s4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(size_t)at);
}

enum : int { kPlain = 0, kEpilogue = 1, kPartial = 2 };

// BM x BN tile of the product by WM x WN waves, NA stages of A in LDS and NB of B.  Lane l of a wave holds, of each 16x16
// tile (it, j) of the wave, row m = 16 it + (l & 15) and four consecutive columns.  Along-the-row B operands (the forward)
// are read so that the column tiles j = 2 q and 2 q + 1 of a lane are eight consecutive columns, one 16-byte store.
// swiglu: half of a wave's columns are gates, the other half the ups beside them, so a lane holds both.
//
// A step of 64 contraction elements is two halves of 32.  While the matrix cores work on one half's fragments the
// other half's are read from LDS into registers and the direct loads of a later step are issued, each
// between two products (in clumps they keep the one wave of a SIMD from issuing products).  The one barrier of a step
// lies between the halves, where every wave has read the step's stages (loads may overwrite them) and the next step's
// have landed.  The 160 KiB of LDS hold two and a half stages of 256 x 256: the half goes to A, whose rows come from HBM and are
// asked for three steps ahead, while B's, which the workgroups of all tile rows share, lie in the caches.
template <typename T, int BM, int BN, int WM, int WN, int NA, int NB, bool DA, bool DB, int MODE, int ACT>
__global__ __launch_bounds__(WM * WN * 64) void product_kernel(const ProductArgs p) {
  constexpr bool GLU = ACT == kActSwiglu;
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr unsigned kA = BM * kStep * 2, kB = BN * kStep * 2, kRing = NA * kA + NB * kB;  // bytes of a stage; of all
  constexpr int HALF = BN / WN / 2;  // swiglu: gates of a wave
  static_assert(!GLU || (!DB && MODE == kEpilogue), "gates and ups of one wave");
  static_assert(TM == TN, "one fragment of each operand between two rows of products");
  constexpr int kPass = TM < 4 ? TM * 16 : 64, kRow = TN * 16 + 4;  // rows of a wave in the epilogue at a time, floats a row
  constexpr unsigned kOut = NW * kPass * kRow * 4;
  __shared__ __attribute__((aligned(1024))) char smem[kRing > kOut ? kRing : kOut];
  const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  constexpr int NT = GLU ? BN / 2 : BN;  // output columns of a tile
  // tile of this workgroup: each XCD (workgroups are handed out round-robin over the 8) takes consecutive tiles, in
  // column order within bands of 8 tile rows, so that its L2 holds what its workgroups share
  const int tm = (int)((p.M + BM - 1) / BM), tn = (int)((p.N + NT - 1) / NT), tiles = tm * tn;
  const int xcd = blockIdx.x & 7, q8 = tiles >> 3, r8 = tiles & 7;
  const int t = xcd * q8 + min(xcd, r8) + (blockIdx.x >> 3);
  const int band = t / (8 * tn), in = t - band * 8 * tn, rows = min(8, tm - band * 8);
  const long m0 = (long)(band * 8 + in % rows) * BM, n0 = (long)(in / rows) * NT;
  // steps of this workgroup: whole ones, and the contraction's end
  const int all = (int)((p.K + kStep - 1) / kStep), per = (all + p.splits - 1) / p.splits;
  const int s0 = blockIdx.y * per, s1 = min(all, s0 + per);
  const int tail = (!DA || !DB) && s1 == all && s0 < s1 ? (int)(p.K & (kStep - 1)) : 0;  // (down both: zeros by the end)
  const int whole = max(0, s1 - s0 - (tail ? 1 : 0));

  const unsigned lds0 = lds_addr(smem);
  typedef TileLoad<BM, DA, false, NW> LoadA;
  typedef TileLoad<BN, DB, !DB, NW> LoadB;
  static_assert(LoadA::PER == TM && LoadB::PER == TN, "one load of each operand between two rows of products");
  LoadA la;
  LoadB lb;
  la.init(lds0, wave, l, p.lda);
  lb.init(lds0 + NA * kA, wave, l, p.ldb);
  // Rows of an operand that lie a multiple of 4 KiB apart meet in one channel of the L2 at any one step.  So the tile
  // rows of a band begin their contraction at different steps, 256 bytes apart, and come round to them at its end;
  // those of one tile row keep together and find its operand in the L2.  (8192^3 forward: 849 -> 788 us; contractions
  // of few steps gain nothing and lose the operands' meeting in the L2: 16384 x 5632 over 1024, 187 -> 193 us.)
  const int turn = BM == 256 && whole >= 32 ? 2 * (int)(in % rows) : 0;
  const long stepA = (DA ? kStep * p.lda : kStep) * 2, stepB = (DB ? kStep * p.ldb : kStep) * 2;
  const size_t pa = (size_t)p.a + (DA ? (long)s0 * kStep * p.lda + m0 : m0 * p.lda + (long)s0 * kStep) * 2;
  size_t pb = (size_t)p.b + (DB ? (long)s0 * kStep * p.ldb + n0 : n0 * p.ldb + (long)s0 * kStep) * 2;
  if constexpr (GLU) {
    // tile row 2 HALF w + c of B: gate n0 + HALF w + c for c < HALF, up n0 + HALF w + c - HALF behind
    static_assert(LoadB::PER * 8 == HALF, "a wave loads gates or ups");
    if (wave & 1) pb += p.N * p.ldb * 2;
#pragma unroll
    for (int i = 0; i < LoadB::PER; ++i) {
      const int r = ((wave * LoadB::PER + i) * 64 + l) >> 3;
      lb.off[i] = (unsigned)((r / (2 * HALF) * HALF + r % HALF) * p.ldb * 2) + (((l & 7) ^ swz_b(r)) << 4);
    }
  }
  // bytes from a tile's first element to the end of the last of `n` rows, which has `cols` columns left and is whole
  // pieces to its end
  auto extent = [](long n, long ld, long cols) { return (unsigned)(((n - 1) * ld + ((cols + 7) & ~7L)) * 2); };
  const long left = p.K - (long)s0 * kStep, end = (long)kStep * (whole - 1);  // contraction from here on; to the last whole step
  const StepStream<DA> first_a(pa, stepA, whole, turn, DA ? extent(kStep, p.lda, p.M - m0) : extent(min((long)BM, p.M - m0), p.lda, left),
                               extent(min((long)kStep, left - end), p.lda, p.M - m0));
  const StepStream<DB> first_b(pb, stepB, whole, turn, DB ? extent(kStep, p.ldb, p.N - n0) : extent(min((long)NT, p.N - n0), p.ldb, left),
                               extent(min((long)kStep, left - end), p.ldb, p.N - n0));
  StepStream<DA> sa = first_a;
  StepStream<DB> sb = first_b;
  u32x4 ra, rb;

  // fragment addresses of this lane in stage 0
  const int r = l & 15, g = l >> 4;
  unsigned fa[DA ? TM : 2], fb[DB ? TN : 2];
  if constexpr (DA) {
    const int k = 8 * g + (r >> 2), s = wm * TM * 2 + ((r >> 1) & 1);
#pragma unroll
    for (int it = 0; it < TM; ++it)
      fa[it] = lds0 + k * (BM * 2) + (((s + 2 * it) ^ swz_down<BM>(k)) << 4) + 8 * (r & 1);
  } else {
    const int row = wm * TM * 16 + r;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) fa[kk] = lds0 + row * 128 + (((4 * kk + g) ^ swz_a(row)) << 4);
  }
  if constexpr (DB) {
    const int k = 8 * g + (r >> 2), s = wn * TN * 2 + ((r >> 1) & 1);
#pragma unroll
    for (int j = 0; j < TN; ++j)
      fb[j] = lds0 + NA * kA + k * (BN * 2) + (((s + 2 * j) ^ swz_down<BN>(k)) << 4) + 8 * (r & 1);
  } else {
    const int row = wn * TN * 16 + 8 * (r >> 2) + (r & 3);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) fb[kk] = lds0 + NA * kA + row * 128 + (((4 * kk + g) ^ swz_b(row)) << 4);
  }
  auto read_a = [&](int it, unsigned stage, int kk) -> s16x8 {
    if constexpr (DA) {
      const unsigned at = fa[it] + stage + kk * 32 * BM * 2;
      return __builtin_shufflevector(read_tr4(at), read_tr4(at + 4 * BM * 2), 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return read16(fa[kk] + stage + it * 16 * 128);
    }
  };
  auto read_b = [&](int j, unsigned stage, int kk) -> s16x8 {
    if constexpr (DB) {
      const unsigned at = fb[j] + stage + kk * 32 * BN * 2;
      return __builtin_shufflevector(read_tr4(at), read_tr4(at + 4 * BN * 2), 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return read16(fb[kk] + stage + (32 * (j >> 1) + 4 * (j & 1)) * 128);
    }
  };

  // fragment k of a half in the order that its products need them: a[0], b[0..], a[1..]
  auto read = [&](s16x8(&a)[TM], s16x8(&b)[TN], int k, unsigned stage_a, unsigned stage_b, int kk) {
    if (k == 0) a[0] = read_a(0, stage_a, kk);
    else if (k <= TN) b[k - 1] = read_b(k - 1, stage_b, kk);
    else a[k - TN] = read_a(k - TN, stage_a, kk);
  };
  // products between two loads, and between two fragment reads: the reads end at three quarters of the half, so that
  // the last ones have arrived by its end
  constexpr int kLoadGap = TM * TN / (TM + TN), kReadGap = std::max(1, TM * TN * 3 / 4 / (TM + TN));

  f32x4 acc[TM][TN];
  auto clear = [&] {
#pragma unroll
    for (int it = 0; it < TM; ++it)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        acc[it][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        asm volatile("" : "+a"(acc[it][j]));
      }
    acc_settled();
  };
  s16x8 a0[TM], b0[TN], a1[TM], b1[TN];  // fragments of the two halves

  if (whole > 0) {
    auto load_a = [&](unsigned stage) {
      ra = sa.next();
      settled(ra);
      la.issue(ra, stage, kStep, wave, l);
    };
    auto load_b = [&](unsigned stage) {
      rb = sb.next();
      settled(rb);
      lb.issue(rb, stage, kStep, wave, l);
    };
#pragma unroll
    for (int i = 0; i < NA; ++i) {  // in the order that the steps ask for them
      if (i >= NA - NB) load_b((i - (NA - NB)) * kB);
      load_a(i * kA);
    }
    clear();  // (while the first loads are on their way)
    // loads that may be on their way behind those of a step: of the steps asked for later, and A's of the same time
    constexpr int kBehind = (NB < NA ? TM : 0) + (NB - 2) * (TM + TN);
    wait_loads<kBehind + TM + TN>();
    lds_barrier();
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      b0[i] = read_b(i, 0, 0);
      a0[i] = read_a(i, 0, 0);
    }
    unsigned st_a = 0, st_b = 0;  // the step's stages
    auto step = [&](auto with_loads) {
      constexpr bool kLoads = decltype(with_loads)::value;
      const unsigned next_a = st_a == (NA - 1) * kA ? 0 : st_a + kA, next_b = st_b == (NB - 1) * kB ? 0 : st_b + kB;
#pragma unroll
      for (int q = 0; q < TM * TN; ++q) {
        product16<T>(b0[q % TN], a0[q / TN], acc[q / TN][q % TN]);
        if (kLoads && q == 0) {
          ra = sa.next();
          settled(ra);
        }
        if (kLoads && q == 2) {
          rb = sb.next();
          settled(rb);
        }
        if (q % kReadGap == kReadGap - 1 && q / kReadGap < TM + TN) read(a1, b1, q / kReadGap, st_a, st_b, 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      wait_loads<kLoads ? kBehind : 0>();
      lds_barrier();  // this step's stages are read, the next step's have landed (not yet A's behind it)
      const unsigned to_a = la.lds + st_a, to_b = lb.lds + st_b;
#pragma unroll
      for (int q = 0; q < TM * TN; ++q) {
        constexpr int kGap = kLoadGap;
        const int k = q / kGap;
        if (kLoads && q % kGap == 0) {
          if (k < TN) load_to(to_b, k);
          else load_to(to_a, k - TN);
        }
        product16<T>(b1[q % TN], a1[q / TN], acc[q / TN][q % TN]);
        if (kLoads && q % kGap == 0) {
          if (k < TN) load_from(rb, lb.off[k < TN ? k : 0]);
          else load_from(ra, la.off[k < TN ? 0 : k - TN]);
        }
        if (q % kReadGap == kReadGap - 1 && q / kReadGap < TM + TN) read(a0, b0, q / kReadGap, next_a, next_b, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      st_a = next_a;
      st_b = next_b;
    };
    for (int s = NB; s < whole; ++s) step(std::true_type{});
    // the last steps ask for nothing (the reads of the very last are of a stage behind, and not used)
    for (int s = max(0, whole - NB); s < whole; ++s) step(std::false_type{});
    lds_barrier();
  } else {
    clear();
  }
  if (tail) {
    const long n = left - (long)kStep * whole;  // elements of the end
    ra = resource(pa + whole * stepA, DA ? extent(n, p.lda, p.M - m0) : extent(min((long)BM, p.M - m0), p.lda, n));
    rb = resource(pb + whole * stepB, DB ? extent(n, p.ldb, p.N - n0) : extent(min((long)NT, p.N - n0), p.ldb, n));
    settled(ra);
    settled(rb);
    la.issue(ra, 0, tail, wave, l);
    lb.issue(rb, 0, tail, wave, l);
    wait_loads<0>();
    lds_barrier();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        a0[i] = read_a(i, 0, kk);
        b0[i] = read_b(i, 0, kk);
      }
#pragma unroll
      for (int it = 0; it < TM; ++it)
#pragma unroll
        for (int j = 0; j < TN; ++j) product16<T>(b0[j], a0[it], acc[it][j]);
    }
  }

  // The epilogue, 64 rows of a wave at a time: through LDS (its own part, rows 16 bytes apart in the banks), so that a
  // lane takes eight consecutive columns of a row whatever the fragments' order was, and its code exists once or twice
  // rather than once for every tile of the wave.
  acc_settled();
  lds_barrier();
  float* mine = (float*)(smem + wave * kPass * kRow * 4);
#pragma unroll
  for (int h = 0; h < TM * 16 / kPass; ++h) {
#pragma unroll
    for (int i = 0; i < kPass / 16; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
        *(f32x4*)(mine + (16 * i + r) * kRow + (DB ? 16 * j + 4 * g : 32 * (j >> 1) + 4 * (j & 1) + 8 * g)) = acc[h * (kPass / 16) + i][j];
    __builtin_amdgcn_wave_barrier();  // (LDS operations of a wave are in order)
    constexpr int WC = GLU ? HALF : TN * 16, PR = WC / 8;  // output columns of the wave, pieces of a row
    constexpr int RI = 64 / PR, NG = kPass / RI < 4 ? kPass / RI : 4;                    // rows at a time, and how often between the residual's loads
    const int c = l % PR * 8;
    const long n = n0 + wn * WC + c, mh = m0 + wm * TM * 16 + h * kPass + l / PR;
    auto row_out = [&](int i, const auto& bias, const RowPiece<T, 8>& res, auto with_res) {
      const long m = mh + i;
      if (m >= p.M || n >= p.N) return;
      float v[8], up[8];
      const float* row = mine + (i + l / PR) * kRow + c;
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        *(f32x4*)(v + e) = *(const f32x4*)(row + e);
        if (GLU) *(f32x4*)(up + e) = *(const f32x4*)(row + HALF + e);
      }
      if constexpr (MODE == kEpilogue) finish<T, 8, ACT, decltype(with_res)::value>(p, m, n, v, up, bias, res);
      else if constexpr (MODE == kPlain) store_row<T, 8>((T*)p.out + m * p.ldo, n, p.N, v);
      else store_row<float, 8>(p.part + ((long)blockIdx.y * p.M + m) * p.N, n, p.N, v);
    };
    ColumnBias<8, GLU> bias;
    RowPiece<T, 8> res[NG], next[NG];
    if constexpr (MODE == kEpilogue) bias.load(p, n);
    if (MODE == kEpilogue && p.res) {
      auto fetch = [&](RowPiece<T, 8>(&q)[NG], int i) {
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          const long m = mh + i + k * RI;
          if (m < p.M && n < p.N) q[k].load((const T*)p.res + m * p.ldr, n, p.N);
        }
      };
      fetch(res, 0);
      for (int i = 0; i < kPass; i += NG * RI) {
        if (i + NG * RI < kPass) fetch(next, i + NG * RI);
#pragma unroll
        for (int k = 0; k < NG; ++k) row_out(i + k * RI, bias, res[k], std::true_type{});
#pragma unroll
        for (int k = 0; k < NG; ++k) res[k] = next[k];
      }
    } else {  // (of its own: waiting for loads that are never made would wait for the stores before them)
#pragma unroll 2
      for (int i = 0; i < kPass; i += RI) row_out(i, bias, res[0], std::false_type{});
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The parts of the contraction added, then the epilogue: by G threads of a workgroup for the same outputs, each every
// G-th part in order, their sums in order (few outputs of many parts: one load after the other is all there is).
template <typename T, int ACT, int G>
__global__ __launch_bounds__(kThreads) void join_kernel(const ProductArgs p) {
  constexpr int C = 4, W = kThreads / G;
  constexpr bool glu = ACT == kActSwiglu;
  constexpr int H = glu ? 2 : 1;
  __shared__ float sums[G > 1 ? G : 1][H][C][G > 1 ? W : 1];
  const long cols = glu ? 2 * p.N : p.N, groups = (p.N + C - 1) / C;
  const int g = threadIdx.x / W, c = threadIdx.x % W;
  const long at = (long)blockIdx.x * W + c;
  const bool live = at < p.M * groups;
  const long m = at / groups, n = at % groups * C;
  float v[C], up[C];
#pragma unroll
  for (int i = 0; i < C; ++i) v[i] = up[i] = 0.f;
  if (live)
#pragma unroll 4
    for (int s = g; s < p.splits; s += G) {
      const float* row = p.part + ((long)s * p.M + m) * cols;
      add_row<float, C>(row, n, p.N, v);
      if (glu) add_row<float, C>(row + p.N, n, p.N, up);
    }
  if constexpr (G > 1) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      sums[g][0][i][c] = v[i];
      if (glu) sums[g][H - 1][i][c] = up[i];
    }
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int k = 1; k < G; ++k)
#pragma unroll
      for (int i = 0; i < C; ++i) {
        v[i] += sums[k][0][i][c];
        if (glu) up[i] += sums[k][H - 1][i][c];
      }
  }
  if (!live) return;
  ColumnBias<C, glu> bias;
  RowPiece<T, C> res;
  bias.load(p, n);
  if (p.res) {
    res.load((const T*)p.res + m * p.ldr, n, p.N);
    finish<T, C, ACT, true>(p, m, n, v, up, bias, res);
  } else {
    finish<T, C, ACT, false>(p, m, n, v, up, bias, res);
  }
}

// ---------------------------------------------------------------------------
// dz = act'(z) dy, with the bias's gradient: a wave takes up to 512 columns, 8 a lane, of a block of rows (narrower
// maps: several rows at once), two rows a lane loaded together; its sums are one partial row of db.  Bound by HBM bytes
// (16384 x 2816 swiglu 104 us, 5.3 TB/s).
// ---------------------------------------------------------------------------
constexpr int kActRows = 2;
template <typename T, bool glu>
__global__ __launch_bounds__(kThreads) void act_bwd_kernel(const ActBwdArgs a) {
  constexpr int C = 8;
  typedef T vec __attribute__((ext_vector_type(C)));
  const int L = a.lanes, l = threadIdx.x & 63, sub = l / L, rows = 64 / L;  // lanes of a row, rows of a wave
  const long n = ((long)blockIdx.x * L + (l & (L - 1))) * C, width = glu ? a.ldz - a.N : a.ldz;  // (with the columns behind)
  const long rb = (long)blockIdx.y * 4 + (threadIdx.x >> 6);
  if (rb >= a.row_blocks) return;  // (whole waves)
  const long per = (a.M + a.row_blocks - 1) / a.row_blocks, r0 = rb * per, r1 = min(a.M, r0 + per);
  float sum[glu ? 2 : 1][C];
#pragma unroll
  for (int i = 0; i < C; ++i) sum[0][i] = sum[glu ? 1 : 0][i] = 0.f;
  for (long m0 = n < width ? r0 + sub : r1; m0 < r1; m0 += kActRows * rows) {
    vec dy[kActRows];
    KeptZ<C> z[kActRows], u[kActRows];
#pragma unroll
    for (int k = 0; k < kActRows; ++k) {
      const long m = min(m0 + k * rows, r1 - 1);
      dy[k] = load_piece((const T*)a.dy + m * a.ldy, (int)n, (int)a.N);
      if (a.z) z[k].load(a.z, a.M, a.ldz, m, n, a.N);
      if (glu) u[k].load(a.z, a.M, a.ldz, m, a.N + n, 2 * a.N);
    }
#pragma unroll
    for (int k = 0; k < kActRows; ++k) {
      const long m = m0 + k * rows;
      if (m >= r1) break;
      float d[C], du[C];
      if constexpr (glu) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const float gate = z[k][i], g = sigmoid(gate), dd = (float)dy[k][i];
          // (behind the columns dy and both halves are 0)
          d[i] = dd * u[k][i] * (g * (1.f + gate * (1.f - g)));
          du[i] = dd * gate * g;
          sum[1][i] += du[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < C; ++i) d[i] = (float)dy[k][i];
        if (a.z) act_slopes<C>(a.act, z[k], d);
      }
#pragma unroll
      for (int i = 0; i < C; ++i) sum[0][i] += d[i];
      if (a.dz) {
        store_row<T, C>((T*)a.dz + m * a.ldz, n, glu ? a.N : a.ldz, d);
        if (glu) store_row<T, C>((T*)a.dz + m * a.ldz + a.N, n, a.ldz - a.N, du);
      }
    }
  }
  if (a.db_part) {
    for (int o = L; o < 64; o <<= 1)
#pragma unroll
      for (int i = 0; i < C; ++i) {
        sum[0][i] += __shfl_xor(sum[0][i], o);
        if (glu) sum[glu ? 1 : 0][i] += __shfl_xor(sum[glu ? 1 : 0][i], o);
      }
    if (sub || n >= width) return;
    float* row = a.db_part + rb * (glu ? 2 * a.N : a.N);
    store_row<float, C>(row, n, a.N, sum[0]);
    if (glu) store_row<float, C>(row + a.N, n, a.N, sum[glu ? 1 : 0]);
  }
}

// db[n] = sum of the partial rows, in their order inside 16 interleaved groups
__global__ __launch_bounds__(1024) void bias_sum_kernel(const ActBwdArgs a) {
  __shared__ float part[16][64];
  const long n = a.act == kActSwiglu ? 2 * a.N : a.N, c = (long)blockIdx.x * 64 + (threadIdx.x & 63);
  const int g = threadIdx.x >> 6;
  float s = 0.f;
  if (c < n)
#pragma unroll 8
    for (int i = g; i < a.row_blocks; i += 16) s += *gmem(a.db_part + i * n + c);
  part[g][threadIdx.x & 63] = s;
  __syncthreads();
  if (g || c >= n) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += part[i][threadIdx.x];
  if (a.bdtype == kF32) ((float*)a.db)[c] = s;
  else if (a.bdtype == kBf16) ((bf16*)a.db)[c] = (bf16)s;
  else ((f16*)a.db)[c] = (f16)s;
}

__global__ __launch_bounds__(kThreads) void pad_rows_kernel(const PadRowsArgs a) {
  const long pieces = a.ldd / 8, end = a.rows * pieces;
  for (long at = (long)blockIdx.x * kThreads + threadIdx.x; at < end; at += (long)gridDim.x * kThreads) {
    const long m = at / pieces, n = at % pieces * 8;
    const short* row = (const short*)a.src + m * a.ld;
    s16x8 v;
    typedef s16x8 any __attribute__((aligned(2)));
    if (n + 8 <= a.K) {
      v = *gmem((const any*)(row + n));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = n + i < a.K ? *gmem(row + n + i) : (short)0;
    }
    *gmem((s16x8*)((short*)a.dst + m * a.ldd + n)) = v;
  }
}

template <typename T, int BM, int BN, int WM, int WN, int NA, int NB, bool DA, bool DB, int MODE, int ACT>
hipError_t launch_tiles(const ProductArgs& p, hipStream_t st) {
  constexpr int NT = ACT == kActSwiglu ? BN / 2 : BN;
  const long tiles = ((p.M + BM - 1) / BM) * ((p.N + NT - 1) / NT);
  hipLaunchKernelGGL((product_kernel<T, BM, BN, WM, WN, NA, NB, DA, DB, MODE, ACT>), dim3((unsigned)tiles, (unsigned)p.splits),
                     dim3(WM * WN * 64), 0, st, p);
  return hipGetLastError();
}

constexpr int kCus = 256;
// Few tiles of 64 x 64: four stages of both operands in LDS instead of three and two, so two workgroups a CU instead of
// four, and twice the bytes on their way (operands from HBM: 16 x 5632 over 1024 12.2 -> 7.7 us, 1024^3 10.5 -> 7.9; out
// of the caches 0.2 slower.  With more tiles four a CU are ahead: 4096 x 2048 over 512 18.6, 23.1 so).
constexpr int kDeepMost = 2 * kCus;

template <typename T, bool DA, bool DB, int MODE, int ACT = kActNone>
hipError_t launch_size(const ProductArgs& p, int side, hipStream_t st) {
  if (side == 256) return launch_tiles<T, 256, 256, 2, 2, 3, 2, DA, DB, MODE, ACT>(p, st);
  if (side == 128) return launch_tiles<T, 128, 128, 2, 2, 3, 2, DA, DB, MODE, ACT>(p, st);
  constexpr int NT = ACT == kActSwiglu ? 32 : 64;
  if (((p.M + 63) / 64) * ((p.N + NT - 1) / NT) * p.splits <= kDeepMost)
    return launch_tiles<T, 64, 64, 2, 2, 4, 4, DA, DB, MODE, ACT>(p, st);
  return launch_tiles<T, 64, 64, 2, 2, 3, 2, DA, DB, MODE, ACT>(p, st);
}

// Eight threads an output where there are few outputs and many parts (both kernels, beside one thread: 16 x 1024 over 2816
// 9.2 -> 7.6 us, 64 x 64 over 65536 25 -> 13, 128 x 128 over 262144 61 -> 46).
template <typename T, int ACT>
hipError_t launch_join(const ProductArgs& p, hipStream_t st) {
  const long threads = p.M * ((p.N + 3) / 4);
  if (p.splits >= 8 && threads <= 65536)
    hipLaunchKernelGGL((join_kernel<T, ACT, 8>), dim3((unsigned)((threads + kThreads / 8 - 1) / (kThreads / 8))), dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL((join_kernel<T, ACT, 1>), dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_typed(int kind, const ProductArgs& p, int side, hipStream_t st) {
  if (p.splits > 1) {
    ProductArgs q = p;  // partial products of all rows of B
    if (p.act == kActSwiglu) q.N = 2 * p.N;
    q.act = kActNone;
    const hipError_t e = kind == 0 ? launch_size<T, false, false, kPartial>(q, side, st)
                         : kind == 1 ? launch_size<T, false, true, kPartial>(q, side, st)
                                     : launch_size<T, true, true, kPartial>(q, side, st);
    if (e != hipSuccess) return e;
    return p.act == kActSwiglu  ? launch_join<T, kActSwiglu>(p, st)
           : p.act == kActNone ? launch_join<T, kActNone>(p, st)
                               : launch_join<T, kActOther>(p, st);
  }
  if (kind == 0)
    return p.act == kActSwiglu ? launch_size<T, false, false, kEpilogue, kActSwiglu>(p, side, st)
           : p.act == kActNone ? launch_size<T, false, false, kEpilogue, kActNone>(p, side, st)
                               : launch_size<T, false, false, kEpilogue, kActOther>(p, side, st);
  if (kind == 1) return launch_size<T, false, true, kPlain>(p, side, st);
  return launch_size<T, true, true, kPlain>(p, side, st);
}

}  // namespace

// Tile side and parts of the contraction of a product of M x N outputs (swiglu: N = all rows of B) over K, by what a
// call is expected to take, in us.  A CU holds one workgroup of 256 x 256 (its LDS), two of 128 x 128, two of 64 x 64
// with deep rings or four without; `step1` a step's time for each of them, `step0` what they share, `fixed` what a
// workgroup takes besides (launch, the first loads, the epilogue), measured:
//   256: 8192 x 4096 over 4096 202 us, 32768 x 1024 over 2816 153, 16384 x 5632 over 1024 189 (128: 243, 191, 193)
//   128: 2048 x 2048 over 2048 21.2, 4096 x 2048 over 1024 20.4 (256: 44, 30.5; 64: 28, 29)
//    64: 1024 x 1024 over 2048 11.9, 2048 x 1024 over 1024 10.5, over 4096 27.8 (128: 19, 12.2, 33; 128 in two parts: 17.5,
//        20, 31)
// Parts of the contraction go through fp32 partial sums: a second launch, and a read of each part, one after the
// other.  512 x 1024 over 4096 by 64 in one part 19.5, in two or four 16.0; 1024 x 1024 over 2048 11.9 and 17.4;
// 2816 x 1024 over 32768 by 256 in five 185, by 128 in one 340.
void product_plan(long M, long N, long K, int* side, int* splits) {
  static const struct {
    int side, per_cu;
    float step0, step1, fixed;
    long most;  // workgroups of the launch
  } kinds[] = {{256, 1, 0.f, 1.5f, 7.5f, kMaxTiles}, {128, 2, 0.1f, 0.43f, 4.5f, kMaxTiles},
               {64, 2, 0.095f, 0.14f, 3.6f, kDeepMost + 1}, {64, 4, 0.1f, 0.19f, 3.5f, kMaxTiles}};
  const long steps = (K + kStep - 1) / kStep;
  float best = 0.f;
  *side = 256;
  *splits = 1;
  if (M <= 0 || N <= 0) return;
  for (const auto& k : kinds) {
    const long tiles = ((M + k.side - 1) / k.side) * ((N + k.side - 1) / k.side);
    for (int sp = 1; sp <= 64 && (sp == 1 || sp * 2 <= steps) && tiles * sp < k.most; ++sp) {
      const long w = (tiles * sp + kCus - 1) / kCus, full = w / k.per_cu, rest = w % k.per_cu, n = (steps + sp - 1) / sp;
      float t = full * (n * (k.step0 + k.step1 * k.per_cu) + k.fixed);
      if (rest) t += n * (k.step0 + k.step1 * rest) + k.fixed;
      if (sp > 1) t += 3.f + sp * (0.1f + 1.2e-6f * M * N);
      if (best == 0.f || t < best) {
        best = t;
        *side = k.side;
        *splits = sp;
      }
    }
  }
}

// kind 0: y = act(x W^T + b) + r; 1: dx = dz W; 2: dW = dz^T x
hipError_t launch_product(int kind, const ProductArgs& p, hipStream_t st) {
  if (p.M <= 0 || p.N <= 0) return hipSuccess;
  int side, splits;
  product_plan(p.M, p.act == kActSwiglu ? 2 * p.N : p.N, p.K, &side, &splits);
  ProductArgs q = p;
  q.splits = splits;
  return p.dtype == kBf16 ? launch_typed<bf16>(kind, q, side, st) : launch_typed<f16>(kind, q, side, st);
}

// Lanes that the rows' columns take of a wave: the next power of two of the pieces of a row, at most all.
static int act_bwd_lanes(long N) {
  int l = 1;
  while (l < 64 && l * 8 < N) l <<= 1;
  return l;
}
// Blocks of rows, a wave and a partial row of db each: about 16 waves a CU, two rounds of loads or more a block.
int act_bwd_row_blocks(long M, long N) {
  const long cols = (N + 511) / 512, rows = 2 * kActRows * (64 / act_bwd_lanes(N));
  return (int)std::max(1L, std::min((M + rows - 1) / rows, std::max(1L, 16 * kCus / cols)));
}

template <typename T>
static void launch_act_typed(const ActBwdArgs& a, hipStream_t st) {
  const bool glu = a.act == kActSwiglu;
  const long width = glu ? a.ldz - a.N : a.ldz;
  const dim3 grid((unsigned)((width + 8 * a.lanes - 1) / (8 * a.lanes)), (unsigned)((a.row_blocks + 3) / 4));
  if (glu) hipLaunchKernelGGL((act_bwd_kernel<T, true>), grid, dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((act_bwd_kernel<T, false>), grid, dim3(kThreads), 0, st, a);
}

hipError_t launch_act_bwd(const ActBwdArgs& args, hipStream_t st) {
  ActBwdArgs a = args;
  const bool glu = a.act == kActSwiglu;
  a.row_blocks = a.M > 0 ? act_bwd_row_blocks(a.M, a.N) : 0;
  a.lanes = act_bwd_lanes(a.N);
  if (a.row_blocks) {
    if (a.dtype == kBf16) launch_act_typed<bf16>(a, st);
    else launch_act_typed<f16>(a, st);
  }
  if (a.db)
    hipLaunchKernelGGL(bias_sum_kernel, dim3((unsigned)(((glu ? 2 * a.N : a.N) + 63) / 64)), dim3(1024), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_pad_rows(const PadRowsArgs& a, hipStream_t st) {
  const long n = a.rows * (a.ldd / 8);
  if (n <= 0) return hipSuccess;
  const long blocks = std::min((n + kThreads - 1) / kThreads, 1L << 20);
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, a);
  return hipGetLastError();
}

}  // namespace ccq
