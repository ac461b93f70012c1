// Serving in 8 bits: rows turned into e4m3 with a scale for each block of 128 (ccq_fp8.h), and the linear map over two
// operands of that form,
//
//   y[m, n] = act(sum over blocks b of 2^(ea[m, b] + eb[n, b]) sum over k in b of a[m, k] b[n, k] + bias[n]) + r[m, n]
//
// with relu, silu, both gelus or swiglu, into bf16, fp16, fp32, or into 8 bits again for the next map.  gfx950's scaled matrix
// instruction multiplies 16 x 128 by 128 x 16 elements with a power of two for each row's 32 and accumulates in fp32, so the
// scales cost no arithmetic.
//
// What that instruction does to a sum (measured): of each eight consecutive products those bits are cut off that lie below
// 2^-13 of the largest one's exponent; the eights and the accumulator add up in fp32.  On normal data that is 1.4e-5 of the
// result, far below the rounding of 16-bit and 8-bit outputs (2e-4 and more), and so these take it.  An output in fp32 is
// computed exactly: e4m3 widened to bf16, whose products fp32 holds and whose instruction adds in fp32 (6e-8), at half the
// rate; the scales are applied to each block's sum.
#include <algorithm>

#include "ccq_block_args.h"
#include "ccq_fp8.h"
#include "ccq_oper.h"
#include "ccq_product.h"
#include "ccq_rows.h"

namespace ccq {

namespace {

// ---------------------------------------------------------------------------
// rows into 8 bits: 16 lanes a block, 8 elements a lane
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const QuantizeArgs a, int lanes) {
  const int l = threadIdx.x & 63, li = l & (lanes - 1), per = 64 / lanes;  // lanes of a row, rows of a wave
  const long units = (a.D + lanes * 8 - 1) / (lanes * 8);                  // of a row
  const long total = (a.rows + per - 1) / per * units;
  for (long u = (long)blockIdx.x * 4 + (threadIdx.x >> 6); u < total; u += (long)gridDim.x * 4) {
    const long row = u / units * per + l / lanes, c = (u % units * lanes + li) * 8;
    if (row >= a.rows) continue;
    const T* x = (const T*)a.x + row * a.ldx;
    float v[8];
    if (c + 8 <= a.D) {
      typedef T vec __attribute__((ext_vector_type(8)));
      typedef vec any __attribute__((aligned(sizeof(T))));
      const vec p = *gmem((const any*)(x + c));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)p[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c + i < a.D ? (float)*gmem(x + c + i) : 0.f;
    }
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, magnitude(v[i]));
    const unsigned byte = scale_byte(lanes_max(m, 16));
    if (c < a.D) {  // (a whole piece: the rows are multiples of 16)
      *gmem((u32x2*)(a.values + row * a.ldv + c)) =
          u32x2{fp8_word(v[0], v[1], v[2], v[3], byte), fp8_word(v[4], v[5], v[6], v[7], byte)};
      if ((li & 15) == 0) a.scales[row * a.lds + c / kFp8Block] = (unsigned char)byte;
    }
  }
}

// ---------------------------------------------------------------------------
// the tiled product
// ---------------------------------------------------------------------------
constexpr int kStep = 128;  // contraction elements a step, one block
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// Fragments of 16 rows come in groups of G (4 where a wave has as many): fragment i of a group holds its rows G r + i, so
// that G consecutive columns of the result lie in one lane.
__device__ __forceinline__ int slot_row(int s, int G) { return s / (16 * G) * (16 * G) + (s & 15) * G + s / 16 % G; }
__device__ __forceinline__ int swz(int s) { return (s >> 1) & 7; }

// eight e4m3 (bytes 8 c .. of a fragment) in bf16, exactly
__device__ __forceinline__ bf16x8 widen(const i32x8& f, int c) {
  bf16x8 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bf16x2 v = (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[2 * c + i / 2], 1.f, true)
                             : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[2 * c + i / 2], 1.f, false);
    o[2 * i] = v[0];
    o[2 * i + 1] = v[1];
  }
  return o;
}

template <int BM, int BN, int WM, int WN, int ACT, bool EXACT>
__global__ __launch_bounds__(WM * WN * 64) void fp8_product_kernel(const Fp8ProductArgs p) {
  constexpr bool GLU = ACT == kActSwiglu;
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, HALF = BN / WN / 2;
  constexpr int GA = std::min(TM, 4), GB = std::min(GLU ? TN / 2 : TN, 4);
  constexpr unsigned kA = BM * kStep, kB = BN * kStep;
  constexpr int kPass = std::min(TM * 16, 64), kPitch = BN + 4;
  constexpr unsigned kRing = 2 * (kA + kB), kOut = WM * kPass * kPitch * 4;
  constexpr int NT = GLU ? BN / 2 : BN;  // output columns of a tile
  constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;
  static_assert(PA >= 1 && PB >= 1 && (!GLU || PB * 8 == HALF), "whole loads a wave, of gates or ups");
  __shared__ __attribute__((aligned(1024))) char smem[std::max(kRing, kOut)];
  const int tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, r = l & 15, g = l >> 4;
  const int tm = (int)((p.M + BM - 1) / BM), tn = (int)((p.N + NT - 1) / NT), tiles = tm * tn;
  const int xcd = blockIdx.x & 7, q8 = tiles >> 3, r8 = tiles & 7;
  const int t = xcd * q8 + min(xcd, r8) + (blockIdx.x >> 3);
  const int band = t / (8 * tn), in = t - band * 8 * tn, band_rows = min(8, tm - band * 8);
  const long m0 = (long)(band * 8 + in % band_rows) * BM, n0 = (long)(in / band_rows) * NT;

  const unsigned lds0 = lds_addr(smem);
  unsigned offa[PA], offb[PB];
#pragma unroll
  for (int i = 0; i < PA; ++i) {
    const int s = (wave * PA + i) * 8 + (l >> 3), row = slot_row(s, GA);
    offa[i] = m0 + row < p.M ? (unsigned)(row * p.lda) + (((l & 7) ^ swz(s)) << 4) : kNowhere;
  }
  // row of B in slot s: swiglu: the gates of a wave's columns, then their ups
  auto b_row = [&](int s) { return GLU ? s / (2 * HALF) * HALF + slot_row(s % HALF, GB) : slot_row(s, GB); };
  auto b_up = [&](int s) { return GLU && s % (2 * HALF) >= HALF; };
#pragma unroll
  for (int i = 0; i < PB; ++i) {
    const int s = (wave * PB + i) * 8 + (l >> 3), row = b_row(s);
    offb[i] = n0 + row < p.N ? (unsigned)(row * p.ldb) + (((l & 7) ^ swz(s)) << 4) : kNowhere;
  }
  const size_t pa = (size_t)p.a + m0 * p.lda, pb = (size_t)p.b + (n0 + (GLU && (wave & 1) ? p.N : 0)) * p.ldb;
  const int steps = (int)((p.K + kStep - 1) / kStep), tail = (int)(p.K & (kStep - 1));
  auto load = [&](int s) {
    const unsigned stage = (s & 1) * (kA + kB);
    u32x4 ra = resource(pa + (long)s * kStep, 0x7fffffffu), rb = resource(pb + (long)s * kStep, 0x7fffffffu);
    settled(ra);
    settled(rb);
    const int left = tail && s == steps - 1 ? tail : kStep;
    auto issue = [&](const u32x4& rs, unsigned off, unsigned to, int i) {
      load_to(to, i);
      asm volatile("s_nop 0");
      load_from(rs, off);
    };
#pragma unroll
    for (int i = 0; i < PA; ++i) {
      const int slot = (wave * PA + i) * 8 + (l >> 3);
      issue(ra, ((l & 7) ^ swz(slot)) * 16 < left ? offa[i] : kNowhere, lds0 + stage + wave * PA * 1024, i);
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const int slot = (wave * PB + i) * 8 + (l >> 3);
      issue(rb, ((l & 7) ^ swz(slot)) * 16 < left ? offb[i] : kNowhere, lds0 + stage + kA + wave * PB * 1024, i);
    }
  };
  // rows of this lane's scales
  const unsigned char *sa[TM], *sb[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) sa[i] = p.sa + std::min(m0 + slot_row((wm * TM + i) * 16 + r, GA), p.M - 1) * p.lsa;
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int s = (wn * TN + j) * 16 + r;
    sb[j] = p.sb + (std::min(n0 + b_row(s), p.N - 1) + (b_up(s) ? p.N : 0)) * p.lsb;
  }
  unsigned ea[TM], eb[TN];
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto frag = [&](unsigned at, int slot) {
    const s16x8 lo = read16(at + slot * 128 + ((g ^ swz(slot)) << 4)), hi = read16(at + slot * 128 + (((g + 4) ^ swz(slot)) << 4));
    const i32x4 x = __builtin_bit_cast(i32x4, lo), y = __builtin_bit_cast(i32x4, hi);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  load(0);
  for (int s = 0; s < steps; ++s) {
    if ((s & 3) == 0) {
#pragma unroll
      for (int i = 0; i < TM; ++i) ea[i] = *gmem((const unsigned*)(sa[i] + s));
#pragma unroll
      for (int j = 0; j < TN; ++j) eb[j] = *gmem((const unsigned*)(sb[j] + s));
    }
    wait_loads<0>();
    lds_barrier();
    if (s + 1 < steps) load(s + 1);
    const unsigned at = lds0 + (s & 1) * (kA + kB);
    i32x8 mask;
    const bool part = tail & 15 && s == steps - 1;
    if (part)
#pragma unroll
      for (int d = 0; d < 8; ++d) {  // bytes of the end: the row's storage goes on behind them
        const int n = tail - (16 * (g + d / 4 * 4) + d % 4 * 4);
        mask[d] = n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1;
      }
    i32x8 b[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      b[j] = frag(at + kA, (wn * TN + j) * 16 + r);
      if (part) b[j] &= mask;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      i32x8 a = frag(at, (wm * TM + i) * 16 + r);
      if (part) a &= mask;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        if constexpr (!EXACT) {
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j], a, acc[i][j], 0, 0, 0, eb[j], 0, ea[i]);
        } else {
          f32x4 sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 4; ++c) sum = mfma16(widen(b[j], c), widen(a, c), sum);
          // the columns' scales lie in the lanes that hold their fragment's rows: column 4 g + q in lane 4 g + q
          const unsigned x = ea[i] & 0xff;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const unsigned y = (unsigned)__shfl((int)eb[j], 4 * g + q) & 0xff;
            acc[i][j][q] += x == kFp8Nan || y == kFp8Nan ? NAN : __builtin_ldexpf(sum[q], (int)(x + y) - 254);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) ea[i] >>= 8;
#pragma unroll
    for (int j = 0; j < TN; ++j) eb[j] >>= 8;
  }

  float* tile = (float*)smem;
  constexpr int PR = NT / 8, RP = NW * 64 / PR;  // threads of a row, rows at a time
  const int c = tid % PR * 8, cw = c / (GLU ? HALF : NT), cs = GLU ? cw * 2 * HALF + c % HALF : c;
  const long n = n0 + c;
  float bias[8], bias_up[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bias[i] = p.bias && n + i < p.N ? bias_at(p.bias, p.bdtype, n + i) : 0.f;
    bias_up[i] = GLU && p.bias && n + i < p.N ? bias_at(p.bias, p.bdtype, p.N + n + i) : 0.f;
  }
#pragma unroll
  for (int h = 0; h < TM * 16 / kPass; ++h) {
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kPass / 16; ++i)
#pragma unroll
      for (int j = 0; j < TN; j += GB)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int k = 0; k < GB; ++k)
            tile[(wm * kPass + i * 16 + r) * kPitch + (wn * TN + j) * 16 + (4 * g + q) * GB + k] = acc[h * (kPass / 16) + i][j + k][q];
    __syncthreads();
    for (int i = tid / PR; i < WM * kPass; i += RP) {
      const long m = m0 + i / kPass * (TM * 16) + slot_row(h * kPass + i % kPass, GA);
      if (m >= p.M || (n >= p.N && !p.os)) continue;
      float v[8], up[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = tile[i * kPitch + cs + e] + bias[e];
        if (GLU) up[e] = tile[i * kPitch + cs + HALF + e] + bias_up[e];
      }
      if (GLU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] * sigmoid(v[e]) * up[e];
      } else if (ACT != kActNone) {
        act_values<8>(p.act, v);
      }
      if (p.os) {  // a row's 16 lanes of a block go together
        unsigned most = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (n + e >= p.N) v[e] = 0.f;
          most = max(most, magnitude(v[e]));
        }
        const unsigned byte = scale_byte(lanes_max(most, 16));
        if (n >= p.N) continue;
        *gmem((u32x2*)((unsigned char*)p.out + m * p.ldo + n)) =
            u32x2{fp8_word(v[0], v[1], v[2], v[3], byte), fp8_word(v[4], v[5], v[6], v[7], byte)};
        if ((tid & 15) == 0) p.os[m * p.los + n / kFp8Block] = (unsigned char)byte;
        continue;
      }
      if (p.dtype == kF32) {
        if (p.res) add_row<float, 8>((const float*)p.res + m * p.ldr, n, p.N, v);
        store_row<float, 8>((float*)p.out + m * p.ldo, n, p.N, v);
      } else if (p.dtype == kBf16) {
        if (p.res) add_row<bf16, 8>((const bf16*)p.res + m * p.ldr, n, p.N, v);
        store_row<bf16, 8>((bf16*)p.out + m * p.ldo, n, p.N, v);
      } else {
        if (p.res) add_row<f16, 8>((const f16*)p.res + m * p.ldr, n, p.N, v);
        store_row<f16, 8>((f16*)p.out + m * p.ldo, n, p.N, v);
      }
    }
  }
}

template <int BM, int BN, int WM, int WN, bool EXACT>
hipError_t launch_tiles(const Fp8ProductArgs& p, hipStream_t st) {
  const int NT = p.act == kActSwiglu ? BN / 2 : BN;
  const dim3 grid((unsigned)(((p.M + BM - 1) / BM) * ((p.N + NT - 1) / NT))), block(WM * WN * 64);
  if (p.act == kActSwiglu) hipLaunchKernelGGL((fp8_product_kernel<BM, BN, WM, WN, kActSwiglu, EXACT>), grid, block, 0, st, p);
  else if (p.act == kActNone) hipLaunchKernelGGL((fp8_product_kernel<BM, BN, WM, WN, kActNone, EXACT>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((fp8_product_kernel<BM, BN, WM, WN, kActOther, EXACT>), grid, block, 0, st, p);
  return hipGetLastError();
}

constexpr int kCus = 256;

}  // namespace

hipError_t launch_quantize(const QuantizeArgs& a, hipStream_t st) {
  if (a.rows <= 0) return hipSuccess;
  int lanes = 16;
  while (lanes < 64 && lanes * 8 < a.D) lanes <<= 1;
  const long per = 64 / lanes, waves = (a.rows + per - 1) / per * ((a.D + lanes * 8 - 1) / (lanes * 8));
  const dim3 grid((unsigned)std::min<long>((waves + 3) / 4, 8192));
  if (a.dtype == kBf16) hipLaunchKernelGGL(quantize_kernel<bf16>, grid, dim3(kThreads), 0, st, a, lanes);
  else if (a.dtype == kF16) hipLaunchKernelGGL(quantize_kernel<f16>, grid, dim3(kThreads), 0, st, a, lanes);
  else hipLaunchKernelGGL(quantize_kernel<float>, grid, dim3(kThreads), 0, st, a, lanes);
  return hipGetLastError();
}

hipError_t launch_fp8_product(const Fp8ProductArgs& p, hipStream_t st) {
  if (p.M <= 0) return hipSuccess;
  const long outs = p.act == kActSwiglu ? 2 * p.N : p.N;
  if (!p.os && p.dtype == kF32) return launch_tiles<64, 64, 2, 2, true>(p, st);
  if (p.os || ((p.M + 255) / 256) * ((outs + 255) / 256) >= kCus / 2) return launch_tiles<256, 256, 2, 2, false>(p, st);
  return launch_tiles<64, 64, 2, 2, false>(p, st);
}

}  // namespace ccq
