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
// 2^-13 of the largest one's exponent; the eights and the accumulator add up in fp32.  On normal data that is 1.5e-5 of the
// result, with channels 100 to 1000 times the others 7e-5 to 9e-5, below the rounding of 16-bit and 8-bit outputs (2e-4 and
// more), and so these take it; where such channels cancel in a sum it is 3e-4 to 4e-3 of what is left.  An output in fp32 is
// computed exactly: e4m3 widened to bf16, whose products fp32 holds and whose instruction adds in fp32 (6e-8), at half the
// rate; the scales go into the widened values, or where they lie far from one are applied to each block's sum.
#include <algorithm>

#include "ccq_block_args.h"
#include "ccq_fp8.h"
#include "ccq_oper.h"
#include "ccq_product.h"
#include "ccq_rows.h"

namespace ccq {

namespace {

// ---------------------------------------------------------------------------
// rows into 8 bits: 16 lanes a block, 8 elements a lane.  Bound by HBM: 16384 x 2048 bf16 18.5 us, 32000 x 1024 fp32 30.0 (both
// 5.5 TB/s); a wave takes one to four rows, so that narrow rows leave few lanes idle, and few rows many waves.
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
    const unsigned byte = scale_byte(lanes_max16(m));
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

// c += a b 2^(ea + eb - 254) on the matrix cores, the accumulator kept where it is (left to itself the register allocator
// moves the accumulators about between the products).  Two wait states lie between a vector instruction that wrote an
// operand and this one, which the compiler does not know of: the operands come straight out of LDS, or operand_settled.
__device__ __forceinline__ void product128(const i32x8& a, int ea, const i32x8& b, int eb, f32x4& c) {
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
               : "+a"(c) : "v"(a), "v"(b), "v"(ea), "v"(eb));
}
__device__ __forceinline__ void operand_settled(i32x8& v) { asm volatile("s_nop 1" : "+v"(v)); }
// an accumulator's value, read where the program says so (left to itself the compiler copies all 256 at once, and spills)
template <bool PINNED>
__device__ __forceinline__ float value_of(float c) {
  if (!PINNED) return c;
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(c));
  return v;
}
__device__ __forceinline__ void accumulator(f32x4& c) { asm volatile("" : "+a"(c)); }
// direct load of 4 bytes a lane from its own address to LDS byte lds + 4 * lane
__device__ __forceinline__ void load4_to(unsigned lds, const void* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(from) : "memory", "m0");
}

// eight e4m3 (bytes 8 c .. of a fragment) times a power of two in bf16, exactly (within bf16's range)
__device__ __forceinline__ bf16x8 widen(const i32x8& f, int c, float scale = 1.f) {
  bf16x8 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bf16x2 v = (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[2 * c + i / 2], scale, true)
                             : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[2 * c + i / 2], scale, false);
    o[2 * i] = v[0];
    o[2 * i + 1] = v[1];
  }
  return o;
}

// The scale of a byte, 2^(e - 127).  Those of bytes 77 .. 177 may go into the widened values: 2^-59 .. 2^59 with them in
// bf16, and their products 2^-118 .. 2^118 in fp32.
constexpr int kNearOne = 77;
constexpr unsigned kNearMost = 100;
__device__ __forceinline__ float scale_of(int byte) { return __uint_as_float((unsigned)byte << 23); }

// c += a b 2^(ea + eb - 254), exactly but for fp32's additions; lane l holds the scales of rows l & 15 of both
__device__ __forceinline__ void exact_product(const i32x8& a, int ea, const i32x8& b, int eb, f32x4& c) {
  f32x4 sum{0.f, 0.f, 0.f, 0.f};
  if (__all(max((unsigned)(ea - kNearOne), (unsigned)(eb - kNearOne)) <= kNearMost)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) sum = mfma16(widen(a, k, scale_of(ea)), widen(b, k, scale_of(eb)), sum);
    c += sum;
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) sum = mfma16(widen(a, k), widen(b, k), sum);
#pragma unroll
  for (int q = 0; q < 4; ++q) {  // (row 4 g + q of the result: its scale lies in lane 4 g + q)
    const int y = __shfl(ea, 4 * (lane_id() >> 4) + q);
    c[q] += eb == (int)kFp8Nan || y == (int)kFp8Nan ? NAN : __builtin_ldexpf(sum[q], eb + y - 254);
  }
}

// stores that a step lets go on, in its first half alone or throughout
template <int STORES, bool FIRST_HALF>
struct Spare {
  static constexpr int stores = STORES;
  static constexpr bool first_half = FIRST_HALF;
};

// The kernel's arguments, read again where they are used: kept over the loop over tiles they and what follows from them
// would not fit the scalar registers.
typedef const __attribute__((address_space(4))) Fp8ProductArgs* ArgsAgain;
__device__ __forceinline__ ArgsAgain args_again() {
  ArgsAgain p = (ArgsAgain)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}
// the same of a value that follows from the lane
__device__ __forceinline__ int again(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// bf16 or fp16 (dtype; of tiles below 256 fp32 too, of 8-bit products, for a workspace); fp32 exactly; e4m3 with scales
enum : int { kOut16 = 0, kOut32 = 1, kOut8 = 2 };

// BM x BN tile of the product by WM x WN waves, two stages of both operands in LDS.  A lane of a wave holds, of each 16 x 16
// tile (i, j), row r = l & 15 of A's fragment and the columns 4 (l >> 4) .. + 3 of B's.
//
// A step is one block of 128.  Its products go in quarters of the wave's tile, (A0, B0), (A0, B1), (A1, B1), (A1, B0), each
// while the half that the next one needs is read from LDS: B1, A1, then the next step's A0 and, into B1's registers, its B0, so that
// the halves of B change places from step to step.  So A0 and B0 of a step have been read when it begins, A1 and B1 at its
// middle: there stand the barriers, and behind each of them those halves of the step after next are loaded, between
// products, a step and a half before they are read.
//
// Bound by the matrix cores: a step of a 256 tile takes 1.4 us, its instructions alone 1.1.  8192^3 387 - 414 us (2.65 - 2.84
// PFLOP/s; fragments read a whole step at a time 727, halves loaded a step ahead 440); 32768 x 1024 over 2816 with residual
// 90 - 97; 16384 x 2816 swiglu over 1024 into 8 bits 99 - 108, of which the outputs' arithmetic, with one wave a SIMD, is a third.
// In fp32 (exactly) the conversions bound it, 64 a step and wave at half rate: 4096^3 184 - 200 us; fragments are held once and
// read between two barriers, so that three workgroups share a CU.
template <int BM, int BN, int WM, int WN, int ACT, int OUT>
__global__ __launch_bounds__(WM * WN * 64, OUT == kOut32 ? 3 : 1) void fp8_product_kernel(const Fp8ProductArgs p) {
  constexpr bool GLU = ACT == kActSwiglu, EXACT = OUT == kOut32;
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, HALF = BN / WN / 2, HM = TM / 2, HN = TN / 2;
  constexpr int GA = std::min(TM, 4), GB = std::min(GLU ? TN / 2 : TN, 4);
  constexpr unsigned kA = BM * kStep, kStage = (BM + BN) * kStep, kScales = (BM + BN) * 4;  // of a step; of four steps
  constexpr int kPass = std::min(TM * 16, 64), kPitch = BN + 4;
  constexpr unsigned kRing = 2 * (kStage + kScales), kOut = WM * kPass * kPitch * 4;
  constexpr int NT = GLU ? BN / 2 : BN;  // output columns of a tile
  constexpr int PA = BM / 16 / NW, PB = BN / 16 / NW, PS = ((BM + BN) / 64 + NW - 1) / NW;
  static_assert(PA >= 1 && PB >= 1, "whole loads a wave of each half");
  static_assert(TM % 2 == 0 && TN % 2 == 0, "halves");
  __shared__ __attribute__((aligned(1024))) char smem[std::max(kRing, kOut)];
  const int tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, r = l & 15, g = l >> 4;
  const int steps = (int)((p.K + kStep - 1) / kStep), tail = (int)(p.K & (kStep - 1)), whole = steps - (tail ? 1 : 0);

  // row of B in slot s: swiglu: the gates of a wave's columns, then their ups
  auto b_row = [&](int s) { return GLU ? s / (2 * HALF) * HALF + slot_row(s % HALF, GB) : slot_row(s, GB); };
  auto b_up = [&](int s) { return GLU && s % (2 * HALF) >= HALF; };
  const unsigned lds0 = lds_addr(smem), lds_scales = lds0 + 2 * kStage;
  // Loads of half h of a step take 8 slots each, a wave's i-th one those from first + 16 H h + 8 i on (H fragments of the
  // operand's wave in a half).  A lane takes piece (l & 7) ^ swz of row l >> 3 of them; of the swizzle two forms occur, as the
  // slot is 0 or 8 in 16.  The rows of a load lie at a distance from the first one's that no wave differs in.
  const int first_a = wave * PA / (2 * HM) * (TM * 16) + wave * PA % (2 * HM) * 8;
  const int first_b = wave * PB / (2 * HN) * (TN * 16) + wave * PB % (2 * HN) * 8;
  constexpr int FA = std::min(PA, 2), FB = std::min(PB, 2);
  int piece_a[FA], piece_b[FB];
  unsigned lane_a[FA], lane_b[FB];
#pragma unroll
  for (int i = 0; i < FA; ++i) {
    piece_a[i] = 16 * ((l & 7) ^ swz(first_a + 8 * i + (l >> 3)));
    lane_a[i] = (unsigned)((slot_row(first_a, GA) + GA * (l >> 3)) * p.lda) + piece_a[i];
  }
#pragma unroll
  for (int i = 0; i < FB; ++i) {
    piece_b[i] = 16 * ((l & 7) ^ swz(first_b + 8 * i + (l >> 3)));
    lane_b[i] = (unsigned)((b_row(first_b) + GB * (l >> 3)) * p.ldb) + piece_b[i];
  }
  const unsigned lds_a = lds0 + first_a * 128, lds_b = lds0 + kA + first_b * 128;
  auto scale_slot = [&](int i) { return (wave * PS + i) % ((BM + BN) / 64) * 64; };
  long m0, n0;  // the tile whose operands are loaded
  size_t pa, pb;
  unsigned enda, endb;  // bytes from there to the end of its last row
  const size_t up = GLU ? p.N * p.ldb : 0;
  const unsigned char* scales[PS];
  // Tiles: each XCD (workgroups are handed out round-robin over the 8) takes consecutive ones, in column order within
  // bands of 8 tile rows, so that its L2 holds what its workgroups share.  A workgroup takes every `stride`-th of its XCD's.
  const int tiles = (int)((p.M + BM - 1) / BM) * (int)((p.N + NT - 1) / NT);
  const int xcd = blockIdx.x & 7, mine = (tiles >> 3) + (xcd < (tiles & 7)), stride = (gridDim.x + 7) >> 3;
  auto place = [&](int k) {
    const ArgsAgain p = args_again();
    const int l = again(tid & 63);
    const int tm = (int)((p->M + BM - 1) / BM), tn = (int)((p->N + NT - 1) / NT), tiles = tm * tn, q8 = tiles >> 3, r8 = tiles & 7;
    const int t = xcd * q8 + min(xcd, r8) + k;
    const int band = t / (8 * tn), in = t - band * 8 * tn, band_rows = min(8, tm - band * 8);
    m0 = (long)(band * 8 + in % band_rows) * BM;
    n0 = (long)(in / band_rows) * NT;
    pa = (size_t)p->a + m0 * p->lda;
    pb = (size_t)p->b + n0 * p->ldb;
    const long row = (p->K + 15) & ~15L;
    enda = (unsigned)((min((long)BM, p->M - m0) - 1) * p->lda + row);
    endb = (unsigned)((min((long)NT, p->N - n0) - 1) * p->ldb + row);
    // scales: A's slots, then B's, 64 a load (of fewer than the waves have, some load the same ones)
#pragma unroll
    for (int i = 0; i < PS; ++i) {  // (rows behind the last one: the last one's)
      const int s = scale_slot(i) + l;
      if (s < BM) scales[i] = p->sa + min(m0 + slot_row(s, GA), p->M - 1) * p->lsa;
      else scales[i] = p->sb + (min(n0 + b_row(s - BM), p->N - 1) + (b_up(s - BM) ? p->N : 0)) * p->lsb;
    }
  };
  auto load_scales = [&](int quad) {  // of steps 4 quad .. + 3
    if (quad * 4 >= steps) return;
#pragma unroll
    for (int i = 0; i < PS; ++i)
      load4_to(lds_scales + (quad & 1) * kScales + scale_slot(i) * 4, scales[i] + 4 * quad);
  };
  // A buffer resource bounds every load by the end of the tile's last row; what lies behind comes as zeros, and all of it
  // behind the last whole step.
  auto step_resource = [&](size_t base, unsigned end, int s) {
    return resource(base + (size_t)s * kStep, s < whole ? end - s * kStep : 0u);
  };

  // fragment addresses of this lane in stage 0, and of its scales
  unsigned fa[2], fb[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    fa[h] = lds0 + (wm * TM * 16 + r) * 128 + (((g + 4 * h) ^ swz(r)) << 4);
    fb[h] = lds0 + kA + (wn * TN * 16 + r) * 128 + (((g + 4 * h) ^ swz(r)) << 4);
  }
  const unsigned ea0 = lds_scales + (wm * TM * 16 + r) * 4, eb0 = lds_scales + (BM + wn * TN * 16 + r) * 4;
  struct Frag {
    i32x8 v;
    int e;
  };
  auto read = [&](Frag& f, const unsigned (&at)[2], unsigned e0, int i, unsigned stage, unsigned scale) {
    const i32x4 x = __builtin_bit_cast(i32x4, read16(at[0] + stage + i * 2048)), y = __builtin_bit_cast(i32x4, read16(at[1] + stage + i * 2048));
    f.v = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    typedef __attribute__((address_space(3))) const unsigned char lds_byte;
    f.e = *(lds_byte*)(size_t)(e0 + scale + i * 64);
  };
  f32x4 acc[TM][TN];
  // Exactly: the columns' scales of a fragment of B, those of 4 g + q (with the byte of the step in their words)
  struct ColumnScales {
    i32x4 word;
  };
  constexpr int kScaleSets = EXACT ? TN : 1;
  auto read_columns = [&](ColumnScales (&c)[kScaleSets], unsigned scale) {
    if constexpr (EXACT) {
      typedef __attribute__((address_space(3))) const i32x4 lds_words;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        c[j].word = *(lds_words*)(size_t)(lds_scales + (BM + (wn * TN + j) * 16 + 4 * g) * 4 + (scale & ~3u));
#pragma unroll
        for (int q = 0; q < 4; ++q) c[j].word[q] = c[j].word[q] >> (8 * (scale & 3)) & 0xff;
      }
    }
  };
  bool nan_row[EXACT ? TM : 1], nan_column[kScaleSets][4];  // a scale that is NaN was met
  // All products of a step, exactly.  Scales near one go into the widened values (4096^3 218 -> 184 us), others are applied
  // to the block's sums.
  auto multiply = [&](const Frag (&a)[TM], const Frag (&b)[TN], unsigned scale) {
    if constexpr (EXACT) {
      unsigned off = 0;
#pragma unroll
      for (int i = 0; i < TM; ++i) off = max(off, (unsigned)(a[i].e - kNearOne));
#pragma unroll
      for (int j = 0; j < TN; ++j) off = max(off, (unsigned)(b[j].e - kNearOne));
      if (__all(off <= kNearMost)) {
        bf16x8 wide[TN][4];
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) wide[j][k] = widen(b[j].v, k, scale_of(b[j].e));
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          bf16x8 row[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) row[k] = widen(a[i].v, k, scale_of(a[i].e));
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            f32x4 sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4; ++k) sum = mfma16(wide[j][k], row[k], sum);
            acc[i][j] += sum;
          }
        }
        return;
      }
      ColumnScales c[kScaleSets];
      read_columns(c, scale);
      bf16x8 wide[TN][4];
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) wide[j][k] = widen(b[j].v, k);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        bf16x8 row[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) row[k] = widen(a[i].v, k);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          f32x4 sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 4; ++k) sum = mfma16(wide[j][k], row[k], sum);
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i][j][q] += __builtin_ldexpf(sum[q], a[i].e + c[j].word[q] - 254);
        }
        nan_row[i] |= a[i].e == (int)kFp8Nan;
      }
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) nan_column[j][q] |= c[j].word[q] == (int)kFp8Nan;
    }
  };

  Frag a0[HM], a1[HM], b0[HN], b1[HN];
  // a quarter of the products, with `reads` between them; f(k) for each k < n, spread over the quarter
  auto quarter = [&](int ih, int jh, const Frag (&a)[HM], const Frag (&b)[HN], auto&& before, auto&& between) {
#pragma unroll
    for (int q = 0; q < HM * HN; ++q) {
      before(q);
      product128(b[q % HN].v, b[q % HN].e, a[q / HN].v, a[q / HN].e, acc[ih * HM + q / HN][jh * HN + q % HN]);
      between(q);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr int Q = HM * HN, PL = PA + PB;
  // A load of half h of a step in two parts, since M0 is read one wait state after it is written: between them stands a
  // product, or a wait.  (swiglu: half 0 of B holds gates, half 1 ups)
  auto to_a = [&](int h, int i, unsigned stage) { load_to(lds_a + stage, (h * HM * 16 + 8 * i) / 8); };
  auto to_b = [&](int h, int i, unsigned stage) { load_to(lds_b + stage, (h * HN * 16 + 8 * i) / 8); };
  auto off_a = [&](int h, int i) { return lane_a[i % FA] + (unsigned)(slot_row(h * HM * 16 + 8 * i, GA) * p.lda); };
  auto off_b = [&](int h, int i) { return lane_b[i % FB] + (unsigned)(b_row(h * HN * 16 + 8 * i) * p.ldb); };
  auto load_half = [&](int h, unsigned stage, const u32x4& ra, const u32x4& rb, int left) {  // zeros from `left` on
#pragma unroll
    for (int k = 0; k < PL; ++k) {
      const int i = k < PA ? k : k - PA;
      if (k < PA) to_a(h, i, stage);
      else to_b(h, i, stage);
      const unsigned off = k < PA ? off_a(h, i) : off_b(h, i);
      const bool on = (k < PA ? piece_a[i % FA] : piece_b[i % FB]) < left;
      asm volatile("s_nop 0");
      load_from(k < PA ? ra : rb, on ? off : kNowhere);
    }
  };
  // Between which of a quarter's products its n reads and its n loads stand: f(k) for the k-th one (where exactly matters
  // little; with the loads beside the reads 8192^3 took 2 to 3 % longer).
  auto reads = [&](int q, int n, auto&& f) {
#pragma unroll
    for (int k = 0; k < n; ++k)
      if (q == k * Q * 3 / 4 / n) f(k);
  };
  static_assert(PA == PB && (PA == 1 || (PA - 2) * Q / PA + 2 < Q - 1), "one load between two products");
  auto loads = [&](int q, int n, auto&& f) {
#pragma unroll
    for (int k = 0; k < n; ++k)
      if (q == std::min(k * Q / n + 2, Q - 1)) f(k);
  };
  auto scale_at = [&](int s) { return (s >> 2 & 1) * kScales + (s & 3); };
  // (spare: the last tile's stores may be on their way behind the loads)
  auto step = [&](auto spare, int s, Frag (&x0)[HN], Frag (&x1)[HN]) {  // x0: this step's B0; x1: its B1, then the next step's B0
    const unsigned stage = (s & 1) * kStage, next = kStage - stage;
    const unsigned scale = scale_at(s), scale_next = scale_at(s + 1);
    constexpr int kWait = 2 * PL + decltype(spare)::stores;
    wait_loads<kWait>();
    lds_barrier();
    if ((s & 3) == 0) load_scales((s >> 2) + 1);
    u32x4 ra = step_resource(pa, enda, s + 2), rb = step_resource(pb, endb, s + 2);
    settled(ra);
    settled(rb);
    quarter(0, 0, a0, x0, [&](int q) {
      loads(q, PA, [&](int k) { to_a(0, k, stage); });
    }, [&](int q) {
      reads(q, HN, [&](int k) { read(x1[k], fb, eb0, HN + k, stage, scale); });
      loads(q, PA, [&](int k) { load_from(ra, off_a(0, k)); });
    });
    quarter(0, 1, a0, x1, [&](int q) {
      loads(q, PB, [&](int k) { to_b(0, k, stage); });
    }, [&](int q) {
      reads(q, HM, [&](int k) { read(a1[k], fa, ea0, HM + k, stage, scale); });
      loads(q, PB, [&](int k) { load_from(rb, off_b(0, k)); });
    });
    wait_loads<decltype(spare)::first_half ? 2 * PL : kWait>();
    lds_barrier();
    if (GLU) {
      rb = step_resource(pb + up, endb, s + 2);
      settled(rb);
    }
    quarter(1, 1, a1, x1, [&](int q) {
      loads(q, PA, [&](int k) { to_a(1, k, stage); });
    }, [&](int q) {
      reads(q, HM, [&](int k) { read(a0[k], fa, ea0, k, next, scale_next); });
      loads(q, PA, [&](int k) { load_from(ra, off_a(1, k)); });
    });
    quarter(1, 0, a1, x0, [&](int q) {
      loads(q, PB, [&](int k) { to_b(1, k, stage); });
    }, [&](int q) {
      reads(q, HN, [&](int k) { read(x1[k], fb, eb0, k, next, scale_next); });
      loads(q, PB, [&](int k) { load_from(rb, off_b(1, k)); });
    });
  };
  auto load_step = [&](int s) {  // all of a whole step
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 ra = step_resource(pa, enda, s), rb = step_resource(pb + h * up, endb, s);
      settled(ra);
      settled(rb);
      load_half(h, (s & 1) * kStage, ra, rb, kStep);
    }
  };
  // Stores of a whole tile, at the least: they follow the next tile's first loads, and go on while its first steps run.
  constexpr int W = 4 * GB, JG = TN / GB / (GLU ? 2 : 1), COLS = GLU ? HALF : TN * 16;
  constexpr int kStores = TM * JG * W * (OUT == kOut8 ? 1 : OUT == kOut32 ? 4 : 2) / 16;
  constexpr bool kMany = BM == 256;  // a workgroup goes over several tiles
  static_assert(3 * PL + (kMany ? kStores : 0) < 64, "operations that a wait can count");
  auto begin = [&] {
    load_scales(0);
    if (whole == 0) return;
    load_step(0);
    load_step(1);
  };
  // Some workgroups begin half a tile later, so that not all of them multiply at once and store at once: where the last
  // round is not full those that have a tile less, otherwise every other one.
  if constexpr (kMany) {
    const int k0 = blockIdx.x >> 3, rounds = (tiles + (int)gridDim.x - 1) / (int)gridDim.x;
    const bool later = tiles % (int)gridDim.x ? k0 + (rounds - 1) * stride >= mine : k0 & 1;
    for (int i = later ? 0 : p.later; i < p.later; ++i) __builtin_amdgcn_s_sleep(16);  // (1024 cycles)
  }
  place(blockIdx.x >> 3);
  begin();
  bool counted = false;  // kStores stores or more follow the loads
  for (int k = blockIdx.x >> 3; k < mine; k += stride) {
  {  // the sums begin with the bias
    const ArgsAgain p = args_again();
    const long nb = n0 + wn * COLS + (again(tid & 63) >> 4) * W;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      f32x4 b{0.f, 0.f, 0.f, 0.f};
      if (p->bias)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const long n = nb + j / GB % JG * 16 * GB + q * GB + j % GB;
          if (n < p->N) b[q] = bias_at(p->bias, p->bdtype, (j / GB >= JG ? p->N : 0) + n);
        }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        acc[i][j] = b;
        if (!EXACT) accumulator(acc[i][j]);
      }
    }
  }
  acc_settled();
  if constexpr (EXACT) {
    for (int i = 0; i < TM; ++i) nan_row[i] = false;
    for (int j = 0; j < kScaleSets; ++j)
      for (int q = 0; q < 4; ++q) nan_column[j][q] = false;
    for (int s = 0; s < whole; ++s) {
      const unsigned stage = (s & 1) * kStage, scale = scale_at(s);
      Frag a[TM], b[TN];
      wait_loads<2 * PL>();
      lds_barrier();
#pragma unroll
      for (int j = 0; j < TN; ++j) read(b[j], fb, eb0, j, stage, scale);
#pragma unroll
      for (int i = 0; i < TM; ++i) read(a[i], fa, ea0, i, stage, scale);
      lds_barrier();
      if ((s & 3) == 0) load_scales((s >> 2) + 1);
      load_step(s + 2);
      multiply(a, b, scale);
    }
    if (whole > 0) {
      wait_loads<0>();
      lds_barrier();
    }
  } else {
    if (!kMany) wait_loads<3 * PL>();
    else if (counted) wait_loads<3 * PL + kStores>();
    else wait_loads<0>();
    lds_barrier();
    if (whole > 0) {
#pragma unroll
      for (int i = 0; i < HM; ++i) read(a0[i], fa, ea0, i, 0, 0);
#pragma unroll
      for (int j = 0; j < HN; ++j) read(b0[j], fb, eb0, j, 0, 0);
      int s = 0;
      if constexpr (kMany) {
        step(Spare<kStores, false>{}, 0, b0, b1);
        if (whole > 1) step(Spare<kStores, true>{}, 1, b1, b0);
        s = 2;
      }
      for (; s + 2 <= whole; s += 2) {
        step(Spare<0, true>{}, s, b0, b1);
        step(Spare<0, true>{}, s + 1, b1, b0);
      }
      if (s < whole) step(Spare<0, true>{}, s, b0, b1);
      wait_loads<0>();
      lds_barrier();
    }
  }
  if (tail) {  // the end of the rows: its elements at and behind `tail` as zeros
    const unsigned stage = (whole & 1) * kStage, scale = scale_at(whole);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const size_t at = (size_t)whole * kStep;
      u32x4 ra = resource(pa + at, enda - (unsigned)at), rb = resource(pb + h * up + at, endb - (unsigned)at);
      settled(ra);
      settled(rb);
      load_half(h, stage, ra, rb, tail);
    }
    wait_loads<0>();
    lds_barrier();
    i32x8 mask;
#pragma unroll
    for (int d = 0; d < 8; ++d) {  // bytes of the end: the row's storage goes on behind them
      const int n = tail - (16 * (g + d / 4 * 4) + d % 4 * 4);
      mask[d] = n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1;
    }
    Frag b[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      read(b[j], fb, eb0, j, stage, scale);
      b[j].v &= mask;
      operand_settled(b[j].v);
    }
    if constexpr (EXACT) {
      Frag a[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        read(a[i], fa, ea0, i, stage, scale);
        a[i].v &= mask;
      }
      multiply(a, b, scale);
    } else {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        Frag a;
        read(a, fa, ea0, i, stage, scale);
        a.v &= mask;
        operand_settled(a.v);
#pragma unroll
        for (int j = 0; j < TN; ++j) product128(b[j].v, b[j].e, a.v, a.e, acc[i][j]);
      }
    }
    lds_barrier();
  }

  if constexpr (EXACT)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (nan_row[i] || nan_column[j][q]) acc[i][j][q] = NAN;
  acc_settled();
  const ArgsAgain p = args_again();
  const int tid = again(threadIdx.x), l = tid & 63, r = l & 15, g = l >> 4;
  const long cm = m0, cn = n0;  // this tile, while the next one's operands are loaded
  const bool direct = ACT != kActOther && cn + NT <= p->N, more = kMany && k + stride < mine;
  if (direct && more) {
    place(k + stride);
    begin();
  }
  counted = direct && cm + BM <= p->M;
  // Tiles that end within the columns: straight from the accumulators.  A lane holds, of each of its rows, W consecutive
  // columns of each group.
  if constexpr (ACT != kActOther) {
    if (direct) {
      const long nw = cn + wn * COLS + g * W;
      auto row_of = [&](int i) { return cm + wm * TM * 16 + slot_row(i * 16 + r, GA); };
      auto values = [&](int i, int j, float (&v)[W]) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          v[e] = value_of<!EXACT>(acc[i][j * GB + e % GB][e / GB]);
          if (GLU) {
            constexpr int U = GLU ? JG : 0;
            v[e] = v[e] * sigmoid(v[e]) * value_of<!EXACT>(acc[i][(j + U) * GB + e % GB][e / GB]);
          }
        }
      };
      if constexpr (OUT == kOut8) {
        // a block's columns lie in the four lanes of a row, of one wave or of two
        constexpr bool kTwo = COLS * 2 == kFp8Block;
        static_assert((kTwo && JG == 1) || COLS == kFp8Block, "blocks of a wave, or of two");
        auto largest = [&](const float (&v)[JG][W]) {
          unsigned most = 0;
#pragma unroll
          for (int j = 0; j < JG; ++j)
#pragma unroll
            for (int e = 0; e < W; ++e) most = max(most, magnitude(v[j][e]));
          most = max(most, (unsigned)__shfl_xor((int)most, 16));
          return max(most, (unsigned)__shfl_xor((int)most, 32));
        };
        auto emit = [&](int i, const float (&v)[JG][W], unsigned most) {
          const unsigned byte = scale_byte(most);
          const long m = row_of(i);
          if (m >= p->M) return;
#pragma unroll
          for (int j = 0; j < JG; ++j) {
            typedef unsigned words __attribute__((ext_vector_type(W / 4)));
            words o;
#pragma unroll
            for (int e = 0; e < W / 4; ++e) o[e] = fp8_word(v[j][4 * e], v[j][4 * e + 1], v[j][4 * e + 2], v[j][4 * e + 3], byte);
            *gmem((words*)((unsigned char*)p->out + m * p->ldo + nw + j * 16 * GB)) = o;
          }
          if (g == 0 && (!kTwo || (wn & 1) == 0)) p->os[m * p->los + (cn + wn * COLS) / kFp8Block] = (unsigned char)byte;
        };
        if constexpr (!kTwo) {
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            float v[JG][W];
#pragma unroll
            for (int j = 0; j < JG; ++j) values(i, j, v[j]);
            emit(i, v, largest(v));
            __builtin_amdgcn_sched_barrier(0);
          }
        } else {
          __shared__ unsigned block_most[WN][BM];
          float v[TM][JG][W];
          unsigned most[TM];
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            values(i, 0, v[i][0]);
            most[i] = largest(v[i]);
            if (g == 0) block_most[wn][(wm * TM + i) * 16 + r] = most[i];
            __builtin_amdgcn_sched_barrier(0);
          }
          __syncthreads();
#pragma unroll
          for (int i = 0; i < TM; ++i) emit(i, v[i], max(most[i], block_most[wn ^ 1][(wm * TM + i) * 16 + r]));
        }
      } else {
        // all of the residual on its way at once: the fragments' registers are free
        auto emit = [&](auto type) {
          typedef decltype(type) T;
          RowPiece<T, W> res[TM][JG];
          if (p->res)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int j = 0; j < JG; ++j)
                if (row_of(i) < p->M) res[i][j].v = *gmem((const typename RowPiece<T, W>::any*)((const T*)p->res + row_of(i) * p->ldr + nw + j * 16 * GB));
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            const long m = row_of(i);
            if (m >= p->M) continue;
#pragma unroll
            for (int j = 0; j < JG; ++j) {
              float v[W];
              values(i, j, v);
              if (p->res)
#pragma unroll
                for (int e = 0; e < W; ++e) v[e] += (float)res[i][j].v[e];
              typename RowPiece<T, W>::vec o;
#pragma unroll
              for (int e = 0; e < W; ++e) o[e] = (T)v[e];
              *gmem((typename RowPiece<T, W>::any*)((T*)p->out + m * p->ldo + nw + j * 16 * GB)) = o;
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        };
        if constexpr (OUT == kOut32) emit(0.f);
        else if (p->dtype == kBf16) emit((bf16)0.f);
        else if (kMany || p->dtype == kF16) emit((f16)0.f);
        else emit(0.f);
      }
      if (kMany) continue;
      return;
    }
  }

  // The others, and the activations that are code of some size, through LDS: a thread takes eight consecutive columns of NG
  // rows at a time.
  float* tile = (float*)smem;
  constexpr int PR = NT / 8, RP = NW * 64 / PR, NG = std::min(4, WM * kPass / RP);  // threads of a row, rows at a time
  static_assert(WM * kPass % (NG * RP) == 0, "whole groups of rows");
  const int c = tid % PR * 8, cw = c / (GLU ? HALF : NT), cs = GLU ? cw * 2 * HALF + c % HALF : c;
  const long n = cn + c;
  auto through = [&](auto type, int h) {
    typedef decltype(type) T;
    for (int i0 = tid / PR; i0 < WM * kPass; i0 += NG * RP) {
      RowPiece<T, 8> res[NG];
      long m[NG];
      float v[NG * 8], up[8];
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        const int i = i0 + k * RP;
        m[k] = cm + i / kPass * (TM * 16) + slot_row(h * kPass + i % kPass, GA);
        if (p->res && m[k] < p->M && n < p->N) res[k].load((const T*)p->res + m[k] * p->ldr, n, p->N);
      }
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        const float* row = tile + (i0 + k * RP) * kPitch + cs;
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          *(f32x4*)(v + 8 * k + e) = *(const f32x4*)(row + e);
          if (GLU) *(f32x4*)(up + e) = *(const f32x4*)(row + HALF + e);
        }
        if (GLU)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[8 * k + e] = v[8 * k + e] * sigmoid(v[8 * k + e]) * up[e];
      }
      if (!GLU && ACT != kActNone) act_values<NG * 8>(p->act, v);
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        float(&w)[8] = *(float(*)[8])(v + 8 * k);
        if constexpr (OUT == kOut8) {  // a row's 16 lanes of a block go together
          unsigned most = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (n + e >= p->N) w[e] = 0.f;
            most = max(most, magnitude(w[e]));
          }
          const unsigned byte = scale_byte(lanes_max16(most));
          const u32x2 o = {fp8_word(w[0], w[1], w[2], w[3], byte), fp8_word(w[4], w[5], w[6], w[7], byte)};
          if (m[k] < p->M && n < p->N) {
            *gmem((u32x2*)((unsigned char*)p->out + m[k] * p->ldo + n)) = o;
            if ((tid & 15) == 0) p->os[m[k] * p->los + n / kFp8Block] = (unsigned char)byte;
          }
        } else if (m[k] < p->M && n < p->N) {
          if (p->res)
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] += (float)res[k].v[e];
          store_row<T, 8>((T*)p->out + m[k] * p->ldo, n, p->N, w);
        }
      }
    }
  };
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
            tile[(wm * kPass + i * 16 + r) * kPitch + (wn * TN + j) * 16 + (4 * g + q) * GB + k] =
                value_of<!EXACT>(acc[h * (kPass / 16) + i][j + k][q]);
    __syncthreads();
    if constexpr (OUT == kOut16) {
      if (p->dtype == kBf16) through((bf16)0.f, h);
      else if (kMany || p->dtype == kF16) through((f16)0.f, h);
      else through(0.f, h);
    } else {
      through(0.f, h);
    }
  }
  if (!kMany) return;
  if (more) {
    lds_barrier();
    place(k + stride);
    begin();
  }
  }
}

// ---------------------------------------------------------------------------
// few rows: the weight's bytes
// ---------------------------------------------------------------------------
// 16 columns (swiglu: 16 gates and their ups) of 16 rows by a group of `parts` waves, each over its part of the
// contraction, through LDS of its own: a wave waits for nothing but its own loads, some steps of which are on their way.
// (Straight into registers a lane's neighbours would lie in other rows, and 16 bytes take a request each: 16 bytes a cycle
// and CU, 64 so.)  The parts' sums meet in LDS, in their order.  An output in 8 bits needs its blocks' largest magnitudes:
// its workgroup is eight groups of one wave, 128 columns.  Bound by latency, or by the weight's bytes: 16 x 1024 over 1024 4.3 us
// (by tiles of 64 5.5), 16 x 2816 swiglu over 1024 into 8 bits, from HBM, 7.5, one row of 32000 over 1024 into fp32 9.0
// (3.7 TB/s; 7.9 where the last-level cache holds the weight).
struct ThinArgs {
  Fp8ProductArgs p;
  int parts;  // waves to a group: 1, 2, 4 or 8
};
constexpr int kThinWaves = 8;
template <int ACT, int OUT>
__global__ __launch_bounds__(kThinWaves * 64) void fp8_thin_kernel(const ThinArgs a) {
  constexpr bool GLU = ACT == kActSwiglu, EXACT = OUT == kOut32;
  constexpr int NW = kThinWaves, C = GLU ? 2 : 1, kAhead = GLU ? 3 : 4, kLoads = 2 * (C + 1);  // of a step
  constexpr unsigned kTile = 16 * kStep, kSlot = (C + 1) * kTile, kMine = kAhead * kSlot + 512;
  const Fp8ProductArgs& p = a.p;
  const int parts = OUT == kOut8 ? 1 : a.parts;
  __shared__ __attribute__((aligned(1024))) char smem[NW * kMine];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, r = l & 15, g = l >> 4;
  const int part = wave & (parts - 1), first = wave - part;
  const long n0 = ((long)blockIdx.x * (NW / parts) + first / parts) * 16, m0 = (long)blockIdx.y * 16;
  const int steps = (int)((p.K + kStep - 1) / kStep), tail = (int)(p.K & (kStep - 1));
  const int per = (steps + parts - 1) / parts, s0 = min(part * per, steps), s1 = min(s0 + per, steps);
  const unsigned lds = lds_addr(smem) + wave * kMine, lds_scales = lds + kAhead * kSlot;
  // rows behind the last one: the last one's, which nothing is made of; operand 0: x, then the weight's gates and ups
  const long na = min(n0, p.N - 1);
  unsigned off[2][2];  // of a lane's piece in a load of x, of the weight
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int slot = 8 * i + (l >> 3), piece = ((l & 7) ^ swz(slot)) << 4;
    off[0][i] = (unsigned)(min((long)slot, p.M - 1 - m0) * p.lda) + piece;
    off[1][i] = (unsigned)(min((long)slot, p.N - 1 - na) * p.ldb) + piece;
  }
  size_t base[C + 1];
  base[0] = (size_t)p.a + m0 * p.lda;
#pragma unroll
  for (int j = 0; j < C; ++j) base[1 + j] = (size_t)p.b + (na + j * p.N) * p.ldb;
  // scales: 16 rows of each operand, a word of four steps a lane (the fourth 16 lanes as the first)
  const int op = g <= C ? g : 0;
  const unsigned char* scales = op ? p.sb + (min(na + r, p.N - 1) + (op - 1) * p.N) * p.lsb : p.sa + min(m0 + r, p.M - 1) * p.lsa;
  auto load_scales = [&](int quad) {
    if (quad * 4 < steps) load4_to(lds_scales + (quad & 1) * 256, scales + 4 * quad);
  };
  auto load_step = [&](int s, int slot) {  // (nothing but zeros behind the part's end)
    const int left = tail && s == steps - 1 ? tail : kStep;
#pragma unroll
    for (int o = 0; o <= C; ++o) {
      u32x4 rs = resource(base[o] + (size_t)s * kStep, s < s1 ? 0x7fffffffu : 0u);
      settled(rs);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        load_to(lds + slot * kSlot + o * kTile, i);
        const unsigned f = off[o ? 1 : 0][i];
        const bool on = (((l & 7) ^ swz(8 * i + (l >> 3))) << 4) < left;
        asm volatile("s_nop 0");
        load_from(rs, on ? f : kNowhere);
      }
    }
  };
  struct Frag {
    i32x8 v;
    int e;
  };
  auto read = [&](Frag& f, int o, int s, int slot) {
    const unsigned at = lds + slot * kSlot + o * kTile + r * kStep;
    const i32x4 x = __builtin_bit_cast(i32x4, read16(at + ((g ^ swz(r)) << 4))),
                y = __builtin_bit_cast(i32x4, read16(at + (((g + 4) ^ swz(r)) << 4)));
    f.v = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    typedef __attribute__((address_space(3))) const unsigned char lds_byte;
    f.e = *(lds_byte*)(size_t)(lds_scales + (s >> 2 & 1) * 256 + (16 * o + r) * 4 + (s & 3));
  };
  f32x4 acc[C];
#pragma unroll
  for (int j = 0; j < C; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (s0 < s1) {
    load_scales(s0 >> 2);
    load_scales((s0 >> 2) + 1);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load_step(s0 + i, i);
    int slot = 0;
    for (int s = s0; s < s1; ++s) {
      wait_loads<(kAhead - 1) * kLoads>();
      Frag x, w[C];
      read(x, 0, s, slot);
#pragma unroll
      for (int j = 0; j < C; ++j) read(w[j], 1 + j, s, slot);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next load arrives there
      if ((s & 3) == 3) load_scales((s >> 2) + 2);
      load_step(s + kAhead, slot);
      slot = slot == kAhead - 1 ? 0 : slot + 1;
      if (tail & 15 && s == steps - 1)
#pragma unroll
        for (int d = 0; d < 8; ++d) {  // bytes of the end: the rows' storage goes on behind them
          const int n = tail - (16 * (g + d / 4 * 4) + d % 4 * 4);
          const int mask = n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1;
          x.v[d] &= mask;
#pragma unroll
          for (int j = 0; j < C; ++j) w[j].v[d] &= mask;
        }
#pragma unroll
      for (int j = 0; j < C; ++j) {
        if constexpr (!EXACT) acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[j].v, x.v, acc[j], 0, 0, 0, w[j].e, 0, x.e);
        else exact_product(w[j].v, w[j].e, x.v, x.e, acc[j]);
      }
    }
    wait_loads<0>();
  }

  if (parts > 1) {
    f32x4* sums = (f32x4*)smem;
    __syncthreads();  // (the sums lie where other waves' steps lay)
#pragma unroll
    for (int j = 0; j < C; ++j) sums[(wave * C + j) * 64 + l] = acc[j];
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int j = 0; j < C; ++j)
      for (int k = 1; k < parts; ++k) acc[j] += sums[((first + k) * C + j) * 64 + l];
  }
  const long n = n0 + 4 * g, row = m0 + r;
  if (OUT != kOut8 && (row >= p.M || n >= p.N)) return;
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const long c = min(n + e, p.N - 1);
    v[e] = acc[0][e] + (p.bias ? bias_at(p.bias, p.bdtype, c) : 0.f);
    if (GLU) v[e] = v[e] * sigmoid(v[e]) * (acc[C - 1][e] + (p.bias ? bias_at(p.bias, p.bdtype, p.N + c) : 0.f));
  }
  if (!GLU && ACT != kActNone) act_values<4>(p.act, v);
  if constexpr (OUT == kOut8) {
    __shared__ unsigned block_most[NW][16];
    unsigned most = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (n + e >= p.N) v[e] = 0.f;
      most = max(most, magnitude(v[e]));
    }
    most = max(most, (unsigned)__shfl_xor((int)most, 16));
    most = max(most, (unsigned)__shfl_xor((int)most, 32));
    if (g == 0) block_most[wave][r] = most;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NW; ++k) most = max(most, block_most[k][r]);
    if (row >= p.M || n >= p.N) return;
    const unsigned byte = scale_byte(most);
    *gmem((unsigned*)((unsigned char*)p.out + row * p.ldo + n)) = fp8_word(v[0], v[1], v[2], v[3], byte);
    if (wave == 0 && g == 0) p.os[row * p.los + n / kFp8Block] = (unsigned char)byte;
    return;
  }
  auto emit = [&](auto type) {
    typedef decltype(type) T;
    if (p.res) add_row<T, 4>((const T*)p.res + row * p.ldr, n, p.N, v);
    store_row<T, 4>((T*)p.out + row * p.ldo, n, p.N, v);
  };
  if (OUT == kOut32 || p.dtype == kF32) emit(0.f);
  else if (p.dtype == kBf16) emit((bf16)0.f);
  else emit((f16)0.f);
}

constexpr int kCus = 256;

template <int OUT>
hipError_t launch_thin(const Fp8ProductArgs& p, int parts, hipStream_t st) {
  const long groups = (p.N + 15) / 16, per = kThinWaves / parts;
  const dim3 grid((unsigned)((groups + per - 1) / per), (unsigned)((p.M + 15) / 16)), block(kThinWaves * 64);
  const ThinArgs a{p, parts};
  if (p.act == kActSwiglu) hipLaunchKernelGGL((fp8_thin_kernel<kActSwiglu, OUT>), grid, block, 0, st, a);
  else if (p.act == kActNone) hipLaunchKernelGGL((fp8_thin_kernel<kActNone, OUT>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((fp8_thin_kernel<kActOther, OUT>), grid, block, 0, st, a);
  return hipGetLastError();
}

// Half a tile of 256 in units of 1024 cycles, by which some workgroups begin later; 0 where that costs more than it gives.
// Where the last round is not full it costs nothing: 16384 x 2816 swiglu over 1024 into 8 bits 111 -> 104 us, into bf16 109 ->
// 106, 16384 x 2816 58.6 -> 55.0.  Full rounds end half a tile later: 65536 x 2816 swiglu over 1024 into 8 bits (22 rounds)
// 413 -> 365, into bf16 390 -> 363, 16384 x 4096 over 1024 (4) 79.9 -> 76.9, but 8192^3 (4) 384 -> 395, 65536 x 1024 over 2816
// (4) 165 -> 177.
int half_tile(long tiles, long steps) {
  const long rounds = (tiles + kCus - 1) / kCus;
  const float tile = 1.4f * steps + 6.f;  // us, each of 2 units
  return rounds > 1 && (tiles % kCus || rounds * 4.5f > tile) ? (int)std::min(tile, 1000.f) : 0;
}

template <int BM, int OUT>
hipError_t launch_tiles(const Fp8ProductArgs& args, hipStream_t st) {
  constexpr int BN = BM, WM = 2, WN = 2;
  Fp8ProductArgs p = args;
  const int NT = p.act == kActSwiglu ? BN / 2 : BN;
  const long tiles = ((p.M + BM - 1) / BM) * ((p.N + NT - 1) / NT);
  p.later = BM == 256 ? half_tile(tiles, (p.K + kStep - 1) / kStep) : 0;
  const dim3 grid((unsigned)(BM == 256 ? std::min<long>(tiles, kCus) : tiles)), block(WM * WN * 64);
  if (BM == 256 && OUT == kOut16 && p.dtype == kF32) return hipErrorInvalidConfiguration;  // (tiles of 256: 16 bits)
  if (p.act == kActSwiglu) {
    if constexpr (OUT == kOut8 && BN < 256) return hipErrorInvalidConfiguration;  // (a tile's outputs: half a block)
    else hipLaunchKernelGGL((fp8_product_kernel<BM, BN, WM, WN, kActSwiglu, OUT>), grid, block, 0, st, p);
  } else if (p.act == kActNone) {
    hipLaunchKernelGGL((fp8_product_kernel<BM, BN, WM, WN, kActNone, OUT>), grid, block, 0, st, p);
  } else {
    hipLaunchKernelGGL((fp8_product_kernel<BM, BN, WM, WN, kActOther, OUT>), grid, block, 0, st, p);
  }
  return hipGetLastError();
}

// How a product runs.
struct Fp8Plan {
  int side;      // of its tiles: 256, 128, 64; 0: 16 rows by 16 columns at a time (fp8_thin_kernel)
  int parts;     // of the contraction (side 0)
  bool through;  // an output in 8 bits is written in fp32 first, and quantised by a second launch
};
// By what a call is expected to take, in us, out of times measured on one card (on another those of many rows were up to 7%
// longer; `steps` of 128; an activation without a gate is code that a tile's outputs pass through: `act`):
//   side 0: a workgroup a CU, 0.29 a step of a wave (swiglu 0.45, exactly 0.46), or the weight's bytes.  1024 over 1024, 64
//     rows: 4.3 in eight parts, 5.9 in one, by 64 tiles 5.5; 4064 over 1728, 40 rows 10.9, 7.8 (two parts 6.0), 7.4; 2816
//     over 1024, 600 rows 78, 20, 6.8
//   64: 0.28 a step where the CUs have few tiles (1024 over 1024, 300 rows: 5.5, 128 tiles 7.3, 256 16.5), 1450 tiles and
//     steps a us (1024 over 1024, 2000 rows 6.9, 128 tiles 7.8; 2188 over 959, 4363 rows 25, 22); exactly: 0.62 and 740
//   128: half a step's microsecond for each tile of a CU (2816 over 1024, 16384 rows 57.3, silu 71, gelu 84; 256 tiles 57.9,
//     90, 111; 3520 over 3008, 25960 rows 316, 317, 344; 255, 302, 350; 2188 over 959, 4363 rows 22, 25, 29; 30, 35, 42;
//     4096 over 4096, 2048 rows 35, 4096 rows 66; 47, 62), more where outputs end inside a tile (1100 over 700, 600 rows
//     9.6, 1024 over 1024 7.8)
//   256: a round of all CUs 1.4 a step (8192^3, four rounds with their outputs, 390; fewer workgroups 1.0), and the outputs,
//     more where they end inside a tile (swiglu 2816 over 1024, 9000 rows 74, 128 tiles 63; 16384 rows 104, 108; 1024 over
//     2816, 30000 rows 78, 91)
//   through fp32: the second launch (its host time too), and 8 bytes an output to and fro
Fp8Plan fp8_plan(long M, long N, long K, int act, int out) {
  const bool glu = act == kActSwiglu, other = !glu && act != kActNone;
  const long outs = glu ? 2 * N : N, steps = (K + kStep - 1) / kStep;
  Fp8Plan best{256, 1, false};
  float least = 0.f;
  auto offer = [&](int side, int parts, bool through, float t) {
    if (through) t += 5.f + 1.3e-6f * M * N;
    if (least == 0.f || t < least) {
      least = t;
      best = {side, parts, through};
    }
  };
  auto tiles = [&](long side) { return ((M + side - 1) / side) * ((outs + side - 1) / side); };
  const bool exact = out == kOut32, through = out == kOut8;
  if (M <= 1024) {
    const long groups = (N + 15) / 16 * ((M + 15) / 16);
    const float step = exact ? 0.46f : glu ? 0.45f : 0.29f, bytes = 1.5f + outs * K / 5e6f;
    auto time = [&](int parts) {
      const long wgs = (groups * parts + kThinWaves - 1) / kThinWaves, rounds = (wgs + kCus - 1) / kCus;
      const float part = step * ((steps + parts - 1) / parts);
      return std::max(bytes, 2.4f + (rounds == 1 ? 1.6f + part : rounds * (2.3f + part)));
    };
    for (int parts = 1; parts <= kThinWaves && (parts == 1 || parts <= steps); parts *= 2) offer(0, parts, through, time(parts));
    if (through) offer(0, 1, false, time(1));
  }
  if (exact) {
    offer(64, 1, false, 3.5f + std::max(0.62f * steps, tiles(64) * (steps + 2) / 740.f));
    return best;
  }
  offer(64, 1, through, 3.f + std::max(0.28f * steps, tiles(64) * (steps + 4) / 1450.f) + (other ? 0.7f : 0.f));
  const long on_one = (tiles(128) + kCus - 1) / kCus;
  offer(128, 1, through && glu, 4.f + (N % 128 || M % 128 ? 2.f : 0.f) + on_one * 0.5f * (steps + (on_one > 1 ? 1 : 0)) + (other ? 1.f + on_one * 1.8f : 0.f));
  const long full = tiles(256) / kCus, rest = tiles(256) % kCus;
  const float ends = 6.f + (other ? 12.f : 0.f) + (N % 256 || M % 256 ? 3.f : 0.f);
  offer(256, 1, false, 4.f + full * (1.4f * steps + ends) + (rest ? (1.f + 0.4f * rest / kCus) * steps + ends : 0.f));
  return best;
}

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

static int out_kind(int dtype, bool into8) { return into8 ? kOut8 : dtype == kF32 ? kOut32 : kOut16; }

// fp32 elements of the workspace that such a call needs
long fp8_product_workspace(long M, long N, long K, int act, int dtype, bool into8) {
  return M > 0 && fp8_plan(M, N, K, act, out_kind(dtype, into8)).through ? M * N : 0;
}

void fp8_product_plan(long M, long N, long K, int act, int dtype, bool into8, int* side, int* parts, int* through) {
  const Fp8Plan plan = fp8_plan(M, N, K, act, out_kind(dtype, into8));
  *side = plan.side;
  *parts = plan.parts;
  *through = plan.through;
}

hipError_t launch_fp8_product(const Fp8ProductArgs& args, float* workspace, hipStream_t st) {
  if (args.M <= 0) return hipSuccess;
  const int out = out_kind(args.dtype, args.os != nullptr);
  const Fp8Plan plan = fp8_plan(args.M, args.N, args.K, args.act, out);
  Fp8ProductArgs p = args;
  if (plan.through) {
    p.out = workspace;
    p.ldo = p.N;
    p.dtype = kF32;
    p.os = nullptr;
  }
  hipError_t e;
  if (plan.side == 0)
    e = out == kOut32 ? launch_thin<kOut32>(p, plan.parts, st) : p.os ? launch_thin<kOut8>(p, 1, st) : launch_thin<kOut16>(p, plan.parts, st);
  else if (out == kOut32) e = launch_tiles<64, kOut32>(p, st);
  else if (plan.side == 64) e = p.os ? hipErrorInvalidConfiguration : launch_tiles<64, kOut16>(p, st);
  else if (plan.side == 128) e = p.os ? launch_tiles<128, kOut8>(p, st) : launch_tiles<128, kOut16>(p, st);
  else e = p.os ? launch_tiles<256, kOut8>(p, st) : launch_tiles<256, kOut16>(p, st);
  if (e != hipSuccess || !plan.through) return e;
  return launch_quantize({workspace, (unsigned char*)args.out, args.os, args.M, args.N, args.N, args.ldo, args.los, kF32}, st);
}

}  // namespace ccq
