// Block norms: layer norm and RMS norm over rows of any width up to 8192, with the residual stream's add in
// the same pass, and their backward with the gradients of weight and bias.
//
//   s = x + r (kept in x's type: the stream as the next block reads it), mu = mean s (RMS: 0),
//   rho = 1 / sqrt(mean (s - mu)^2 + eps), h = (s - mu) rho, y = h w + b
//   a = dy w, ds = rho (a - mean a - h mean(a h)) + (the stream's own gradient)   (RMS: without mean a)
//   dw = sum over rows of dy h, db = sum over rows of dy
//
// Bound by HBM bytes: every row is read once and held in registers between the statistics and the output, so
// the variance is the mean of squared deviations (two passes over registers, no cancellation).  A row belongs
// to part of a wave, a wave, 4 waves or 16 waves, whichever holds it in one or two 16-byte pieces a lane; the
// workgroups walk the rows with the next row's pieces already in flight, weights stay in registers.  The
// backward keeps the sums over its rows in registers and leaves one partial row a workgroup, added in a fixed
// order by a second kernel: no atomics, the same bits on every run.
#include <algorithm>

#include "ccq_block_args.h"
#include "ccq_fp8.h"
#include "ccq_rows.h"

namespace ccq {

namespace {

constexpr int kNormFwdBlocks = 2048;  // workgroups of 256 that walk the rows (8 per CU)

// N values of a vector of WT from column c on, at its element's alignment; zeros past its end
template <typename WT, int N>
__device__ __forceinline__ void load_values(const WT* w, int c, int D, float (&v)[N]) {
  typedef WT vec __attribute__((ext_vector_type(N)));
  typedef vec any __attribute__((aligned(sizeof(WT))));
  if (c + N <= D) {
    const vec x = *gmem((const any*)(w + c));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)x[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = c + i < D ? (float)*gmem(w + c + i) : 0.f;
}
template <int N>
__device__ __forceinline__ void load_weight(const void* w, int wdtype, int c, int D, float otherwise, float (&v)[N]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = otherwise;
  } else if (wdtype == kF32) {
    load_values((const float*)w, c, D, v);
  } else if (wdtype == kBf16) {
    load_values((const bf16*)w, c, D, v);
  } else {
    load_values((const f16*)w, c, D, v);
  }
}

// The threads of one row: WPR waves, or L lanes of one wave (WPR == 1; L < 64 only with P == 1).
template <int WPR>
struct RowTeam {
  int li, L;         // index inside the row's team, lanes of a team inside one wave
  long row, stride;  // first row, rows between this team's rows
  __device__ RowTeam(int lanes, int tid) {
    if (WPR == 1) {
      L = lanes;
      const int per_wave = 64 / L, waves = kThreads / 64;
      li = tid & (L - 1);
      row = ((long)blockIdx.x * waves + (tid >> 6)) * per_wave + (tid & 63) / L;
      stride = (long)gridDim.x * waves * per_wave;
    } else {
      L = 64;
      li = tid;
      row = blockIdx.x;
      stride = gridDim.x;
    }
  }
};

// Sums of K values over the team.  The slots alternate between calls (phase), so one barrier a call is enough:
// a wave writes a slot again only after every wave has passed the next call's barrier.
template <int WPR, int K>
__device__ __forceinline__ void team_sum(float (&v)[K], int L, int tid, float (*slots)[K][WPR], int& phase) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = lanes_sum(v[k], L);
  if constexpr (WPR > 1) {
    float(*sl)[WPR] = slots[phase];
    phase ^= 1;
    if ((tid & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) sl[k][tid >> 6] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) t += sl[k][i];
      v[k] = t;
    }
  }
}

// the piece as it lies packed in registers: what was computed from it before is not kept for use behind this
template <typename V>
__device__ __forceinline__ void keep_packed(V& v) {
  u32x4 u = __builtin_bit_cast(u32x4, v);
  asm volatile("" : "+v"(u));
  v = __builtin_bit_cast(V, u);
}

// Q8: y in 8 bits (ccq_fp8.h); 128 / N consecutive lanes hold a block, all of the team where it has fewer.
template <typename T, bool LAYER, int WPR, int P, bool Q8>
__global__ __launch_bounds__(WPR > 4 ? WPR * 64 : kThreads) void norm_fwd_kernel(const NormArgs a, int lanes) {
  constexpr int N = Piece<T>::N;
  typedef typename Piece<T>::vec vec;
  __shared__ float slots[2][1][WPR];
  const int tid = threadIdx.x, D = a.D;
  const RowTeam<WPR> t(lanes, tid);
  const int step = WPR == 1 ? t.L * N : WPR * 64 * N, c0 = t.li * N;
  const T *x = (const T*)a.x, *r = (const T*)a.r;
  float w[P][N], b[P][N];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    load_weight<N>(a.w, a.wdtype, c0 + j * step, D, 1.f, w[j]);
    load_weight<N>(a.b, a.wdtype, c0 + j * step, D, 0.f, b[j]);
  }
  const float inv = 1.f / (float)D;
  int phase = 0;
  vec nx[P], nr[P];
  const long first = min(t.row, a.rows - 1);  // (teams past the last row repeat it and store nothing)
#pragma unroll
  for (int j = 0; j < P; ++j) {
    nx[j] = load_piece(x + first * a.ldx, c0 + j * step, D);
    if (r) nr[j] = load_piece(r + first * a.ldr, c0 + j * step, D);
  }
  // whole workgroups go round together: the barriers of team_sum need every wave
  const long rounds = WPR == 1 ? (a.rows + t.stride - 1) / t.stride : (a.rows - blockIdx.x + t.stride - 1) / t.stride;
  long row = t.row;
  for (long k = 0; k < rounds; ++k, row += t.stride) {
    float f[P][N];
    float s1[1] = {0.f};
#pragma unroll
    for (int j = 0; j < P; ++j) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[j][i] = (float)nx[j][i];
      if (r) {
        vec sv;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sv[i] = (T)(f[j][i] + (float)nr[j][i]);
          f[j][i] = (float)sv[i];
        }
        if (row < a.rows) store_piece((T*)a.s + row * D, c0 + j * step, D, sv);
      }
    }
    if (k + 1 < rounds) {
      const long next = min(row + t.stride, a.rows - 1);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        nx[j] = load_piece(x + next * a.ldx, c0 + j * step, D);
        if (r) nr[j] = load_piece(r + next * a.ldr, c0 + j * step, D);
      }
    }
    float mu = 0.f;
    if (LAYER) {
#pragma unroll
      for (int j = 0; j < P; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) s1[0] += f[j][i];
      team_sum<WPR, 1>(s1, t.L, tid, slots, phase);
      mu = s1[0] * inv;
    }
    float s2[1] = {0.f};
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (LAYER) f[j][i] = c0 + j * step + i < D ? f[j][i] - mu : 0.f;
        s2[0] += f[j][i] * f[j][i];
      }
    team_sum<WPR, 1>(s2, t.L, tid, slots, phase);
    const float rstd = 1.f / sqrtf(s2[0] * inv + a.eps);
    if constexpr (Q8) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const int c = c0 + j * step, block = kFp8Block / N;
        float v[N];
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {  // (zeros behind D)
          v[i] = f[j][i] * rstd * w[j][i];
          m = max(m, magnitude(v[i]));
        }
        const unsigned byte = scale_byte(lanes_max(m, min(t.L, block)));
        if (row >= a.rows || c >= D) continue;
        typedef unsigned words __attribute__((ext_vector_type(N / 4)));
        words o;
#pragma unroll
        for (int i = 0; i < N / 4; ++i) o[i] = fp8_word(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], byte);
        *gmem((words*)((unsigned char*)a.y + row * a.ldy + c)) = o;
        if ((t.li & (block - 1)) == 0) a.scales[row * a.lds + c / kFp8Block] = (unsigned char)byte;
      }
    } else if (row < a.rows) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        vec y;
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = (T)(f[j][i] * rstd * w[j][i] + b[j][i]);
        store_piece((T*)a.y + row * D, c0 + j * step, D, y);
      }
      if (t.li == 0 && a.rstd) {
        a.rstd[row] = rstd;
        if (LAYER) a.mean[row] = mu;
      }
    }
  }
}

template <typename T, bool LAYER, int WPR, int P>
__global__ __launch_bounds__(WPR > 4 ? WPR * 64 : kThreads) void norm_bwd_kernel(const NormArgs a, int lanes) {
  constexpr int N = Piece<T>::N;
  typedef typename Piece<T>::vec vec;
  __shared__ float slots[2][2][WPR];
  __shared__ float cols[WPR == 1 ? 64 * P * N : 1];
  const int tid = threadIdx.x, D = a.D;
  const RowTeam<WPR> t(lanes, tid);
  const int step = WPR == 1 ? t.L * N : WPR * 64 * N, c0 = t.li * N;
  const T *x = (const T*)a.x, *dy = (const T*)a.dy, *ds = (const T*)a.ds;
  float w[P][N], dw[P][N], db[P][N];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    load_weight<N>(a.w, a.wdtype, c0 + j * step, D, 1.f, w[j]);
#pragma unroll
    for (int i = 0; i < N; ++i) dw[j][i] = db[j][i] = 0.f;
  }
  const float inv = 1.f / (float)D;
  int phase = 0;
  vec nx[P], ny[P], ns[P];
  float nmu = 0.f, nrho = 0.f;
  auto fetch = [&](long row) {
    row = min(row, a.rows - 1);
    nrho = a.rstd[row];
    if (LAYER) nmu = a.mean[row];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      nx[j] = load_piece(x + row * a.ldx, c0 + j * step, D);
      ny[j] = load_piece(dy + row * a.ldy, c0 + j * step, D);
      if (ds) ns[j] = load_piece(ds + row * a.ldds, c0 + j * step, D);
    }
  };
  constexpr bool kAhead = WPR < 16;  // (16 waves hide each other's loads, and their registers hold one row)
  if (kAhead) fetch(t.row);
  const long rounds = WPR == 1 ? (a.rows + t.stride - 1) / t.stride : (a.rows - blockIdx.x + t.stride - 1) / t.stride;
  long row = t.row;
  for (long k = 0; k < rounds; ++k, row += t.stride) {
    if (!kAhead) fetch(row);
    const bool on = row < a.rows;  // (a team past the last row adds nothing)
    const float mu = nmu, rho = nrho;
    vec cx[P], cy[P], cs[P];
    float sums[2] = {0.f, 0.f};  // of a h, of a
#pragma unroll
    for (int j = 0; j < P; ++j) {
      cx[j] = nx[j];
      cy[j] = on ? ny[j] : vec{};
      if (ds) cs[j] = ns[j];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = (float)cy[j][i], h = ((float)cx[j][i] - mu) * rho;
        if (on) dw[j][i] += d * h;
        db[j][i] += d;
        sums[0] += d * w[j][i] * h;
        if (LAYER) sums[1] += d * w[j][i];
      }
    }
    if (kAhead && k + 1 < rounds) fetch(row + t.stride);
    if (!a.dx) continue;
    team_sum<WPR, 2>(sums, t.L, tid, slots, phase);
    const float m1 = sums[0] * inv, m0 = LAYER ? sums[1] * inv : 0.f;
    if (on) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        // h and a are formed again from the pieces: kept in fp32 over the sums they would take four times the
        // registers and leave one wave a SIMD
        keep_packed(cx[j]);
        keep_packed(cy[j]);
        vec o;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float h = ((float)cx[j][i] - mu) * rho, v = rho * ((float)cy[j][i] * w[j][i] - m0 - h * m1);
          o[i] = (T)(ds ? v + (float)cs[j][i] : v);
        }
        store_piece((T*)a.dx + row * D, c0 + j * step, D, o);
      }
    }
  }
  // one partial row a workgroup: the teams of a wave by lane moves, the waves one after the other through LDS
  auto leave = [&](float (&v)[P][N], float* part) {
    if constexpr (WPR == 1) {
#pragma unroll
      for (int j = 0; j < P; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i)
          for (int o = t.L; o < 64; o <<= 1) v[j][i] += __shfl_xor(v[j][i], o);
      for (int wv = 0; wv < kThreads / 64; ++wv) {
        if (tid >> 6 == wv && (tid & 63) < t.L)
#pragma unroll
          for (int j = 0; j < P; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) {
              float* p = cols + (j * 64 + t.li) * N + i;
              *p = wv ? *p + v[j][i] : v[j][i];
            }
        __syncthreads();
      }
      if (tid < t.L)
#pragma unroll
        for (int j = 0; j < P; ++j)
#pragma unroll
          for (int i = 0; i < N; ++i) v[j][i] = cols[(j * 64 + t.li) * N + i];
      __syncthreads();
      if (tid >= t.L) return;
    }
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c0 + j * step + i < D) part[(long)blockIdx.x * D + c0 + j * step + i] = v[j][i];
  };
  if (a.dw) leave(dw, a.dw_part);
  if (a.db) leave(db, a.db_part);
}

// out[c] = sum over the nb partial rows, in their order inside 16 interleaved groups
__global__ __launch_bounds__(1024) void norm_sum_kernel(const NormArgs a, int nb) {
  __shared__ float part[16][64];
  const bool first = a.dw && blockIdx.y == 0;
  const float* p = first ? a.dw_part : a.db_part;
  void* out = first ? a.dw : a.db;
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), g = threadIdx.x >> 6;
  float s = 0.f;
  if (c < a.D)
#pragma unroll 8
    for (int i = g; i < nb; i += 16) s += *gmem(p + (long)i * a.D + c);
  part[g][threadIdx.x & 63] = s;
  __syncthreads();
  if (g || c >= a.D) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += part[i][threadIdx.x];
  if (a.wdtype == kF32) ((float*)out)[c] = s;
  else if (a.wdtype == kBf16) ((bf16*)out)[c] = (bf16)s;
  else ((f16*)out)[c] = (f16)s;
}

// Pieces of a row, and by them the team: part of a wave, a wave, 4 or 16 waves, one or two pieces a lane.  Into 8 bits (no
// bias, nothing kept for a backward) 4 waves hold four pieces a lane as well, and more rows are in flight: 32768 x 8192 fp16
// 217 -> 155 us, 8000 x 4104 52 -> 29, 2048 x 8192 14.9 -> 12.2, 600 x 8000 8.3 -> 6.8 (with 2048 workgroups in place of 1024
// 152, 30.5, 12.6, 6.8).
struct NormShape {
  int wpr, p, lanes;
};
NormShape norm_shape(int D, int dtype, bool q8 = false) {
  const int n = dtype == kF32 ? 4 : 8, np = (D + n - 1) / n;
  if (np <= 64) {
    int l = 1;
    while (l < np) l <<= 1;
    return {1, 1, l};
  }
  if (np <= 128) return {1, 2, 64};
  if (np <= 512) return {4, np <= 256 ? 1 : 2, 64};
  if (q8 && np <= 1024) return {4, 4, 64};
  return {16, np <= 1024 ? 1 : 2, 64};
}
long norm_groups(const NormShape& s, long rows) {  // workgroups that give every team one row
  const long per = s.wpr == 1 ? 4L * (64 / s.lanes) : 1;
  return (rows + per - 1) / per;
}

// A shape for which no kernel is compiled is an error, not a call that leaves its outputs as they were.
template <typename T, bool LAYER>
hipError_t launch_typed(bool bwd, const NormArgs& a, const NormShape& s, unsigned blocks, hipStream_t st) {
  const dim3 block(s.wpr == 16 ? 1024 : kThreads);
#define CCQ_NORM(W, PP)                                                                                        \
  if (s.wpr == W && s.p == PP) {                                                                               \
    constexpr bool Q8 = !LAYER && (W != 16 || PP != 1); /* (4 waves hold those rows) */                        \
    if (a.scales && (bwd || !Q8)) return hipErrorInvalidConfiguration;                                         \
    if (bwd)                                                                                                   \
      hipLaunchKernelGGL((norm_bwd_kernel<T, LAYER, W, PP>), dim3(blocks), block, 0, st, a, s.lanes);          \
    else if (!a.scales)                                                                                        \
      hipLaunchKernelGGL((norm_fwd_kernel<T, LAYER, W, PP, false>), dim3(blocks), block, 0, st, a, s.lanes);   \
    else                                                                                                       \
      hipLaunchKernelGGL((norm_fwd_kernel<T, LAYER, W, PP, Q8>), dim3(blocks), block, 0, st, a, s.lanes);      \
    return hipGetLastError();                                                                                  \
  }
  CCQ_NORM(1, 1) CCQ_NORM(1, 2) CCQ_NORM(4, 1) CCQ_NORM(4, 2) CCQ_NORM(16, 1)
  if constexpr (sizeof(T) == 4) {  // (8192 of two bytes are one piece a thread)
    CCQ_NORM(16, 2)
  }
#undef CCQ_NORM
  if constexpr (!LAYER)
    if (s.wpr == 4 && s.p == 4 && a.scales && !bwd) {
      hipLaunchKernelGGL((norm_fwd_kernel<T, false, 4, 4, true>), dim3(blocks), block, 0, st, a, s.lanes);
      return hipGetLastError();
    }
  return hipErrorInvalidConfiguration;
}

hipError_t launch_norm(bool bwd, const NormArgs& a, unsigned blocks, hipStream_t st) {
  const NormShape s = norm_shape(a.D, a.dtype, a.scales);
  if (a.layer) {
    if (a.dtype == kBf16) return launch_typed<bf16, true>(bwd, a, s, blocks, st);
    if (a.dtype == kF16) return launch_typed<f16, true>(bwd, a, s, blocks, st);
    return launch_typed<float, true>(bwd, a, s, blocks, st);
  }
  if (a.dtype == kBf16) return launch_typed<bf16, false>(bwd, a, s, blocks, st);
  if (a.dtype == kF16) return launch_typed<f16, false>(bwd, a, s, blocks, st);
  return launch_typed<float, false>(bwd, a, s, blocks, st);
}

}  // namespace

// Workgroups of the backward, so partial rows of the weight's and the bias's gradient: 2 a CU have enough pieces in
// flight where a lane holds two; with one piece a lane 4 a CU do, once the rows are many enough to pay for the
// partial rows (32768 x 2048 bf16 layer norm 111 -> 92 us; 32768 x 1024 with two pieces 55 -> 64, 1531 x 777 fp32
// 14.5 -> 17).
int norm_bwd_blocks(long rows, int D, int dtype) {
  const NormShape s = norm_shape(D, dtype);
  const long groups = norm_groups(s, rows);
  const long most = s.p == 1 && s.wpr <= 4 ? std::min(1024L, std::max(512L, groups / 4)) : 512;
  return (int)std::max(1L, std::min(most, groups));
}

hipError_t launch_norm_fwd(const NormArgs& a, hipStream_t st) {
  if (a.rows <= 0) return hipSuccess;
  const NormShape s = norm_shape(a.D, a.dtype, a.scales);
  // 16 waves: each workgroup goes over several rows, so that it loads the weights once and a row's pieces while it works on the
  // one before.  Of 16-bit rows and fp32 rows of two pieces a CU holds one such workgroup (66 to 78 registers), of fp32 rows of
  // one piece two.  2048 -> 512 workgroups, us: RMS norm 2048 x 8192 bf16 20.6 -> 16.6, fp32 30.0 -> 26.5, 8000 x 8192 bf16
  // 52.8 -> 50.3, 2048 x 4104 bf16 20.2 -> 15.0; layer norm 24.9 -> 20.9, 34.0 -> 28.2, 71.6 -> 70.4, 27.1 -> 20.0; into 8
  // bits 2048 x 8192 fp32 24.9 -> 20.2.  Up to 3 % more where HBM is busy with a residual's rows: 8000 x 8192 RMS norm bf16
  // 94.6 -> 95.3, fp32 192.8 -> 195.1.  256 would give 16-bit rows little more (16.3, 50.3, 14.3) and take from fp32 rows of
  // one piece (8000 x 2056 37.6, with 512 35.2, with 256 50.9).
  const long most = s.wpr == 16 ? 512 : s.p == 4 ? 1024 : kNormFwdBlocks;
  return launch_norm(false, a, (unsigned)std::min(most, norm_groups(s, a.rows)), st);
}

hipError_t launch_norm_bwd(const NormArgs& a, hipStream_t st) {
  const int nb = a.rows > 0 ? norm_bwd_blocks(a.rows, a.D, a.dtype) : 0;
  if (nb)
    if (hipError_t e = launch_norm(true, a, (unsigned)nb, st)) return e;
  if (a.dw || a.db)  // (no rows: sums of nothing, zeros)
    hipLaunchKernelGGL(norm_sum_kernel, dim3((unsigned)((a.D + 63) / 64), a.dw && a.db ? 2 : 1), dim3(1024), 0, st, a, nb);
  return hipGetLastError();
}

}  // namespace ccq
