// Log probabilities of given tokens, with the entropy and the k likeliest alternatives of every row, and the
// gradient of the logits.
//
//   m = max x, Z = sum e^(x - m), log p = (x - m) - log Z, logp = log p[id]
//   H = log Z - sum e^(x - m) (x - m) / Z
//   d logits_j = dlogp ([j = id] - p_j) - dH p_j (log p_j + H)
//
// Bound by HBM bytes: the forward reads the logits once (a running maximum with the two sums rescaled when it
// moves, in fp32), the backward reads them once more and writes their gradient.  Both sums of H have terms of
// one sign, so nothing cancels; m and log Z are kept apart, since their sum would lose log Z beside a large m (a row
// masked to the type's lowest value is uniform).  A row belongs to one workgroup.
//
// The alternatives come out of the same pass.  The 64 lanes stand for 64 parts of the row; after a thread's first few
// pieces, which it holds in registers, the k-th largest of the 64 maxima (k <= 64) is a lower bound of the row's k-th
// largest logit, and the pieces with a logit that reaches it are listed, those behind as they are read: about 24 for
// k = 20 where the first pieces are the whole row, 24 / f where they are a fraction f.  Their candidates are listed in
// turn, and every one counts those before it.  A row with more than kTopPieces is read again with the bound of the whole
// row's maxima, and one that still has more, or more than kTopList candidates (equal logits), is ranked by k passes over
// it.  (A second pass for all rows, as first built: 53.8 us against 31 now on 1531 x 32007 fp32 with half the rows
// skipped, k = 5: 98 MB, whose copy would take 20; the start, the bound and the ranks of a row are about 8.)
#include <algorithm>

#include "ccq_block_args.h"
#include "ccq_rows.h"

namespace ccq {

namespace {

constexpr int kTopParts = 64;    // parts of a row, so the largest k
constexpr int kTopPieces = 512;  // pieces that may hold candidates
constexpr int kTopList = 1024;   // candidates
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFar = -1e4f;    // e^(x - m) is 0 long before: stands for -inf in the products with it

// 2^x, one instruction: results below 2^-126 are 0 (beside a sum of at least 1 they are nothing)
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Running maximum m of a part of a row, s = sum e^(x - m), t = sum e^(x - m) (x - m).
struct Part {
  float m, s, t;
};
// NaN enters s alone (comparisons and maxima pass it over), and makes every result of the row NaN.
// Rounded the same whichever comes first, so that the lanes that merge with each other hold the same bits.
__device__ __forceinline__ Part merge(const Part& a, const Part& b) {
#pragma clang fp contract(off)
  const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
  const float da = fmaxf(a.m - ref, kFar), db = fmaxf(b.m - ref, kFar);
  const float ca = exp2_(da * kLog2e), cb = exp2_(db * kLog2e);
  return {m, ca * a.s + cb * b.s, ca * (a.t + a.s * da) + cb * (b.t + b.s * db)};
}

// the values of a piece into p; returns their maximum
template <int N>
__device__ __forceinline__ float add_values(Part& p, const float (&v)[N]) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
  if (m > p.m) {
    if (p.m != -INFINITY) {
      const float d = fmaxf(p.m - m, kFar), c = exp2_(d * kLog2e);
      p.t = c * (p.t + p.s * d);
      p.s *= c;
    }
    p.m = m;
  }
  const float ref = p.m == -INFINITY ? 0.f : p.m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = v[i] - ref, e = exp2_(d * kLog2e);
    p.s += e;
    p.t += e * fmaxf(d, kFar);
  }
  return m;
}

// Order of the alternatives: NaN before any number, the larger logit first, the lower index first.  A key lies above 0
// and below 2^64 - 1, where the passes over a row begin: +inf's upper half is 0xff800000, -inf's 0x007fffff.
__device__ __forceinline__ unsigned long long rank_key(float x, int i) {
  const int b = __float_as_int(x + 0.f);  // (-0 as +0)
  unsigned u = b < 0 ? ~(unsigned)b : (unsigned)b | 0x80000000u;
  if (x != x) u = 0xfffffffeu;
  return (unsigned long long)u << 32 | (unsigned)~i;
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)~(unsigned)k; }
__device__ __forceinline__ float key_value(unsigned long long k) {
  const unsigned u = (unsigned)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

constexpr int kAhead = 4;  // pieces loaded together

// f(column, piece) over the thread's pieces of a row, one at a time (for rows that are read again: its registers are the
// main loop's loss)
template <typename T, typename F>
__device__ __forceinline__ void over_row(const T* row, int V, int tid, int threads, F&& f) {
  constexpr int N = Piece<T>::N;
#pragma unroll 1
  for (int c = tid * N; c < V; c += threads * N) f(c, load_piece(row, c, V));
}

// The candidates of a row: pieces that hold a logit at or above the bound, then those logits in rank order.  (Whole
// pieces, since a thread that looked at every element there and then took twice the registers: four workgroups a CU for
// seven, and 50 us for 41 on 2000 x 32000 bf16, k = 5; 29 for 25 on 1000.)
template <int THREADS>
struct TopList {
  u32x4 piece[kTopPieces];
  unsigned long long list[kTopList];
  int column[kTopPieces];
  float pm[THREADS / 64][kTopParts];
  float bound;
  int pieces, count;
};

// the k-th largest of the lanes' maxima over the workgroup's waves
template <int THREADS>
__device__ float top_bound(TopList<THREADS>& s, int k, float mine) {
  const int l = threadIdx.x & 63;
  __syncthreads();  // (the last use of pm and the counts)
  s.pm[threadIdx.x >> 6][l] = mine;
  if (threadIdx.x == 0) s.pieces = s.count = 0;
  __syncthreads();
  if (threadIdx.x < 64) {  // (one wave: sixteen at once would share the SIMDs for the same answer)
    float v = s.pm[0][l];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) v = fmaxf(v, s.pm[w][l]);
    int before = 0;
#pragma unroll
    for (int i = 0; i < kTopParts; ++i) {
      const float u = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), i));
      before += u > v || (u == v && i < l);
    }
    if (before == k - 1) s.bound = v;  // one lane: the ranks are distinct
  }
  __syncthreads();
  return s.bound;
}

template <typename T, int THREADS>
__device__ __forceinline__ void list_piece(TopList<THREADS>& s, const typename Piece<T>::vec& v, int c) {
  const int at = atomicAdd(&s.pieces, 1);
  if (at < kTopPieces) {
    s.piece[at] = __builtin_bit_cast(u32x4, v);
    s.column[at] = c;
  }
}

// The k first of the row in rank order, into out / ids.  The pieces listed hold every logit that reaches some bound below
// the k-th largest, unless they overflowed; most: the maximum of this thread's logits; m, logz: the row's.
template <typename T, int THREADS>
__device__ void top_of_row(TopList<THREADS>& s, const T* row, int V, int k, float most, float m, float logz, float* out,
                           int64_t* ids) {
  constexpr int N = Piece<T>::N, W = THREADS / 64;
  const int tid = threadIdx.x;
  const bool bad = logz != logz;  // (a NaN is listed by no comparison)
  __syncthreads();
  int n = s.pieces;
  if (n > kTopPieces && !bad) {
    const float bound = top_bound<THREADS>(s, k, most);
    over_row(row, V, tid, THREADS, [&](int c, const typename Piece<T>::vec& v) {
      bool reach = false;
#pragma unroll
      for (int i = 0; i < N; ++i) reach |= c + i < V && (float)v[i] >= bound;
      if (reach) list_piece<T, THREADS>(s, v, c);
    });
    __syncthreads();
    n = s.pieces;
  }
  if (n <= kTopPieces && !bad) {
    const float bound = s.bound;
    for (int a = tid; a < n * N; a += THREADS) {
      const int c = s.column[a / N] + a % N;
      const float x = (float)((const T*)s.piece)[a];
      if (c < V && x >= bound) {
        const int at = atomicAdd(&s.count, 1);
        if (at < kTopList) s.list[at] = rank_key(x, c);
      }
    }
    __syncthreads();
    n = s.count;
    if (n <= kTopList) {
      for (int a = tid; a < n; a += THREADS) {
        const unsigned long long mine = s.list[a];
        int before = 0;
#pragma unroll 4
        for (int i = 0; i < n; ++i) before += s.list[i] > mine;
        if (before < k) {
          out[before] = (key_value(mine) - m) - logz;
          ids[before] = key_index(mine);
        }
      }
      return;
    }
  }
  // the first of the row behind the last one found, k times
  unsigned long long last = ~0ull;
  for (int j = 0; j < k; ++j) {
    __syncthreads();
    unsigned long long best = 0;
    over_row(row, V, tid, THREADS, [&](int c, const typename Piece<T>::vec& v) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const unsigned long long key = c + i < V ? rank_key((float)v[i], c + i) : 0;
        if (key < last && key > best) best = key;
      }
    });
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned long long other = __shfl_xor(best, o);
      best = other > best ? other : best;
    }
    if ((tid & 63) == 0) s.list[tid >> 6] = best;
    __syncthreads();
    for (int i = 0; i < W; ++i) best = s.list[i] > best ? s.list[i] : best;
    last = best;
    if (tid == 0) {
      out[j] = (key_value(best) - m) - logz;
      ids[j] = key_index(best);
    }
  }
}

// grid: (rows up to kRowsX, whole kRowsX of rows), since a launch's work items in x stay within 32 bits
constexpr long kRowsX = 1L << 20;
// waves a SIMD that the registers are held to (left to itself the compiler takes LDS for the bound and 121 registers)
template <typename T, int THREADS>
constexpr int kFwdWaves = THREADS == 1024 || sizeof(T) == 4 ? 8 : 6;
template <typename T, int THREADS, bool TOP>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(kFwdWaves<T, THREADS>)))
void logprob_fwd_kernel(const LogprobArgs a) {
  constexpr int N = Piece<T>::N, W = THREADS / 64;
  __shared__ Part parts[W];
  __shared__ TopList<TOP ? THREADS : 64> top;
  const int tid = threadIdx.x, V = a.V;
  const long r = (long)blockIdx.y * kRowsX + blockIdx.x;
  if (r >= a.rows) return;
  const int64_t id = a.ids[r];
  if (id == a.ignore) {
    if (tid == 0) a.logp[r] = a.ent[r] = 0.f;
    if (TOP && tid < a.k) {
      a.top[r * a.k + tid] = 0.f;
      a.top_ids[r * a.k + tid] = -1;
    }
    return;
  }
  const T* row = (const T*)a.x + r * a.ldx;
  Part p{-INFINITY, 0.f, 0.f};
  float bound = NAN;  // (reached by nothing, +inf neither: the list begins with the first bound)
  constexpr int step = THREADS * N;
  constexpr bool kNext = THREADS < 1024;  // the next pieces on their way too (sixteen waves have the registers for one set)
  typename Piece<T>::vec x[kAhead], y[kAhead];
  auto fetch = [&](typename Piece<T>::vec(&v)[kAhead], int c) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (c + j * step < V) v[j] = load_piece(row, c + j * step, V);
  };
  fetch(x, tid * N);
  // a token outside the vocabulary has no log probability
  const float given = tid == 0 && id >= 0 && id < V ? (float)*gmem(row + id) : NAN;
  for (int c0 = 0; c0 < V; c0 += kAhead * step) {  // (the same rounds for every thread)
    const int c = c0 + tid * N;
    if (kNext) fetch(y, c + kAhead * step);
    float first[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) first[j] = NAN;  // (reaches no bound)
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int at = c + j * step;
      if (at >= V) break;
      float v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (float)x[j][i];
      if (at + N > V)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = at + i < V ? v[i] : -INFINITY;
      const float most = add_values<N>(p, v);
      if constexpr (TOP) {
        first[j] = most;
        if (most >= bound) list_piece<T, THREADS>(top, x[j], at);
      }
    }
    if constexpr (TOP) {
      if (c0 == 0) {
        bound = top_bound<THREADS>(top, a.k, p.m);
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
          if (first[j] >= bound) list_piece<T, THREADS>(top, x[j], c + j * step);
      }
    }
    if (!kNext) fetch(x, c + kAhead * step);
    else
#pragma unroll
      for (int j = 0; j < kAhead; ++j) x[j] = y[j];
  }
  const float mine = p.m;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) p = merge(p, Part{__shfl_xor(p.m, o), __shfl_xor(p.s, o), __shfl_xor(p.t, o)});
  if ((tid & 63) == 0) parts[tid >> 6] = p;
  __syncthreads();
  p = parts[tid & (W - 1)];
#pragma unroll
  for (int o = 1; o < W; o <<= 1) p = merge(p, Part{__shfl_xor(p.m, o), __shfl_xor(p.s, o), __shfl_xor(p.t, o)});
  const float logz = logf(p.s);
  if (tid == 0) {
    a.logp[r] = (given - p.m) - logz;
    a.ent[r] = logz - p.t / p.s;
    if (a.stats) {
      a.stats[2 * r] = p.m;
      a.stats[2 * r + 1] = logz;
    }
  }
  if constexpr (TOP)
    top_of_row<T, THREADS>(top, row, V, a.k, mine, p.m, logz, a.top + r * a.k, a.top_ids + r * a.k);
}

// grid: (parts of a row, rows).  The rows from the last one on, whose logits the forward left in the last-level cache, and
// neither these nor the gradients put there again: 16384 x 32000 bf16 forward and backward 566 -> 537 us, 4096 rows
// 160 -> 137 (the products that read the gradients next take what they took).
constexpr int kBwdPieces = 8;  // 16-byte pieces a thread, all in flight together
template <typename T>
__global__ __launch_bounds__(kThreads) void logprob_bwd_kernel(const LogprobArgs a) {
  constexpr int N = Piece<T>::N;
  typedef typename Piece<T>::vec vec;
  const int V = a.V;
  const long r = a.rows - 1 - (long)blockIdx.y - (long)blockIdx.z * 32768;
  if (r < 0) return;
  const int64_t id = a.ids[r];
  T* out = (T*)a.dx + r * V;
  const int c0 = (blockIdx.x * kBwdPieces * kThreads + threadIdx.x) * N;
  constexpr int step = kThreads * N;
  if (id == a.ignore) {
    for (int j = 0; j < kBwdPieces; ++j)
      if (c0 + j * step < V) store_piece(out, c0 + j * step, V, vec{});
    return;
  }
  const T* row = (const T*)a.x + r * a.ldx;
  vec x[kBwdPieces];
#pragma unroll
  for (int j = 0; j < kBwdPieces; ++j)
    if (c0 + j * step < V) x[j] = load_last(row, c0 + j * step, V);
  const float m = a.stats[2 * r], logz = a.stats[2 * r + 1], dent = a.dent ? a.dent[r] : 0.f;
  float dlogp = a.dlogp ? a.dlogp[r] : 0.f;
  // such a row has no gradient either (log Z is NaN beside a NaN or +inf, -inf where nothing but -inf is)
  if (id < 0 || id >= V || !(logz > -INFINITY)) dlogp = NAN;
  const float c = -(dlogp + dent * (dent != 0.f ? a.ent[r] : 0.f));
#pragma unroll
  for (int j = 0; j < kBwdPieces; ++j) {
    const int at = c0 + j * step;
    if (at >= V) break;
    float g[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float v = fmaxf(((float)x[j][i] - m) - logz, kFar);
      g[i] = exp2_(v * kLog2e) * (c - dent * v);
    }
    if (id >= at && id < at + N)
#pragma unroll
      for (int i = 0; i < N; ++i) g[i] += id == at + i ? dlogp : 0.f;
    vec o;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = (T)g[i];
    store_past(out, at, V, o);
  }
}

// Fewer than two rows a CU: sixteen waves to a row, otherwise four (32000 bf16, k = 5: 16 rows 8.9 us by sixteen and 12.3
// by four, 256 rows 11.5 and 14.2, 512 16.3 and 17.1, 1000 28 and 25, 2000 50 and 40; without alternatives 16 rows 6.2
// and 7.7, 512 12.5 and 12.0, 2000 36 and 34).
constexpr long kFewRows = 512;
template <typename T>
void launch_typed(bool bwd, const LogprobArgs& a, hipStream_t st) {
  if (bwd) {
    const int per = kBwdPieces * kThreads * Piece<T>::N;
    const dim3 grid((unsigned)((a.V + per - 1) / per), (unsigned)std::min<long>(a.rows, 32768),
                    (unsigned)((a.rows + 32767) / 32768));
    hipLaunchKernelGGL(logprob_bwd_kernel<T>, grid, dim3(kThreads), 0, st, a);
  } else if (a.rows < kFewRows) {
    if (a.k) hipLaunchKernelGGL((logprob_fwd_kernel<T, 1024, true>), dim3((unsigned)a.rows), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((logprob_fwd_kernel<T, 1024, false>), dim3((unsigned)a.rows), dim3(1024), 0, st, a);
  } else {
    const dim3 grid((unsigned)std::min(a.rows, kRowsX), (unsigned)((a.rows + kRowsX - 1) / kRowsX));
    if (a.k) hipLaunchKernelGGL((logprob_fwd_kernel<T, 256, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((logprob_fwd_kernel<T, 256, false>), grid, dim3(256), 0, st, a);
  }
}

}  // namespace

hipError_t launch_logprobs(bool bwd, const LogprobArgs& a, hipStream_t st) {
  if (a.rows <= 0) return hipSuccess;
  if (a.dtype == kBf16) launch_typed<bf16>(bwd, a, st);
  else if (a.dtype == kF16) launch_typed<f16>(bwd, a, st);
  else launch_typed<float>(bwd, a, st);
  return hipGetLastError();
}

}  // namespace ccq
