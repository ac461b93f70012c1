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
// The alternatives: pass one also leaves the maximum of each of 64 parts of the row; the k-th largest of those
// (k <= 64) is a lower bound of the k-th largest logit, and few logits reach it (about 24 for k = 20).  Pass two
// reads the row again (it lies in the L2) and lists those, and every listed logit counts those before it.  A
// row with more than kTopList of them (equal logits) is ranked by k passes over it.
#include <algorithm>

#include "ccq_block_args.h"
#include "ccq_rows.h"

namespace ccq {

namespace {

constexpr int kTopParts = 64;    // parts of a row, so the largest k
constexpr int kTopList = 1024;   // listed candidates
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFar = -1e4f;    // e^(x - m) is 0 long before: stands for -inf in the products with it

// Running maximum m of a part of a row, s = sum e^(x - m), t = sum e^(x - m) (x - m).
struct Part {
  float m, s, t;
};
// NaN enters s alone (comparisons and maxima pass it over), and makes every result of the row NaN.
__device__ __forceinline__ Part merge(const Part& a, const Part& b) {
  const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
  const float da = fmaxf(a.m - ref, kFar), db = fmaxf(b.m - ref, kFar);
  const float ca = exp2f(da * kLog2e), cb = exp2f(db * kLog2e);
  return {m, ca * a.s + cb * b.s, ca * (a.t + a.s * da) + cb * (b.t + b.s * db)};
}

template <int N>
__device__ __forceinline__ void add_values(Part& p, const float (&v)[N]) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
  if (m > p.m) {
    if (p.m != -INFINITY) {
      const float d = fmaxf(p.m - m, kFar), c = exp2f(d * kLog2e);
      p.t = c * (p.t + p.s * d);
      p.s *= c;
    }
    p.m = m;
  }
  const float ref = p.m == -INFINITY ? 0.f : p.m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = v[i] - ref, e = exp2f(d * kLog2e);
    p.s += e;
    p.t += e * fmaxf(d, kFar);
  }
}

// Order of the alternatives: NaN before any number, the larger logit first, the lower index first.
__device__ __forceinline__ unsigned long long rank_key(float x, int i) {
  const int b = __float_as_int(x + 0.f);  // (-0 as +0)
  unsigned u = b < 0 ? ~(unsigned)b : (unsigned)b | 0x80000000u;
  if (x != x) u = 0xffffffffu;
  return (unsigned long long)u << 32 | (unsigned)~i;
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)~(unsigned)k; }

template <typename T, typename F>
__device__ __forceinline__ void over_row(const T* row, int V, int tid, int threads, F&& f) {
  constexpr int N = Piece<T>::N;
  for (int c = tid * N; c < V; c += threads * N) f(c, load_piece(row, c, V));
}

// The k first of the row in rank order, into out / ids.  part: the maximum of this thread's logits; m, logz: the row's.
template <typename T, int THREADS>
__device__ void top_of_row(const T* row, int V, int k, float part, float m, float logz, float* out, int64_t* ids) {
  constexpr int N = Piece<T>::N, W = THREADS / 64;
  __shared__ unsigned long long list[kTopList];
  __shared__ float pm[kTopParts];
  __shared__ int count;
  const int tid = threadIdx.x;
  constexpr int G = THREADS / kTopParts;  // threads of a part
#pragma unroll
  for (int o = 1; o < G; o <<= 1) part = fmaxf(part, __shfl_xor(part, o));
  if (tid % G == 0) pm[tid / G] = part;
  if (tid == 0) count = 0;
  __syncthreads();
  float bound = -INFINITY;
  {
    const int l = tid & 63;
    const float v = pm[l];
    int before = 0;
    for (int i = 0; i < kTopParts; ++i) {
      const float u = pm[i];
      before += u > v || (u == v && i < l);
    }
    const unsigned long long hit = __ballot(before == k - 1);  // one lane: the ranks are distinct
    bound = __shfl(v, __ffsll(hit) - 1);
  }
  over_row(row, V, tid, THREADS, [&](int c, const typename Piece<T>::vec& v) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < V && !((float)v[i] < bound)) {
        const int at = atomicAdd(&count, 1);
        if (at < kTopList) list[at] = rank_key((float)v[i], c + i);
      }
  });
  __syncthreads();
  const int n = count;
  if (n <= kTopList) {
    for (int a = tid; a < n; a += THREADS) {
      const unsigned long long mine = list[a];
      int before = 0;
      for (int i = 0; i < n; ++i) before += list[i] > mine;
      if (before < k) {
        const int id = key_index(mine);
        out[before] = ((float)row[id] - m) - logz;
        ids[before] = id;
      }
    }
    __syncthreads();
    return;
  }
  // more candidates than the list holds: the first of the row behind the last one found, k times
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
    if ((tid & 63) == 0) list[tid >> 6] = best;
    __syncthreads();
    for (int i = 0; i < W; ++i) best = list[i] > best ? list[i] : best;
    last = best;
    if (tid == 0) {
      const int id = key_index(best);
      out[j] = ((float)row[id] - m) - logz;
      ids[j] = id;
    }
  }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void logprob_fwd_kernel(const LogprobArgs a) {
  constexpr int N = Piece<T>::N, W = THREADS / 64;
  __shared__ Part parts[W];
  const int tid = threadIdx.x, V = a.V;
  const long r = blockIdx.x;
  const int64_t id = a.ids[r];
  if (id == a.ignore) {
    if (tid == 0) {
      a.logp[r] = a.ent[r] = 0.f;
    }
    if (tid < a.k) {
      a.top[r * a.k + tid] = 0.f;
      a.top_ids[r * a.k + tid] = -1;
    }
    return;
  }
  const T* row = (const T*)a.x + r * a.ldx;
  Part p{-INFINITY, 0.f, 0.f};
  over_row(row, V, tid, THREADS, [&](int c, const typename Piece<T>::vec& x) {
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = c + i < V ? (float)x[i] : -INFINITY;
    add_values<N>(p, v);
  });
  const float mine = p.m;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) p = merge(p, Part{__shfl_xor(p.m, o), __shfl_xor(p.s, o), __shfl_xor(p.t, o)});
  if ((tid & 63) == 0) parts[tid >> 6] = p;
  __syncthreads();
  p = parts[0];
#pragma unroll
  for (int i = 1; i < W; ++i) p = merge(p, parts[i]);
  const float logz = logf(p.s);
  if (tid == 0) {
    // a token outside the vocabulary has no log probability
    a.logp[r] = id >= 0 && id < V ? ((float)row[id] - p.m) - logz : NAN;
    a.ent[r] = logz - p.t / p.s;
    if (a.stats) {
      a.stats[2 * r] = p.m;
      a.stats[2 * r + 1] = logz;
    }
  }
  if (a.k) top_of_row<T, THREADS>(row, V, a.k, mine, p.m, logz, a.top + r * a.k, a.top_ids + r * a.k);
}

// grid: (parts of a row, rows)
constexpr int kBwdPieces = 8;  // 16-byte pieces a thread, all in flight together
template <typename T>
__global__ __launch_bounds__(kThreads) void logprob_bwd_kernel(const LogprobArgs a) {
  constexpr int N = Piece<T>::N;
  typedef typename Piece<T>::vec vec;
  const int V = a.V;
  const long r = (long)blockIdx.y + (long)blockIdx.z * 32768;
  if (r >= a.rows) return;
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
    if (c0 + j * step < V) x[j] = load_piece(row, c0 + j * step, V);
  const float m = a.stats[2 * r], logz = a.stats[2 * r + 1], dent = a.dent ? a.dent[r] : 0.f;
  float dlogp = a.dlogp ? a.dlogp[r] : 0.f;
  if (id < 0 || id >= V || logz != logz) dlogp = NAN;  // such a row has no gradient either
  const float c = -(dlogp + dent * (dent != 0.f ? a.ent[r] : 0.f));
#pragma unroll
  for (int j = 0; j < kBwdPieces; ++j) {
    const int at = c0 + j * step;
    if (at >= V) break;
    float g[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float v = fmaxf(((float)x[j][i] - m) - logz, kFar);
      g[i] = exp2f(v * kLog2e) * (c - dent * v);
    }
    if (id >= at && id < at + N)
#pragma unroll
      for (int i = 0; i < N; ++i) g[i] += id == at + i ? dlogp : 0.f;
    vec o;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = (T)g[i];
    store_piece(out, at, V, o);
  }
}

template <typename T>
void launch_typed(bool bwd, const LogprobArgs& a, hipStream_t st) {
  if (bwd) {
    const int per = kBwdPieces * kThreads * Piece<T>::N;
    const dim3 grid((unsigned)((a.V + per - 1) / per), (unsigned)std::min<long>(a.rows, 32768),
                    (unsigned)((a.rows + 32767) / 32768));
    hipLaunchKernelGGL(logprob_bwd_kernel<T>, grid, dim3(kThreads), 0, st, a);
  } else if (a.rows < 512) {
    hipLaunchKernelGGL((logprob_fwd_kernel<T, 1024>), dim3((unsigned)a.rows), dim3(1024), 0, st, a);
  } else {
    hipLaunchKernelGGL((logprob_fwd_kernel<T, 256>), dim3((unsigned)a.rows), dim3(256), 0, st, a);
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
