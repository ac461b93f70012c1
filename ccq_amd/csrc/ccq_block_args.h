// Arguments of the kernels around the token mixers: block norms (ccq_norm.hip), log probabilities of given
// tokens (ccq_logprobs.hip), projections with an epilogue (ccq_linear.hip).
#pragma once

#include <stdint.h>

namespace ccq {

// Element types as the C ABI numbers them (CCQ_DTYPE_*).
enum : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

struct NormArgs {
  const void* x;       // [rows, D], row stride ldx (backward: the normalised stream)
  const void* r;       // forward: residual added to x (nullable), row stride ldr
  const void* w;       // [D] of wdtype (nullable: ones)
  const void* b;       // [D] of wdtype (nullable: none)
  void* y;             // forward: [rows, D]
  void* s;             // forward: x + r (with r)
  float* mean;         // [rows] (layer norm; forward: nullable)
  float* rstd;         // [rows] (forward: nullable)
  const void* dy;      // backward: [rows, D], row stride ldy
  const void* ds;      // backward: gradient of the stream itself (nullable), row stride ldds
  void* dx;            // backward: [rows, D] (nullable)
  void* dw;            // backward: [D] of wdtype (nullable)
  void* db;            // backward: [D] of wdtype (nullable)
  float* dw_part;      // backward: [blocks, D] (with dw)
  float* db_part;      // backward: [blocks, D] (with db)
  long rows, ldx, ldr, ldy, ldds;
  int D, dtype, wdtype, layer;
  float eps;
};

struct LogprobArgs {
  const void* x;       // logits [rows, V], row stride ldx
  const int64_t* ids;  // [rows]; ignore: the row is skipped
  float* logp;         // [rows]
  float* ent;          // [rows] entropy (backward: as the forward left it)
  float* stats;        // [rows, 2] maximum m, log of sum e^(x - m) (forward: nullable; not of skipped rows)
  float* top;          // [rows, k] (nullable with k == 0)
  int64_t* top_ids;    // [rows, k]
  const float* dlogp;  // backward: [rows] (nullable)
  const float* dent;   // backward: [rows] (nullable)
  void* dx;            // backward: [rows, V]
  long rows, ldx, ignore;
  int V, k, dtype;
};

}  // namespace ccq
