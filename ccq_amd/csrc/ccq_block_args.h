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

// Activations of the linear map as the C ABI numbers them (CCQ_ACT_*).
enum : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4, kActSwiglu = 5 };

// Tiles of a product's launch: workgroups of 256 whose work items in x stay within 32 bits.
constexpr long kMaxTiles = 1L << 24;

// One product out[M, N] = A B^T over K, its operands stored with the contraction running along the rows
// (A [M, K], B [N, K]) or down them (A [K, M], B [K, N]), and what is done with the result.
struct ProductArgs {
  const void* a;       // row stride lda elements, rows 16-byte aligned
  const void* b;       // row stride ldb
  long lda, ldb;
  long M, N, K;        // (swiglu: N outputs of 2 N rows of B)
  void* out;           // [M, ldo]
  long ldo;
  const void* bias;    // [N] (swiglu: [2 N]) of bdtype (nullable)
  const void* res;     // [M, N] row stride ldr (nullable)
  void* z;             // [M, ldz] the values before the activation, 16 bits, then 8 (nullable)
  long ldr, ldz;
  float* part;         // [splits, M, N (swiglu: 2 N)] partial sums (splits > 1)
  int splits;          // parts of the contraction, whole steps each
  int act, bdtype, dtype;
};

struct ActBwdArgs {
  const void* z;       // [M, ldz] 16 bits, then 8 (nullable: no activation)
  const void* dy;      // [M, N] row stride ldy
  void* dz;            // [M, ldz], zeros behind the Nz columns (nullable: only db is wanted)
  float* db_part;      // [row blocks, Nz] (nullable)
  void* db;            // [Nz] of bdtype
  long M, N, ldz, ldy;
  int act, bdtype, dtype, row_blocks, lanes;
};

struct PadRowsArgs {
  const void* src;     // [rows, K] row stride ld
  void* dst;           // [rows, ldd], zeros behind the K columns
  long rows, K, ld, ldd;
};

}  // namespace ccq
