// What the shared-prefix read's kernels have in common: their arguments, and how a prefix is cut
// into pieces.
#pragma once

#include "lsa_read_dev.h"

namespace lsa {

constexpr int kPieceTile = 64;  // keys; a piece is a multiple of it
constexpr int kMaxPieces = 128;
constexpr int kMaxOwn = 64;

struct PrefixArgs {
  const void* q;
  const void* kp;
  const void* vp;
  const int32_t* prefix_rows;     // [B] or nullptr: the only prefix, or prefix b of B
  const int32_t* prefix_lengths;  // [P] or nullptr: Tp
  const int32_t* slots;           // [P, Tp] cache rows of a pool, or nullptr
  int64_t slot_stride, pool;      // rows the prefix cache holds a batch entry
  int64_t p_sb, p_st, p_sh;
  const void* k;
  const void* v;
  int64_t kv_sb, kv_st, kv_sh, Tk;
  const int32_t* ids;
  const int32_t* lengths;
  int W, per_head;
  int64_t B, Tq, Tp;
  int P, Hq, Hkv;
  float scale_log2;
  int splits;      // pieces of a prefix at most (how many parts a unit has room for)
  int* plan;       // pieces of a prefix at most for the rows' own spread over prefixes, or nullptr: splits (at
                   // most 1024 prefixes)
  int own_splits;  // spans of an own list at most
  int own_span;    // list slots of a span
  int* counters;   // [units]: cleared by the prefix kernel, arrivals of the own spans
  float* parts;    // [units][splits + own_splits][GQ (D + 2)]
  float* sums;     // [units][splits][GQ]: the pieces' sums for lse (where lse is wanted)
  void* out;
  float* lse;      // [B, Tq, Hq] or nullptr
};

struct Pieces {
  int n;      // keys
  int count;  // pieces with keys in them
  int keys;   // of a piece
};

__device__ __forceinline__ Pieces prefix_pieces(const PrefixArgs& a, int p, int splits) {
  Pieces x{0, 0, kPieceTile};
  if (p < 0 || p >= a.P) return x;  // no prefix
  const int64_t n = a.prefix_lengths ? (int64_t)a.prefix_lengths[p] : a.Tp;
  x.n = (int)(n < 0 ? 0 : (n > a.Tp ? a.Tp : n));
  const int tiles = (x.n + kPieceTile - 1) / kPieceTile;
  const int per = (tiles + splits - 1) / splits;
  x.keys = (per > 0 ? per : 1) * kPieceTile;
  x.count = (x.n + x.keys - 1) / x.keys;
  return x;
}
__device__ __forceinline__ int prefix_of(const PrefixArgs& a, int64_t b) {
  return a.prefix_rows ? a.prefix_rows[b] : (a.P > 1 ? (int)b : 0);
}

// On the matrix cores a workgroup has a CU to itself: as many pieces as make one workgroup a CU, given the
// column blocks of all prefixes.
__host__ __device__ __forceinline__ int prefix_mfma_pieces(int64_t blocks, int Hkv) {
  const int64_t n = blocks * Hkv;
  return n > 256 ? 1 : 256 / (n > 0 ? (int)n : 1);
}

// Partials of the prefixes from the matrix cores (16-bit rows, head dim 64 or 128); clears the
// counters too, and writes *plan. `columns`: query columns a prefix on average. False, and nothing
// launched, where the sizes do not fit.
bool prefix_mfma_ok(int dtype, int D);
int64_t prefix_mfma_columns(int64_t columns);  // of a workgroup
bool launch_prefix_mfma(const PrefixArgs& a, int dtype, int D, int64_t columns, hipStream_t s);

}  // namespace lsa
