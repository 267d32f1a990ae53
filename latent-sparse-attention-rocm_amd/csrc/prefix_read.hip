// Attention of a batch over prefixes that its rows share, and over each row's own read list,
// for gfx950.
//
// The softmax over both parts is one: each part leaves partials (running maximum m, sum l and
// weighted value row, in fp32, log2 domain), and the usual rescaling joins them.
//
//   prefix_mfma_kernel,  (prefix_mfma.hip) a prefix's partials for up to 256 query columns at once,
//   prefix_wide_kernel   16-bit rows of head dim 64 or 128;
//   prefix_rows_kernel   row by row with the gather read's span loop: the pieces of a prefix (any type and
//                        head dim), a row's own list, and the join, by the last of a unit to finish.
//
// A prefix of n keys is cut into pieces of whole 64-key tiles, a workgroup a piece, the same for
// all of them (prefix_pieces). Partials of (row, kv-head) unit i: piece s of n_p at
// [i][splits - n_p + s], the own list's spans behind them, so the join finds them in a line.
#include <math.h>

#include <algorithm>

#include "lsa_abi_common.h"
#include "lsa_prefix_dev.h"

using namespace lsa;

namespace {

// grid (row * Hkv, span): spans [0, splits) are the pieces of the row's prefix, the rest its own list's.
enum Arrive { kNone, kOwn, kAll };  // whose arrival the join waits for (kNone: another launch joins)
template <typename T, int D, int GQ>
__global__ __launch_bounds__(LSA_BLOCK) void prefix_rows_kernel(PrefixArgs a, int first, int arrive) {
  __shared__ ReadLds<D, GQ, kMaxPieces + kMaxOwn> sh;
  constexpr int PSTRIDE = GQ * (D + 2);
  const int64_t i = blockIdx.x, row = i / a.Hkv;
  const int g = (int)(i % a.Hkv), s = (int)blockIdx.y + first;
  const int64_t b = row / a.Tq;
  if (arrive == kNone && s == 0 && threadIdx.x == 0) a.counters[i] = 0;
  const bool piece = s < a.splits;
  const int p = prefix_of(a, b);
  const int most = a.plan ? *a.plan : a.splits;
  int n = 0;
  const int32_t* ids = nullptr;  // the keys' rows (a prefix's own order without)
  if (a.W > 0 && !(arrive == kNone && piece)) {
    const int64_t li = a.per_head ? row * a.Hkv + g : row;
    n = a.lengths[li];
    n = (n < 0 || a.Tk <= 0) ? 0 : (n > a.W ? a.W : n);
    ids = a.ids + li * a.W;
  }
  const Pieces pc = prefix_pieces(a, p, most);
  const int n_own = (n + a.own_span - 1) / a.own_span, total = pc.count + n_own;
  const int at = piece ? s : s - a.splits;
  const bool active = at < (piece ? pc.count : n_own);
  float* own = a.parts + (i * (a.splits + a.own_splits) + a.splits) * (int64_t)PSTRIDE;
  if (!active) {  // a unit without spans to wait for still joins: its first workgroup
    if (arrive == kNone || blockIdx.y != 0 || (arrive == kAll ? total : n_own) > 0) return;
  } else {
    const int span = piece ? pc.keys : a.own_span;
    const int lo = at * span, hi = min(lo + span, piece ? pc.n : n);
    const int lp = (threadIdx.x & (LSA_WAVE - 1)) % ReadShape<T, D, GQ>::LPT;
    if (piece) ids = a.slots ? a.slots + p * a.slot_stride : nullptr;
    const int64_t off = (piece ? (a.slots ? 0 : p * a.p_sb) + g * a.p_sh : b * a.kv_sb + g * a.kv_sh) +
                        lp * ReadShape<T, D, GQ>::VEC;
    AttnState<T, D, GQ> st;
    attend_span<T, D, GQ, true>((const T*)a.q + (row * a.Hq + (int64_t)g * GQ) * D,
                                (const T*)(piece ? a.kp : a.k) + off, (const T*)(piece ? a.vp : a.v) + off,
                                piece ? a.p_st : a.kv_st, piece ? a.pool : a.Tk, lo, hi,
                                [&](int j) {
                                  const int jc = j < hi ? j : hi - 1;
                                  const int32_t id = ids ? ids[jc] : jc;
                                  return j < hi ? id : -1;
                                },
                                a.scale_log2, st);
    finish_span<T, D, GQ, kMaxPieces + kMaxOwn, true>(sh, st, false, (T*)nullptr,
                                                      own + (int64_t)(piece ? at - pc.count : at) * PSTRIDE, 0);
    if (arrive == kNone) return;
    // the partials complete before they are read back, by this workgroup or the last one
    if (!arrive_last(&a.counters[i], arrive == kAll ? total : n_own, &sh.flag)) return;
  }
  const float* parts = own - pc.count * PSTRIDE;
  T* outp = (T*)a.out + (row * a.Hq + (int64_t)g * GQ) * D;
  if (total == 0) {
    for (int j = threadIdx.x; j < GQ * D; j += LSA_BLOCK) store_out<T>(outp + j, 0.0f);
  } else {
    combine_partials<T, D, GQ>(sh, parts, total, outp, 0);
  }
  if (a.lse) {
    const int lane = threadIdx.x & (LSA_WAVE - 1);
    const float* sums = a.sums ? a.sums + (i * a.splits + a.splits - pc.count) * GQ : nullptr;
    for (int h = threadIdx.x / LSA_WAVE; h < GQ; h += LSA_WAVES) {
      float M = kNegBig, L = 0.0f;
      for (int x = lane; x < total; x += LSA_WAVE) M = fmaxf(M, coherent_load(parts + (int64_t)x * PSTRIDE + h));
      M = wave_max(M);
      for (int x = lane; x < total; x += LSA_WAVE) {
        const float* part = parts + (int64_t)x * PSTRIDE;
        L += (sums && x < pc.count ? sums[x * GQ + h] : coherent_load(part + GQ + h)) * fast_exp2(coherent_load(part + h) - M);
      }
      L = wave_sum(L);
      if (lane == 0) {
        // no keys, or a sum that is not a number, which counts as none
        a.lse[row * a.Hq + g * GQ + h] = L > 0.0f ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
      }
    }
  }
}

struct PrefixPlan {
  int splits, own_splits, own_span;
  size_t parts, sums, total;
};

// The query columns of a prefix if the rows are spread evenly over as many as they may read.
int64_t mean_columns(int64_t B, int64_t Tq, int64_t P, int32_t Hq, int32_t Hkv) {
  const int64_t n = std::max<int64_t>(1, std::min(B, P));
  return (B * Tq * (Hq / Hkv) + n - 1) / n;
}

// Pieces and own spans by size. On the matrix cores room for the pieces, of at least 256 keys, that a prefix is
// cut into if every row reads the same one (how the rows are spread is known on the device alone). The
// gather: about 512 workgroups. Own spans of at least 256 slots, as many as make 512 workgroups.
PrefixPlan prefix_plan(int dtype, int64_t B, int64_t Tq, int64_t P, int64_t Tp, int32_t Hq, int32_t Hkv, int32_t D, int32_t W) {
  PrefixPlan p;
  const int64_t units = B * Tq * Hkv;
  const int64_t tiles = (Tp + kPieceTile - 1) / kPieceTile;
  int64_t most = tiles, want_p = 512 / std::max<int64_t>(units, 1);
  if (prefix_mfma_ok(dtype, D)) {
    const int64_t wg = prefix_mfma_columns(mean_columns(B, Tq, P, Hq, Hkv));
    most = (tiles + 3) / 4;
    want_p = prefix_mfma_pieces((B * Tq * (Hq / Hkv) + wg - 1) / wg, Hkv);
  }
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({most, kMaxPieces, want_p}));
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(kMaxOwn, 512 / std::max<int64_t>(units, 1)));
  const int64_t per = std::max<int64_t>((W + want - 1) / want, 256);
  p.own_span = (int)((per + 63) / 64 * 64);
  p.own_splits = std::max(1, (W + p.own_span - 1) / p.own_span);
  const int64_t gq = Hq / Hkv;
  p.parts = (size_t)units * (p.splits + p.own_splits) * (size_t)(gq * (D + 2)) * sizeof(float);
  p.sums = (size_t)units * p.splits * gq * sizeof(float);
  p.total = p.parts + p.sums + (size_t)(units + 1) * sizeof(int);
  return p;
}

bool prefix_shape_ok(int dtype, int64_t B, int64_t Tq, int64_t P, int64_t Tp, int32_t Hq, int32_t Hkv, int32_t D,
                     int32_t W) {
  if (!(dtype == LSA_F32 || dtype == LSA_BF16 || dtype == LSA_F16)) return false;
  if (!(D == 32 || D == 64 || D == 128 || D == 256) || Hq < 1 || Hkv < 1 || Hq % Hkv) return false;
  const int gq = Hq / Hkv;
  if (!(gq == 1 || gq == 2 || gq == 4 || gq == 8)) return false;
  // a launch holds fewer than 2^32 threads along an axis
  return B >= 0 && Tq >= 0 && B <= 0x7FFFFFFF && Tq <= 0x7FFFFFFF && B * Tq <= 0x7FFFFFFF / Hq &&
         B * Tq * Hkv <= 0xFFFFFFFFll / LSA_BLOCK && P >= 1 && P <= 65535 && Tp >= 0 &&
         Tp <= 0x7FFFFFC0 && W >= 0 && W <= 0x7FFFFFC0;
}

template <typename T, int D>
void launch_prefix_gq(PrefixArgs a, int gq, int64_t units, int* counters, hipStream_t s) {
  const dim3 pieces((unsigned)units, (unsigned)a.splits), own((unsigned)units, (unsigned)a.own_splits);
  const dim3 all((unsigned)units, (unsigned)(a.splits + a.own_splits));
  const bool mfma = launch_prefix_mfma(a, __is_same(T, float) ? LSA_F32 : (__is_same(T, bf16_t) ? LSA_BF16 : LSA_F16), D,
                                       mean_columns(a.B, a.Tq, a.P, a.Hq, a.Hkv), s);
  if (!mfma) a.plan = nullptr;
  if (!mfma) a.sums = nullptr;  // row by row the weights are fp32: one sum serves both
  if (!mfma && counters) a.counters = counters;
#define LSA_PREFIX(GQ)                                                                        \
  if (mfma) {                                                                                 \
    prefix_rows_kernel<T, D, GQ><<<own, LSA_BLOCK, 0, s>>>(a, a.splits, kOwn);                \
  } else if (counters) {                                                                      \
    prefix_rows_kernel<T, D, GQ><<<all, LSA_BLOCK, 0, s>>>(a, 0, kAll);                       \
  } else {                                                                                    \
    prefix_rows_kernel<T, D, GQ><<<pieces, LSA_BLOCK, 0, s>>>(a, 0, kNone);                   \
    prefix_rows_kernel<T, D, GQ><<<own, LSA_BLOCK, 0, s>>>(a, a.splits, kOwn);                \
  }
  switch (gq) {
    case 1: LSA_PREFIX(1); break;
    case 2: LSA_PREFIX(2); break;
    case 4: LSA_PREFIX(4); break;
    default: LSA_PREFIX(8); break;
  }
#undef LSA_PREFIX
}

template <typename T>
void launch_prefix(const PrefixArgs& a, int D, int gq, int64_t units, int* counters, hipStream_t s) {
  switch (D) {
    case 32: launch_prefix_gq<T, 32>(a, gq, units, counters, s); break;
    case 64: launch_prefix_gq<T, 64>(a, gq, units, counters, s); break;
    case 128: launch_prefix_gq<T, 128>(a, gq, units, counters, s); break;
    default: launch_prefix_gq<T, 256>(a, gq, units, counters, s); break;
  }
}

}  // namespace

extern "C" size_t lsa_prefix_read_scratch_bytes(int dtype, int64_t B, int64_t Tq, int64_t P, int64_t Tp, int32_t Hq,
                                                int32_t Hkv, int32_t D, int32_t W) {
  if (!prefix_shape_ok(dtype, B, Tq, P, Tp, Hq, Hkv, D, W) || B * Tq == 0) return 0;
  return prefix_plan(dtype, B, Tq, P, Tp, Hq, Hkv, D, W).total;
}

extern "C" int lsa_prefix_read(const void* q, const void* k_prefix, const void* v_prefix, int dtype, int64_t B,
                               int64_t Tq, int64_t P, int64_t Tp, int64_t prefix_cache_rows, int32_t Hq, int32_t Hkv,
                               int32_t D, int64_t prefix_batch_stride, int64_t prefix_token_stride,
                               int64_t prefix_head_stride, const int32_t* prefix_rows, const int32_t* prefix_lengths,
                               const int32_t* prefix_slots, int64_t prefix_slot_stride, const void* k, const void* v,
                               int64_t Tk, int64_t kv_batch_stride, int64_t kv_token_stride, int64_t kv_head_stride,
                               const int32_t* ids, const int32_t* lengths, int32_t W, int ids_per_head, float scale,
                               int32_t* counters, void* scratch, size_t scratch_bytes, void* out, float* lse,
                               void* stream) {
  LSA_REQUIRE(q && out && (Tp == 0 || (k_prefix && v_prefix)), LSA_ERR_NULL, "lsa_prefix_read: NULL pointer");
  LSA_TRY(check_dtype(dtype));
  LSA_REQUIRE(prefix_shape_ok(dtype, B, Tq, P, Tp, Hq, Hkv, D, W), LSA_ERR_SHAPE,
              "lsa_prefix_read: B %lld Tq %lld P %lld Tp %lld Hq %d Hkv %d D %d W %d (D in {32,64,128,256}, groups of "
              "1/2/4/8, 1..65535 prefixes, rows x kv-heads under 2^24)", (long long)B, (long long)Tq, (long long)P, (long long)Tp, Hq, Hkv, D, W);
  LSA_REQUIRE(prefix_rows || P == 1 || P == B, LSA_ERR_NULL, "lsa_prefix_read: %lld prefixes for %lld rows need "
              "prefix_rows", (long long)P, (long long)B);
  LSA_REQUIRE(W == 0 || (k && v && ids && lengths && Tk >= 0 && Tk <= 0x7FFFFFFF), LSA_ERR_NULL,
              "lsa_prefix_read: own lists need K, V, ids and lengths");
  LSA_REQUIRE(prefix_cache_rows >= 0 && prefix_cache_rows <= 0x7FFFFFFF && (prefix_slots || prefix_cache_rows >= Tp),
              LSA_ERR_SHAPE, "lsa_prefix_read: a prefix cache of %lld rows for prefixes of %lld",
              (long long)prefix_cache_rows, (long long)Tp);
  LSA_REQUIRE(!prefix_slots || (prefix_slot_stride >= Tp && prefix_cache_rows >= 1), LSA_ERR_SHAPE,
              "lsa_prefix_read: slot rows of stride %lld for %lld positions", (long long)prefix_slot_stride, (long long)Tp);
  const int64_t e = dtype == LSA_F32 ? 4 : 2;
  const bool own = W > 0;
  LSA_REQUIRE(prefix_batch_stride >= 0 && prefix_token_stride >= D && prefix_head_stride >= D &&
                  (!own || (kv_batch_stride >= 0 && kv_token_stride >= D && kv_head_stride >= D)),
              LSA_ERR_SHAPE, "lsa_prefix_read: K/V strides must leave rows of %d elements apart", D);
  LSA_REQUIRE((((uintptr_t)q | (uintptr_t)k_prefix | (uintptr_t)v_prefix | (own ? (uintptr_t)k | (uintptr_t)v : 0)) & 15) == 0 &&
                  ((prefix_batch_stride | prefix_token_stride | prefix_head_stride |
                    (own ? kv_batch_stride | kv_token_stride | kv_head_stride : 0)) * e) % 16 == 0,
              LSA_ERR_ALIGN, "lsa_prefix_read: q and K/V rows must be 16-byte aligned");
  // the span loop multiplies a 32-bit row by a 32-bit stride
  LSA_REQUIRE(prefix_token_stride <= 0x7FFFFFFF && (!own || kv_token_stride <= 0x7FFFFFFF), LSA_ERR_SHAPE,
              "lsa_prefix_read: token strides past 2^31 elements");
  if (B * Tq == 0) return LSA_OK;
  const PrefixPlan p = prefix_plan(dtype, B, Tq, P, Tp, Hq, Hkv, D, W);
  LSA_REQUIRE(scratch && scratch_bytes >= p.total && ((uintptr_t)scratch & 15) == 0, LSA_ERR_WORKSPACE,
              "lsa_prefix_read: scratch missing, not 16-byte aligned or %zu < %zu bytes", scratch_bytes, p.total);
  PrefixArgs a = {};
  a.q = q; a.kp = k_prefix; a.vp = v_prefix; a.prefix_rows = prefix_rows; a.prefix_lengths = prefix_lengths;
  a.slots = prefix_slots; a.slot_stride = prefix_slot_stride; a.pool = prefix_slots ? prefix_cache_rows : Tp;
  a.p_sb = prefix_batch_stride; a.p_st = prefix_token_stride; a.p_sh = prefix_head_stride;
  a.k = k; a.v = v; a.kv_sb = kv_batch_stride; a.kv_st = kv_token_stride; a.kv_sh = kv_head_stride; a.Tk = Tk;
  a.ids = ids; a.lengths = lengths; a.W = W; a.per_head = ids_per_head ? 1 : 0;
  a.B = B; a.Tq = Tq; a.Tp = Tp; a.P = (int)P; a.Hq = Hq; a.Hkv = Hkv; a.scale_log2 = scale * kLog2e;
  a.splits = p.splits; a.own_splits = p.own_splits; a.own_span = p.own_span;
  a.parts = (float*)scratch;
  a.sums = (float*)((char*)scratch + p.parts);
  a.counters = (int*)((char*)scratch + p.parts + p.sums);
  a.out = out; a.lse = lse;
  hipStream_t s = (hipStream_t)stream;
  const int64_t units = B * Tq * Hkv;
  const int gq = Hq / Hkv;
  if (P > 1 && prefix_mfma_ok(dtype, D)) {
    const int64_t cols = mean_columns(B, Tq, P, Hq, Hkv), wg = prefix_mfma_columns(cols);
    const int spread = prefix_mfma_pieces(std::min(B, P) * ((cols + wg - 1) / wg), Hkv);  // rows spread evenly
    if (!prefix_rows) a.splits = std::min(p.splits, spread);  // a row each
    // by the rows' own spread, unless it cuts them alike however they are spread (the plan costs 0.9 us: 32 rows on
    // 8 prefixes of 2048 keys 20.5 us without and 21.4 with it)
    else if (spread < p.splits || P > 1024) a.plan = a.counters + units;
  }
  if (dtype == LSA_BF16) launch_prefix<bf16_t>(a, D, gq, units, counters, s);
  else if (dtype == LSA_F16) launch_prefix<_Float16>(a, D, gq, units, counters, s);
  else launch_prefix<float>(a, D, gq, units, counters, s);
  LSA_LAUNCHED("lsa_prefix_read");
  return LSA_OK;
}
