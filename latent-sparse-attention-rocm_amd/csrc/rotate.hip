// Norms of the heads of q and k and their rotary positions, in one pass (gfx950). The mathematics is
// lsa_turn_dev.h's.
//
// Memory bounds it: every row is read and written once, and about 60 instructions an 8-element lane hide
// behind that. A workgroup takes 4 tokens, a wave each, or, where there are few tokens, one token and a part of
// its heads. Its threads take the sines of the tokens' pairs first, once for all heads, through LDS; each lane
// keeps those of its 8 dims in registers and walks the heads of its token, so a wave reads and writes
// consecutive heads of one token.
#include <math.h>

#include <algorithm>

#include "lsa_abi_common.h"
#include "lsa_turn_dev.h"

using namespace lsa;

namespace {

struct RotateArgs {
  const void* q;
  const void* k;
  void* q_out;  // [B, T, Hq, D]
  void* k_out;
  const void* pos;
  int pos64;
  int64_t pos_sb;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh;
  int Hq, Hkv;
  int T, tokens;   // tokens = B T
  int heads;       // of a workgroup
  TurnArgs turn;
};

template <typename T, int D, int TOKENS>
__global__ __launch_bounds__(LSA_BLOCK) void rotate_kernel(RotateArgs a) {
  using L = HeadLanes<D>;
  constexpr int ROWS = L::SLOTS / TOKENS;  // heads at a time
  constexpr int AHEAD = 4;                 // rows a lane loads before it works on them
  __shared__ __attribute__((aligned(16))) float stage[LSA_BLOCK * 8];
  __shared__ float2 angles[TOKENS][D / 2];
  const int tid = threadIdx.x, lp = tid % L::LPT, slot = tid / L::LPT;
  const int t0 = blockIdx.x * TOKENS;
  const int mine = t0 + slot / ROWS;
  const int token = mine < a.tokens ? mine : a.tokens - 1;
  const int b = token / a.T, t = token - b * a.T;
  const T* q = (const T*)a.q + b * a.q_sb + t * a.q_st + 8 * lp;
  const T* k = (const T*)a.k + b * a.k_sb + t * a.k_st + 8 * lp;
  T* qo = (T*)a.q_out + (int64_t)token * a.Hq * D + 8 * lp;
  T* ko = (T*)a.k_out + (int64_t)token * a.Hkv * D + 8 * lp;
  const int first = blockIdx.y * a.heads + slot % ROWS;
  const int end = mine < a.tokens ? min(a.Hq + a.Hkv, (int)(blockIdx.y + 1) * a.heads) : 0;

  Raw8<T> raw[AHEAD];
  auto fetch = [&](int h, Raw8<T>& r) {
    if (h < end) r.load(h < a.Hq ? q + h * a.q_sh : k + (h - a.Hq) * a.k_sh);
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) fetch(first + i * ROWS, raw[i]);
  for (int i = tid; i < TOKENS * a.turn.pairs; i += LSA_BLOCK) {
    const int n = i / a.turn.pairs, j = i - n * a.turn.pairs;
    const int at = min(t0 + n, a.tokens - 1);
    const int64_t p = (at / a.T) * a.pos_sb + at % a.T;
    angles[n][j] = turn_angle(a.turn, a.pos64 ? ((const int64_t*)a.pos)[p] : (int64_t)((const int32_t*)a.pos)[p], j);
  }
  float wq[8], wk[8];
  load_weights<T>(a.turn.qw, a.turn.w32, lp, wq);
  load_weights<T>(a.turn.kw, a.turn.w32, lp, wk);
  __syncthreads();
  LaneTurn turn;
  if (a.turn.pairs > 0) turn.load(a.turn, angles[slot / ROWS], lp);
  for (int h0 = first; h0 < end; h0 += AHEAD * ROWS) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int h = h0 + i * ROWS;
      if (h >= end) break;
      float y[8];
      raw[i].get(y);
      fetch(h + AHEAD * ROWS, raw[i]);
      const bool is_q = h < a.Hq;
      if (is_q ? a.turn.qw != nullptr : a.turn.kw != nullptr) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = is_q ? wq[e] : wk[e];
        norm8<D>(y, w, a.turn.eps);
      }
      if (a.turn.pairs > 0) turn8(a.turn, y, turn, stage + slot * D, lp);
      store8(is_q ? qo + (int64_t)h * D : ko + (int64_t)(h - a.Hq) * D, y);
    }
  }
}

template <typename T, int D>
void launch_rotate(RotateArgs a, hipStream_t s) {
  const int heads = a.Hq + a.Hkv;
  constexpr int SLOTS = HeadLanes<D>::SLOTS;
  if (a.tokens >= 1024) {  // a workgroup a CU and more
    a.heads = heads;
    rotate_kernel<T, D, 4><<<dim3((a.tokens + 3) / 4), LSA_BLOCK, 0, s>>>(a);
    return;
  }
  // one token a workgroup; its heads over several while that leaves CUs idle
  const int most = (heads + SLOTS - 1) / SLOTS;
  const int parts = std::max(1, std::min(most, 512 / a.tokens));
  a.heads = ((heads + parts - 1) / parts + SLOTS - 1) / SLOTS * SLOTS;
  rotate_kernel<T, D, 1><<<dim3(a.tokens, (heads + a.heads - 1) / a.heads), LSA_BLOCK, 0, s>>>(a);
}

}  // namespace

extern "C" int lsa_rotate(const void* q, const void* k, int dtype, int64_t B, int64_t T, int32_t Hq, int32_t Hkv,
                          int32_t D, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride,
                          int64_t k_batch_stride, int64_t k_token_stride, int64_t k_head_stride, const void* positions,
                          int positions_i64, int64_t position_stride, const lsa_turn* turn, void* q_out, void* k_out,
                          void* stream) {
  LSA_REQUIRE(q && q_out && turn && (Hkv == 0 || (k && k_out)), LSA_ERR_NULL, "lsa_rotate: NULL pointer");
  LSA_TRY(check_dtype(dtype));
  LSA_REQUIRE(B >= 0 && T >= 0 && Hq >= 1 && Hkv >= 0 && Hq <= 65536 && Hkv <= 65536, LSA_ERR_SHAPE,
              "lsa_rotate: B %lld T %lld Hq %d Hkv %d", (long long)B, (long long)T, Hq, Hkv);
  LSA_REQUIRE(B == 0 || T <= 0x3FFFFFFF / B, LSA_ERR_SHAPE, "lsa_rotate: more than 2^30 tokens");
  TurnArgs t;
  LSA_TRY(check_turn("lsa_rotate", turn, D, &t));
  LSA_REQUIRE(t.pairs == 0 || positions, LSA_ERR_NULL, "lsa_rotate: NULL positions");
  LSA_REQUIRE(position_stride >= 0, LSA_ERR_SHAPE, "lsa_rotate: position stride %lld", (long long)position_stride);
  const int64_t e = dtype == LSA_F32 ? 4 : 2;
  LSA_REQUIRE((((uintptr_t)q | (uintptr_t)q_out | (Hkv ? (uintptr_t)k | (uintptr_t)k_out : 0)) & 15) == 0 &&
                  ((q_batch_stride | q_token_stride | q_head_stride |
                    (Hkv ? k_batch_stride | k_token_stride | k_head_stride : 0)) * e) % 16 == 0,
              LSA_ERR_ALIGN, "lsa_rotate: rows of q and k must be 16-byte aligned");
  if (B * T == 0) return LSA_OK;
  RotateArgs a = {};
  a.q = q; a.k = Hkv ? k : q; a.q_out = q_out; a.k_out = Hkv ? k_out : q_out;
  a.pos = positions; a.pos64 = positions_i64 ? 1 : 0; a.pos_sb = position_stride;
  a.q_sb = q_batch_stride; a.q_st = q_token_stride; a.q_sh = q_head_stride;
  a.k_sb = k_batch_stride; a.k_st = k_token_stride; a.k_sh = k_head_stride;
  a.Hq = Hq; a.Hkv = Hkv; a.T = (int)T; a.tokens = (int)(B * T); a.turn = t;
  hipStream_t s = (hipStream_t)stream;
  LSA_DISPATCH_QT(dtype, {
    switch (D) {
      case 32: launch_rotate<QT, 32>(a, s); break;
      case 64: launch_rotate<QT, 64>(a, s); break;
      case 128: launch_rotate<QT, 128>(a, s); break;
      default: launch_rotate<QT, 256>(a, s); break;
    }
  });
  LSA_LAUNCHED("lsa_rotate");
  return LSA_OK;
}
