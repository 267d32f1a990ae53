// Norms of the heads of q and k and their rotary positions, in one pass (gfx950). The mathematics is
// lsa_turn_dev.h's, and so is a workgroup's work (rotate_rows).
//
// Memory bounds it: every row is read and written once, and some 60 instructions a lane of 8 elements hide behind
// that. A workgroup takes 4 tokens, a wave each, or, where there are few tokens, one token and a part of its heads.
// 32768 bf16 tokens of 40 heads of 128 (671 MB): 120 us, 5.6 TB/s (a large copy: 5.1). It took 152 with the norms'
// weights in registers (4 waves a SIMD for 5) and 138 with stores that stay in the caches: outputs of more than
// 64 MB, twice the caches' 32, go past them. One token: 3.4 us on the device.
#include <math.h>

#include <algorithm>

#include "lsa_abi_common.h"
#include "lsa_turn_dev.h"

using namespace lsa;

namespace {

template <typename T, int D, int TOKENS, bool STREAM>
__global__ __launch_bounds__(LSA_BLOCK) void rotate_kernel(RotateArgs a) {
  __shared__ RotateLds<D, TOKENS> sh;
  rotate_rows<T, D, TOKENS, STREAM>(a, blockIdx.x, blockIdx.y, sh);
}

template <typename T, int D>
void launch_rotate_of(RotateArgs a, hipStream_t s) {
  const int heads = a.Hq + a.Hkv;
  constexpr int SLOTS = HeadLanes<D>::SLOTS;
  if (a.tokens >= 1024) {  // a workgroup a CU and more
    a.heads = heads;
    const dim3 grid((a.tokens + 3) / 4);
    if ((int64_t)a.tokens * heads * D * sizeof(T) > (64 << 20)) rotate_kernel<T, D, 4, true><<<grid, LSA_BLOCK, 0, s>>>(a);
    else rotate_kernel<T, D, 4, false><<<grid, LSA_BLOCK, 0, s>>>(a);
    return;
  }
  // one token a workgroup; its heads over several while that leaves CUs idle
  const int most = (heads + SLOTS - 1) / SLOTS;
  const int parts = std::max(1, std::min(most, 512 / a.tokens));
  a.heads = ((heads + parts - 1) / parts + SLOTS - 1) / SLOTS * SLOTS;
  rotate_kernel<T, D, 1, false><<<dim3(a.tokens, (heads + a.heads - 1) / a.heads), LSA_BLOCK, 0, s>>>(a);
}

void launch_rotate(const RotateArgs& a, int dtype, int D, hipStream_t s) {
  LSA_DISPATCH_QT(dtype, {
    switch (D) {
      case 32: launch_rotate_of<QT, 32>(a, s); break;
      case 64: launch_rotate_of<QT, 64>(a, s); break;
      case 128: launch_rotate_of<QT, 128>(a, s); break;
      default: launch_rotate_of<QT, 256>(a, s); break;
    }
  });
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
  LSA_REQUIRE(B == 0 || T <= 4 * kMaxGroups / B, LSA_ERR_SHAPE, "lsa_rotate: 2^26 tokens or more");
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
  launch_rotate(a, dtype, D, (hipStream_t)stream);
  LSA_LAUNCHED("lsa_rotate");
  return LSA_OK;
}
