// A cache of 8-bit codes with a scale for each block of tokens and kv-head: writing to it and reading it back as
// numbers (gfx950). The rotation is lsa_turn_dev.h's.
//
// byte_append_kernel. A workgroup takes a tile of 64 positions (whole blocks) of one batch row and a part of the
// kv-heads, K and V of a head in turn: its lanes hold the tile's new tokens in registers (fp32, normed and rotated),
// the largest magnitude of each block meets in LDS (an integer maximum: its order changes nothing), one barrier,
// and every lane divides, rounds and stores. The block belongs to one workgroup, so its scale and the codes that
// were there before are read and rewritten with no atomics on memory. The sines of the tile's tokens are taken once
// for all heads of the workgroup. The rows of q, if any, go through workgroups of the same launch.
// 32768 bf16 tokens of 32 + 8 + 8 heads of 128 (738 MB): 151 us a call among others, 4.9 TB/s; K and V alone (201 MB)
// take 69: 513 workgroups, two a CU, each with 16 units (K or V of a head) one after the other and a barrier a unit.
// Five pieces of 300 tokens: 16 us (13 without q): a head a workgroup there, so that a tile's sines are taken eight
// times over, in front of two units. 32 decode tokens: 8 us, the launch and four round trips to memory (start, slot,
// the block's old scale, K and V beside them).
//
// byte_values_kernel copies: codes in, numbers out, 8 a lane. A whole cache of 32768 tokens (201 MB): 34 us, 5.9 TB/s.
#include <math.h>

#include <algorithm>

#include "lsa_abi_common.h"
#include "lsa_turn_dev.h"

using namespace lsa;

namespace {

constexpr int kTile = 64;
constexpr int kValueLanes = 512;  // 8-element lanes of a workgroup that reads back, about
constexpr int kPartHeads = 64;  // kv-heads of a workgroup at most
constexpr float kLeast = 7.888609052210118e-31f;  // 2^-100, the smallest scale: its reciprocal is finite

struct CacheArgs {
  uint8_t* k;
  uint8_t* v;
  float* scales;
  int block_shift;
  int64_t tokens, sb, st, sh;  // sb 0: one pool
  int64_t scale_sb;            // scale pairs of a cache, times kv-heads
};

enum QueryMode { kFew, kMany, kStream };

struct AppendArgs {
  CacheArgs c;
  const void* k;
  const void* v;
  int64_t k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  const int32_t* starts;
  const int32_t* lengths;
  SlotMap slots;
  int Hkv, T;
  int B, tiles;      // tiles of a row
  int parts, heads;  // workgroups of a tile, kv-heads of one
  int64_t kv_groups; // workgroups before the first of q's
  TurnArgs turn;
  RotateArgs q;      // rows of q, in workgroups behind the others:
  int q_mode;        // of a token (and a part of its heads), or of 4
  uint32_t q_parts;  // workgroups of a token
};

__device__ __forceinline__ int new_tokens(const AppendArgs& a, int b) {
  const int n = a.lengths ? a.lengths[b] : a.T;
  return n < 0 ? 0 : (n > a.T ? a.T : n);
}

template <int D>
struct alignas(16) AppendLds {
  float stage[LSA_BLOCK * 8 + 8];
  Angles<D> angles[kTile];
  uint32_t most[3][kTile];       // of a unit's blocks, as integers; three units take turns
  float before[2 * kPartHeads];  // the first block's scales, where it holds earlier tokens
  int32_t block_row[kTile];
};

template <typename T, int D, typename C>
__global__ __launch_bounds__(LSA_BLOCK) void byte_append_kernel(AppendArgs a) {
  using L = HeadLanes<D>;
  constexpr int STEPS = kTile / L::SLOTS;  // tokens of a lane
  __shared__ union {
    AppendLds<D> kv;
    RotateLds<D, 1> q;
    RotateLds<D, 4> q4;
  } sh;
  if ((int64_t)blockIdx.x >= a.kv_groups) {
    const uint32_t g = (uint32_t)(blockIdx.x - a.kv_groups), token = g / a.q_parts;
    if (a.q_mode == kStream) rotate_rows<T, D, 4, true>(a.q, g, 0, sh.q4);
    else if (a.q_mode == kMany) rotate_rows<T, D, 4, false>(a.q, g, 0, sh.q4);
    else rotate_rows<T, D, 1, false>(a.q, token, g - token * a.q_parts, sh.q);
    return;
  }
  const int tid = threadIdx.x;
  auto& most = sh.kv.most;
  auto& block_row = sh.kv.block_row;
  float* before = sh.kv.before;
  float* stage = sh.kv.stage;
  auto& angles = sh.kv.angles;
  if (tid < 8) stage[LSA_BLOCK * 8 + tid] = 0.0f;
  const int part = blockIdx.x % a.parts, tile = blockIdx.x / a.parts % a.tiles;
  const int b = blockIdx.x / a.parts / a.tiles;
  const SlotRow map = slot_row_of(a.slots, b);  // beside the start's load
  const int64_t start = a.starts[b];
  const int64_t end = min(start + new_tokens(a, b), a.slots.table ? (int64_t)map.width : a.c.tokens);  // what is past it is dropped
  const int64_t p0 = (start >= 0 ? start / kTile : 0) * kTile + (int64_t)tile * kTile;
  const int64_t from = start > p0 ? start : p0;  // the tile's new positions: [from, to)
  const int64_t to = end < p0 + kTile ? end : p0 + kTile;
  if (from >= to) return;
  const int shift = a.c.block_shift, block = 1 << shift;
  const int lo = (int)(from - p0), hi = (int)(to - p0);
  const int begin = lo >> shift << shift;  // the first written block's first token
  const int h0 = part * a.heads, h1 = min(h0 + a.heads, a.Hkv), units = 2 * (h1 - h0);
  const int lp = tid % L::LPT, slot = tid / L::LPT;
  const int first = slot * STEPS;  // a lane's tokens are consecutive
  const int64_t n0 = p0 - start;   // token of the tile's first position
  const T* k_row[STEPS];  // where a lane's tokens lie
  const T* v_row[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int x = first + i;
    const int64_t n = x >= lo && x < hi ? n0 + x : 0;
    k_row[i] = (const T*)a.k + b * a.k_sb + n * a.k_st + 8 * lp;
    v_row[i] = (const T*)a.v + b * a.v_sb + n * a.v_st + 8 * lp;
  }
  Raw8<T> raw[STEPS];
  auto fetch = [&](int u) {  // unit u: K (even) or V of a head
    const int64_t off = (h0 + (u >> 1)) * ((u & 1) ? a.v_sh : a.k_sh);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int x = first + i;
      if (u < units && x >= lo && x < hi) raw[i].load(((u & 1) ? v_row[i] : k_row[i]) + off);
      else raw[i].zero();
    }
  };
  fetch(0);
  float* scales = a.c.scales + (b * a.c.scale_sb) * 2;
  auto usable = [&](int64_t row) {  // a block's first slot, or -1
    return row < 0 || row >= a.c.tokens || (row & (block - 1)) ? -1 : (int32_t)row;
  };
  // a wave, a position a lane: a block is written to where its slots are a whole block of the pool (those behind the
  // new tokens may name no row yet)
  if (tid < kTile) {
    const int off = tid & (block - 1);
    const int64_t p = p0 + tid;
    int64_t row = p;
    bool whole = true;
    if (map.row) {
      const int32_t slot = p < map.width ? map.row[p] : -1;
      const int64_t first_slot = __shfl(slot, tid - off);
      row = slot;
      whole = p >= map.width || row == first_slot + off || (tid >= hi && (row < 0 || row >= a.c.tokens));
    }
    const uint64_t bad = __ballot(!whole) >> (tid - off) << (kTile - block);  // of this lane's block
    if (off == 0) block_row[tid >> shift] = bad ? -1 : usable(row);
  }
  if (tid >= kTile && tid < kTile + units) {
    const int u = tid - kTile;
    const int64_t p = p0 + begin;
    const int32_t row = begin < lo ? usable(!map.row ? p : (p < map.width ? map.row[p] : -1)) : -1;
    before[u] = row < 0 ? 0.0f : scales[((int64_t)(row >> shift) * a.Hkv + h0 + (u >> 1)) * 2 + (u & 1)];
  }
  for (int i = tid; i < 3 * kTile; i += LSA_BLOCK) (&most[0][0])[i] = 0u;
  // the sines of the tile's tokens: a pair a thread (64 or 128 threads a token), the tile's first angle and a
  // multiple of the pair's frequency, in fp64 turns
  {
    const int wide = a.turn.pairs > 64 ? 7 : 6, j = tid & ((1 << wide) - 1);
    if (j < a.turn.pairs) {
      const double f = turn_frequency(a.turn, j), each = f * kPerTurn;
      double base = (double)p0 * f * kPerTurn;
      base -= rint(base);
#pragma unroll 4
      for (int x = lo + (tid >> wide); x < hi; x += LSA_BLOCK >> wide) angles[x].put(j, turn_angle(a.turn, fma((double)x, each, base)));
    }
  }
  float wk[8];
  load_weights<T>(a.turn.kw, a.turn.w32, lp, wk);
  __syncthreads();

  const bool had = begin < lo;  // the first block holds earlier tokens
  int64_t to_row[STEPS];  // where their codes go, or -1: nowhere; earlier tokens of the first block among them
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int x = first + i;
    const int64_t row0 = block_row[x >> shift], row = row0 + (x & (block - 1));
    to_row[i] = x < begin || x >= hi || row0 < 0 || row >= a.c.tokens ? -1 : b * a.c.sb + row * a.c.st + 8 * lp;
  }
  for (int u = 0; u < units; ++u) {
    const int h = h0 + (u >> 1), kv = u & 1, turn_no = u % 3;
    float y[STEPS][8];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) raw[i].get(y[i]);
    fetch(u + 1);
    uint32_t tops[STEPS];  // a token's largest magnitude, as an integer: infinities and NaN are the largest of all
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int x = first + i;
      if (kv == 0 && x >= lo && x < hi) {  // uniform over the lanes of a row
        if (a.turn.kw) norm8<D>(y[i], wk, a.turn.eps);
        if (a.turn.pairs > 0) {
          LaneTurn turn;
          turn.load(a.turn, angles[x], lp);
          turn8(a.turn, y[i], turn, stage + slot * D, stage + LSA_BLOCK * 8, lp);
        }
      }
      uint32_t m = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(y[i][e]) & 0x7FFFFFFFu);
      tops[i] = to_row[i] < 0 ? 0u : m;  // a dropped one has no part in the scale
    }
    bool strange = false;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) strange |= tops[i] >= 0x7F800000u;
    const bool odd = __ballot(strange) != 0ull;  // wave-uniform, and rare
    if (odd) {  // the finite ones' maximum
      asm volatile("; kept a branch");
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        tops[i] = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t z = __float_as_uint(y[i][e]) & 0x7FFFFFFFu;
          tops[i] = z < 0x7F800000u && z > tops[i] && to_row[i] >= 0 ? z : tops[i];
        }
      }
    }
    // tokens that are not new are zeros, here and in their blocks' maxima
    if (block >= STEPS) {  // a lane's tokens are of one block
      uint32_t m = 0u;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) m = max(m, tops[i]);
      const float top = group_max<L::LPT>(__uint_as_float(m));
      if (lp == 0) atomicMax(&most[turn_no][first >> shift], __float_as_uint(top));
    } else {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const float top = group_max<L::LPT>(__uint_as_float(tops[i]));
        if (lp == 0) atomicMax(&most[turn_no][(first + i) >> shift], __float_as_uint(top));
      }
    }
    if (tid < kTile) most[(u + 1) % 3][tid] = 0u;  // unit u - 2's: every thread read it before the last barrier
    __syncthreads();
    const float held = before[u];
    uint8_t* cache = (kv ? a.c.v : a.c.k) + h * a.c.sh;
    float scale = 0.0f, inv = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int x = first + i, blk = x >> shift;
      if (i == 0 || block < STEPS) {  // else the lane's tokens are of one block
        scale = fmaxf(__uint_as_float(most[turn_no][blk]) / C::kMost, kLeast);
        if (had && blk == begin >> shift) scale = fmaxf(scale, held);
        inv = 1.0f / scale;
      }
      if (to_row[i] < 0) continue;
      uint2* at = (uint2*)(cache + to_row[i]);
      if (x >= lo) {
        uint2 codes;
        if (odd) {
          asm volatile("; kept a branch");
          codes = put8<C>(y[i], scale, inv, true);
        } else {
          codes = put8<C>(y[i], scale, inv, false);
        }
        *at = codes;
      } else if (scale != held) {  // the block's earlier tokens, where its scale grew
        const float ratio = held / scale;
        float z[8];
        C::get8(*at, z);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = C::odd(z[e] * ratio);
        *at = make_uint2(C::put4(z), C::put4(z + 4));
      }
      if (lp == 0 && x == max(blk << shift, lo))  // the block's first new token
        scales[((int64_t)(block_row[blk] >> shift) * a.Hkv + h) * 2 + kv] = scale;
    }
  }
}

struct ValueArgs {
  CacheArgs c;
  const int32_t* rows;
  int64_t row_stride;
  const int32_t* lengths;
  int64_t R, W;
  int Hkv;
  void* k_out;
  void* v_out;
  uint32_t many, chunks;  // rows of a workgroup, workgroups of a list
};

// A workgroup takes `many` consecutive rows of a list, 8 codes of K and of V a lane.
template <typename T, int D, typename C>
__global__ __launch_bounds__(LSA_BLOCK) void byte_values_kernel(ValueArgs a) {
  const uint32_t per = (uint32_t)a.Hkv * (D / 8);  // lanes of a row
  const uint32_t r = blockIdx.x / a.chunks;
  const int64_t w0 = (int64_t)(blockIdx.x - r * a.chunks) * a.many;
  const int64_t n = a.lengths ? (int64_t)a.lengths[r] : a.W;
  const uint32_t lanes = (uint32_t)min((int64_t)a.many, a.W - w0) * per;
  const int64_t out = ((int64_t)r * a.W + w0) * per;
  for (uint32_t i = threadIdx.x; i < lanes; i += LSA_BLOCK) {
    const uint32_t dw = i / per, x = i - dw * per, h = x / (D / 8), lp = x % (D / 8);
    const int64_t w = w0 + dw;
    const int64_t row = a.rows ? (int64_t)a.rows[r * a.row_stride + w] : w;
    float k[8], v[8];
    if (w < n && row >= 0 && row < a.c.tokens) {
      const int64_t at = r * a.c.sb + row * a.c.st + h * a.c.sh + 8 * lp;
      const float2 s = ((const float2*)a.c.scales)[r * a.c.scale_sb + (row >> a.c.block_shift) * a.Hkv + h];
      C::get8(*(const uint2*)(a.c.k + at), k);
      C::get8(*(const uint2*)(a.c.v + at), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        k[e] *= s.x;
        v[e] *= s.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) k[e] = v[e] = 0.0f;
    }
    store8((T*)a.k_out + 8 * (out + i), k);
    store8((T*)a.v_out + 8 * (out + i), v);
  }
}

template <typename T, int D, typename C>
void launch_append(const AppendArgs& a, int64_t groups, hipStream_t s) {
  byte_append_kernel<T, D, C><<<dim3((unsigned)groups), LSA_BLOCK, 0, s>>>(a);
}

template <typename T, int D, typename C>
void launch_values(const ValueArgs& a, hipStream_t s) {
  byte_values_kernel<T, D, C><<<dim3((unsigned)(a.R * a.chunks)), LSA_BLOCK, 0, s>>>(a);
}

CacheArgs cache_args(const lsa_byte_cache* c, int32_t Hkv) {
  const int64_t pairs = (c->tokens + c->block - 1) / c->block * Hkv;
  return CacheArgs{(uint8_t*)c->k, (uint8_t*)c->v, c->scales, __builtin_ctz((unsigned)c->block), c->tokens, c->caches == 1 ? 0 : c->batch_stride,
                   c->token_stride, c->head_stride, c->caches == 1 ? 0 : pairs};
}

}  // namespace

#define LSA_DISPATCH_CODES(D, code, LAUNCH, ...)                                   \
  switch (D) {                                                                     \
    case 32: code == LSA_INT8 ? LAUNCH<QT, 32, Int8Code>(__VA_ARGS__) : LAUNCH<QT, 32, E4m3Code>(__VA_ARGS__); break;    \
    case 64: code == LSA_INT8 ? LAUNCH<QT, 64, Int8Code>(__VA_ARGS__) : LAUNCH<QT, 64, E4m3Code>(__VA_ARGS__); break;    \
    case 128: code == LSA_INT8 ? LAUNCH<QT, 128, Int8Code>(__VA_ARGS__) : LAUNCH<QT, 128, E4m3Code>(__VA_ARGS__); break; \
    default: code == LSA_INT8 ? LAUNCH<QT, 256, Int8Code>(__VA_ARGS__) : LAUNCH<QT, 256, E4m3Code>(__VA_ARGS__); break;  \
  }

extern "C" int lsa_byte_append(const lsa_byte_cache* cache, const void* k, const void* v, const void* q, int dtype,
                               int64_t B, int64_t T, int32_t Hq, int32_t Hkv, int32_t D, int64_t k_batch_stride,
                               int64_t k_token_stride, int64_t k_head_stride, int64_t v_batch_stride,
                               int64_t v_token_stride, int64_t v_head_stride, int64_t q_batch_stride,
                               int64_t q_token_stride, int64_t q_head_stride, const int32_t* starts,
                               const int32_t* lengths, const lsa_slot_map* slots, const lsa_turn* turn, void* q_out,
                               void* stream) {
  LSA_REQUIRE(k && v && starts && turn && (!q || q_out), LSA_ERR_NULL, "lsa_byte_append: NULL pointer");
  LSA_TRY(check_dtype(dtype));
  LSA_REQUIRE(B >= 0 && T >= 0 && (!q || (Hq >= 1 && Hq <= 65536)) && (B == 0 || T <= kMaxGroups / B), LSA_ERR_SHAPE,
              "lsa_byte_append: B %lld T %lld Hq %d (under 2^24 tokens)", (long long)B, (long long)T, Hq);
  LSA_TRY(check_byte_cache("lsa_byte_append", cache, B, Hkv, D));
  TurnArgs t;
  LSA_TRY(check_turn("lsa_byte_append", turn, D, &t));
  AppendArgs a = {};
  LSA_TRY(check_slots("lsa_byte_append", slots, &a.slots));
  LSA_REQUIRE(slots || cache->caches == B, LSA_ERR_SHAPE, "lsa_byte_append: a pool for %lld rows needs a slot map", (long long)B);
  const int64_t e = dtype == LSA_F32 ? 4 : 2;
  LSA_REQUIRE((((uintptr_t)k | (uintptr_t)v | (q ? (uintptr_t)q | (uintptr_t)q_out : 0)) & 15) == 0 &&
                  ((k_batch_stride | k_token_stride | k_head_stride | v_batch_stride | v_token_stride | v_head_stride |
                    (q ? q_batch_stride | q_token_stride | q_head_stride : 0)) * e) % 16 == 0,
              LSA_ERR_ALIGN, "lsa_byte_append: rows of q, k and v must be 16-byte aligned");
  if (B * T == 0) return LSA_OK;
  a.c = cache_args(cache, Hkv);
  a.k = k; a.v = v;
  a.k_sb = k_batch_stride; a.k_st = k_token_stride; a.k_sh = k_head_stride;
  a.v_sb = v_batch_stride; a.v_st = v_token_stride; a.v_sh = v_head_stride;
  a.starts = starts; a.lengths = lengths; a.Hkv = Hkv; a.T = (int)T; a.B = (int)B;
  a.tiles = (int)((T + kTile - 2) / kTile + 1);  // from any start
  a.turn = t;
  // kv-heads of a tile over several workgroups while those leave CUs idle; q's tokens likewise
  const int64_t tiles = B * a.tiles;
  a.parts = (int)std::max<int64_t>((Hkv + kPartHeads - 1) / kPartHeads, std::min<int64_t>(Hkv, 1024 / tiles));
  a.heads = (Hkv + a.parts - 1) / a.parts;
  a.parts = (Hkv + a.heads - 1) / a.heads;
  a.kv_groups = tiles * a.parts;
  RotateArgs& r = a.q;
  r.q = r.k = q; r.q_out = r.k_out = q_out; r.starts = starts; r.lengths = lengths;
  r.q_sb = q_batch_stride; r.q_st = q_token_stride; r.q_sh = q_head_stride;
  r.Hq = Hq; r.T = (int)T; r.tokens = (int)(B * T); r.turn = t;
  // q in the same launch: its workgroups wait for memory while those of K and V wait for barriers and each other
  // (32768 tokens: 151 us, and 96 for q and 69 for K and V one after the other). Its outputs go past the caches as rotate's.
  a.q_mode = B * T < 1024 ? kFew : (B * T * Hq * D * e > (64 << 20) ? kStream : kMany);
  const int rows = 256 / (D / 8);
  r.heads = a.q_mode == kFew && B * T * ((Hq + rows - 1) / rows) <= 512 ? rows : std::max(Hq, 1);
  a.q_parts = (uint32_t)((Hq + r.heads - 1) / r.heads);
  const int64_t groups = a.kv_groups + (!q ? 0 : (a.q_mode == kFew ? B * T * a.q_parts : (B * T + 3) / 4));
  LSA_REQUIRE(groups <= kMaxGroups, LSA_ERR_SHAPE, "lsa_byte_append: %lld tokens of %d kv-heads (2^24 workgroups)",
              (long long)(B * T), Hkv);
  hipStream_t s = (hipStream_t)stream;
  const int code = cache->code;
  LSA_DISPATCH_QT(dtype, { LSA_DISPATCH_CODES(D, code, launch_append, a, groups, s) });
  LSA_LAUNCHED("lsa_byte_append");
  return LSA_OK;
}

extern "C" int lsa_byte_values(const lsa_byte_cache* cache, const int32_t* rows, int64_t row_stride,
                               const int32_t* lengths, int64_t R, int64_t W, int32_t Hkv, int32_t D, int dtype,
                               void* k_out, void* v_out, void* stream) {
  LSA_REQUIRE(k_out && v_out, LSA_ERR_NULL, "lsa_byte_values: NULL pointer");
  LSA_TRY(check_dtype(dtype));
  LSA_REQUIRE(R >= 0 && W >= 0 && R <= 0x7FFFFFFF && W <= 0x7FFFFFFF && (!rows || row_stride >= 0), LSA_ERR_SHAPE,
              "lsa_byte_values: R %lld W %lld", (long long)R, (long long)W);
  LSA_TRY(check_byte_cache("lsa_byte_values", cache, R, Hkv, D));
  LSA_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, LSA_ERR_ALIGN, "lsa_byte_values: outputs must be 16-byte aligned");
  if (R * W == 0) return LSA_OK;
  ValueArgs a = {cache_args(cache, Hkv), rows, row_stride, lengths, R, W, Hkv, k_out, v_out};
  a.many = (uint32_t)std::max(1, kValueLanes / (Hkv * (D / 8)));
  const int64_t chunks = (W + a.many - 1) / a.many;
  LSA_REQUIRE(chunks <= kMaxGroups / R, LSA_ERR_SHAPE, "lsa_byte_values: %lld rows", (long long)(R * W));
  a.chunks = (uint32_t)chunks;
  hipStream_t s = (hipStream_t)stream;
  const int code = cache->code;
  LSA_DISPATCH_QT(dtype, { LSA_DISPATCH_CODES(D, code, launch_values, a, s) });
  LSA_LAUNCHED("lsa_byte_values");
  return LSA_OK;
}
