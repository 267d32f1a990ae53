// The sparse read over a cache of 8-bit codes (gfx950): softmax attention of every query row over its listed rows,
//   o = sum_i w_i vs_i vc_i / sum_i w_i,   w_i = exp2(scale log2(e) ks_i (q . kc_i) - m),
// with codes kc, vc and a scale ks, vs of each block of tokens and kv-head.
//
// A workgroup (4 waves) takes one (query row, kv-head, up to 16 of its query heads) and a span of its list; a wave
// takes every fourth tile of 32 keys by itself, with no barrier until the end. K, V, the scales and the list go
// from memory straight to LDS, a tile (the list two tiles) ahead of the one that is computed: 8 KB a wave in flight
// at head dim 128, in two buffers of LDS and no registers. Both products are matrix instructions in bf16, whose 8
// bits of mantissa hold every code exactly: S^T = K Q^T, and O^T += V^T P^T with V's columns by the transposing LDS
// read. q enters exactly too: bf16 as it is, fp16 in two parts, fp32 in three. A weight times V's scale goes in as
// two parts (16 bits), for fp32 rows as three, so that rounding it costs nothing beside the output's own rounding.
// The keys of a tile are dealt to the rows of S^T so that a lane's 8 scores are those of the 8 keys whose V codes
// it holds (keys 8 row .. + 8): weights go from one product to the other in their registers.
//
// An id outside the cache reads zeros in place of codes and scales and weighs nothing, so what the cache holds
// elsewhere never enters. Spans of a list leave fp32 partials (m, l, o) that the last of them to finish joins, in
// the list's order.
#include <math.h>

#include <algorithm>

#include "lsa_abi_common.h"
#include "lsa_mfma_dev.h"
#include "lsa_turn_dev.h"

using namespace lsa;

namespace {

constexpr int kKeys = 32;                   // of a wave's tile
constexpr int kStep = kKeys * LSA_WAVES;    // of a workgroup's
constexpr int kByteSplits = 64;
constexpr int kHeads = 16;                  // query heads of a workgroup

__device__ const uint4 g_zeros[16] = {};  // a row of codes, or a pair of scales, of nothing

struct ByteReadArgs {
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  const float* scales;
  int64_t sb, st, sh, scale_sb;
  int64_t tokens;
  int block_shift;
  const int32_t* ids;
  const int32_t* lengths;
  int W, per_head;
  int64_t Tq;
  int Hq, Hkv, group, blocks;  // query heads a kv-head, in blocks of 16
  float scale_log2;
  int span, splits;
  int* counters;  // or nullptr: another launch joins
  float* parts;
  void* out;
};

__host__ __device__ constexpr int part_floats(int heads, int D) { return heads * D + (2 * heads + 3) / 4 * 4; }

// A workgroup's unit: query row, kv-head, its query heads, and its list.
struct Unit {
  int64_t row, list;
  int g, h0, heads, n;
  __device__ __forceinline__ Unit(const ByteReadArgs& a, int64_t i) {
    const int cb = (int)(i % a.blocks);
    const int64_t rg = i / a.blocks;
    row = rg / a.Hkv;
    g = (int)(rg % a.Hkv);
    h0 = g * a.group + cb * kHeads;
    heads = min(kHeads, a.group - cb * kHeads);
    list = a.per_head ? rg : row;
    const int len = a.lengths[list];
    n = len < 0 ? 0 : (len > a.W ? a.W : len);
  }
};

// 8 codes as bf16, exactly.
template <typename C> __device__ __forceinline__ uint4 codes_bf16(const uint2& u);
template <> __device__ __forceinline__ uint4 codes_bf16<E4m3Code>(const uint2& u) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.x, 1.0f, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.x, 1.0f, true)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.y, 1.0f, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.y, 1.0f, true)));
}
template <> __device__ __forceinline__ uint4 codes_bf16<Int8Code>(const uint2& u) {
  float f[8];
  Int8Code::get8(u, f);
  uint32_t r[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)  // whole numbers under 2^8: the low half of the fp32 word is zero
    r[e] = __builtin_amdgcn_perm(__float_as_uint(f[2 * e + 1]), __float_as_uint(f[2 * e]), 0x07060302u);
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// Which 16-byte segment of LDS row r holds the row's segment 0 (XOR). S^T reads rows 8 a + u (u < 4 or u >= 4) of
// one segment in 16 lanes, V^T rows 8 a .. + 8: either way they spread over the 256 bytes of a bank cycle.
template <int D> __device__ __forceinline__ int swizzle(int r) {
  const int x = ((r >> 3) ^ (r >> 2)) & 1;
  if constexpr (D == 256) return (r & 3) | x << 2 | (r >> 4 & 1) << 3;
  if constexpr (D == 128) return (r >> 1 & 1) | x << 1 | (r >> 4 & 1) << 2;
  if constexpr (D == 64) return x | (r >> 4 & 1) << 1;
  return ((r >> 3) ^ (r >> 4)) & 1;
}

template <int D>
struct WaveLds {
  uint8_t k[2][kKeys * D];
  uint8_t v[2][kKeys * D];
  float scales[2][64];  // K's 32, V's 32
  int32_t ids[2][64];   // 32 and their copies
};
template <int D>
struct ByteLds {
  WaveLds<D> wave[LSA_WAVES];
  float m[LSA_WAVES][kHeads], l[LSA_WAVES][kHeads];
  int flag;
};

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) u32x2_t lds_u2;
typedef __attribute__((address_space(3))) u32x4_t lds_u4;
typedef __attribute__((address_space(3))) i32x2_t lds_i2;
typedef __attribute__((address_space(3))) float lds_float;
typedef __attribute__((address_space(3))) int32_t lds_int;

__device__ __forceinline__ void dma16_far(uint32_t lds, const void* p) {  // a lane's own 64-bit address
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
__device__ __forceinline__ void dma4_far(uint32_t lds, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}

// x and y as N bf16 parts each that add up to them (to 8 N bits).
template <int N>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t* out) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    out[i] = pack_bf16(x, y);
    if (i + 1 < N) {
      x -= __uint_as_float(out[i] << 16);
      y -= __uint_as_float(out[i] & 0xFFFF0000u);
    }
  }
}
// The same where they may be infinite: nothing is left of an infinity.
template <int N>
__device__ __forceinline__ void split_any(float x, float y, uint32_t* out) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    out[i] = pack_bf16(x, y);
    if (i + 1 < N) {
      const float a = __uint_as_float(out[i] << 16), b = __uint_as_float(out[i] & 0xFFFF0000u);
      x = isinf(a) ? 0.0f : x - a;
      y = isinf(b) ? 0.0f : y - b;
    }
  }
}

template <typename T> struct Parts;
template <> struct Parts<bf16_t> { static constexpr int Q = 1, P = 2; };
template <> struct Parts<_Float16> { static constexpr int Q = 2, P = 2; };
template <> struct Parts<float> { static constexpr int Q = 3, P = 3; };

// The partials of a unit's n_act spans into its output rows. Every thread calls it.
template <typename T, int D>
__device__ __forceinline__ void join(const ByteReadArgs& a, const Unit& u, const float* parts, int n_act, float* w, float* ltot) {
  const int tid = threadIdx.x, heads = u.heads, stride = part_floats(heads, D);
  const CoherentRows rows(parts);  // under 2 GiB
  __syncthreads();
  for (int t = tid; t < n_act * heads; t += LSA_BLOCK) {
    const int s = t / heads, h = t % heads;
    w[t] = coherent_load(parts + (int64_t)s * stride + heads * D + h);
    w[kByteSplits * kHeads + t] = coherent_load(parts + (int64_t)s * stride + heads * D + heads + h);
  }
  __syncthreads();
  if (tid < heads) {
    float m = kNegBig, l = 0.0f;
    for (int s = 0; s < n_act; ++s) m = fmaxf(m, w[s * heads + tid]);
    for (int s = 0; s < n_act; ++s) {
      const float f = fast_exp2(w[s * heads + tid] - m);
      l += f * w[kByteSplits * kHeads + s * heads + tid];
      w[s * heads + tid] = f;
    }
    ltot[tid] = l;
  }
  __syncthreads();
  T* out = (T*)a.out + (u.row * a.Hq + u.h0) * D;
  for (int c = tid; c < heads * D / 4; c += LSA_BLOCK) {
    const int h = 4 * c / D;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < n_act; s0 += 8) {
      float4 x[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) x[s] = rows.load4(4 * (min(s0 + s, n_act - 1) * stride + 4 * c));
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float f = s0 + s < n_act ? w[(s0 + s) * heads + h] : 0.0f;
        acc.x += f * x[s].x; acc.y += f * x[s].y; acc.z += f * x[s].z; acc.w += f * x[s].w;
      }
    }
    const float l = ltot[h], inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const float r[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
    for (int e = 0; e < 4; ++e) store_out<T>(out + 4 * c + e, r[e]);
  }
}

template <typename T, int D, typename C>
__global__ __launch_bounds__(LSA_BLOCK) void byte_read_kernel(ByteReadArgs a) {
  constexpr int SEGS = D / 16, NI = D / 32;     // 16-byte segments of a row; DMAs of a tile, K and V each
  constexpr int KS = D / 32, DB = D / 16;       // matrix steps over the dims; 16-dim blocks of the output
  constexpr int RPI = 64 / SEGS;                // rows of a DMA
  constexpr int NV = 2 * NI + 1;                // memory operations of a tile
  constexpr int QP = Parts<T>::Q, PP = Parts<T>::P;
  __shared__ __attribute__((aligned(1024))) ByteLds<D> sh;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int row = lane >> 4, col = lane & 15;
  const Unit u(a, blockIdx.x);
  const int s = blockIdx.y, n_act = (u.n + a.span - 1) / a.span;
  if (s >= max(n_act, 1)) return;
  T* out = (T*)a.out + (u.row * a.Hq + u.h0) * D;
  if (u.n == 0) {
    for (int j = tid; j < u.heads * D; j += LSA_BLOCK) store_out<T>(out + j, 0.0f);
    return;
  }
  const int lo = s * a.span + kKeys * w, hi = min((s + 1) * a.span, u.n);
  const int n_tiles = hi > lo ? (hi - lo + kStep - 1) / kStep : 0;
  const int32_t* ids = a.ids + u.list * a.W;
  const int64_t b = u.row / a.Tq;
  const uint8_t* kb = a.k + b * a.sb + u.g * a.sh;
  const uint8_t* vb = a.v + b * a.sb + u.g * a.sh;
  const float* scales = a.scales + (b * a.scale_sb + u.g) * 2;
  WaveLds<D>& mem = sh.wave[w];
  const lds_char* base = (const lds_char*)&mem;
  const uint32_t lds = (uint32_t)(uintptr_t)base;
  constexpr uint32_t V_AT = 2 * kKeys * D, S_AT = 4 * kKeys * D, I_AT = S_AT + 512;

  auto load_ids = [&](int i) {
    const int j = lo + kStep * i + (lane & 31);
    dma4_far(lds + I_AT + (uint32_t)(i & 1) * 256u, ids + min(j, hi - 1));
  };
  uint32_t live[2] = {0u, 0u};  // which keys of the two buffers' tiles count
  auto load = [&](int i) {
    const uint32_t buf = (uint32_t)(i & 1);
    const lds_int* at = (const lds_int*)(base + I_AT + buf * 256u);
    const int left = hi - (lo + kStep * i);  // keys from the tile's first on
    auto good = [&](int id, int x) { return x < left && id >= 0 && id < a.tokens; };
    {
      const int x = lane & 31, id = at[x];
      const bool ok = good(id, x);
      live[i & 1] = (uint32_t)__ballot(ok);
      const float* p = scales + ((int64_t)((uint32_t)id >> a.block_shift) * a.Hkv) * 2 + (lane >> 5);
      dma4_far(lds + S_AT + buf * 256u, ok ? (const void*)p : (const void*)g_zeros);
    }
#pragma unroll
    for (int y = 0; y < NI; ++y) {
      const int r = y * RPI + lane / SEGS, id = at[r];
      const int sg = (lane % SEGS) ^ swizzle<D>(r);
      const bool ok = good(id, r);
      const uint64_t off = (uint64_t)(uint32_t)id * (uint32_t)a.st + 16 * sg;
      dma16_far(lds + buf * (kKeys * D) + 1024u * y, ok ? (const void*)(kb + off) : (const void*)g_zeros);
      dma16_far(lds + V_AT + buf * (kKeys * D) + 1024u * y, ok ? (const void*)(vb + off) : (const void*)g_zeros);
    }
  };

  // this lane's part of Q^T: head col, dims 16 (row + 4 j) .. + 16 for steps 2 j, 2 j + 1 (D = 32: 8 row .. + 8)
  uint4 q[KS][QP];
  float m = kNegBig, l = 0.0f;
  f32x4_t o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  if (n_tiles > 0) {  // wave-uniform
    load_ids(0);
    if (n_tiles > 1) load_ids(1);
    const T* qr = (const T*)a.q + (u.row * a.Hq + u.h0 + (col < u.heads ? col : 0)) * D;
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      Raw8<T> raw;
      raw.load(qr + (D == 32 ? 8 * row : 16 * (row + 4 * (j >> 1)) + 8 * (j & 1)));
      float f[8];
      raw.get(f);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = col < u.heads ? f[e] : 0.0f;
      uint32_t p[4][QP];
#pragma unroll
      for (int e = 0; e < 4; ++e) split_any<QP>(f[2 * e], f[2 * e + 1], p[e]);
#pragma unroll
      for (int x = 0; x < QP; ++x) {
        q[j][x] = make_uint4(p[0][x], p[1][x], p[2][x], p[3][x]);
        asm volatile("" : "+v"(q[j][x].x), "+v"(q[j][x].y), "+v"(q[j][x].z), "+v"(q[j][x].w));  // here, before the DMAs
      }
    }
    wait_vm<0>();
    load(0);
  }
  for (int i = 0; i < n_tiles; ++i) {
    if (i + 1 < n_tiles) {
      wait_vm<NV>();  // the list of tile i + 1
      if (i + 2 < n_tiles) {
        load_ids(i + 2);
        load(i + 1);
        wait_vm<NV + 1>();  // tile i
      } else {
        load(i + 1);
        wait_vm<NV>();
      }
    } else {
      wait_vm<0>();
    }
    const uint32_t buf = (uint32_t)(i & 1);
    const uint32_t mine = (i & 1 ? live[1] : live[0]) >> (8 * row);
    // S^T: rows 4 a + u of the first product are keys 8 a + u, of the second 8 a + 4 + u
    f32x4_t c[2];
    const lds_char* kt = base + buf * (kKeys * D);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      c[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      const int r = 8 * (col >> 2) + 4 * t + (col & 3);
      if constexpr (D == 32) {
        const u32x2_t x = *(const lds_u2*)(kt + r * D + 16 * ((row >> 1) ^ swizzle<D>(r)) + 8 * (row & 1));
        const uint4 kc = codes_bf16<C>(make_uint2(x[0], x[1]));
#pragma unroll
        for (int p = 0; p < QP; ++p) c[t] = Mfma16<bf16_t>::run(kc, q[0][p], c[t]);
      } else {
#pragma unroll
        for (int j = 0; j < KS / 2; ++j) {
          const u32x4_t x = *(const lds_u4*)(kt + r * D + 16 * ((row + 4 * j) ^ swizzle<D>(r)));
          const uint4 k0 = codes_bf16<C>(make_uint2(x[0], x[1])), k1 = codes_bf16<C>(make_uint2(x[2], x[3]));
#pragma unroll
          for (int p = 0; p < QP; ++p) {
            c[t] = Mfma16<bf16_t>::run(k0, q[2 * j][p], c[t]);
            c[t] = Mfma16<bf16_t>::run(k1, q[2 * j + 1][p], c[t]);
          }
        }
      }
    }
    const lds_float* sc = (const lds_float*)(base + S_AT + buf * 256u) + 8 * row;
    float x[8], top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = (mine >> e & 1u) ? c[e >> 2][e & 3] * (sc[e] * a.scale_log2) : -INFINITY;
      top = fmaxf(top, x[e]);
    }
    top = fmaxf(top, lane_xor(top, 16));
    top = fmaxf(top, lane_xor(top, 32));
    if (__ballot(top > m + 8.0f) != 0) {  // the reference moves where a head's maximum passes it by 2^8
      const float to = fmaxf(m, top), f = fast_exp2(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] = f32x4_t{o[d][0] * f, o[d][1] * f, o[d][2] * f, o[d][3] * f};
    }
    uint32_t pr[4][PP];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p0 = fast_exp2(x[2 * e] - m), p1 = fast_exp2(x[2 * e + 1] - m);
      l += p0 + p1;
      split_pair<PP>(p0 * sc[32 + 2 * e], p1 * sc[32 + 2 * e + 1], pr[e]);
    }
    const lds_char* vt = base + V_AT + buf * (kKeys * D);
    const int vr = 8 * row + (col >> 1);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const i32x2_t y = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2*)(vt + vr * D + 16 * (d ^ swizzle<D>(vr)) + 8 * (col & 1)));
      const uint4 vc = codes_bf16<C>(make_uint2((uint32_t)y[0], (uint32_t)y[1]));
#pragma unroll
      for (int p = 0; p < PP; ++p)
        o[d] = Mfma16<bf16_t>::run(vc, make_uint4(pr[0][p], pr[1][p], pr[2][p], pr[3][p]), o[d]);
    }
  }

  // the waves' states meet in LDS, each in its wave's own buffers: [16][D]
  l += lane_xor(l, 16);
  l += lane_xor(l, 32);
  float* mo = (float*)&mem;
  if (lane < kHeads) {
    sh.m[w][lane] = m;
    sh.l[w][lane] = l;
  }
#pragma unroll
  for (int d = 0; d < DB; ++d) *(float4*)(mo + col * D + 16 * d + 4 * row) = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
  __syncthreads();
  const int64_t unit = blockIdx.x;
  const int stride = part_floats(u.heads, D);
  float* parts = a.parts + unit * a.splits * (int64_t)part_floats(min(kHeads, a.group), D);
  float* part = parts + (int64_t)s * stride;
  for (int t = tid; t < u.heads * D / 4; t += LSA_BLOCK) {
    const int h = 4 * t / D, d = 4 * t % D;
    float top = kNegBig;
#pragma unroll
    for (int y = 0; y < LSA_WAVES; ++y) top = fmaxf(top, sh.m[y][h]);
    float ll = 0.0f, r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int y = 0; y < LSA_WAVES; ++y) {
      const float f = fast_exp2(sh.m[y][h] - top);
      const float4 z = *(const float4*)((const float*)&sh.wave[y] + h * D + d);
      ll += f * sh.l[y][h];
      r[0] += f * z.x; r[1] += f * z.y; r[2] += f * z.z; r[3] += f * z.w;
    }
    if (n_act == 1) {
      const float inv = ll > 0.0f || ll != ll ? 1.0f / ll : 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) store_out<T>(out + 4 * t + e, r[e] * inv);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) coherent_store(part + 4 * t + e, r[e]);
      if (d == 0) {
        coherent_store(part + u.heads * D + h, top);
        coherent_store(part + u.heads * D + u.heads + h, ll);
      }
    }
  }
  if (n_act == 1 || a.counters == nullptr) return;
  if (!arrive_last(&a.counters[unit], n_act, &sh.flag)) return;
  join<T, D>(a, u, parts, n_act, (float*)&sh.wave[0], &sh.m[0][0]);
}

// The join as a launch of its own, where there are no counters.
template <typename T, int D>
__global__ __launch_bounds__(LSA_BLOCK) void byte_join_kernel(ByteReadArgs a) {
  __shared__ float w[2 * kByteSplits * kHeads];
  __shared__ float ltot[kHeads];
  const Unit u(a, blockIdx.x);
  const int n_act = (u.n + a.span - 1) / a.span;
  if (n_act <= 1) return;
  join<T, D>(a, u, a.parts + (int64_t)blockIdx.x * a.splits * part_floats(min(kHeads, a.group), D), n_act, w, ltot);
}

template <typename T, int D>
void launch_byte_read(const ByteReadArgs& a, int code, int64_t units, hipStream_t s) {
  const dim3 grid((unsigned)units, (unsigned)a.splits);
  if (code == LSA_INT8) byte_read_kernel<T, D, Int8Code><<<grid, LSA_BLOCK, 0, s>>>(a);
  else byte_read_kernel<T, D, E4m3Code><<<grid, LSA_BLOCK, 0, s>>>(a);
  if (a.splits > 1 && a.counters == nullptr) byte_join_kernel<T, D><<<dim3((unsigned)units), LSA_BLOCK, 0, s>>>(a);
}

int64_t head_blocks(int32_t Hq, int32_t Hkv) { return (Hq / Hkv + kHeads - 1) / kHeads; }

}  // namespace

extern "C" size_t lsa_byte_read_scratch_bytes(int64_t rows, int32_t Hq, int32_t Hkv, int32_t D, int32_t splits) {
  if (splits <= 1 || rows <= 0 || Hkv <= 0 || Hq < Hkv || Hq % Hkv || D <= 0) return 0;
  return (size_t)rows * Hkv * (size_t)head_blocks(Hq, Hkv) * splits * part_floats(std::min(kHeads, Hq / Hkv), D) * sizeof(float);
}

extern "C" int lsa_byte_read(const void* q, const lsa_byte_cache* cache, int dtype, int64_t B, int64_t Tq, int32_t Hq,
                             int32_t Hkv, int32_t D, const int32_t* ids, const int32_t* lengths, int32_t W,
                             int ids_per_head, float scale, int32_t splits, int32_t* counters, void* scratch,
                             size_t scratch_bytes, void* out, void* stream) {
  LSA_REQUIRE(q && out && (ids || W == 0) && lengths, LSA_ERR_NULL, "lsa_byte_read: NULL pointer");
  LSA_TRY(check_dtype(dtype));
  LSA_REQUIRE(B >= 0 && Tq >= 0 && W >= 0, LSA_ERR_SHAPE, "lsa_byte_read: negative size");
  LSA_TRY(check_byte_cache("lsa_byte_read", cache, B, Hkv, D));
  LSA_REQUIRE(Hq >= Hkv && Hq % Hkv == 0 && Hq <= 65536, LSA_ERR_SHAPE, "lsa_byte_read: Hq %d must group onto Hkv %d", Hq, Hkv);
  LSA_REQUIRE(splits >= 1 && splits <= kByteSplits, LSA_ERR_SHAPE, "lsa_byte_read: splits in [1, %d], got %d", kByteSplits, splits);
  const int64_t blocks = head_blocks(Hq, Hkv);
  LSA_REQUIRE(B == 0 || Tq <= 0x3FFFFFF / B, LSA_ERR_SHAPE, "lsa_byte_read: too many rows");
  const int64_t units = B * Tq * Hkv * blocks;
  LSA_REQUIRE(units < (1 << 24), LSA_ERR_SHAPE, "lsa_byte_read: %lld rows x kv-heads (under 2^24)", (long long)units);
  LSA_REQUIRE((((uintptr_t)q | (uintptr_t)out) & 15) == 0, LSA_ERR_ALIGN, "lsa_byte_read: q and out must be 16-byte aligned");
  const size_t need = lsa_byte_read_scratch_bytes(B * Tq, Hq, Hkv, D, splits);
  LSA_REQUIRE(need == 0 || (scratch && scratch_bytes >= need && ((uintptr_t)scratch & 15) == 0), LSA_ERR_WORKSPACE,
              "lsa_byte_read: scratch missing, not 16-byte aligned or %zu < %zu bytes", scratch_bytes, need);
  if (units == 0) return LSA_OK;
  ByteReadArgs a = {};
  a.q = q; a.k = (const uint8_t*)cache->k; a.v = (const uint8_t*)cache->v; a.scales = cache->scales;
  a.sb = cache->caches == 1 ? 0 : cache->batch_stride; a.st = cache->token_stride; a.sh = cache->head_stride;
  a.scale_sb = cache->caches == 1 ? 0 : (cache->tokens + cache->block - 1) / cache->block * Hkv;
  a.tokens = cache->tokens; a.block_shift = __builtin_ctz((unsigned)cache->block);
  a.ids = ids; a.lengths = lengths; a.W = W; a.per_head = ids_per_head ? 1 : 0; a.Tq = Tq;
  a.Hq = Hq; a.Hkv = Hkv; a.group = Hq / Hkv; a.blocks = (int)blocks; a.scale_log2 = scale * kLog2e;
  a.span = (int)(((int64_t)(W + splits - 1) / splits + kStep - 1) / kStep * kStep);
  a.span = std::max(a.span, kStep);
  a.splits = splits; a.counters = counters; a.parts = (float*)scratch; a.out = out;
  hipStream_t s = (hipStream_t)stream;
  const int code = cache->code;
  LSA_DISPATCH_QT(dtype, {
    switch (D) {
      case 32: launch_byte_read<QT, 32>(a, code, units, s); break;
      case 64: launch_byte_read<QT, 64>(a, code, units, s); break;
      case 128: launch_byte_read<QT, 128>(a, code, units, s); break;
      default: launch_byte_read<QT, 256>(a, code, units, s); break;
    }
  });
  LSA_LAUNCHED("lsa_byte_read");
  return LSA_OK;
}
