// The sparse read over a cache of 8-bit codes (gfx950): softmax attention of every query row over its listed rows,
//   o = sum_i w_i vs_i vc_i / sum_i w_i,   w_i = exp2(scale log2(e) ks_i (q . kc_i) - m),
// with codes kc, vc and a scale ks, vs of each block of tokens and kv-head.
//
// A workgroup (4 waves) takes one (query row, kv-head, up to 16 of its query heads) and a span of its list; a wave
// takes every fourth tile of 32 keys by itself, with no barrier until the end. K, V, the scales and the list go
// from memory straight to LDS, so that what is in flight takes no registers. A wave has one buffer each of K and V
// and fills it again as soon as its product is through: K of the next tile loads while the softmax and V's product
// run, V while it waits for K (8 KB a wave in flight at head dim 128, four waves a SIMD). Both products are matrix
// instructions in bf16, whose 8 bits of mantissa hold every code exactly: S^T = K Q^T, and O^T += V^T P^T with V's
// columns by the transposing LDS read. q enters exactly too: bf16 as it is, fp16 in two parts, fp32 in three. A weight
// times V's scale goes in as two parts (16 bits), for fp32 rows as three, so that rounding it costs nothing beside the
// output's own rounding.
// The keys of a tile are dealt to the rows of S^T so that a lane's 8 scores are those of the 8 keys whose V codes
// it holds (keys 8 row .. + 8): weights go from one product to the other in their registers.
//
// What bounds it: memory. Measured at bf16, head dim 128, 32 query heads on 8: 32 lists of about 2048 keys a kv-head
// (134 MB, spans of 64 keys at 128 bytes a key) 29 us, where the loads alone take 28; sixteen whole caches of about
// 24600 keys (805 MB) 170 us a call among others, 4.7 TB/s, and no less with the products left out (a plain read of as
// much in one piece reaches 6.2); one list of 2048, 9.3 us: the launch, five round trips to memory and the join. One
// buffer and four waves a SIMD against two and two, measured together: 29 for 32, 168 for 163, 9.2 for 9.0. What a
// decode batch reads, many short spans, gains a tenth, the others lose 3%: one form for all of them.
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

constexpr int kKeys = 32;                 // of a wave's tile
constexpr int kStep = kKeys * LSA_WAVES;  // of a workgroup's
constexpr int kByteSplits = 64;
constexpr int kXcds = 8;
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
  uint32_t Tq, rows;
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
  int g, h0, heads;
  __device__ __forceinline__ Unit(const ByteReadArgs& a, uint32_t i) {  // units are fewer than 2^24
    const uint32_t rg = i / (uint32_t)a.blocks, r = rg / (uint32_t)a.Hkv;
    const int cb = (int)(i - rg * (uint32_t)a.blocks);
    row = r;
    g = (int)(rg - r * (uint32_t)a.Hkv);
    h0 = g * a.group + cb * kHeads;
    heads = min(kHeads, a.group - cb * kHeads);
    list = a.per_head ? rg : row;
  }
  __device__ __forceinline__ int keys(const ByteReadArgs& a) const {
    const int n = a.lengths[list];
    return n < 0 ? 0 : (n > a.W ? a.W : n);
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
  uint8_t k[kKeys * D];
  uint8_t v[kKeys * D];
  float scales[2][64];  // K's 32, V's 32
  int32_t ids[2][64];   // 32 and their copies
  uint64_t rows[kKeys][2];  // where the codes of the tile that is being fetched lie, K's and V's
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
typedef uint64_t u64x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) u64x2_t lds_u64x2;
typedef __attribute__((address_space(3))) uint64_t lds_u64;
typedef __attribute__((address_space(3))) f32x4_t lds_f4;
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

// What the weighted sum is divided by: no keys give zeros.
__device__ __forceinline__ float inverse(float l) { return l > 0.0f || l != l ? 1.0f / l : 0.0f; }
template <typename T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d);
template <> __device__ __forceinline__ void store4<float>(float* p, float a, float b, float c, float d) { *(float4*)p = make_float4(a, b, c, d); }
template <> __device__ __forceinline__ void store4<bf16_t>(bf16_t* p, float a, float b, float c, float d) { *(uint2*)p = make_uint2(pack_bf16(a, b), pack_bf16(c, d)); }
template <> __device__ __forceinline__ void store4<_Float16>(_Float16* p, float a, float b, float c, float d) { *(uint2*)p = make_uint2(pack_f16(a, b), pack_f16(c, d)); }

__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// v_max3_f32 as it is: fmaxf quiets its operands first.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
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

// Waves a SIMD holds: as many as LDS does (a wave takes 1.5 KB and 64 D bytes of a CU's 160 KB), or fewer for the registers of
// fp32 rows' parts.
template <typename T, int D> constexpr int waves_per_simd() { return D == 256 ? (sizeof(T) == 4 ? 1 : 2) : (sizeof(T) == 4 && D == 128 ? 2 : 4); }

template <typename T> struct Parts;
template <> struct Parts<bf16_t> { static constexpr int Q = 1, P = 2; };
template <> struct Parts<_Float16> { static constexpr int Q = 2, P = 2; };
template <> struct Parts<float> { static constexpr int Q = 3, P = 3; };

// The partials of n_act spans into `heads` output rows that follow each other. Every thread calls it. w: [64][16]
// floats, ltot: [16].
template <typename T, int D>
__device__ __forceinline__ void join(T* out, int heads, const float* parts, int n_act, float* w, float* ltot) {
  constexpr int BATCH = 8;
  const int tid = threadIdx.x, lane = tid & 63, stride = part_floats(heads, D), columns = heads * D / 4;
  const CoherentRows rows(parts);  // under 2 GiB
  float4 x[BATCH];
  auto fetch = [&](int c, int s0) {
#pragma unroll
    for (int s = 0; s < BATCH; ++s) x[s] = rows.load4(4 * (min(s0 + s, n_act - 1) * stride + 4 * c));
  };
  if (tid < columns) fetch(tid, 0);  // beside the weights' loads
  __syncthreads();
  for (int h = tid / 64; h < heads; h += LSA_WAVES) {  // a head a wave, a span a lane
    const float* p = parts + (int64_t)min(lane, n_act - 1) * stride + heads * D + h;
    const float m = coherent_load(p), l = coherent_load(p + heads);
    const float f = lane < n_act ? fast_exp2(m - wave_max(m)) : 0.0f;
    const float ll = wave_sum(f * l);
    if (lane < n_act) w[lane * kHeads + h] = f;
    if (lane == 0) ltot[h] = ll;
  }
  __syncthreads();
  for (int c = tid; c < columns; c += LSA_BLOCK) {
    const int h = 4 * c / D;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < n_act; s0 += BATCH) {
      if (c != tid || s0 > 0) fetch(c, s0);
#pragma unroll
      for (int s = 0; s < BATCH; ++s) {
        const float f = s0 + s < n_act ? w[(s0 + s) * kHeads + h] : 0.0f;
        acc.x += f * x[s].x; acc.y += f * x[s].y; acc.z += f * x[s].z; acc.w += f * x[s].w;
      }
    }
    const float inv = inverse(ltot[h]);
    store4<T>(out + 4 * c, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  }
}

template <typename T, int D, typename C>
__global__ __launch_bounds__(LSA_BLOCK) __attribute__((amdgpu_waves_per_eu(waves_per_simd<T, D>(), waves_per_simd<T, D>())))
void byte_read_kernel(ByteReadArgs a) {
  constexpr int SEGS = D / 16, NI = D / 32;     // 16-byte segments of a row; DMAs of a tile, K and V each
  constexpr int KS = D / 32, DB = D / 16;       // matrix steps over the dims; 16-dim blocks of the output
  constexpr int RPI = 64 / SEGS;                // rows of a DMA
  constexpr int QP = Parts<T>::Q, PP = Parts<T>::P;
  __shared__ __attribute__((aligned(1024))) ByteLds<D> sh;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int row = lane >> 4, col = lane & 15;
  // Workgroup x is on XCD x % 8. The heads of a span follow each other on one XCD: their rows are neighbours in
  // memory, so that the lines of a page are asked for together (sixteen whole caches with a head an XCD: 191 us).
  // The spans of a row are dealt over the XCDs (its place moves by one from span to span), so that rows of many
  // lengths keep all of them busy.
  const uint32_t units = (uint32_t)(a.Hkv * a.blocks), x8 = blockIdx.x / kXcds;  // workgroups of a query row's span
  const uint32_t pair = x8 / units * kXcds + blockIdx.x % kXcds;  // of a span and a query row, span by span
  const uint32_t s0 = pair / a.rows, at = pair - s0 * a.rows + s0 % a.rows;
  const int s = (int)s0;
  if (s >= a.splits) return;
  const uint32_t unit = (at < a.rows ? at : at - a.rows) * units + x8 % units;
  const Unit u(a, unit);
  const int32_t* ids = a.ids + u.list * a.W;
  const int lo = s * a.span + kKeys * w, end = min((s + 1) * a.span, a.W);  // of the list's slots
  const int64_t b = (uint32_t)u.row / a.Tq;
  const uint8_t* kb = a.k + b * a.sb + u.g * a.sh;
  const uint8_t* vb = a.v + b * a.sb + u.g * a.sh;
  const float* scales = a.scales + (b * a.scale_sb + u.g) * 2;
  WaveLds<D>& mem = sh.wave[w];
  lds_char* base = (lds_char*)&mem;
  const uint32_t lds = (uint32_t)(uintptr_t)base;
  constexpr uint32_t V_AT = kKeys * D, S_AT = 2 * kKeys * D, I_AT = S_AT + 512, R_AT = I_AT + 512;

  auto load_ids = [&](int i) {
    const int j = lo + kStep * i + (lane & 31);
    dma4_far(lds + I_AT + (uint32_t)(i & 1) * 256u, ids + min(j, end - 1));
  };
  int hi = 0;                   // past the list's last key here
  uint32_t live[2] = {0u, 0u};  // which keys of tiles of even and odd number count
  uint64_t seg[NI];  // the lane's 16 bytes of a row, by DMA
#pragma unroll
  for (int y = 0; y < NI; ++y) seg[y] = 16u * (uint32_t)((lane % SEGS) ^ swizzle<D>(y * RPI + lane / SEGS));
  auto load_k = [&](int i) {  // and the tile's scales
    const uint32_t buf = (uint32_t)(i & 1);
    const int x = lane & 31, id = ((const lds_int*)(base + I_AT + buf * 256u))[x];
    const bool ok = x < hi - (lo + kStep * i) && id >= 0 && id < a.tokens;
    live[i & 1] = (uint32_t)__ballot(ok);
    const float* p = scales + ((int64_t)((uint32_t)id >> a.block_shift) * a.Hkv) * 2 + (lane >> 5);
    const uint64_t zeros = (uint64_t)(uintptr_t)g_zeros;
    const uint64_t off = (uint64_t)(uint32_t)id * (uint32_t)a.st;
    const uint64_t kr = ok ? (uint64_t)(uintptr_t)kb + off : zeros, vr = ok ? (uint64_t)(uintptr_t)vb + off : zeros;
    *(lds_u64x2*)(base + R_AT + 16 * x) = u64x2_t{kr, vr};
    wait_lds();  // the reads of K's buffer, too
    dma4_far(lds + S_AT + buf * 256u, ok ? (const void*)p : (const void*)g_zeros);
#pragma unroll
    for (int y = 0; y < NI; ++y)
      dma16_far(lds + 1024u * y, (const void*)(uintptr_t)(*(const lds_u64*)(base + R_AT + 16 * (y * RPI + lane / SEGS)) + seg[y]));
  };
  auto load_v = [&]() {  // of the tile whose K was loaded last
    wait_lds();  // the reads of V's buffer
#pragma unroll
    for (int y = 0; y < NI; ++y)
      dma16_far(lds + V_AT + 1024u * y,
                (const void*)(uintptr_t)(*(const lds_u64*)(base + R_AT + 8 + 16 * (y * RPI + lane / SEGS)) + seg[y]));
  };

  // The list's first entries and q come in beside its length.
  if (lo < end) {  // wave-uniform
    load_ids(0);
    load_ids(1);
  }
  // this lane's part of Q^T: head col, dims 16 (row + 4 j) .. + 16 for steps 2 j, 2 j + 1 (D = 32: 8 row .. + 8)
  uint4 q[KS][QP];
  {
    const T* qr = (const T*)a.q + (u.row * a.Hq + u.h0 + (col < u.heads ? col : 0)) * D;
    Raw8<T> raw[KS];
#pragma unroll
    for (int j = 0; j < KS; ++j) raw[j].load(qr + (D == 32 ? 8 * row : 16 * (row + 4 * (j >> 1)) + 8 * (j & 1)));
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      float f[8];
      raw[j].get(f);
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
  }
  wait_vm<0>();  // also where there is nothing to do: no DMA outlives its workgroup
  const int n = u.keys(a), n_act = (n + a.span - 1) / a.span;
  if (s >= max(n_act, 1)) return;
  T* out = (T*)a.out + (u.row * a.Hq + u.h0) * D;
  if (n == 0) {
    for (int j = tid; j < u.heads * D; j += LSA_BLOCK) store_out<T>(out + j, 0.0f);
    return;
  }
  hi = min(end, n);
  const int n_tiles = hi > lo ? (hi - lo + kStep - 1) / kStep : 0;
  float m = kNegBig, l = 0.0f;
  f32x4_t o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  if (n_tiles > 0) {  // wave-uniform
    load_k(0);
    load_v();
  }
  // Memory operations retire in order. V of tile i is the newest at the loop's head; the list of tile i + 1 came before it.
  for (int i = 0; i < n_tiles; ++i) {
    const uint32_t buf = (uint32_t)(i & 1);
    const uint32_t mine = i & 1 ? live[1] : live[0];
    wait_vm<NI>();  // K and scales of tile i, the list of tile i + 1
    // S^T: rows 4 a + u of the first product are keys 8 a + u, of the second 8 a + 4 + u
    f32x4_t c[2];
    const lds_char* kt = base;
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
    const bool more = i + 1 < n_tiles;
    if (more) {
      load_k(i + 1);
      load_ids(i + 2);
      wait_vm<NI + 2>();  // V of tile i
    } else {
      wait_vm<0>();
    }
    f32x4_t ks[2], vs[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      ks[h] = ((const lds_f4*)(base + S_AT + buf * 256u + 32 * row))[h];
      vs[h] = ((const lds_f4*)(base + S_AT + buf * 256u + 128 + 32 * row))[h];
    }
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = c[e >> 2][e & 3] * (ks[e >> 2][e & 3] * a.scale_log2);
    if (mine != ~0u) {  // wave-uniform
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = mine >> (8 * row + e) & 1u ? x[e] : -INFINITY;
    }
    float top = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), fmaxf(x[6], x[7]));
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
      split_pair<PP>(p0 * vs[e >> 1][2 * (e & 1)], p1 * vs[e >> 1][2 * (e & 1) + 1], pr[e]);
    }
    const lds_char* vt = base + V_AT;
    const int vr = 8 * row + (col >> 1);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const i32x2_t y = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2*)(vt + vr * D + 16 * (d ^ swizzle<D>(vr)) + 8 * (col & 1)));
      const uint4 vc = codes_bf16<C>(make_uint2((uint32_t)y[0], (uint32_t)y[1]));
#pragma unroll
      for (int p = 0; p < PP; ++p)
        o[d] = Mfma16<bf16_t>::run(vc, make_uint4(pr[0][p], pr[1][p], pr[2][p], pr[3][p]), o[d]);
    }
    if (more) load_v();
  }

  l += lane_xor(l, 16);
  l += lane_xor(l, 32);
  const int stride = part_floats(u.heads, D);
  float* parts = a.parts + (int64_t)unit * a.splits * (int64_t)part_floats(min(kHeads, a.group), D);
  float* part = parts + (int64_t)s * stride;
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(part, 0, 4 * stride, 0x00020000);
  // the waves' states meet in LDS, each in its wave's own buffers: [16][D]
  float* mo = (float*)&mem;
  if (lane < kHeads) {
    sh.m[w][lane] = m;
    sh.l[w][lane] = l;
  }
#pragma unroll
  for (int d = 0; d < DB; ++d) *(float4*)(mo + col * D + 16 * d + 4 * row) = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
  __syncthreads();
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
      const float inv = inverse(ll);
      store4<T>(out + 4 * t, r[0] * inv, r[1] * inv, r[2] * inv, r[3] * inv);
    } else {
      const f32x4_t z = {r[0], r[1], r[2], r[3]};  // past the XCD's cache (sc1), as CoherentRows reads it
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, z), rsrc, 16 * t, 0, 16);
      if (d == 0) {
        coherent_store(part + u.heads * D + h, top);
        coherent_store(part + u.heads * D + u.heads + h, ll);
      }
    }
  }
  if (n_act == 1 || a.counters == nullptr) return;
  if (!arrive_last(&a.counters[unit], n_act, &sh.flag)) return;
  join<T, D>(out, u.heads, parts, n_act, (float*)&sh.wave[0], &sh.m[0][0]);
}

// The join as a launch of its own, where there are no counters.
template <typename T, int D>
__global__ __launch_bounds__(LSA_BLOCK) void byte_join_kernel(ByteReadArgs a) {
  __shared__ float w[kByteSplits * kHeads];
  __shared__ float ltot[kHeads];
  const Unit u(a, blockIdx.x);
  const int n_act = (u.keys(a) + a.span - 1) / a.span;
  if (n_act <= 1) return;
  join<T, D>((T*)a.out + (u.row * a.Hq + u.h0) * D, u.heads,
             a.parts + (int64_t)blockIdx.x * a.splits * part_floats(min(kHeads, a.group), D), n_act, w, ltot);
}

template <typename T, int D>
void launch_byte_read(const ByteReadArgs& a, int code, int64_t units, hipStream_t s) {
  const int64_t pairs = ((int64_t)a.rows * a.splits + kXcds - 1) / kXcds * kXcds;
  const dim3 grid((unsigned)(pairs * a.Hkv * a.blocks));
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
                             int ids_per_head, float scale, int32_t splits, int32_t* counters,
                             void* scratch, size_t scratch_bytes, void* out, void* stream) {
  LSA_REQUIRE(q && out && (ids || W == 0) && lengths, LSA_ERR_NULL, "lsa_byte_read: NULL pointer");
  LSA_TRY(check_dtype(dtype));
  LSA_REQUIRE(B >= 0 && Tq >= 0 && W >= 0 && W <= 1 << 30, LSA_ERR_SHAPE, "lsa_byte_read: negative size, or a list of more than 2^30");
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
  LSA_REQUIRE((B * Tq * splits + kXcds) * Hkv * blocks <= kMaxGroups, LSA_ERR_SHAPE,
              "lsa_byte_read: %d spans of %lld rows x kv-heads (2^24 workgroups)", splits, (long long)units);
  if (units == 0) return LSA_OK;
  ByteReadArgs a = {};
  a.q = q; a.k = (const uint8_t*)cache->k; a.v = (const uint8_t*)cache->v; a.scales = cache->scales;
  a.sb = cache->caches == 1 ? 0 : cache->batch_stride; a.st = cache->token_stride; a.sh = cache->head_stride;
  a.scale_sb = cache->caches == 1 ? 0 : (cache->tokens + cache->block - 1) / cache->block * Hkv;
  a.tokens = cache->tokens; a.block_shift = __builtin_ctz((unsigned)cache->block);
  a.ids = ids; a.lengths = lengths; a.W = W; a.per_head = ids_per_head ? 1 : 0; a.Tq = (uint32_t)Tq; a.rows = (uint32_t)(B * Tq);
  a.Hq = Hq; a.Hkv = Hkv; a.group = Hq / Hkv; a.blocks = (int)blocks; a.scale_log2 = scale * kLog2e;
  a.span = std::max((int)(((int64_t)W + splits - 1) / splits + kStep - 1) / kStep * kStep, kStep);
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
