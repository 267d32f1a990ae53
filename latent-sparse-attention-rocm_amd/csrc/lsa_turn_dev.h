// Norms and rotary positions of head rows, and 8-bit codes: what rotate.hip and byte_cache.hip share.
//
// A head row of D elements is held by D / 8 lanes, 8 elements a lane, as fp32:
//   y = x / sqrt(mean(x^2) + eps) * w,
//   (y_a, y_b) -> m (y_a cos t - y_b sin t, y_a sin t + y_b cos t),  t = position * frequency_j
// for pair j = (2j, 2j + 1) or (j, j + pairs); dims past 2 * pairs stay. Written for one element i with
// its pair's other one as y' = c y + s y_other, c and s hold the cosine and the signed sine.
// The angle is taken in fp64 as turns (position * frequency / 2 pi less its nearest integer), so that far
// positions lose nothing, and its sine and cosine in fp32.
#pragma once

#include "lsa_read_dev.h"

namespace lsa {

struct TurnArgs {
  const void* freq;
  const void* qw;
  const void* kw;
  int pairs;
  int freq64, interleaved, w32;
  float eps, magnitude;
};

template <int D>
struct HeadLanes {
  static constexpr int LPT = D / 8;             // lanes of a row
  static constexpr int RPW = LSA_WAVE / LPT;    // rows of a wave
  static constexpr int SLOTS = LSA_WAVES * RPW; // rows of a workgroup
};

// Maximum over each group of N consecutive lanes, in every lane of the group (as group_sum).
template <int N>
__device__ __forceinline__ float group_max(float x) {
  if constexpr (N >= 2) x = fmaxf(x, dpp_mov<0xB1>(x));
  if constexpr (N >= 4) x = fmaxf(x, dpp_mov<0x4E>(x));
  if constexpr (N >= 8) x = fmaxf(x, dpp_mov<0x141>(x));
  if constexpr (N >= 16) x = fmaxf(x, dpp_mov<0x140>(x));
  if constexpr (N >= 32) x = fmaxf(x, lane_xor(x, 16));
  return x;
}

// 8 elements, raw.
template <typename T> struct Raw8 {
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = *(const uint4*)p; }
  __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void get(float* f) const { Row16<T>::cvt(u, f); }
};
template <> struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = ((const float4*)p)[0]; b = ((const float4*)p)[1]; }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {  // v_cvt_pk_bf16_f32 (RNE)
  typedef __bf16 v2_t __attribute__((ext_vector_type(2)));
  typedef float f2_t __attribute__((ext_vector_type(2)));
  const f2_t f = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2_t));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  typedef _Float16 v2_t __attribute__((ext_vector_type(2)));
  const v2_t h = {(_Float16)lo, (_Float16)hi};
  return __builtin_bit_cast(uint32_t, h);
}
// 8 numbers to memory. STREAM: past the caches, for outputs that they could not hold.
typedef uint32_t words4_t __attribute__((ext_vector_type(4)));
template <bool STREAM> __device__ __forceinline__ void store_words(void* p, words4_t x) {
  if constexpr (STREAM) __builtin_nontemporal_store(x, (words4_t*)p);
  else *(words4_t*)p = x;
}
template <bool STREAM = false> __device__ __forceinline__ void store8(float* p, const float* f) {
  const words4_t lo = {__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
  const words4_t hi = {__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])};
  store_words<STREAM>(p, lo);
  store_words<STREAM>(p + 4, hi);
}
template <bool STREAM = false> __device__ __forceinline__ void store8(bf16_t* p, const float* f) {
  store_words<STREAM>(p, words4_t{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])});
}
template <bool STREAM = false> __device__ __forceinline__ void store8(_Float16* p, const float* f) {
  store_words<STREAM>(p, words4_t{pack_f16(f[0], f[1]), pack_f16(f[2], f[3]), pack_f16(f[4], f[5]), pack_f16(f[6], f[7])});
}

constexpr double kPerTurn = 0.15915494309189533577;  // 1 / (2 pi)

__device__ __forceinline__ double turn_frequency(const TurnArgs& a, int j) {
  return a.freq64 ? ((const double*)a.freq)[j] : (double)((const float*)a.freq)[j];
}
// (cos, sin) * magnitude of an angle in turns.
__device__ __forceinline__ float2 turn_angle(const TurnArgs& a, double turns) {
  const float x = (float)(turns - rint(turns));
  float s, c;
  sincospif(2.0f * x, &s, &c);
  return make_float2(c * a.magnitude, s * a.magnitude);
}

// A token's angles in LDS: the cosines of its pairs, then their sines.
template <int D>
struct alignas(16) Angles {
  float c[D / 2], s[D / 2];
  __device__ __forceinline__ void put(int j, float2 cs) {
    c[j] = cs.x;
    s[j] = cs.y;
  }
};

// This lane's dims 8 lp .. + 8 of the row's rotation; those that stay: cosine 1, sine 0.
struct LaneTurn {
  float c[8], s[8];
  template <int D>
  __device__ __forceinline__ void load(const TurnArgs& a, const Angles<D>& angles, int lp) {
    if (!a.interleaved && (a.pairs & 7) == 0) {  // eight angles in a row, one side of their pairs
      const bool in = 8 * lp < 2 * a.pairs, low = 8 * lp < a.pairs;
      const int j = in ? (low ? 8 * lp : 8 * lp - a.pairs) : 0;
      const float4 c0 = *(const float4*)&angles.c[j], c1 = *(const float4*)&angles.c[j + 4];
      const float4 s0 = *(const float4*)&angles.s[j], s1 = *(const float4*)&angles.s[j + 4];
      const float cc[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
      const float ss[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
      const uint32_t sign = low ? 0x80000000u : 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        c[e] = in ? cc[e] : 1.0f;
        s[e] = in ? __uint_as_float(__float_as_uint(ss[e]) ^ sign) : 0.0f;
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = 8 * lp + e;
      const bool in = i < 2 * a.pairs;
      const bool low = a.interleaved ? (i & 1) == 0 : i < a.pairs;
      const int j = in ? (a.interleaved ? i >> 1 : (low ? i : i - a.pairs)) : 0;
      c[e] = in ? angles.c[j] : 1.0f;
      s[e] = in ? (low ? -angles.s[j] : angles.s[j]) : 0.0f;
    }
  }
};

// The norm's factors of this lane's dims (ones without weights).
template <typename T>
__device__ __forceinline__ void load_weights(const void* w, int w32, int lp, float* f) {
  if (w == nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 1.0f;
  } else if (w32) {
    Raw8<float> r;
    r.load((const float*)w + 8 * lp);
    r.get(f);
  } else {
    Raw8<T> r;
    r.load((const T*)w + 8 * lp);
    r.get(f);
  }
}

template <int D>
__device__ __forceinline__ void norm8(float* y, const float* w, float eps) {
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
  ss = group_sum<HeadLanes<D>::LPT>(ss);
  const float r = rsqrtf(ss * (1.0f / D) + eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = y[e] * r * w[e];
}

// Rotates the row whose dims 8 lp .. + 8 this lane holds. stage: LDS of the row's D floats, where the lanes
// of a row (of one wave) show each other their elements; none: eight zeros, the others of a dim that stays.
__device__ __forceinline__ void turn8(const TurnArgs& a, float* y, const LaneTurn& t, float* stage, const float* none, int lp) {
  if (a.interleaved) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float y0 = y[e], y1 = y[e + 1];
      if (8 * lp + e < 2 * a.pairs) {
        y[e] = t.c[e] * y0 + t.s[e] * y1;
        y[e + 1] = t.c[e + 1] * y1 + t.s[e + 1] * y0;
      }
    }
    return;
  }
  ((float4*)(stage + 8 * lp))[0] = make_float4(y[0], y[1], y[2], y[3]);
  ((float4*)(stage + 8 * lp))[1] = make_float4(y[4], y[5], y[6], y[7]);
  __builtin_amdgcn_wave_barrier();
  float other[8];
  if ((a.pairs & 7) == 0) {  // the lane's other elements are eight in a row
    const float* at = 8 * lp < a.pairs ? stage + 8 * lp + a.pairs : (8 * lp < 2 * a.pairs ? stage + 8 * lp - a.pairs : none);
    const float4 u = ((const float4*)at)[0], v = ((const float4*)at)[1];
    other[0] = u.x; other[1] = u.y; other[2] = u.z; other[3] = u.w;
    other[4] = v.x; other[5] = v.y; other[6] = v.z; other[7] = v.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = 8 * lp + e;
      other[e] = *(i < a.pairs ? stage + i + a.pairs : (i < 2 * a.pairs ? stage + i - a.pairs : none));
    }
  }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = t.c[e] * y[e] + t.s[e] * other[e];
}

// ---------------------------------------------------------------- rows of q and k

struct RotateArgs {
  const void* q;
  const void* k;
  void* q_out;  // [B, T, Hq, D]
  void* k_out;
  const void* pos;  // positions, int32 or int64 at b pos_sb + t, or, without, those from starts[b] on
  int pos64;
  int64_t pos_sb;
  const int32_t* starts;
  const int32_t* lengths;  // or nullptr: T. Zeros are written behind a row's length
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh;
  int Hq, Hkv;
  int T, tokens;   // tokens = B T
  int heads;       // of a workgroup
  TurnArgs turn;
};

template <int D, int TOKENS>
struct alignas(16) RotateLds {
  float stage[LSA_BLOCK * 8 + 8];
  float weights[2][D];
  Angles<D> angles[TOKENS];
};

// The heads [part, part + 1) * heads of TOKENS tokens from TOKENS * group on: a workgroup's work. Its threads take the
// sines of the tokens' pairs first, once for all heads, through LDS; a lane keeps those of its 8 dims in registers
// and walks the heads of its token, so that a wave reads and writes consecutive heads of one token.
template <typename T, int D, int TOKENS, bool STREAM>
__device__ __forceinline__ void rotate_rows(const RotateArgs& a, uint32_t group, uint32_t part, RotateLds<D, TOKENS>& sh) {
  using L = HeadLanes<D>;
  constexpr int ROWS = L::SLOTS / TOKENS;  // heads at a time
  constexpr int AHEAD = 4;                 // rows a lane loads before it works on them
  const int tid = threadIdx.x, lp = tid % L::LPT, slot = tid / L::LPT;
  const int t0 = group * TOKENS;
  const int mine = t0 + slot / ROWS;
  const int token = mine < a.tokens ? mine : a.tokens - 1;
  const int b = token / a.T, t = token - b * a.T;
  const T* q = (const T*)a.q + b * a.q_sb + t * a.q_st + 8 * lp;
  const T* k = (const T*)a.k + b * a.k_sb + t * a.k_st + 8 * lp;
  T* qo = (T*)a.q_out + (int64_t)token * a.Hq * D + 8 * lp;
  T* ko = (T*)a.k_out + (int64_t)token * a.Hkv * D + 8 * lp;
  const int first = part * a.heads + slot % ROWS;
  const int end = mine < a.tokens ? min(a.Hq + a.Hkv, (int)(part + 1) * a.heads) : 0;
  const bool live = a.lengths == nullptr || t < a.lengths[b];

  Raw8<T> raw[AHEAD];
  auto fetch = [&](int h, Raw8<T>& r) {
    if (h >= end) return;
    if (live) r.load(h < a.Hq ? q + h * a.q_sh : k + (h - a.Hq) * a.k_sh);
    else r.zero();
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) fetch(first + i * ROWS, raw[i]);
  for (int i = tid; i < TOKENS * a.turn.pairs; i += LSA_BLOCK) {
    const int n = i / a.turn.pairs, j = i - n * a.turn.pairs;
    const int at = min(t0 + n, a.tokens - 1), row = at / a.T, x = at - row * a.T;
    const int64_t p = row * a.pos_sb + x;
    const int64_t pos = a.pos == nullptr ? (int64_t)a.starts[row] + x
                                         : (a.pos64 ? ((const int64_t*)a.pos)[p] : (int64_t)((const int32_t*)a.pos)[p]);
    sh.angles[n].put(j, turn_angle(a.turn, (double)pos * turn_frequency(a.turn, j) * kPerTurn));
  }
  if (tid < 8) sh.stage[LSA_BLOCK * 8 + tid] = 0.0f;
  if (tid < 2 * L::LPT) {  // the norms' weights, q's and k's: in LDS they leave the registers to a fifth wave a SIMD
    float w[8];
    load_weights<T>(tid < L::LPT ? a.turn.qw : a.turn.kw, a.turn.w32, lp, w);
    store8(&sh.weights[tid / L::LPT][8 * lp], w);
  }
  __syncthreads();
  LaneTurn turn;
  if (a.turn.pairs > 0) turn.load(a.turn, sh.angles[slot / ROWS], lp);
  for (int h0 = first; h0 < end; h0 += AHEAD * ROWS) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int h = h0 + i * ROWS;
      if (h >= end) break;
      float y[8];
      raw[i].get(y);
      fetch(h + AHEAD * ROWS, raw[i]);
      const bool is_q = h < a.Hq;
      if (live) {
        if (is_q ? a.turn.qw != nullptr : a.turn.kw != nullptr) {
          Raw8<float> r;
          float w[8];
          r.load(&sh.weights[is_q ? 0 : 1][8 * lp]);
          r.get(w);
          norm8<D>(y, w, a.turn.eps);
        }
        if (a.turn.pairs > 0) turn8(a.turn, y, turn, sh.stage + slot * D, sh.stage + LSA_BLOCK * 8, lp);
      }
      store8<STREAM>(is_q ? qo + (int64_t)h * D : ko + (int64_t)(h - a.Hq) * D, y);
    }
  }
}

// ---------------------------------------------------------------- 8-bit codes

// put8: the codes of 8 numbers x / scale, inv = 1 / scale. The quotient is rounded as a division rounds it (one
// residual step behind the product), then to the nearest code, ties to even. Finite numbers of at most kMost scales.
struct Int8Code {
  static constexpr float kMost = 127.0f;
  static __device__ __forceinline__ void get8(const uint2& u, float* f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = (float)(int8_t)(u.x >> (8 * e));
      f[4 + e] = (float)(int8_t)(u.y >> (8 * e));
    }
  }
  static __device__ __forceinline__ uint32_t put4(const float* z) {
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(z[e] + 12582912.0f);  // 1.5 2^23: a whole number's low byte is its code
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u),
                                 0x05040100u);
  }
  static __device__ __forceinline__ float odd(float z) { return z != z ? 0.0f : fminf(fmaxf(z, -kMost), kMost); }
};
struct E4m3Code {
  static constexpr float kMost = 448.0f;
  static __device__ __forceinline__ void get8(const uint2& u, float* f) {
    typedef float f2_t __attribute__((ext_vector_type(2)));
    const f2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(u.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(u.x, true);
    const f2_t c = __builtin_amdgcn_cvt_pk_f32_fp8(u.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(u.y, true);
    f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1]; f[4] = c[0]; f[5] = c[1]; f[6] = d[0]; f[7] = d[1];
  }
  static __device__ __forceinline__ uint32_t put4(const float* z) {
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], r, true);
  }
  static __device__ __forceinline__ float odd(float z) { return z != z ? z : fminf(fmaxf(z, -kMost), kMost); }
};

// strange: some of the numbers may be infinite (the largest code) or NaN (e4m3's own, int8's 0).
template <typename C>
__device__ __forceinline__ uint2 put8(const float* x, float scale, float inv, bool strange) {
  float z[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = x[e] * inv;
    z[e] = fmaf(fmaf(-y, scale, x[e]), inv, y);
    if (strange) z[e] = C::odd(fabsf(y) < 3.0e38f ? z[e] : y);  // an infinity has no residual
  }
  return make_uint2(C::put4(z), C::put4(z + 4));
}

}  // namespace lsa
