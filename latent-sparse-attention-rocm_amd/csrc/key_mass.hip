// The attention weight that each listed key received, added up over query rows, for gfx950.
//
//   mass[b, g, key] += sum over batch row b's query rows and the group's heads of
//                      2^(s - m) / l,   s = q . k scale log2(e),
// with m and l the row's own (the softmax over its list) or, from a given lse, a wider
// softmax's. K alone is read.
//
//   mass_scores_kernel  gathers the listed K rows and leaves their scores and each span's
//                       (maximum, sum) a head;
//   mass_add_kernel     turns the scores into weights and adds them. With one query row a cache the last span
//                       of a list to finish does that within the first launch, if it has counters
//                       to tell which that is (a launch costs the host 3 us, as much as the rest of a small
//                       call). A small call is one chain of latencies: 2564 keys of 8 kv-heads, 9.5 us (1.2
//                       until the keys' rows are asked for, 2 for their scores, 1.6 to tell who is last, 1 for
//                       the sums, 4 to add), 640 fp32 keys of 2 kv-heads 7.4.
//                       32 such rows: 35.5 us, the gather's 4.8 TB/s.
//
// A key that a list names twice counts twice; several query rows of one cache add to the same
// keys. Sums must not depend on the order in which workgroups arrive. With one query row a cache, all
// additions to a key come from one list and are the same number, so fp32 atomics will do.
// With more, the weights go to 64-bit integers of 2^-44 first (integer sums have no order;
// 2^-45 of rounding a weight, against 2^-24 of the fp32 sum: a weight below that counts as none), and
// mass_fold_kernel adds those to the fp32 weights. The weights that a softmax gives a key are 1 together at most,
// and 2^19 softmaxes fit. Those by a given lse are so only if it is a wider softmax's: each is held to 1, and
// the integers' unit is as large as it has to be for every slot of every list to hold 1 for one key (2^-44 up to
// 2^19 slots times heads a cache, 2^-37 at 2^26).
#include <math.h>

#include <algorithm>

#include "lsa_abi_common.h"
#include "lsa_read_dev.h"

using namespace lsa;

namespace {

constexpr int kFixBits = 44;           // a key's weights add up to less than 2^20 in units of 2^-44
constexpr int64_t kMaxRows = 1 << 19;  // so of softmaxes (one a row and head) at most this a cache
constexpr float kMaxWeight = 1.0f;     // a given lse may be off; a weight is at most this

struct MassArgs {
  const void* q;
  const void* k;
  const int32_t* ids;
  const int32_t* lengths;
  const float* lse;       // [rows, Hq] or nullptr
  int64_t Tq, Tk;
  int64_t k_sb, k_st, k_sh;
  int Hq, Hkv, W, per_head;
  float scale_log2;
  int span;               // list slots of a workgroup of mass_scores_kernel
  int n_span;
  float* scores;          // [units, W, GQ], log2 domain
  float* stats;           // [units, n_span, GQ, 2]
  float* mass;
  int64_t m_sb, m_sh;     // batch stride 0: one pool for every batch row
  int64_t m_n;            // caches * Hkv * Tk (zero: fresh weights are written whole)
  int caches;
  int* counters;          // one launch: arrivals of a unit's spans, zero before and after; or nullptr
  int zero;               // the weights begin at zero
  uint64_t* fixed;        // [caches, Hkv, Tk] or nullptr
  float fix;              // of them, one over the unit
  int whole;              // fixed is cleared and folded whole, not by the lists
};

// 16 bytes written through (visible to the workgroup that adds), from a workgroup-uniform base
struct CoherentOut {
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ __forceinline__ explicit CoherentOut(float* base)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(base, 0, 0x7FFFFFFF, 0x00020000)) {}
  __device__ __forceinline__ void store4(int byte_offset, const float (&x)[4]) const {
    typedef int i4v __attribute__((ext_vector_type(4)));
    const i4v v = {__float_as_int(x[0]), __float_as_int(x[1]), __float_as_int(x[2]), __float_as_int(x[3])};
    __builtin_amdgcn_raw_buffer_store_b128(v, rsrc, byte_offset, 0, 16 /* sc1 */);
  }
};

struct MassList {
  const int32_t* ids;
  int n;
};

__device__ __forceinline__ MassList mass_list(const MassArgs& a, int64_t row, int g) {
  const int64_t li = a.per_head ? row * a.Hkv + g : row;
  int n = a.lengths[li];
  n = n < 0 ? 0 : (n > a.W ? a.W : n);
  return {a.ids + li * a.W, n};
}

// (maximum, sum of 2^(x - maximum)) joined with another's
__device__ __forceinline__ void join(float& m, float& l, float mo, float lo) {
  const float mn = fmaxf(m, mo);
  l = l * fast_exp2(m - mn) + lo * fast_exp2(mo - mn);
  m = mn;
}

template <int GQ>
struct WeighLds {
  float pm[LSA_WAVES][GQ], pl[LSA_WAVES][GQ];
  float m[GQ], inv[GQ];  // the reference, and one over the sum
};

// What the unit's weights are measured by, the spans' statistics a span and head a thread. Every thread calls
// it; a barrier before `sh` is read.
template <int GQ, bool COHERENT>
__device__ __forceinline__ void weigh_by(const MassArgs& a, int64_t unit, int64_t row, int g, const MassList& list,
                                         WeighLds<GQ>& sh) {
  const int tid = threadIdx.x, lane = tid & (LSA_WAVE - 1), w = tid / LSA_WAVE;
  float m = kNegBig, l = 0.0f;
  if (a.lse) {
    if (tid < GQ) {
      m = a.lse[row * a.Hq + g * GQ + tid] * kLog2e;
      l = m > -INFINITY ? 1.0f : 0.0f;  // no keys at all, or not a number: no weight
    }
  } else {
    const int n_act = (list.n + a.span - 1) / a.span;
    const float* st = a.stats + unit * a.n_span * (GQ * 2);
    for (int i = tid; i < n_act * GQ; i += LSA_BLOCK) {
      if constexpr (COHERENT) join(m, l, coherent_load(st + 2 * i), coherent_load(st + 2 * i + 1));
      else join(m, l, st[2 * i], st[2 * i + 1]);
    }
#pragma unroll
    for (int x = GQ; x < LSA_WAVE; x <<= 1) join(m, l, lane_xor(m, x), lane_xor(l, x));
    if (n_act * GQ > LSA_WAVE) {  // uniform: more than the first wave's
      if (lane < GQ) {
        sh.pm[w][lane] = m;
        sh.pl[w][lane] = l;
      }
      __syncthreads();
      if (tid < GQ) {
#pragma unroll
        for (int y = 1; y < LSA_WAVES; ++y) join(m, l, sh.pm[y][tid], sh.pl[y][tid]);
      }
    }
  }
  if (tid < GQ) {
    sh.m[tid] = m;
    sh.inv[tid] = l > 0.0f ? 1.0f / l : 0.0f;  // a sum that is not a number counts as none, as in the read
  }
}

// Slot j's scores, and its weight, the heads together.
template <int GQ, bool COHERENT>
__device__ __forceinline__ void scores_of(const float* scores, int64_t j, float (&s)[GQ]) {
  if constexpr (COHERENT && GQ % 4 == 0) {
#pragma unroll
    for (int h = 0; h < GQ; h += 4) {
      const float4 x = CoherentRows(scores).load4(4 * ((int)j * GQ + h));
      s[h] = x.x; s[h + 1] = x.y; s[h + 2] = x.z; s[h + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int h = 0; h < GQ; ++h) s[h] = COHERENT ? coherent_load(scores + j * GQ + h) : scores[j * GQ + h];
  }
}
template <int GQ>
__device__ __forceinline__ float weight_of(const float (&s)[GQ], const WeighLds<GQ>& sh) {
  float sum = 0.0f;
#pragma unroll
  for (int h = 0; h < GQ; ++h) {
    const float x = fast_exp2(s[h] - sh.m[h]) * sh.inv[h];
    sum += sh.inv[h] > 0.0f && x > 0.0f ? fminf(x, kMaxWeight) : 0.0f;
  }
  return sum;
}

typedef uint32_t raw_t __attribute__((ext_vector_type(4)));  // 16 bytes of a row, kept in registers

template <typename T, int D>
struct MassShape {
  static constexpr bool MM = sizeof(T) == 2;             // scores on the matrix cores
  static constexpr int VEC = Row16<T>::N;
  static constexpr int LPT = D / VEC;                    // lanes that load a token
  static constexpr int TPW = MM ? 16 : LSA_WAVE / LPT;   // tokens of a wave's step
  static constexpr int LD = MM ? D / 32 : 1;             // 16-byte loads a lane a step
  static constexpr int U = MM ? (D == 256 ? 2 : 4) : 4;  // steps in flight
  static constexpr int TW = TPW * U;                     // tokens of a wave's turn
  static constexpr int NT = LSA_WAVES * TW;
};

// grid (row * Hkv, span). Matrix-core form: 16 tokens a wave's step, Q as the A operand (heads
// past the group are zero rows), K as the B operand: lane (row, col) holds dims 32 i + 8 row .. + 8 of
// token col and receives the scores of heads 4 row .. + 3 against it. Loading K so would touch 16 tokens
// with every 16 lanes, which the cache serves a line a lane: 53 cycles a load of 1 KB where 16 would do,
// 69 us for 64 rows of 4096 keys on 8 kv-heads. So lanes load whole rows, D / 8 lanes a token, and the wave
// turns them through LDS of its own: 50 us.
template <typename T, int D, int GQ>
__global__ __launch_bounds__(LSA_BLOCK) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 2 && D <= 128 ? 4 : 1)))
void mass_scores_kernel(MassArgs a) {
  using S = MassShape<T, D>;
  constexpr int U = S::U, TPW = S::TPW, NT = S::NT, TW = S::TW;
  constexpr int HL = S::MM ? (GQ < 4 ? GQ : 4) : GQ;  // heads of a lane
  __shared__ float sm[LSA_WAVES][GQ], sl[LSA_WAVES][GQ];
  __shared__ __attribute__((aligned(16))) uint16_t turn[S::MM ? LSA_WAVES : 1][16][S::MM ? D + 8 : 8];
  const int tid = threadIdx.x, lane = tid & (LSA_WAVE - 1), w = tid / LSA_WAVE;
  const int64_t unit = blockIdx.x;
  const int sp = blockIdx.y;
  const int64_t row = unit / a.Hkv;
  const int g = (int)(unit % a.Hkv);
  const MassList list = mass_list(a, row, g);
  const int lo = sp * a.span, hi = min(lo + a.span, list.n);
  const int n_act = (list.n + a.span - 1) / a.span;
  if (a.counters) {
    if (sp >= max(n_act, 1)) return;
    if (a.zero) {  // this span's share of the unit's own weights, which no other unit adds to
      float* m = a.mass + (a.caches > 1 ? row / a.Tq : 0) * a.m_sb + g * a.m_sh;
      const uint32_t n_all = (uint32_t)a.Tk, share = (n_all - 1) / (uint32_t)max(n_act, 1) + 1;  // 32 bits
      const int64_t k0 = (int64_t)share * sp, k1 = min(k0 + share, a.Tk);
      for (int64_t i = k0 + tid; i < k1; i += LSA_BLOCK) coherent_store(m + i, 0.0f);
    }
  } else if (a.zero || a.whole) {  // this workgroup's share of the weights, and of the integers
    const int64_t grid = (int64_t)gridDim.x * gridDim.y * LSA_BLOCK;
    const int64_t at = ((int64_t)sp * gridDim.x + unit) * LSA_BLOCK + tid;
    if (a.zero) {
      for (int64_t i = at; i < a.m_n; i += grid) a.mass[i] = 0.0f;
    }
    if (a.whole) {
      for (int64_t i = at; i < a.m_n; i += grid) a.fixed[i] = 0;
    }
  }
  if (lo >= hi) return;
  const int64_t b = row / a.Tq;
  const int64_t c = a.caches > 1 ? b : 0;
  const T* kb = (const T*)a.k + b * a.k_sb + g * a.k_sh;
  const T* qrow = (const T*)a.q + (row * a.Hq + (int64_t)g * GQ) * D;
  float* scores = a.scores + unit * (int64_t)a.W * GQ;
  uint64_t* fixed = a.fixed && !a.whole ? a.fixed + (c * a.Hkv + g) * a.Tk : nullptr;

  float m[HL], l[HL];
#pragma unroll
  for (int h = 0; h < HL; ++h) {
    m[h] = kNegBig;
    l[h] = 0.0f;
  }
  const int rowq = lane >> 4, col = lane & 15;                   // matrix-core form
  const int tg = S::MM ? col : lane / S::LPT, lp = lane % S::LPT;
  uint4 qm[S::LD];
  float qf[S::MM ? 1 : GQ][S::VEC];
  if constexpr (S::MM) {
#pragma unroll
    for (int i = 0; i < S::LD; ++i) {
      const uint4 x = *(const uint4*)(qrow + (int64_t)(col < GQ ? col : 0) * D + 32 * i + 8 * rowq);
      qm[i] = col < GQ ? x : make_uint4(0u, 0u, 0u, 0u);
    }
  } else {
#pragma unroll
    for (int h = 0; h < GQ; ++h) Row16<T>::cvt(*(const uint4*)(qrow + (int64_t)h * D + lp * S::VEC), qf[h]);
  }
  // slot of token tg of step u: the wave's turn of TW slots (matrix cores), or steps of all waves
  auto slot = [&](int base, int u) {
    return S::MM ? base + w * TW + u * TPW + tg : base + (u * LSA_WAVES + w) * TPW + tg;
  };
  auto id_of = [&](int base) {  // matrix-core form: one id a lane, fetched a turn ahead
    const int j = base + w * TW + lane % TW;
    return list.ids[j < hi ? j : hi - 1];
  };
  int32_t next = S::MM ? id_of(lo) : 0;
  for (int base = lo; base < hi; base += NT) {
    bool ok[U];
    raw_t kr[U][S::LD];
    if constexpr (S::MM) {
      // handed to the lanes that load its row
      int32_t id = next;
      const bool in = base + w * TW + lane % TW < hi && id >= 0 && id < a.Tk;
      if (fixed && in && lane < TW) fixed[id] = 0;
      const uint64_t live = __ballot(in);
      id = in ? id : 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ok[u] = live >> (u * TPW + col) & 1;
#pragma unroll
        for (int i = 0; i < S::LD; ++i) {
          const int32_t mine = __shfl(id, u * TPW + i * (16 / S::LD) + lane / S::LPT, LSA_WAVE);
          kr[u][i] = *(const raw_t*)(kb + (int64_t)mine * a.k_st + 8 * lp);
        }
      }
      next = id_of(base + NT);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = slot(base, u);
        const int32_t id = list.ids[j < hi ? j : hi - 1];
        ok[u] = j < hi && id >= 0 && id < a.Tk;
        kr[u][0] = *(const raw_t*)(kb + (int64_t)(ok[u] ? id : 0) * a.k_st + S::VEC * lp);
        if (fixed && ok[u] && lp == 0) fixed[id] = 0;
      }
    }
    float s[U][HL];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (S::MM) {
        __builtin_amdgcn_wave_barrier();  // the last step's reads before these writes
#pragma unroll
        for (int i = 0; i < S::LD; ++i)
          *(raw_t*)&turn[w][i * (16 / S::LD) + lane / S::LPT][8 * lp] = kr[u][i];
        __builtin_amdgcn_wave_barrier();  // and these before the reads (a wave's LDS operations keep their order)
        f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < S::LD; ++i) x = Mfma16<T>::run(qm[i], __builtin_bit_cast(uint4, *(const raw_t*)&turn[w][col][32 * i + 8 * rowq]), x);
#pragma unroll
        for (int h = 0; h < HL; ++h) s[u][h] = ok[u] ? x[h] * a.scale_log2 : -INFINITY;
      } else {
        float kf[S::VEC];
        Row16<T>::cvt(__builtin_bit_cast(uint4, kr[u][0]), kf);
#pragma unroll
        for (int h = 0; h < HL; ++h) {
          float p = 0.0f;
#pragma unroll
          for (int e = 0; e < S::VEC; ++e) p = fmaf(qf[h][e], kf[e], p);
          p = group_sum<S::LPT>(p);
          s[u][h] = ok[u] ? p * a.scale_log2 : -INFINITY;
        }
      }
    }
#pragma unroll
    for (int h = 0; h < HL; ++h) {
      float mt = m[h];
#pragma unroll
      for (int u = 0; u < U; ++u) mt = fmaxf(mt, s[u][h]);
      float sum = l[h] * fast_exp2(m[h] - mt);
#pragma unroll
      for (int u = 0; u < U; ++u) sum += fast_exp2(s[u][h] - mt);
      m[h] = mt;
      l[h] = sum;
    }
    if (S::MM ? HL * rowq < GQ : lp == 0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = slot(base, u);
        if (j < hi) {
          const int h0 = S::MM ? HL * rowq : 0;
          if (a.counters) {
            if constexpr (HL % 4 == 0) {
#pragma unroll
              for (int h = 0; h < HL; h += 4) {
                const float x[4] = {s[u][h], s[u][h + 1], s[u][h + 2], s[u][h + 3]};
                CoherentOut(scores).store4(4 * (j * GQ + h0 + h), x);
              }
            } else {
#pragma unroll
              for (int h = 0; h < HL; ++h) coherent_store(scores + (int64_t)j * GQ + h0 + h, s[u][h]);
            }
          } else {
            float* to = scores + (int64_t)j * GQ + h0;
#pragma unroll
            for (int h = 0; h < HL; ++h) to[h] = s[u][h];
          }
        }
      }
    }
  }
  // the wave's tokens, then the four waves
  constexpr int FIRST = S::MM ? 1 : S::LPT, LAST = S::MM ? 16 : LSA_WAVE;
#pragma unroll
  for (int x = FIRST; x < LAST; x <<= 1) {
#pragma unroll
    for (int h = 0; h < HL; ++h) join(m[h], l[h], lane_xor(m[h], x), lane_xor(l[h], x));
  }
  if (S::MM ? (col == 0 && HL * rowq < GQ) : lane == 0) {
#pragma unroll
    for (int h = 0; h < HL; ++h) {
      sm[w][(S::MM ? HL * rowq : 0) + h] = m[h];
      sl[w][(S::MM ? HL * rowq : 0) + h] = l[h];
    }
  }
  __syncthreads();
  if (tid < GQ) {
    float mm = sm[0][tid], ll = sl[0][tid];
#pragma unroll
    for (int x = 1; x < LSA_WAVES; ++x) join(mm, ll, sm[x][tid], sl[x][tid]);
    float* st = a.stats + ((unit * a.n_span + sp) * GQ + tid) * 2;
    if (a.counters) {
      coherent_store(st, mm);
      coherent_store(st + 1, ll);
    } else {
      st[0] = mm;
      st[1] = ll;
    }
  }
  if (!a.counters) return;
  __shared__ int flag;
  __shared__ WeighLds<GQ> by;
  if (!arrive_last(&a.counters[unit], n_act, &flag)) return;
  // E slots of a thread at once, and two steps' scores loaded ahead: a load comes back after the atomics
  // issued before it (one slot at a time: 8 us of 12 for a list of 2564)
  constexpr int E = GQ == 8 ? 2 : 4, AHEAD = 3, STEP = E * LSA_BLOCK;
  float* mass = a.mass + c * a.m_sb + g * a.m_sh;
  int32_t id[AHEAD][E];
  float s[AHEAD][E][GQ];
  auto load = [&](int j0, int (&id)[E], float (&s)[E][GQ]) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = min(j0 + e * LSA_BLOCK + tid, list.n - 1);
      id[e] = list.ids[j];
      scores_of<GQ, true>(scores, j, s[e]);
    }
  };
  load(0, id[0], s[0]);
  load(STEP, id[1], s[1]);
  weigh_by<GQ, true>(a, unit, row, g, list, by);
  __syncthreads();
  for (int i = 0; i < list.n; i += AHEAD * STEP) {
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) {
      const int j0 = i + x * STEP;
      if (j0 >= list.n) break;  // uniform
      load(j0 + 2 * STEP, id[(x + 2) % AHEAD], s[(x + 2) % AHEAD]);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float sum = weight_of<GQ>(s[x][e], by);
        if (j0 + e * LSA_BLOCK + tid < list.n && id[x][e] >= 0 && id[x][e] < a.Tk && sum > 0.0f)
          atomicAdd(mass + id[x][e], sum);
      }
    }
  }
}

// grid (row * Hkv, slots / 256). Bound by the rate of 64-bit atomics: 64 rows of about 4096 keys on 8
// kv-heads, 2.1 M additions, take 19 us (four slots a thread 20).
template <int GQ>
__global__ __launch_bounds__(LSA_BLOCK) void mass_add_kernel(MassArgs a) {
  __shared__ WeighLds<GQ> by;
  const int tid = threadIdx.x;
  const int64_t unit = blockIdx.x;
  const int64_t row = unit / a.Hkv;
  const int g = (int)(unit % a.Hkv);
  const MassList list = mass_list(a, row, g);
  const int j = blockIdx.y * LSA_BLOCK + tid;
  if (blockIdx.y * LSA_BLOCK >= list.n) return;
  float s[GQ];
  const int at = min(j, list.n - 1);
  const int32_t id = list.ids[at];
  scores_of<GQ, false>(a.scores + unit * (int64_t)a.W * GQ, at, s);
  weigh_by<GQ, false>(a, unit, row, g, list, by);
  __syncthreads();
  if (j >= list.n || id < 0 || id >= a.Tk) return;
  const float sum = weight_of<GQ>(s, by);
  if (!(sum > 0.0f)) return;
  const int64_t c = a.caches > 1 ? row / a.Tq : 0;
  if (a.fixed) {
    atomicAdd((unsigned long long*)a.fixed + (c * a.Hkv + g) * a.Tk + id,
              (unsigned long long)__float2ull_rn(sum * a.fix));
  } else {
    atomicAdd(a.mass + c * a.m_sb + g * a.m_sh + id, sum);
  }
}

// The integers into the weights: whole (grid-stride over the caches), or by the lists, where the first
// to take a key's integer (leaving zero) adds it.
__global__ __launch_bounds__(LSA_BLOCK) void mass_fold_kernel(MassArgs a) {
  if (a.whole) {
    const int64_t grid = (int64_t)gridDim.x * LSA_BLOCK;
    for (int64_t i = (int64_t)blockIdx.x * LSA_BLOCK + threadIdx.x; i < a.m_n; i += grid) {
      const uint64_t x = a.fixed[i];
      if (x == 0) continue;
      const int64_t cg = i / a.Tk;
      float* m = a.mass + (cg / a.Hkv) * a.m_sb + (cg % a.Hkv) * a.m_sh + i % a.Tk;
      *m += (float)((double)x / (double)a.fix);
    }
    return;
  }
  const int64_t unit = blockIdx.x;
  const int64_t row = unit / a.Hkv;
  const int g = (int)(unit % a.Hkv);
  const MassList list = mass_list(a, row, g);
  const int j = blockIdx.y * LSA_BLOCK + threadIdx.x;
  if (j >= list.n) return;
  const int32_t id = list.ids[j];
  if (id < 0 || id >= a.Tk) return;
  const int64_t c = a.caches > 1 ? row / a.Tq : 0;
  const uint64_t x = atomicExch((unsigned long long*)a.fixed + (c * a.Hkv + g) * a.Tk + id, 0ull);
  if (x) a.mass[c * a.m_sb + g * a.m_sh + id] += (float)((double)x / (double)a.fix);
}

// Bits below one of the integers. rows: query rows of a cache.
int mass_fix_bits(int64_t rows, int gq, int32_t W, bool given) {
  int slots = 0;
  if (given) {
    while (slots < 62 && (int64_t)1 << slots < rows * gq * W) ++slots;
  }
  return std::min(kFixBits, 63 - slots);
}

int mass_span(int dtype, int D, int64_t units, int W) {
  const int nt = LSA_WAVES * (dtype == LSA_F32 ? LSA_WAVE / (D / 4) * 4 : (D == 256 ? 32 : 64));  // MassShape::NT
  const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(units, 1));  // workgroups a list
  const int tiles = (W + nt - 1) / nt;
  const int per = (int)((tiles + want - 1) / want);
  return (per > 0 ? per : 1) * nt;
}

struct MassPlan {
  int span, n_span;
  bool fixed, whole;
  size_t scores, stats, fix, total;
};

MassPlan mass_plan(int dtype, int64_t B, int64_t Tq, int64_t caches, int64_t Tk, int32_t Hq, int32_t Hkv, int32_t D,
                   int32_t W) {
  MassPlan p;
  const int64_t units = B * Tq * Hkv, gq = Hq / Hkv;
  p.span = mass_span(dtype, D, units, W);
  p.n_span = std::max(1, (W + p.span - 1) / p.span);
  p.fixed = B * Tq > caches;
  const int64_t cells = caches * Hkv * Tk;
  p.whole = p.fixed && cells <= 4 * units * (int64_t)W;
  auto up = [](size_t x) { return (x + 15) / 16 * 16; };
  p.scores = up((size_t)units * W * gq * 4);
  p.stats = up((size_t)units * p.n_span * gq * 8);
  p.fix = p.fixed ? (size_t)cells * 8 : 0;
  p.total = p.scores + p.stats + p.fix;
  return p;
}

template <typename T, int D>
void launch_scores(const MassArgs& a, int gq, dim3 grid, hipStream_t s) {
  switch (gq) {
    case 1: mass_scores_kernel<T, D, 1><<<grid, LSA_BLOCK, 0, s>>>(a); break;
    case 2: mass_scores_kernel<T, D, 2><<<grid, LSA_BLOCK, 0, s>>>(a); break;
    case 4: mass_scores_kernel<T, D, 4><<<grid, LSA_BLOCK, 0, s>>>(a); break;
    default: mass_scores_kernel<T, D, 8><<<grid, LSA_BLOCK, 0, s>>>(a); break;
  }
}

template <typename T>
void launch_scores_d(const MassArgs& a, int D, int gq, dim3 grid, hipStream_t s) {
  switch (D) {
    case 32: launch_scores<T, 32>(a, gq, grid, s); break;
    case 64: launch_scores<T, 64>(a, gq, grid, s); break;
    case 128: launch_scores<T, 128>(a, gq, grid, s); break;
    default: launch_scores<T, 256>(a, gq, grid, s); break;
  }
}

bool mass_shape_ok(int dtype, int64_t B, int64_t Tq, int64_t caches, int64_t Tk, int32_t Hq, int32_t Hkv, int32_t D,
                   int32_t W) {
  if (!(dtype == LSA_F32 || dtype == LSA_BF16 || dtype == LSA_F16)) return false;
  if (!(D == 32 || D == 64 || D == 128 || D == 256) || Hq < 1 || Hkv < 1 || Hq % Hkv) return false;
  const int gq = Hq / Hkv;
  if (!(gq == 1 || gq == 2 || gq == 4 || gq == 8)) return false;
  // a launch holds fewer than 2^32 threads along an axis
  return B >= 0 && Tq >= 0 && B <= 0x7FFFFFFF && Tq <= 0x7FFFFFFF && Tk >= 0 && Tk <= 0x7FFFFFFF && W >= 0 &&
         (caches == B || caches == 1) && B * Tq <= 0xFFFFFFFFll / LSA_BLOCK / Hkv &&
         (B * Tq <= caches || B * Tq <= caches * (kMaxRows / gq));
}

}  // namespace

extern "C" size_t lsa_key_mass_scratch_bytes(int dtype, int64_t B, int64_t Tq, int64_t caches, int64_t Tk, int32_t Hq,
                                             int32_t Hkv, int32_t D, int32_t W) {
  if (!mass_shape_ok(dtype, B, Tq, caches, Tk, Hq, Hkv, D, W) || B * Tq == 0 || W == 0 || Tk == 0) return 0;
  return mass_plan(dtype, B, Tq, caches, Tk, Hq, Hkv, D, W).total;
}

extern "C" int lsa_key_mass(const void* q, const void* k, int dtype, int64_t B, int64_t Tq, int64_t caches, int64_t Tk,
                            int32_t Hq, int32_t Hkv, int32_t D, int64_t k_batch_stride, int64_t k_token_stride,
                            int64_t k_head_stride, const int32_t* ids, const int32_t* lengths, int32_t W,
                            int ids_per_head, float scale, const float* lse, int zero_first, int32_t* counters,
                            void* scratch, size_t scratch_bytes, float* mass, int64_t mass_batch_stride, int64_t mass_head_stride,
                            void* stream) {
  LSA_REQUIRE(q && k && ids && lengths && mass, LSA_ERR_NULL, "lsa_key_mass: NULL pointer");
  LSA_TRY(check_dtype(dtype));
  LSA_REQUIRE(mass_shape_ok(dtype, B, Tq, caches, Tk, Hq, Hkv, D, W), LSA_ERR_SHAPE,
              "lsa_key_mass: B %lld Tq %lld caches %lld Tk %lld Hq %d Hkv %d D %d W %d (D in {32,64,128,256}, groups of "
              "1/2/4/8, B caches or 1, rows x kv-heads under 2^24, rows x group of a cache up to 2^19)", (long long)B, (long long)Tq, (long long)caches, (long long)Tk, Hq, Hkv, D, W);
  const int64_t e = dtype == LSA_F32 ? 4 : 2;
  LSA_REQUIRE(k_batch_stride >= 0 && k_token_stride >= D && k_head_stride >= D && mass_batch_stride >= 0 &&
                  mass_head_stride >= 0, LSA_ERR_SHAPE, "lsa_key_mass: strides must leave rows apart");
  LSA_REQUIRE((((uintptr_t)q | (uintptr_t)k) & 15) == 0 &&
                  ((k_batch_stride | k_token_stride | k_head_stride) * e) % 16 == 0, LSA_ERR_ALIGN,
              "lsa_key_mass: q and K rows must be 16-byte aligned");
  LSA_REQUIRE(!zero_first || (mass_head_stride == Tk && mass_batch_stride == Hkv * Tk), LSA_ERR_SHAPE,
              "lsa_key_mass: weights that begin at zero must be dense");
  if (B * Tq == 0 || W == 0 || Tk == 0) return LSA_OK;
  const MassPlan p = mass_plan(dtype, B, Tq, caches, Tk, Hq, Hkv, D, W);
  LSA_REQUIRE(scratch && scratch_bytes >= p.total && ((uintptr_t)scratch & 15) == 0, LSA_ERR_WORKSPACE,
              "lsa_key_mass: scratch missing, not 16-byte aligned or %zu < %zu bytes", scratch_bytes, p.total);
  const int64_t units = B * Tq * Hkv;
  const int64_t chunks = ((int64_t)W + LSA_BLOCK - 1) / LSA_BLOCK;
  LSA_REQUIRE(p.n_span <= 65535 && chunks <= 65535, LSA_ERR_SHAPE, "lsa_key_mass: lists of %d slots are too wide", W);
  MassArgs a = {};
  a.q = q; a.k = k; a.ids = ids; a.lengths = lengths; a.lse = lse; a.Tq = Tq; a.Tk = Tk;
  a.k_sb = caches > 1 ? k_batch_stride : 0; a.k_st = k_token_stride; a.k_sh = k_head_stride;
  a.Hq = Hq; a.Hkv = Hkv; a.W = W; a.per_head = ids_per_head ? 1 : 0; a.scale_log2 = scale * kLog2e;
  a.span = p.span; a.n_span = p.n_span;
  a.scores = (float*)scratch;
  a.stats = (float*)((char*)scratch + p.scores);
  a.fixed = p.fixed ? (uint64_t*)((char*)scratch + p.scores + p.stats) : nullptr;
  a.fix = ldexpf(1.0f, mass_fix_bits(B * Tq / caches, Hq / Hkv, W, lse != nullptr));
  a.whole = p.whole ? 1 : 0;
  a.mass = mass; a.m_sb = caches > 1 ? mass_batch_stride : 0; a.m_sh = mass_head_stride;
  // offsets within a unit's scores are 32 bits of bytes
  a.counters = !p.fixed && (int64_t)W * (Hq / Hkv) * 4 <= 0x7FFFFFFF ? counters : nullptr;
  a.m_n = caches * Hkv * Tk; a.caches = (int)caches; a.zero = zero_first ? 1 : 0;
  hipStream_t s = (hipStream_t)stream;
  const int gq = Hq / Hkv;
  const dim3 grid((unsigned)units, (unsigned)p.n_span);
  if (dtype == LSA_BF16) launch_scores_d<bf16_t>(a, D, gq, grid, s);
  else if (dtype == LSA_F16) launch_scores_d<_Float16>(a, D, gq, grid, s);
  else launch_scores_d<float>(a, D, gq, grid, s);
  LSA_LAUNCHED("lsa_key_mass");
  if (a.counters) return LSA_OK;
  const dim3 add((unsigned)units, (unsigned)chunks);
  switch (gq) {
    case 1: mass_add_kernel<1><<<add, LSA_BLOCK, 0, s>>>(a); break;
    case 2: mass_add_kernel<2><<<add, LSA_BLOCK, 0, s>>>(a); break;
    case 4: mass_add_kernel<4><<<add, LSA_BLOCK, 0, s>>>(a); break;
    default: mass_add_kernel<8><<<add, LSA_BLOCK, 0, s>>>(a); break;
  }
  LSA_LAUNCHED("lsa_key_mass");
  if (p.fixed) {
    const dim3 fold = p.whole ? dim3((unsigned)std::min<int64_t>((a.m_n + LSA_BLOCK - 1) / LSA_BLOCK, 4096)) : add;
    mass_fold_kernel<<<fold, LSA_BLOCK, 0, s>>>(a);
    LSA_LAUNCHED("lsa_key_mass");
  }
  return LSA_OK;
}
