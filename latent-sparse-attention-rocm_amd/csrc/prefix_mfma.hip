// A shared prefix's partials on the matrix cores (16-bit rows, head dim 64 or 128).
//
// The query rows of a prefix's batch rows, times the kv-head's query group, are the columns of
// S^T = K Q^T and O^T += V^T P^T. A workgroup takes up to 128 columns and one piece of the
// prefix, so every key is read once per 128 columns, where the gather reads it once a row.
//
// KG groups of CG waves, 32 columns a wave, take the piece's tiles in turn, each group with tile
// buffers of its own (two of K and V, filled straight from memory a tile ahead): four groups on
// 32-key tiles for up to 32 or 64 columns, two on 64-key tiles for up to 128. So few columns, too,
// have 64 KB in flight a CU (D = 128), and what bounds them is memory. At the end the groups'
// states meet in LDS and leave as one partial.
//
// A weight enters the matrix cores as one 16-bit number: half a step of it (2^-9 in bf16, 2^-12
// in fp16), independent from key to key; the output is rounded by as much when it is stored.
// The sum l, which lse shows, adds the weights before that rounding. fp16 weights are kept high
// in their range (the largest is 2^12 when the reference moves and stays below 2^15), so the smallest step
// is 2^-36 of it and many small weights beside a large one are not lost.
#include <math.h>

#include <algorithm>

#include "lsa_abi_common.h"
#include "lsa_mfma_dev.h"
#include "lsa_prefix_dev.h"

using namespace lsa;

namespace {

constexpr int kXcds = 8;

template <int KG> constexpr int tile_keys() { return 128 / KG; }

template <int D, int KG, int CG>
struct alignas(1024) PrefixLds {
  union {
    struct {
      uint16_t k[KG][2][tile_keys<KG>() * D];  // 16-byte segments of a row permuted by kseg
      uint16_t v[KG][2][tile_keys<KG>() * D];  // by vseg
    };
    float o[KG][CG][32][D + 4];  // every wave's state (rows 4 banks apart)
  };
  float m[KG][CG][32], l[KG][CG][32];
  int32_t ids[KG][CG][4][64];    // paged: cache rows of the tiles ahead, a wave's own
  int32_t member[32 * CG];       // batch rows whose columns these are
  int count[KG * CG];
};

__device__ __forceinline__ void dma16_far(uint32_t lds, const void* p) {  // a lane's own 64-bit address
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}

// grid: (kv-head, prefix, piece) units in groups of 8, the column blocks of a unit 8 apart, so that
// those which read the same keys share an XCD and its L2.
template <typename T, int D, int KG, int CG, bool PAGED>
__global__ __launch_bounds__(64 * KG * CG) __attribute__((amdgpu_waves_per_eu(KG * CG / 4, KG * CG / 4)))
void prefix_mfma_kernel(PrefixArgs a, int n_cb) {
  using M = Mfma<T>;
  using op_t = typename M::op_t;
  constexpr int KS = D / 16, DB = D / 32, SEGS = D / 8, ROWB = 2 * D;
  constexpr int KT = tile_keys<KG>(), HT = KT / 32;
  constexpr int KPI = 1024 / ROWB;             // keys a dma16 moves
  constexpr int NI = KT / KPI / CG;            // dma16s a wave a tile, K and V each
  constexpr int NW = KG * CG, THREADS = 64 * NW, COLS = 32 * CG;
  constexpr bool HALF = !__is_same(T, bf16_t);
  constexpr float BIAS = HALF ? 12.0f : 0.0f, TOP = HALF ? 15.0f : 8.0f;
  __shared__ PrefixLds<D, KG, CG> sh;

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int kg = w % KG, cg = w / KG;
  const int hh = lane / 32, ln = lane % 32;
  const int GQ = a.Hq / a.Hkv;
  const int64_t clear = (int64_t)gridDim.x * THREADS;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + tid; i < a.B * a.Tq * a.Hkv; i += clear) a.counters[i] = 0;
  const int64_t x = blockIdx.x;
  const int cb = (int)(x / kXcds % n_cb);
  int64_t u = x / kXcds / n_cb * kXcds + x % kXcds;
  const int s = (int)(u % a.splits); u /= a.splits;
  const int g = (int)(u % a.Hkv);
  const int64_t pp = u / a.Hkv;
  if (pp >= a.P) return;
  const int p = (int)pp;
  const Pieces pc = prefix_pieces(a, p);
  if (s >= pc.count) return;

  // the batch rows of this block's columns (column: batch row of the prefix, query row, head)
  const int64_t per = a.Tq * GQ, c0 = (int64_t)cb * COLS;
  const int64_t first = c0 / per;
  int found;
  if (a.prefix_rows == nullptr) {
    if (first >= a.B) return;
    found = (int)min(a.B - first, (int64_t)COLS);
    if (tid < found) sh.member[tid] = (int32_t)(first + tid);
  } else {
    int64_t seen = 0;
    for (int64_t b0 = 0; b0 < a.B && seen < first + COLS; b0 += THREADS) {
      const int64_t b = b0 + tid;
      const bool is = b < a.B && a.prefix_rows[b < a.B ? b : 0] == p;
      const uint64_t mask = __ballot(is);
      if (lane == 0) sh.count[w] = __popcll(mask);
      __syncthreads();
      int64_t at = seen;
#pragma unroll
      for (int y = 0; y < NW; ++y) {
        at += y < w ? sh.count[y] : 0;
        seen += sh.count[y];
      }
      at += __popcll(mask & ((1ull << lane) - 1)) - first;
      if (is && at >= 0 && at < COLS) sh.member[at] = (int32_t)b;
      __syncthreads();
    }
    found = (int)max((int64_t)0, min(seen - first, (int64_t)COLS));
    if (found == 0) return;
  }
  __syncthreads();
  // column c of the block: its query row (b * Tq + t) and head in the group, or row -1
  auto column = [&](int c, int& h) -> int64_t {
    const int64_t e = c0 + c - first * per;  // 32-bit: below COLS + per
    const int mi = (int)((uint32_t)e / (uint32_t)per), r = (int)((uint32_t)e % (uint32_t)per);
    h = r % GQ;
    return mi < found ? (int64_t)sh.member[mi] * a.Tq + r / GQ : -1;
  };
  op_t qop[KS];
  {
    int h;
    int64_t row = column(cg * 32 + ln, h);
    if (row < 0) row = (int64_t)sh.member[0] * a.Tq, h = 0;
    const T* src = (const T*)a.q + (row * a.Hq + (int64_t)g * GQ + h) * D + 8 * hh;
#pragma unroll
    for (int y = 0; y < KS; ++y) qop[y] = __builtin_bit_cast(op_t, *(const uint4*)(src + 16 * y));
  }
#pragma unroll
  for (int y = 0; y < KS; ++y) asm volatile("" ::"v"(qop[y]));  // here: below, waits are counted by hand
  f32x16_t o[DB];
  float m_run = kNegBig, l_run = 0.0f;
#pragma unroll
  for (int d = 0; d < DB; ++d) {
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  }

  const int k0 = s * pc.keys, n_keys = min(pc.keys, pc.n - k0);
  const int n_tiles = (n_keys + KT - 1) / KT;
  const int64_t head = (PAGED ? 0 : p * a.p_sb) + g * a.p_sh;
  const T* kb = (const T*)a.kp + head;
  const T* vb = (const T*)a.vp + head;
  const int32_t* slots = PAGED ? a.slots + p * a.slot_stride + k0 : nullptr;
  const uint32_t k_lds = (uint32_t)(uintptr_t)(lds_char*)&sh.k[kg][0][0];
  const uint32_t v_lds = (uint32_t)(uintptr_t)(lds_char*)&sh.v[kg][0][0];
  const uint32_t i_lds = (uint32_t)(uintptr_t)(lds_char*)&sh.ids[kg][cg][0][0];
  const int64_t st = a.p_st * 2;  // bytes
  const float scale = a.scale_log2;
  uint64_t live[2] = {0ull, 0ull};  // which keys of the two tiles in the buffers count

  // Tile i of the group's (i-th of its turn) into buffer i & 1; this wave moves its share of the rows.
  auto load_ids = [&](int i) {
    const int t = kg + KG * i;
    const int j = min(t, n_tiles - 1) * KT + lane % KT;
    dma4(i_lds + (uint32_t)(i & 3) * 256u, slots, 4u * (uint32_t)min(j, n_keys - 1));
  };
  auto load = [&](int i) {
    const int t = kg + KG * i;
    if (t >= n_tiles) return;  // wave-uniform
    const int n = min(KT, n_keys - t * KT);
    uint64_t ok = ~0ull >> (64 - n);
    int32_t mine = 0;
    if constexpr (PAGED) {
      typedef __attribute__((address_space(3))) const int32_t lds_int;
      const lds_char* at = (const lds_char*)&sh.ids[kg][cg][i & 3][0];
      mine = *(lds_int*)(at + 4 * lane);
      const bool in = mine >= 0 && mine < a.pool && lane < n;
      ok = __ballot(in);
      mine = in ? mine : 0;
    }
    live[i & 1] = ok;
    const uint32_t to = (uint32_t)(i & 1) * (KT * ROWB);
#pragma unroll
    for (int y = 0; y < NI; ++y) {
      const int part = cg * NI + y;
      const int r = part * KPI + lane / SEGS, sg = lane % SEGS;
      const uint32_t ko = (uint32_t)((sg ^ kseg<D>(r)) * 16), vo = (uint32_t)((sg ^ vseg<D>(r)) * 16);
      const uint32_t dst = to + (uint32_t)part * 1024u;
      if constexpr (PAGED) {
        const int64_t off = (int64_t)__shfl(mine, r, 64) * st;
        dma16_far(k_lds + dst, (const char*)kb + off + ko);
        dma16_far(v_lds + dst, (const char*)vb + off + vo);
      } else {
        const uint32_t off = (uint32_t)min(r, n - 1) * (uint32_t)st;
        const int64_t row0 = (int64_t)(k0 + t * KT) * st;
        dma16(k_lds + dst, (const char*)kb + row0, off + ko);
        dma16(v_lds + dst, (const char*)vb + row0, off + vo);
      }
    }
  };
  // Rows that do not count read as zeros, whatever their place in memory holds (every wave of a
  // group writes the same).
  auto blank = [&](int i) {
    const uint64_t ok = live[i & 1];
    const uint32_t at = (uint32_t)(i & 1) * (KT * ROWB);
    for (int y = lane; y < KT * SEGS; y += 64) {
      if (!(ok >> (y / SEGS) & 1u)) {
        *(uint4*)((char*)&sh.k[kg][0][0] + at + 16 * y) = make_uint4(0u, 0u, 0u, 0u);
        *(uint4*)((char*)&sh.v[kg][0][0] + at + 16 * y) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };

  const int jj = (lane % 16) / 4;
  const uint32_t kbase = (uint32_t)(ln * ROWB) + (uint32_t)((hh ^ kseg<D>(ln)) * 16);
  const uint32_t vbase = (uint32_t)((4 * hh + jj) * ROWB + 32 * (ln / 16) + 8 * (lane % 4));
  auto compute = [&](int i) {
    typedef __attribute__((address_space(3))) const op_t lds_op;
#pragma unroll
    for (int half = 0; half < HT; ++half) {
      const uint32_t ok = (uint32_t)(live[i & 1] >> (32 * half));
      const lds_char* kt = (const lds_char*)&sh.k[kg][i & 1][0] + half * 32 * ROWB;
      const lds_char* vt = (const lds_char*)&sh.v[kg][i & 1][0] + half * 32 * ROWB + vbase;
      f32x16_t sc;
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = 0.0f;
#pragma unroll
      for (int y = 0; y < KS; ++y) sc = M::run(*(lds_op*)(kt + (kbase ^ (uint32_t)(32 * y))), qop[y], sc);
      if (ok != ~0u) {  // uniform
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = ok >> (8 * (r / 4) + 4 * hh + r % 4) & 1u ? sc[r] : -INFINITY;
      }
      float mt = sc[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mt = fmaxf(mt, sc[r]);
      mt = fmaxf(mt, lane_xor(mt, 32)) * scale;
      const bool moves = mt > m_run + TOP;
      if (__any(moves)) {
        const float mn = moves ? mt - BIAS : m_run;
        const float alpha = fast_exp2(m_run - mn);
        m_run = mn;
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
        }
      }
      float ls[2] = {0.0f, 0.0f};
      uint32_t ph[8];
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = fast_exp2(fmaf(sc[r], scale, -m_run)), p1 = fast_exp2(fmaf(sc[r + 1], scale, -m_run));
        ls[0] += p0;
        ls[1] += p1;
        ph[r / 2] = M::pack2(p0, p1);
      }
      l_run += ls[0] + ls[1];
#pragma unroll
      for (int sp = 0; sp < 2; ++sp) {
        const op_t pb = __builtin_bit_cast(op_t, make_uint4(ph[4 * sp], ph[4 * sp + 1], ph[4 * sp + 2], ph[4 * sp + 3]));
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const lds_char* vd = vt + (uint32_t)(64 * (D == 128 ? (d ^ jj) : (d ^ (jj >> 1))));
          const uint2 lo = v_column4(vd, 16 * sp * ROWB), hi = v_column4(vd, (16 * sp + 8) * ROWB);
          o[d] = M::run(__builtin_bit_cast(op_t, make_uint4(lo.x, lo.y, hi.x, hi.y)), pb, o[d]);
        }
      }
    }
  };

  const int turns = (n_tiles + KG - 1) / KG;
  if constexpr (PAGED) {
    load_ids(0);
    load_ids(1);
    wait_vm<0>();
  }
  load(0);
  for (int i = 0; i < turns; ++i) {
    // tile i (and the cache rows of the next) landed, by this wave and its neighbour, and both
    // through with tile i - 1
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    if constexpr (CG > 1) phase_barrier();
    if (i + 1 < turns) {
      load(i + 1);
      if constexpr (PAGED) load_ids(i + 2);
    }
    if (kg + KG * i < n_tiles) {  // wave-uniform
      if (live[i & 1] != ~0ull >> (64 - KT)) {
        blank(i);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      compute(i);
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // nothing lands after this
  __syncthreads();

  // the groups' states into one partial a column
  {
    const float l = l_run + lane_xor(l_run, 32);
    if (hh == 0) {
      sh.m[kg][cg][ln] = m_run;
      sh.l[kg][cg][ln] = l;
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) {
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        *(float4*)&sh.o[kg][cg][ln][32 * d + 8 * r4 + 4 * hh] =
            make_float4(o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]);
    }
  }
  __syncthreads();
  const int pstride = GQ * (D + 2);
  for (int y = tid; y < COLS * (D / 4); y += THREADS) {
    const int c = y / (D / 4), d4 = y % (D / 4), oc = c / 32, cl = c % 32;
    int h;
    const int64_t row = column(c, h);
    if (row < 0) continue;
    float mm = kNegBig;
#pragma unroll
    for (int z = 0; z < KG; ++z) mm = fmaxf(mm, sh.m[z][oc][cl]);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float ll = 0.0f;
#pragma unroll
    for (int z = 0; z < KG; ++z) {
      const float f = fast_exp2(sh.m[z][oc][cl] - mm);
      const float4 v = *(const float4*)&sh.o[z][oc][cl][4 * d4];
      acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
      ll += f * sh.l[z][oc][cl];
    }
    float* part = a.parts + ((row * a.Hkv + g) * (a.splits + a.own_splits) + a.splits - pc.count + s) * (int64_t)pstride;
    float* to = part + 2 * GQ + h * D + 4 * d4;  // 8-byte aligned
    *(float2*)to = make_float2(acc.x, acc.y);
    *(float2*)(to + 2) = make_float2(acc.z, acc.w);
    if (d4 == 0) {
      part[h] = mm;
      part[GQ + h] = ll;
    }
  }
}

int64_t prefix_units(const PrefixArgs& a) { return ((int64_t)a.P * a.Hkv * a.splits + kXcds - 1) / kXcds * kXcds; }

// Column blocks of a prefix, at most (it has as many as it has rows).
int64_t column_blocks(const PrefixArgs& a, int64_t columns) {
  const int64_t wg = prefix_mfma_columns(columns);
  return (a.B * a.Tq * (a.Hq / a.Hkv) + wg - 1) / wg;
}

template <typename T, int D, int KG, int CG>
void launch_mfma(const PrefixArgs& a, int n_cb, hipStream_t s) {
  const dim3 grid((unsigned)(prefix_units(a) * n_cb));
  if (a.slots) prefix_mfma_kernel<T, D, KG, CG, true><<<grid, 64 * KG * CG, 0, s>>>(a, n_cb);
  else prefix_mfma_kernel<T, D, KG, CG, false><<<grid, 64 * KG * CG, 0, s>>>(a, n_cb);
}

template <typename T, int D>
void launch_mfma_cols(const PrefixArgs& a, int64_t columns, hipStream_t s) {
  const int64_t wg = prefix_mfma_columns(columns);
  const int n_cb = (int)column_blocks(a, columns);
  if (wg == 32) launch_mfma<T, D, 4, 1>(a, n_cb, s);
  else if (wg == 64) launch_mfma<T, D, 4, 2>(a, n_cb, s);
  else launch_mfma<T, D, 2, 4>(a, n_cb, s);
}

}  // namespace

namespace lsa {

bool prefix_mfma_ok(int dtype, int D) { return dtype != LSA_F32 && (D == 64 || D == 128); }

int64_t prefix_mfma_columns(int64_t columns) { return columns <= 32 ? 32 : (columns <= 64 ? 64 : 128); }

bool launch_prefix_mfma(const PrefixArgs& a, int dtype, int D, int64_t columns, hipStream_t s) {
  // a lane's offset within a tile is 32 bits of bytes
  if (!prefix_mfma_ok(dtype, D) || a.p_st >= (int64_t)1 << 25 || prefix_units(a) * column_blocks(a, columns) > 0x7FFFFFFF)
    return false;
  if (dtype == LSA_BF16) {
    if (D == 64) launch_mfma_cols<bf16_t, 64>(a, columns, s);
    else launch_mfma_cols<bf16_t, 128>(a, columns, s);
  } else {
    if (D == 64) launch_mfma_cols<_Float16, 64>(a, columns, s);
    else launch_mfma_cols<_Float16, 128>(a, columns, s);
  }
  return true;
}

}  // namespace lsa
