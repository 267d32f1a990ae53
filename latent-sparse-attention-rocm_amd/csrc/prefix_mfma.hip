// A shared prefix's partials on the matrix cores (16-bit rows, head dim 64 or 128).
//
// The query rows of a prefix's batch rows, times the kv-head's query group, are the columns of
// S^T = K Q^T and O^T += V^T P^T. A workgroup takes up to 256 columns and one piece of the
// prefix, so every key is read once per block of columns, where the gather reads it once a row.
//
// Up to 128 columns: KG groups of CG waves, 32 columns a wave, take the piece's tiles in turn, each
// group with tile buffers of its own (two of K and V, filled straight from memory a tile ahead): four
// groups on 32-key tiles for up to 32 or 64 columns, two on 64-key tiles for up to 128. So few columns,
// too, have 64 KB in flight a CU (D = 128), and what bounds them is memory: 32768 bf16 keys of 128 on 8
// kv-heads (134 MB) for 128 columns take 34 to 36 us, 10 of them the start and the joining of states.
// (128 columns as four waves of 64 spilled 45 registers: 102 us.) At the end the groups' states meet in
// LDS and leave as one partial. More than 128 columns: the second kernel below.
//
// A weight enters the matrix cores as one 16-bit number: off by at most half a step of it (2^-8 in bf16,
// 2^-11 in fp16), independent from key to key; the output is rounded by as much when it is stored. The
// sum it is divided by adds the same rounded weights, so a row that one key fills returns that key's
// value; the sum that lse shows adds them unrounded, in fp32. fp16 weights are kept high in their range
// (the largest is 2^12 when the reference moves and stays below 2^15), so the smallest step is 2^-36 of
// it and many small weights beside a large one are not lost.
#include <math.h>

#include <algorithm>

#include "lsa_abi_common.h"
#include "lsa_mfma_dev.h"
#include "lsa_prefix_dev.h"

using namespace lsa;

namespace {

constexpr int kXcds = 8;

// A workgroup's place: kv-head, piece, prefix, and the batch rows whose query rows times heads are
// its columns (column: batch row of the prefix, query row, head). The column blocks of all prefixes
// stand in one line, and the grid is that line times the (kv-head, piece) units: which prefix a block
// belongs to follows from how many rows each has, counted here. (A grid of every prefix times the most
// blocks one may have is nearly all empty where prefixes are many: 512 rows over 128 prefixes of 2048
// keys took 820 us so, and take 242; 64 rows over 4000 of 256 keys 1922 and 42.) Into how many pieces a prefix
// is cut follows from the blocks there are, so rows that all read one prefix of a table of many fill the chip
// too (32 rows on one of 32 prefixes of 32768 keys: 48 us, and 259 in as many pieces as if they were spread; 39
// where the table holds that prefix alone, whose rows then stand in wider blocks). Units come in groups of 8, the
// blocks of a unit 8 apart, so that those which read the same keys share an XCD and its L2.
template <int COLS>
struct PrefixBlock {
  static constexpr int kCount = 1024;  // prefixes counted at once
  struct Lds {
    int32_t member[COLS];  // the batch rows
    int32_t row[COLS];     // a column's query row (b * Tq + t), -1 past the prefix's rows
    int32_t head[COLS];    // and head in the group
    int count[16];
  };
  int GQ, g, p, s;
  Pieces pc;

  uint32_t cb;  // the prefix's column block

  // How many rows read each of the kCount prefixes from p0 on. Ends with a barrier.
  __device__ __forceinline__ void count(const PrefixArgs& a, int p0, int threads, int* rows) const {
    const int tid = threadIdx.x, np = min(kCount, a.P - p0);
    for (int i = tid; i < np; i += threads) rows[i] = 0;
    __syncthreads();
    for (int64_t b = tid; b < a.B; b += threads) {
      const int64_t r = (int64_t)a.prefix_rows[b] - p0;
      if (r >= 0 && r < np) atomicAdd(&rows[r], 1);
    }
    __syncthreads();
  }
  // The column blocks of the i-th of them (none past the last).
  __device__ __forceinline__ static int blocks_of(const PrefixArgs& a, int p0, int i, uint32_t per, const int* rows) {
    return i < min(kCount, a.P - p0) ? (int)(((uint32_t)rows[i] * per + COLS - 1) / COLS) : 0;
  }

  // False: nothing to do (the whole workgroup). Clears the grid's share of the counters. Contains
  // barriers; `rows`: kCount ints of LDS, free again after it.
  __device__ __forceinline__ bool place(const PrefixArgs& a, uint32_t blocks, int threads, int* rows) {
    const int tid = threadIdx.x, lane = tid & 63;
    GQ = a.Hq / a.Hkv;
    const int64_t clear = (int64_t)gridDim.x * threads;
    for (int64_t i = (int64_t)blockIdx.x * threads + tid; i < a.B * a.Tq * a.Hkv; i += clear) a.counters[i] = 0;
    const uint32_t per = (uint32_t)a.Tq * (uint32_t)GQ;  // columns of a batch row; all are fewer than 2^31
    int splits = a.splits, own = 0, to = 0;
    int of = 0;  // lane c: the blocks of the c-th kCount prefixes (64 times as many at most)
    const bool counted = a.prefix_rows != nullptr && a.P > 1, few = a.P <= 64;
    if (counted && a.P <= kCount) count(a, 0, threads, rows);
    if (counted && few) {  // uniform from here on, as every wave finds the same
      own = blocks_of(a, 0, lane, per, rows);
      to = wave_inclusive_sum(own);
    }
    if (a.plan) {
      blocks = few ? (uint32_t)__builtin_amdgcn_readlane(to, 63) : 0u;
      for (int c = 0; !few && c * kCount < a.P; ++c) {
        if (a.P > kCount) count(a, c * kCount, threads, rows);
        own = 0;
        for (int i0 = 0; i0 < kCount && c * kCount + i0 < a.P; i0 += 64) own += blocks_of(a, c * kCount, i0 + lane, per, rows);
        own = wave_sum(own);
        of = lane == c ? own : of;
        blocks += (uint32_t)own;
        if (a.P > kCount) __syncthreads();  // before the counts' place is used again
      }
      splits = min(splits, prefix_mfma_pieces(blocks, a.Hkv));
      if (blockIdx.x == 0 && tid == 0) *a.plan = splits;
      if (blocks == 0) return false;
    }
    const uint32_t units = (uint32_t)(a.Hkv * splits), together = min(units, (uint32_t)kXcds);
    const uint32_t x = blockIdx.x, xu = x / together;
    cb = xu % blocks;
    const uint32_t u = xu / blocks * together + x % together;
    s = (int)(u % (uint32_t)splits);
    g = (int)(u / (uint32_t)splits);
    if (g >= a.Hkv) return false;
    p = 0;
    if (counted) {
      int p0 = 0;
      if (a.P > kCount) {
        to = wave_inclusive_sum(of);
        const int c = __builtin_ctzll(__ballot((uint32_t)to > cb));
        cb -= (uint32_t)__shfl(to - of, c, 64);
        p0 = c * kCount;
        count(a, p0, threads, rows);
      }
      for (int i0 = 0;; i0 += 64) {
        if (i0 >= min(kCount, a.P - p0)) return false;  // unplanned: fewer blocks than there may be
        if (!few) {
          own = blocks_of(a, p0, i0 + lane, per, rows);
          to = wave_inclusive_sum(own);
        }
        const uint64_t after = __ballot((uint32_t)to > cb);
        if (after != 0ull) {
          const int l = __builtin_ctzll(after);
          p = p0 + i0 + l;
          cb -= (uint32_t)__shfl(to - own, l, 64);
          break;
        }
        cb -= (uint32_t)__shfl(to, 63, 64);
      }
      __syncthreads();  // the counts are read
    } else if (a.prefix_rows == nullptr && a.P > 1) {
      const uint32_t each = (per + COLS - 1) / COLS;
      p = (int)(cb / each);
      cb %= each;
    }
    pc = prefix_pieces(a, p, splits);
    return s < pc.count;
  }
  // The columns; false: none. Contains barriers.
  __device__ __forceinline__ bool columns(const PrefixArgs& a, int threads, Lds& sh) const {
    const int tid = threadIdx.x, lane = tid & 63, w = tid / 64;
    // columns and rows are fewer than 2^31
    const uint32_t per = (uint32_t)a.Tq * (uint32_t)GQ, c0 = cb * COLS, first = c0 / per;
    int found;
    if (a.prefix_rows == nullptr) {
      const int64_t of = a.P > 1 ? 1 : a.B;  // batch rows: p, or all of them
      if (first >= of) return false;
      found = (int)min(of - first, (int64_t)COLS);
      if (tid < found) sh.member[tid] = (a.P > 1 ? p : (int32_t)first) + tid;
    } else {
      int64_t seen = 0;
      for (int64_t b0 = 0; b0 < a.B && seen < (int64_t)first + COLS; b0 += threads) {
        const int64_t b = b0 + tid;
        const bool is = b < a.B && a.prefix_rows[b < a.B ? b : 0] == p;
        const uint64_t mask = __ballot(is);
        if (lane == 0) sh.count[w] = __popcll(mask);
        __syncthreads();
        int64_t at = seen;
        for (int y = 0; y < threads / 64; ++y) {
          at += y < w ? sh.count[y] : 0;
          seen += sh.count[y];
        }
        at += __popcll(mask & ((1ull << lane) - 1)) - (int64_t)first;
        if (is && at >= 0 && at < COLS) sh.member[at] = (int32_t)b;
        __syncthreads();
      }
      found = (int)max((int64_t)0, min(seen - (int64_t)first, (int64_t)COLS));
      if (found == 0) return false;
    }
    __syncthreads();
    if (tid < COLS) {
      const uint32_t e = c0 + tid - first * per, r = e % per;
      const int mi = (int)(e / per);
      sh.row[tid] = mi < found ? sh.member[mi] * (int32_t)a.Tq + (int32_t)(r / (uint32_t)GQ) : -1;
      sh.head[tid] = (int)(r % (uint32_t)GQ);
    }
    __syncthreads();
    return true;
  }
  // Column c's query row in q; past the prefix's rows the first column's.
  template <typename T, int D>
  __device__ __forceinline__ const T* query(const PrefixArgs& a, const Lds& sh, int c) const {
    const int e = sh.row[c] < 0 ? 0 : c;
    return (const T*)a.q + ((int64_t)sh.row[e] * a.Hq + (int64_t)g * GQ + sh.head[e]) * D;
  }
};

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
  float m[KG][CG][32], l[KG][CG][32], l32[KG][CG][32];
  int32_t ids[KG][CG][4][64];    // paged: cache rows of the tiles ahead, a wave's own
  typename PrefixBlock<32 * CG>::Lds block;
};

__device__ __forceinline__ void dma16_far(uint32_t lds, const void* p) {  // a lane's own 64-bit address
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}

// The wave groups' states into one partial a column. Every thread calls it, after a barrier.
template <int D, int KG, int CG, typename Lds>
__device__ __forceinline__ void store_partials(const PrefixArgs& a, Lds& sh, const PrefixBlock<32 * CG>& blk, int kg, int cg,
                                               const f32x16_t (&o)[D / 32], float m_run, float l_run, float l32_run) {
  const int tid = threadIdx.x, lane = tid & 63, hh = lane / 32, ln = lane % 32;
  const float l = l_run + lane_xor(l_run, 32), l32 = l32_run + lane_xor(l32_run, 32);
  if (hh == 0) {
    sh.m[kg][cg][ln] = m_run;
    sh.l[kg][cg][ln] = l;
    sh.l32[kg][cg][ln] = l32;
  }
#pragma unroll
  for (int d = 0; d < D / 32; ++d) {
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4)
      *(float4*)&sh.o[kg][cg][ln][32 * d + 8 * r4 + 4 * hh] =
          make_float4(o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]);
  }
  __syncthreads();
  const int GQ = blk.GQ, pstride = GQ * (D + 2);
  constexpr int STEP = 64 * KG * CG / (D / 4);  // columns of the workgroup at once
  const int d4 = tid % (D / 4);
#pragma unroll 4
  for (int n = 0; n < 32 * CG / STEP; ++n) {
    const int c = tid / (D / 4) + STEP * n, oc = c / 32, cl = c % 32;
    const int h = sh.block.head[c];
    const int64_t row = sh.block.row[c];
    if (row < 0) continue;
    float mm = kNegBig;
#pragma unroll
    for (int z = 0; z < KG; ++z) mm = fmaxf(mm, sh.m[z][oc][cl]);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float ll = 0.0f, ll32 = 0.0f;
#pragma unroll
    for (int z = 0; z < KG; ++z) {
      const float f = fast_exp2(sh.m[z][oc][cl] - mm);
      const float4 v = *(const float4*)&sh.o[z][oc][cl][4 * d4];
      acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
      ll += f * sh.l[z][oc][cl];
      ll32 += f * sh.l32[z][oc][cl];
    }
    const int64_t unit = row * a.Hkv + blk.g;
    const int at = a.splits - blk.pc.count + blk.s;
    float* part = a.parts + (unit * (a.splits + a.own_splits) + at) * (int64_t)pstride;
    float* to = part + 2 * GQ + h * D + 4 * d4;  // 8-byte aligned
    *(float2*)to = make_float2(acc.x, acc.y);
    *(float2*)(to + 2) = make_float2(acc.z, acc.w);
    if (d4 == 0) {
      part[h] = mm;
      part[GQ + h] = ll;
      if (a.lse) a.sums[(unit * a.splits + at) * GQ + h] = ll32;
    }
  }
}

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
  PrefixBlock<COLS> blk;
  if (!blk.place(a, (uint32_t)n_cb, THREADS, (int*)&sh)) return;
  const int g = blk.g, p = blk.p, s = blk.s;
  const Pieces pc = blk.pc;
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

  // a block past the first may have no columns: looked up before anything loads
  if (blk.cb != 0 && !blk.columns(a, THREADS, sh.block)) return;
  if constexpr (PAGED) {
    load_ids(0);
    load_ids(1);
    wait_vm<0>();
  }
  load(0);
  // the first tile is on its way while the columns are looked up
  if (blk.cb == 0 && !blk.columns(a, THREADS, sh.block)) {
    wait_vm<0>();  // nothing lands after the workgroup's LDS is given back
    return;
  }
  op_t qop[KS];
  {
    const T* src = blk.template query<T, D>(a, sh.block, cg * 32 + ln) + 8 * hh;
#pragma unroll
    for (int y = 0; y < KS; ++y) qop[y] = __builtin_bit_cast(op_t, *(const uint4*)(src + 16 * y));
  }
#pragma unroll
  for (int y = 0; y < KS; ++y) asm volatile("" ::"v"(qop[y]));  // here: below, waits are counted by hand
  f32x16_t o[DB];
  float m_run = kNegBig, l_run = 0.0f, l32_run = 0.0f;
#pragma unroll
  for (int d = 0; d < DB; ++d) {
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  }

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
        l32_run *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
        }
      }
      float ls[2] = {0.0f, 0.0f}, l32[2] = {0.0f, 0.0f};
      uint32_t ph[8];
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = fast_exp2(fmaf(sc[r], scale, -m_run)), p1 = fast_exp2(fmaf(sc[r + 1], scale, -m_run));
        l32[0] += p0;
        l32[1] += p1;
        ph[r / 2] = M::pack2(p0, p1);
        ls[r / 2 & 1] = M::sum2(ph[r / 2], ls[r / 2 & 1]);
      }
      l_run += ls[0] + ls[1];
      l32_run += l32[0] + l32[1];
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

  store_partials<D, KG, CG>(a, sh, blk, kg, cg, o, m_run, l_run, l32_run);
}

// ---------------------------------------------------------------- 256 columns
//
// Eight waves of 32 columns share 64-key tiles, four buffers each of K and V. A wave's step is two
// phases: M, the last tile's P V products and this tile's scores (matrix cores and LDS reads), and V, the
// loads ahead and this tile's weights (vector unit). Two groups of four waves, one of each on every SIMD, run
// half a step apart (a barrier after each phase), so one's matrix work runs beside the other's vector work.
//
// A load straight to LDS holds its wave for about 155 cycles (four waves at once: 39 cycles a KB of the
// CU). In M, between the matrix operations, four of them cost 500 cycles; in V they fill time that V has
// left. 131072 keys, 512 columns of 128 on 8 kv-heads: a step takes 4850 cycles with them in M, 3720 in V
// (2048 of them matrix work). At that load the card lowers its clock as the cycles fall, and both take 310
// us, 920 TFLOP/s: power bounds it. A tile is shared by all waves for the same reason: 32 KB a step,
// where two groups on tiles of their own load 64 KB (350 us).
//
// V(i) loads K(i + 3) over K(i - 1) and V(i + 2) over V(i - 2), both read for the last time in M(i - 1) of
// either group. K(i) is read in M(i), V(i) from the end of V(i) on: both were loaded in V(i - 2) or
// earlier, and at the end of V(i - 1) only the loads of that phase may be outstanding.
constexpr int kWideBuf = 4;

template <int D>
struct alignas(1024) WideLds {
  union {
    struct {
      uint16_t k[kWideBuf][64 * D];  // 16-byte segments of a row permuted by kseg
      uint16_t v[kWideBuf][64 * D];  // by vseg
    };
    float o[1][8][32][D + 4];
  };
  float m[1][8][32], l[1][8][32], l32[1][8][32];
  int32_t ids[8][8][64];  // paged: cache rows of eight tiles, a wave's own
  typename PrefixBlock<256>::Lds block;
};

template <typename T, int D, bool PAGED>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void prefix_wide_kernel(PrefixArgs a, int n_cb) {
  using M = Mfma<T>;
  using op_t = typename M::op_t;
  constexpr int KG = 1, CG = 8, KT = 64, COLS = 256, THREADS = 512, NB = kWideBuf;
  constexpr int KS = D / 16, DB = D / 32, SEGS = D / 8, ROWB = 2 * D;
  constexpr int KPI = 1024 / ROWB, NI = KT / KPI / CG;
  constexpr int PER = 2 * NI + (PAGED ? 1 : 0);  // loads of a step
  constexpr int NG = 4 + KS / 2;                 // groups of matrix operations of an M: 4 of P V, the scores
  constexpr bool HALF = !__is_same(T, bf16_t);
  constexpr float BIAS = HALF ? 12.0f : 0.0f, TOP = HALF ? 15.0f : 8.0f;
  typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
  __shared__ WideLds<D> sh;

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid / 64);
  const int hh = lane / 32, ln = lane % 32;
  PrefixBlock<COLS> blk;
  if (!blk.place(a, (uint32_t)n_cb, THREADS, (int*)&sh)) return;
  const int k0 = blk.s * blk.pc.keys, n_keys = min(blk.pc.keys, blk.pc.n - k0);
  const int n_tiles = (n_keys + KT - 1) / KT;
  const int64_t head = (PAGED ? 0 : blk.p * a.p_sb) + blk.g * a.p_sh;
  const T* kb = (const T*)a.kp + head;
  const T* vb = (const T*)a.vp + head;
  const int32_t* slots = PAGED ? a.slots + blk.p * a.slot_stride + k0 : nullptr;
  const uint32_t k_lds = (uint32_t)(uintptr_t)(lds_char*)&sh.k[0][0];
  const uint32_t v_lds = (uint32_t)(uintptr_t)(lds_char*)&sh.v[0][0];
  const uint32_t i_lds = (uint32_t)(uintptr_t)(lds_char*)&sh.ids[w][0][0];
  const int64_t st = a.p_st * 2;  // bytes
  const float scale = a.scale_log2;
  typedef __attribute__((address_space(3))) const int32_t lds_int;

  // past the last tile: that one again, loaded and not used
  auto tile_of = [&](int i) { return min(i, n_tiles - 1); };
  auto keys_of = [&](int t) { return min(KT, n_keys - t * KT); };
  auto load_ids = [&](int i) {
    dma4(i_lds + (uint32_t)(i & 7) * 256u, slots, 4u * (uint32_t)min(tile_of(i) * KT + lane, n_keys - 1));
  };
  // Move y of this wave's eighth of tile i's K or V rows. A lane's offset within the rows of one move is the
  // same for every move but for two bits of K's segment.
  const uint32_t lrow = (uint32_t)(lane / SEGS) * (uint32_t)st;
  const uint32_t kseg0 = (uint32_t)(((lane % SEGS) ^ kseg<D>(lane / SEGS)) * 16);
  const uint32_t vseg0 = (uint32_t)(((lane % SEGS) ^ vseg<D>(lane / SEGS)) * 16);
  auto load = [&](bool values, int i, int y) {
    static_assert(KPI == 512 / D && (D == 64 || D == 128), "moves differ by 64-byte steps of K's segment");
    const int t = tile_of(i), n = keys_of(t), part = w * NI + y;
    const char* src = (const char*)(values ? vb : kb);
    const uint32_t dst = (values ? v_lds : k_lds) + (uint32_t)(i & (NB - 1)) * (KT * ROWB) + (uint32_t)part * 1024u;
    const uint32_t seg = values ? vseg0 : kseg0 ^ (uint32_t)(part % (D == 128 ? 4 : 2) * 64);
    if constexpr (PAGED) {
      const int32_t id = *(lds_int*)((const lds_char*)&sh.ids[w][i & 7][0] + 4 * (part * KPI + lane / SEGS));
      dma16_far(dst, src + (int64_t)(id >= 0 && id < a.pool ? id : 0) * st + seg);
    } else {
      const int64_t row0 = (int64_t)(k0 + t * KT) * st;
      if (n == KT) {  // uniform
        dma16(dst, src + row0 + (int64_t)(part * KPI) * st, lrow + seg);
      } else {  // rows past the last read the last
        dma16(dst, src + row0, (uint32_t)min(part * KPI + lane / SEGS, n - 1) * (uint32_t)st + seg);
      }
    }
  };
  // which keys of tile i count
  auto live_of = [&](int i) -> uint64_t {
    const int n = keys_of(tile_of(i));
    if constexpr (PAGED) {
      const int32_t id = *(lds_int*)((const lds_char*)&sh.ids[w][i & 7][0] + 4 * lane);
      return __ballot(id >= 0 && id < a.pool && lane < n);
    }
    return ~0ull >> (64 - n);
  };
  // V rows of tile i that do not count become zeros, whatever their place in memory holds: this
  // wave's own eighth, landed.
  auto blank = [&](int i) {
    const uint64_t ok = live_of(i);
    if (ok == ~0ull) return;  // uniform
    for (int y = lane; y < KT / CG * SEGS; y += 64) {
      const int r = w * (KT / CG) + y / SEGS;
      if (!(ok >> r & 1u))
        *(uint4*)((char*)&sh.v[i & (NB - 1)][0] + r * ROWB + 16 * (y % SEGS)) = make_uint4(0u, 0u, 0u, 0u);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };

  // a block past the first may have no columns: looked up before anything loads
  if (blk.cb != 0 && !blk.columns(a, THREADS, sh.block)) return;
  if constexpr (PAGED) {
#pragma unroll
    for (int i = 0; i < 6; ++i) load_ids(i);
    wait_vm<0>();
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
#pragma unroll
    for (int y = 0; y < NI; ++y) {
      load(false, i, y);
      if (i < 2) load(true, i, y);
    }
  }
  // the first tiles are on their way while the columns are looked up
  if (blk.cb == 0 && !blk.columns(a, THREADS, sh.block)) {
    wait_vm<0>();  // nothing lands after the workgroup's LDS is given back
    return;
  }
  op_t qop[KS];
  {
    const T* src = blk.template query<T, D>(a, sh.block, w * 32 + ln) + 8 * hh;
#pragma unroll
    for (int y = 0; y < KS; ++y) qop[y] = __builtin_bit_cast(op_t, *(const uint4*)(src + 16 * y));
  }
#pragma unroll
  for (int y = 0; y < KS; ++y) asm volatile("" ::"v"(qop[y]));  // here: below, waits are counted by hand

  f32x16_t o[DB], sc[2];
  uint32_t ph[2][8];  // a tile's weights, two a word
  float m_run = kNegBig, l_run = 0.0f, l32_run = 0.0f;
#pragma unroll
  for (int d = 0; d < DB; ++d) {
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  }
  const int jj = (lane % 16) / 4;
  const uint32_t kbase = (uint32_t)(ln * ROWB) + (uint32_t)((hh ^ kseg<D>(ln)) * 16);
  const uint32_t vbase = (uint32_t)((4 * hh + jj) * ROWB + 32 * (ln / 16) + 8 * (lane % 4));
  // Groups of matrix operations with their LDS operands, read while the two groups before compute:
  // 0 .. 3 are O^T += V^T P^T of 16 keys each, 4 .. the scores at two 16-dim steps each.
  op_t op[3][4];
  auto load_group = [&](int gi, int tile_v, int tile_k) {
    if (gi < 4) {
      const lds_char* vt = (const lds_char*)&sh.v[tile_v & (NB - 1)][0] + vbase;
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const lds_char* vd = vt + (uint32_t)(64 * (D == 128 ? (d ^ jj) : (d ^ (jj >> 1))));
        const uint2 lo = v_column4(vd, 16 * gi * ROWB), hi = v_column4(vd, (16 * gi + 8) * ROWB);
        op[gi % 3][d] = __builtin_bit_cast(op_t, make_uint4(lo.x, lo.y, hi.x, hi.y));
      }
    } else if (gi < NG) {
      typedef __attribute__((address_space(3))) const op_t lds_op;
      const lds_char* kt = (const lds_char*)&sh.k[tile_k & (NB - 1)][0];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        op[gi % 3][e] = *(lds_op*)(kt + (kbase ^ (uint32_t)(32 * (2 * (gi - 4) + e / 2))) + (e % 2) * 32 * ROWB);
    }
  };
  auto run_group = [&](int gi) {
    if (gi < 4) {
      const uint32_t* x = &ph[gi / 2][4 * (gi % 2)];
      const op_t pb = __builtin_bit_cast(op_t, make_uint4(x[0], x[1], x[2], x[3]));
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] = M::run(op[gi % 3][d], pb, o[d]);
    } else {
      f32x16_t none;
#pragma unroll
      for (int r = 0; r < 16; ++r) none[r] = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sc[e % 2] = M::run(op[gi % 3][e], qop[2 * (gi - 4) + e / 2], gi == 4 && e < 2 ? none : sc[e % 2]);
    }
  };
  auto run_groups = [&](int g0, int g1, int tile_v, int tile_k) {  // g0 .. g1 - 1, the first two's operands loaded
#pragma unroll
    for (int gi = g0; gi < g1; ++gi) {
      load_group(gi + 2, tile_v, tile_k);
      __builtin_amdgcn_sched_barrier(0);
      run_group(gi);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // p = exp2(s scale - m) against the reference as it is, eight at a time (one wave a SIMD makes weights:
  // a chain of dependent instructions would leave the unit idle), and their sum. top: fp16, the largest
  // of the packed halves as bits.
  u16x2_t top;
  const bool want_lse = a.lse != nullptr;
  float l32;
  auto weights = [&](float (&ls)[2]) {
    ls[0] = ls[1] = l32 = 0.0f;
    top = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int r0 = 0; r0 < 16; r0 += 8) {
        float x[8];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(sc[h][r0 + e], scale, -m_run);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fast_exp2(x[e]);
        __builtin_amdgcn_sched_barrier(0);
        uint32_t* pair = &ph[h][r0 / 2];
#pragma unroll
        for (int e = 0; e < 8; e += 2) pair[e / 2] = M::pack2(x[e], x[e + 1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) ls[e & 1] = M::sum2(pair[e], ls[e & 1]);
        if (want_lse) l32 += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));  // uniform
        if constexpr (HALF) {
#pragma unroll
          for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, pair[e]));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // The reference moves lazily: weights are made against it as it is, and only where one may have
  // reached 2^TOP (bf16: a lane's 32 together) are the column maxima taken, the state rescaled and
  // the weights made again. Most tiles take no maximum.
  auto softmax = [&](uint64_t ok) {
    if (ok != ~0ull) {  // uniform: a tile with keys that do not count
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t wd = (uint32_t)(ok >> (32 * h)) >> (4 * hh);
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[h][r] = wd >> (8 * (r / 4) + r % 4) & 1u ? sc[h][r] : -INFINITY;
      }
    }
    float ls[2];
    weights(ls);
    static_assert(TOP == (HALF ? 15.0f : 8.0f), "the test is against 2^TOP");
    const bool over = HALF ? max(top.x, top.y) >= 0x7800 : !(ls[0] + ls[1] < 256.0f);
    if (__builtin_expect(__any(over), 0)) {
      float mx = sc[0][0];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[h][r]);
      }
      const float mt = fmaxf(mx, lane_xor(mx, 32)) * scale;
      const bool moves = mt > m_run + TOP;
      if (__any(moves)) {
        const float mn = moves ? mt - BIAS : m_run;
        const float alpha = fast_exp2(m_run - mn);
        m_run = mn;
        l_run *= alpha;
        l32_run *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
        }
        weights(ls);
      }
    }
    l_run += ls[0] + ls[1];
    l32_run += l32;
  };

  wait_vm<0>();
  blank(0);
  phase_barrier();
  const bool late = w >= 4;
  if (late) phase_barrier();
  load_group(4, 0, 0);
  load_group(5, 0, 0);
  for (int i = 0;;) {
    run_groups(4, NG, i, i);
    phase_barrier();
#pragma unroll
    for (int y = 0; y < NI; ++y) {
      load(false, i + 3, y);
      load(true, i + 2, y);
    }
    if constexpr (PAGED) load_ids(i + 6);
    softmax(live_of(i));
    __builtin_amdgcn_sched_barrier(0);
    load_group(0, i, i);
    load_group(1, i, i);
    wait_vm<PER>();
    blank(i + 1);
    phase_barrier();
    run_groups(0, 4, i, i + 1);
    if (++i == n_tiles) break;
  }
  if (!late) phase_barrier();
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // nothing lands after this
  __syncthreads();
  store_partials<D, KG, CG>(a, sh, blk, 0, w, o, m_run, l_run, l32_run);
}

// Column blocks of all prefixes, at most.
int64_t column_blocks(const PrefixArgs& a, int64_t wg) {
  const int64_t per = a.Tq * (a.Hq / a.Hkv);
  if (a.prefix_rows == nullptr && a.P > 1) return a.P * ((per + wg - 1) / wg);
  return (a.B * per + std::min<int64_t>(a.P, a.B) * (wg - 1)) / wg;
}

// Workgroups of `blocks` column blocks, a prefix in `splits` pieces (PrefixBlock::place).
int64_t placed(const PrefixArgs& a, int64_t blocks, int64_t splits) {
  const int64_t units = (int64_t)a.Hkv * splits, together = std::min<int64_t>(units, kXcds);
  return (units + together - 1) / together * together * blocks;
}
int64_t prefix_grid(const PrefixArgs& a, int64_t wg) {
  const int64_t blocks = column_blocks(a, wg);
  if (!a.plan) return placed(a, blocks, a.splits);
  int64_t most = placed(a, blocks, 1);  // whichever spread of the rows needs most
  for (int64_t n = 2; n <= a.splits; ++n) most = std::max(most, placed(a, std::min<int64_t>(blocks, 256 / (n * a.Hkv)), n));
  return most;
}

template <typename T, int D, int KG, int CG>
void launch_mfma(const PrefixArgs& a, int n_cb, hipStream_t s) {
  const dim3 grid((unsigned)prefix_grid(a, 32 * CG));
  if (a.slots) prefix_mfma_kernel<T, D, KG, CG, true><<<grid, 64 * KG * CG, 0, s>>>(a, n_cb);
  else prefix_mfma_kernel<T, D, KG, CG, false><<<grid, 64 * KG * CG, 0, s>>>(a, n_cb);
}

template <typename T, int D>
void launch_mfma_cols(const PrefixArgs& a, int64_t columns, hipStream_t s) {
  const int64_t wg = prefix_mfma_columns(columns);
  const int n_cb = (int)column_blocks(a, wg);
  if (wg == 32) launch_mfma<T, D, 4, 1>(a, n_cb, s);
  else if (wg == 64) launch_mfma<T, D, 4, 2>(a, n_cb, s);
  else if (wg == 128) launch_mfma<T, D, 2, 4>(a, n_cb, s);
  else {
    const dim3 grid((unsigned)prefix_grid(a, wg));
    if (a.slots) prefix_wide_kernel<T, D, true><<<grid, 512, 0, s>>>(a, n_cb);
    else prefix_wide_kernel<T, D, false><<<grid, 512, 0, s>>>(a, n_cb);
  }
}

}  // namespace

namespace lsa {

bool prefix_mfma_ok(int dtype, int D) { return dtype != LSA_F32 && (D == 64 || D == 128); }

int64_t prefix_mfma_columns(int64_t columns) {
  return columns <= 32 ? 32 : (columns <= 64 ? 64 : (columns <= 128 ? 128 : 256));
}

bool launch_prefix_mfma(const PrefixArgs& a, int dtype, int D, int64_t columns, hipStream_t s) {
  // a lane's offset within a tile is 32 bits of bytes; a column's largest score is its largest dot product
  if (!prefix_mfma_ok(dtype, D) || !(a.scale_log2 > 0.0f && a.scale_log2 < INFINITY) ||
      a.p_st >= (int64_t)1 << 25 || prefix_grid(a, prefix_mfma_columns(columns)) > 0xFFFFFFFFll / 512)
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
