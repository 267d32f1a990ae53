// A cache cut down to the keys that carried attention weight, for gfx950.
//
// Of a row's n positions the first `sink` and the last `window` stay, and of the others the
// budget - sink - window of largest weight (ties: the lower position; a NaN weighs least).
// The kept positions come out ascending. n <= budget keeps everything.
//
//   seen_keys_kernel  the weights as 32-bit keys of the same order, summed over the kv-heads
//                     (fp64 in head order, rounded to fp32 once) and, for a paged cache, looked
//                     up through the slot table;
//   keep_kernel       a radix select of the threshold, then one pass that ranks what stays;
//   keep_rows_kernel  (dense caches) moves the kept K, V and weight rows.
#include "lsa_abi_common.h"
#include "lsa_device.h"

using namespace lsa;

namespace {

constexpr int kKeepThreads = 1024;
constexpr int kKeepWaves = kKeepThreads / LSA_WAVE;

// A weight as an unsigned key of the same order: NaN (0) below -inf, -0 as +0.
__device__ __forceinline__ uint32_t seen_key(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

struct KeepArgs {
  const float* mass;      // [B or 1, Hkv, T or pool] (strides below)
  int64_t mass_sb, mass_sh;
  const uint32_t* keys;   // [units, T]: summed weights' keys (seen_keys_kernel), or nullptr
  const int32_t* lengths; // [B], or nullptr: T
  int64_t T;
  int G;                  // selections a batch row: Hkv, or 1 shared by the heads
  int Hkv;
  int budget, window, sink;
  int32_t* kept;          // [B, G, budget]
  int32_t* new_lengths;   // [B]
  const int32_t* table;   // paged: the slot table and its new rows
  int64_t table_stride;
  int32_t* new_table;
  int64_t new_stride;
  int64_t pool;           // paged: cache rows the weights hold
  uint32_t* keys_out;
  int* hist;              // rows in slabs: [3][units][slabs][2048]
  int2* state;            // [units][2]
};

__device__ __forceinline__ int row_length(const KeepArgs& a, int64_t b) {
  const int64_t n = a.lengths ? (int64_t)a.lengths[b] : a.T;
  return (int)(n < 0 ? 0 : (n > a.T ? a.T : n));
}

// grid (chunks of T, B). A paged cache's weights are gathered, one 64-byte sector a page and head.
__global__ __launch_bounds__(LSA_BLOCK) void seen_keys_kernel(KeepArgs a) {
  const int64_t b = blockIdx.y;
  const int64_t i = (int64_t)blockIdx.x * LSA_BLOCK + threadIdx.x;
  if (i >= row_length(a, b)) return;
  int64_t at = i;
  bool ok = true;
  if (a.table) {
    at = a.table[b * a.table_stride + i];
    ok = at >= 0 && at < a.pool;
  }
  const float* m = a.mass + b * a.mass_sb + (ok ? at : 0);
  double sum = 0.0;
  for (int h0 = 0; h0 < a.Hkv; h0 += 8) {  // eight heads' loads in flight
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = m[min(h0 + e, a.Hkv - 1) * a.mass_sh];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += h0 + e < a.Hkv ? (double)f[e] : 0.0;
  }
  a.keys_out[b * a.T + i] = ok ? seen_key((float)sum) : 0u;
}

// One workgroup a selection.
//
// The threshold, the budget's last key, comes from three histograms (11, 11 and 10 bits from the
// top), each over the keys that share the digits found so far. Weights crowd into few bins (a third
// of a cache may be exactly zero), and lanes that meet in one bin of LDS wait for each other, so there are eight
// copies of each histogram, a lane's by its number, side by side: a bin's copies lie in banks of their own.
//
//   keep_kernel       rows of up to 32768 positions: a thread holds R in a line, turned through LDS
//                     after coalesced loads. A CU's vector unit is what bounds it (one CU works on
//                     a selection), so a key costs few instructions: the first and last positions
//                     are the largest key, those past the row the least, and no loop asks which is
//                     which; one scan over the threads' counts ranks everything.
//   keep_slab_kernel  longer rows, a workgroup a slab of 32768, four launches: a histogram each, then the
//                     ranks.
constexpr int kBins = 2048, kCopies = 8;

struct KeepLds {
  alignas(16) int hist[kBins][kCopies];
  int wave_gt[kKeepWaves], wave_eq[kKeepWaves];
  uint32_t digit;
  int need;
};

// Exclusive sums over the workgroup's threads of two counts; every thread calls it.
__device__ __forceinline__ void keep_scan(KeepLds& sh, int& gt, int& eq, int& all_gt, int& all_eq) {
  const int lane = threadIdx.x & (LSA_WAVE - 1), w = threadIdx.x / LSA_WAVE;
  const int ig = wave_inclusive_sum(gt), ie = wave_inclusive_sum(eq);
  if (lane == LSA_WAVE - 1) {
    sh.wave_gt[w] = ig;
    sh.wave_eq[w] = ie;
  }
  __syncthreads();
  int bg = 0, be = 0;
  all_gt = all_eq = 0;
#pragma unroll
  for (int y = 0; y < kKeepWaves; ++y) {
    const int cg = sh.wave_gt[y], ce = sh.wave_eq[y];
    bg += y < w ? cg : 0;
    be += y < w ? ce : 0;
    all_gt += cg;
    all_eq += ce;
  }
  __syncthreads();
  gt = bg + ig - gt;
  eq = be + ie - eq;
}

// The bin that the `need`-th key from the top is in, given every thread's counts (bins 2047 - 2 t and
// 2046 - 2 t): its digit, and how many of its keys are needed.
__device__ __forceinline__ void keep_digit(KeepLds& sh, int need, const int (&c)[2]) {
  const int tid = threadIdx.x;
  int none = 0, mine = c[0] + c[1], total, unused;
  const int own = mine;
  keep_scan(sh, mine, none, total, unused);
  if (mine < need && need <= mine + own) {
    const int e = mine + c[0] < need ? 1 : 0;
    sh.digit = (uint32_t)(kBins - 1 - 2 * tid - e);
    sh.need = need - mine - (e ? c[0] : 0);
  }
  __syncthreads();
}
__device__ __forceinline__ void keep_clear(KeepLds& sh) {
  int4* h = (int4*)&sh.hist[0][0];
#pragma unroll
  for (int i = 0; i < kCopies * kBins / 4 / kKeepThreads; ++i) h[i * kKeepThreads + threadIdx.x] = make_int4(0, 0, 0, 0);
  __syncthreads();
}

template <int R>
struct KeepTurn {
  static constexpr int PAD = R > 4 ? 4 : 0;  // dwords a thread's run is kept apart: 16-byte reads without conflicts
  static __host__ __device__ constexpr int at(int i) { return i + (int)((unsigned)i / R) * PAD; }
  union {
    uint32_t key[kKeepThreads * (R + PAD)];
    int32_t place[kKeepThreads * R];  // the positions in their new order
    KeepLds sh;
  };
};

// The thread's run of R keys of the positions from p0 on: the first and last of the row are the largest
// key, which no weight equals, positions past it the least. Contains barriers.
template <int R>
__device__ __forceinline__ void keep_load(KeepTurn<R>& turn, const KeepArgs& a, int64_t u, int64_t b, int g, int n, int p0,
                                          uint32_t (&x)[R]) {
  using Turn = KeepTurn<R>;
  const int tid = threadIdx.x;
  const float* mass = a.mass + b * a.mass_sb + g * a.mass_sh;
  const uint32_t* keys = a.keys ? a.keys + u * a.T : nullptr;
  uint32_t in[R];
#pragma unroll
  for (int e = 0; e < R; ++e) {  // unconditional (clamped): all in flight
    const int i = min(p0 + e * kKeepThreads + tid, n - 1);
    in[e] = keys ? keys[i] : __float_as_uint(mass[i]);
  }
  uint32_t* to = &turn.key[Turn::at(tid)];
#pragma unroll
  for (int e = 0; e < R; ++e)
    to[Turn::at(e * kKeepThreads)] = keys ? in[e] : seen_key(__uint_as_float(in[e]));
  __syncthreads();
  const int end = R * kKeepThreads;
  for (int i = tid; i < min(a.sink - p0, end); i += kKeepThreads) turn.key[Turn::at(i)] = 0xFFFFFFFFu;
  for (int i = max(n - a.window - p0, 0) + tid; i < end; i += kKeepThreads)
    turn.key[Turn::at(i)] = p0 + i < n ? 0xFFFFFFFFu : 0u;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < R; e += 4) {
    const uint4 y = *(const uint4*)&turn.key[tid * (R + Turn::PAD) + e];
    x[e] = y.x; x[e + 1] = y.y; x[e + 2] = y.z; x[e + 3] = y.w;
  }
  __syncthreads();
}

// Counts the digits at `shift` of the keys that share `thr` under `mask`. Ends with a barrier. Positions past the
// row are counted, as the least key; there are enough of the row's own before they would matter.
template <int R>
__device__ __forceinline__ void keep_count(KeepLds& sh, const uint32_t (&x)[R], uint32_t mask, uint32_t thr, int shift) {
  int* hist = &sh.hist[0][threadIdx.x % kCopies];
#pragma unroll
  for (int e = 0; e < R; ++e) {
    if ((x[e] & mask) == thr) atomicAdd(&hist[((x[e] >> shift) & (kBins - 1)) * kCopies], 1);
  }
  __syncthreads();
}

template <int R, bool TABLE>
__global__ __launch_bounds__(kKeepThreads) void keep_kernel(KeepArgs a) {
  using Turn = KeepTurn<R>;
  __shared__ __attribute__((aligned(16))) Turn turn;
  KeepLds& sh = turn.sh;
  const int tid = threadIdx.x;
  const int64_t u = blockIdx.x;
  const int64_t b = u / a.G;
  const int g = (int)(u % a.G);
  const int n = row_length(a, b);
  const int keep = n < a.budget ? n : a.budget;
  if (g == 0 && tid == 0) a.new_lengths[b] = keep;
  int32_t* kept = a.kept + u * a.budget;
  const int32_t* table = a.table ? a.table + b * a.table_stride : nullptr;
  int32_t* new_table = a.new_table ? a.new_table + b * a.new_stride : nullptr;
  if (n <= a.budget) {  // uniform: all of it
    for (int i = tid; i < a.budget; i += kKeepThreads) kept[i] = i < n ? i : -1;
    if (TABLE) {
      for (int64_t i = tid; i < a.T; i += kKeepThreads) new_table[i] = table[i];
    }
    return;
  }
  uint32_t x[R];
  keep_load<R>(turn, a, u, b, g, n, 0, x);
  uint32_t thr = 0, mask = 0;
  int ties = a.budget;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    keep_clear(sh);
    keep_count<R>(sh, x, mask, thr, shift);
    int c[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int y = 0; y < kCopies; y += 4) {
        const int4 z = *(const int4*)&sh.hist[kBins - 1 - 2 * tid - e][y];
        c[e] += z.x + z.y + z.z + z.w;
      }
    }
    keep_digit(sh, ties, c);
    thr |= sh.digit << shift;
    ties = sh.need;
    mask |= (pass == 2 ? 1023u : 2047u) << shift;
  }
  int gt = 0, eq = 0, all_gt, all_eq;
#pragma unroll
  for (int e = 0; e < R; ++e) {
    gt += x[e] > thr;
    eq += x[e] == thr;
  }
  keep_scan(sh, gt, eq, all_gt, all_eq);  // kept, and at the threshold, before this thread's positions
  // positions past the row tie with NaN alone, and come after every position of the row
  int rank = gt + min(eq, ties);  // kept positions before this one
#pragma unroll
  for (int e = 0; e < R; ++e) {
    const int i = tid * R + e;
    const bool same = x[e] == thr;
    const bool in = x[e] > thr || (same && eq < ties);
    if (TABLE) {
      if (i < n) turn.place[in ? rank : keep + (i - rank)] = i;
    } else if (in) {
      turn.place[rank] = i;
    }
    rank += in;
    eq += same;
  }
  __syncthreads();
  for (int j = tid; j < keep; j += kKeepThreads) kept[j] = turn.place[j];
  if (TABLE) {
    constexpr int E = 8;  // entries of a thread in flight
    for (int64_t i0 = tid; i0 < a.T; i0 += E * kKeepThreads) {
      int32_t y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int64_t i = min(i0 + e * kKeepThreads, a.T - 1);
        y[e] = table[i < n ? turn.place[i] : i];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int64_t i = i0 + e * kKeepThreads;
        if (i < a.T) new_table[i] = y[e];
      }
    }
  }
}

// A row in slabs of 32768 positions, a workgroup a slab; grid (selection, slab). Phases 0, 1 and 2 leave
// each slab's histogram of their digit, and phases 1, 2 and 3 add the slabs' up and find the digit
// (slab 0 keeps it for the phases after the next). Phase 3 ranks: what is kept before a slab follows from
// the earlier slabs' histograms.
constexpr int kSlabRun = 32, kSlab = kSlabRun * kKeepThreads;

template <int PHASE, bool TABLE>
__global__ __launch_bounds__(kKeepThreads) void keep_slab_kernel(KeepArgs a) {
  constexpr int R = kSlabRun;
  using Turn = KeepTurn<R>;
  __shared__ __attribute__((aligned(16))) Turn turn;
  KeepLds& sh = turn.sh;
  const int tid = threadIdx.x, lane = tid & (LSA_WAVE - 1);
  const int64_t u = blockIdx.x;
  const int slab = blockIdx.y, slabs = gridDim.y;
  const int64_t b = u / a.G;
  const int g = (int)(u % a.G);
  const int n = row_length(a, b), p0 = slab * kSlab, p1 = (int)min((int64_t)p0 + kSlab, a.T);
  const int keep = n < a.budget ? n : a.budget;
  int32_t* kept = a.kept + u * a.budget;
  const int32_t* table = a.table ? a.table + b * a.table_stride : nullptr;
  int32_t* new_table = a.new_table ? a.new_table + b * a.new_stride : nullptr;
  if (PHASE == 3) {
    if (g == 0 && slab == 0 && tid == 0) a.new_lengths[b] = keep;
    for (int i = max(p0, keep) + tid; i < min(p1, a.budget); i += kKeepThreads) kept[i] = -1;
    if (TABLE) {
      for (int i = max(p0, n) + tid; i < p1; i += kKeepThreads) new_table[i] = table[i];
    }
    if (n <= a.budget) {  // uniform: all of it
      for (int i = p0 + tid; i < min(p1, n); i += kKeepThreads) {
        kept[i] = i;
        if (TABLE) new_table[i] = table[i];
      }
    }
  }
  if (n <= a.budget) return;
  int* hist = a.hist + u * slabs * kBins;             // of phase 0, [slab][bin]
  const int64_t phase_hist = (int64_t)gridDim.x * slabs * kBins;
  int2* state = a.state + u * 2;                      // digits (and what they leave needed) of phases 0, 1
  uint32_t thr = 0, mask = 0;
  int ties = a.budget, gt0 = 0, eq0 = 0;  // phase 3: above and at the threshold in the slabs before
#pragma unroll
  for (int q = 0; q < PHASE; ++q) {
    const int shift = q == 0 ? 21 : (q == 1 ? 10 : 0);
    int c[2] = {0, 0}, before[2] = {0, 0};
    if (q == PHASE - 1 || PHASE == 3) {  // bins 2047 - 2 t and 2046 - 2 t of all slabs, and of the ones before
      const int2* h = (const int2*)(hist + q * phase_hist + kBins - 2 - 2 * tid);
      for (int y = 0; y < slabs; ++y) {
        const int2 x = h[(int64_t)y * kBins / 2];
        c[0] += x.y;
        c[1] += x.x;
        before[0] += y < slab ? x.y : 0;
        before[1] += y < slab ? x.x : 0;
      }
    }
    if (q == PHASE - 1) {
      keep_digit(sh, ties, c);
      if (PHASE < 3 && slab == 0 && tid == 0) state[q] = make_int2((int)sh.digit, sh.need);
    } else {
      if (tid == 0) {
        const int2 x = state[q];
        sh.digit = (uint32_t)x.x;
        sh.need = x.y;
      }
      __syncthreads();
    }
    const uint32_t digit = sh.digit;
    ties = sh.need;
    thr |= digit << shift;
    mask |= (q == 2 ? 1023u : 2047u) << shift;
    if (PHASE == 3) {
      int more = 0, same = 0, all_more, all_same;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t bin = (uint32_t)(kBins - 1 - 2 * tid - e);
        more += bin > digit ? before[e] : 0;
        same += q == 2 && bin == digit ? before[e] : 0;
      }
      keep_scan(sh, more, same, all_more, all_same);
      gt0 += all_more;
      eq0 += all_same;
    }
    __syncthreads();  // the digit is read before the next takes its place
  }
  uint32_t x[R];
  keep_load<R>(turn, a, u, b, g, n, p0, x);
  if (PHASE < 3) {
    const int shift = PHASE == 0 ? 21 : (PHASE == 1 ? 10 : 0);
    keep_clear(sh);
    keep_count<R>(sh, x, mask, thr, shift);
    int* out = hist + PHASE * phase_hist + (int64_t)slab * kBins;
    for (int i = tid; i < kBins; i += kKeepThreads) {
      int c = 0;
#pragma unroll
      for (int y = 0; y < kCopies; y += 4) {
        const int4 z = *(const int4*)&sh.hist[i][y];
        c += z.x + z.y + z.z + z.w;
      }
      out[i] = c;
    }
    return;
  }
  int gt = 0, eq = 0, all_gt, all_eq;
#pragma unroll
  for (int e = 0; e < R; ++e) {
    gt += x[e] > thr;
    eq += x[e] == thr;
  }
  keep_scan(sh, gt, eq, all_gt, all_eq);
  const int first = gt0 + min(eq0, ties);                                  // kept before this slab,
  const int mine = gt0 + all_gt + min(eq0 + all_eq, ties) - first;         // and in it
  eq += eq0;
  int rank = gt0 + gt + min(eq, ties) - first;
#pragma unroll
  for (int e = 0; e < R; ++e) {
    const int i = tid * R + e;
    const bool same = x[e] == thr;
    const bool in = x[e] > thr || (same && eq < ties);
    if (TABLE) {
      if (p0 + i < n) turn.place[in ? rank : mine + (i - rank)] = p0 + i;
    } else if (in) {
      turn.place[rank] = p0 + i;
    }
    rank += in;
    eq += same;
  }
  __syncthreads();
  for (int j = tid; j < mine; j += kKeepThreads) kept[first + j] = turn.place[j];
  if (TABLE) {
    const int live = max(0, min(p1, n) - p0), rest = keep + (p0 - first) - mine;  // where what it gives up goes
    for (int j = tid; j < live; j += kKeepThreads) new_table[j < mine ? first + j : rest + j] = table[turn.place[j]];
  }
}

struct RowsArgs {
  const char* k;
  const char* v;
  const float* mass;
  char* k2;
  char* v2;
  float* mass2;
  int64_t sb, st, sh;     // bytes
  int64_t o_sb, o_st, o_sh;
  int64_t m_sb, m_sh, mo_sb, mo_sh;
  const int32_t* kept;    // [B, G, budget]
  const int32_t* lengths; // [B], or nullptr: T
  int64_t T;
  int G, Hkv, budget;
  int segs;               // 16-byte segments of a row
  int zero;               // rows past the new length: zeros (else left as they were)
};

// HBM-bound: each kept row read and written once. grid (rows of the new cache a workgroup, B).
__global__ __launch_bounds__(LSA_BLOCK) void keep_rows_kernel(RowsArgs a, int rows_per_block) {
  const int64_t b = blockIdx.y;
  const int j0 = blockIdx.x * rows_per_block;
  const int per = a.Hkv * a.segs;
  const int total = min(rows_per_block, a.budget - j0) * per;
  for (int x = threadIdx.x; x < total; x += LSA_BLOCK) {
    const int j = j0 + x / per, rest = x % per;
    const int h = rest / a.segs, seg = rest % a.segs;
    const int32_t src = a.kept[(b * a.G + (a.G > 1 ? h : 0)) * a.budget + j];
    if (src < 0 && !a.zero) continue;
    uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
    float m = 0.0f;
    if (src >= 0) {
      const int64_t off = b * a.sb + src * a.st + h * a.sh + 16 * seg;
      kx = *(const uint4*)(a.k + off);
      vx = *(const uint4*)(a.v + off);
      if (seg == 0) m = a.mass[b * a.m_sb + h * a.m_sh + src];
    }
    const int64_t to = b * a.o_sb + j * a.o_st + h * a.o_sh + 16 * seg;
    *(uint4*)(a.k2 + to) = kx;
    *(uint4*)(a.v2 + to) = vx;
    if (seg == 0) a.mass2[b * a.mo_sb + h * a.mo_sh + j] = m;
  }
}

template <int R>
void launch_keep(const KeepArgs& a, dim3 grid, hipStream_t s) {
  if (a.table) keep_kernel<R, true><<<grid, kKeepThreads, 0, s>>>(a);
  else keep_kernel<R, false><<<grid, kKeepThreads, 0, s>>>(a);
}

int64_t keep_slabs(int64_t T) { return T > kSlab ? (T + kSlab - 1) / kSlab : 0; }

template <bool TABLE>
void launch_keep_slabs(const KeepArgs& a, int64_t units, hipStream_t s) {
  const dim3 grid((unsigned)units, (unsigned)keep_slabs(a.T));
  keep_slab_kernel<0, TABLE><<<grid, kKeepThreads, 0, s>>>(a);
  keep_slab_kernel<1, TABLE><<<grid, kKeepThreads, 0, s>>>(a);
  keep_slab_kernel<2, TABLE><<<grid, kKeepThreads, 0, s>>>(a);
  keep_slab_kernel<3, TABLE><<<grid, kKeepThreads, 0, s>>>(a);
}

size_t summed_bytes(int64_t B, int64_t T, int shared) {
  return shared ? ((size_t)B * (size_t)T * sizeof(uint32_t) + 15) / 16 * 16 : 0;
}

int check_keep(const char* who, const void* mass, int64_t B, int32_t Hkv, int64_t T, int64_t mass_sb, int64_t mass_sh,
               int32_t budget, int32_t window, int32_t sink, const void* kept, const void* new_lengths) {
  LSA_REQUIRE(mass && kept && new_lengths, LSA_ERR_NULL, "%s: NULL pointer", who);
  LSA_REQUIRE(B >= 0 && B <= 65535 && Hkv >= 1 && T >= 1 && T <= 1 << 30, LSA_ERR_SHAPE,
              "%s: needs 0..65535 rows of 1..2^30 positions and a kv-head", who);
  LSA_REQUIRE(mass_sb >= 0 && mass_sh >= 0, LSA_ERR_SHAPE, "%s: weight strides must be >= 0", who);
  LSA_REQUIRE(budget >= 1 && budget <= T, LSA_ERR_SHAPE, "%s: budget %d not in 1..%lld", who, budget, (long long)T);
  LSA_REQUIRE(window >= 0 && sink >= 0 && (int64_t)window + sink <= budget, LSA_ERR_SHAPE,
              "%s: window %d and sink %d must fit the budget %d", who, window, sink, budget);
  // a launch holds fewer than 2^32 threads along an axis
  LSA_REQUIRE(B * (int64_t)Hkv <= 0xFFFFFFFFll / kKeepThreads, LSA_ERR_SHAPE, "%s: %lld rows of %d kv-heads are too many",
              who, (long long)B, Hkv);
  return LSA_OK;
}

}  // namespace

extern "C" size_t lsa_evict_scratch_bytes(int64_t B, int32_t Hkv, int64_t T, int shared) {
  if (B <= 0 || T <= 0 || Hkv <= 0) return 0;
  const size_t units = (size_t)B * (shared ? 1 : Hkv), slabs = (size_t)keep_slabs(T);
  return summed_bytes(B, T, shared) + units * (3 * slabs * kBins * sizeof(int) + (slabs ? 2 * sizeof(int2) : 0));
}

extern "C" int lsa_evict_keep(const float* mass, int64_t B, int32_t Hkv, int64_t T, int64_t mass_batch_stride,
                              int64_t mass_head_stride, const int32_t* lengths, int32_t budget, int32_t window,
                              int32_t sink, int shared, const int32_t* table, int64_t table_stride, int64_t pool_rows,
                              void* scratch, size_t scratch_bytes, int32_t* kept, int32_t* new_lengths,
                              int32_t* new_table, int64_t new_table_stride, void* stream) {
  LSA_TRY(check_keep("lsa_evict_keep", mass, B, Hkv, T, mass_batch_stride, mass_head_stride, budget, window, sink, kept,
                     new_lengths));
  LSA_REQUIRE((table == nullptr) == (new_table == nullptr), LSA_ERR_NULL,
              "lsa_evict_keep: a slot table and its new rows come together");
  LSA_REQUIRE(table == nullptr || (shared && table_stride >= T && new_table_stride >= T && pool_rows >= 1),
              LSA_ERR_SHAPE, "lsa_evict_keep: a slot table needs shared selection, strides >= %lld and a pool",
              (long long)T);
  const size_t need = lsa_evict_scratch_bytes(B, Hkv, T, shared);
  LSA_REQUIRE(need == 0 || (scratch && scratch_bytes >= need && ((uintptr_t)scratch & 15) == 0), LSA_ERR_WORKSPACE,
              "lsa_evict_keep: scratch missing, not 16-byte aligned or %zu < %zu bytes", scratch_bytes, need);
  if (B == 0) return LSA_OK;
  KeepArgs a = {};
  a.mass = mass; a.mass_sb = mass_batch_stride; a.mass_sh = mass_head_stride; a.lengths = lengths; a.T = T;
  a.G = shared ? 1 : Hkv; a.Hkv = Hkv; a.budget = budget; a.window = window; a.sink = sink;
  a.kept = kept; a.new_lengths = new_lengths; a.table = table; a.table_stride = table_stride;
  a.new_table = new_table; a.new_stride = new_table_stride; a.pool = pool_rows;
  hipStream_t s = (hipStream_t)stream;
  a.hist = (int*)((char*)scratch + summed_bytes(B, T, shared));
  a.state = (int2*)(a.hist + 3 * B * a.G * keep_slabs(T) * kBins);
  if (shared) {
    a.keys = a.keys_out = (uint32_t*)scratch;
    const dim3 grid((unsigned)((T + LSA_BLOCK - 1) / LSA_BLOCK), (unsigned)B);
    seen_keys_kernel<<<grid, LSA_BLOCK, 0, s>>>(a);
    LSA_LAUNCHED("lsa_evict_keep");
  }
  const int64_t units = B * a.G;
  const dim3 grid((unsigned)units);
  if (T <= 4 * kKeepThreads) launch_keep<4>(a, grid, s);
  else if (T <= 8 * kKeepThreads) launch_keep<8>(a, grid, s);
  else if (T <= 16 * kKeepThreads) launch_keep<16>(a, grid, s);
  else if (T <= 32 * kKeepThreads) launch_keep<32>(a, grid, s);
  else if (a.table) launch_keep_slabs<true>(a, units, s);
  else launch_keep_slabs<false>(a, units, s);
  LSA_LAUNCHED("lsa_evict_keep");
  return LSA_OK;
}

extern "C" int lsa_evict_rows(const void* k, const void* v, const float* mass, int dtype, int64_t B, int64_t T,
                              int32_t Hkv, int32_t D, int64_t kv_batch_stride, int64_t kv_token_stride,
                              int64_t kv_head_stride, int64_t mass_batch_stride, int64_t mass_head_stride,
                              const int32_t* kept, int shared, int32_t budget, void* k_out, void* v_out,
                              int64_t out_batch_stride, int64_t out_token_stride, int64_t out_head_stride,
                              float* mass_out, int64_t mass_out_batch_stride, int64_t mass_out_head_stride,
                              int zero_tail, void* stream) {
  LSA_REQUIRE(k && v && mass && kept && k_out && v_out && mass_out, LSA_ERR_NULL, "lsa_evict_rows: NULL pointer");
  LSA_TRY(check_dtype(dtype));
  const int64_t e = dtype == LSA_F32 ? 4 : 2;
  LSA_REQUIRE(B >= 0 && B <= 65535 && T >= 1 && T <= 0x7FFFFFFF && Hkv >= 1 && D >= 1 && budget >= 1 && budget <= T,
              LSA_ERR_SHAPE, "lsa_evict_rows: B %lld T %lld Hkv %d D %d budget %d", (long long)B, (long long)T, Hkv, D,
              budget);
  LSA_REQUIRE(kv_batch_stride >= 0 && kv_token_stride >= D && kv_head_stride >= D && out_batch_stride >= 0 &&
                  out_token_stride >= D && out_head_stride >= D && mass_batch_stride >= 0 && mass_head_stride >= 0 &&
                  mass_out_batch_stride >= 0 && mass_out_head_stride >= 0,
              LSA_ERR_SHAPE, "lsa_evict_rows: strides must leave rows of %d elements apart", D);
  const uintptr_t at = (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_out | (uintptr_t)v_out;
  LSA_REQUIRE(at % 16 == 0 && ((int64_t)D * e) % 16 == 0 &&
                  ((kv_batch_stride | kv_token_stride | kv_head_stride | out_batch_stride | out_token_stride |
                    out_head_stride) * e) % 16 == 0,
              LSA_ERR_ALIGN, "lsa_evict_rows: K/V rows must be 16-byte aligned, and a multiple of 16 bytes");
  LSA_REQUIRE((int64_t)Hkv * D * e / 16 <= 1 << 20, LSA_ERR_SHAPE, "lsa_evict_rows: rows of more than 16 MB");
  if (B == 0) return LSA_OK;
  RowsArgs a;
  a.k = (const char*)k; a.v = (const char*)v; a.mass = mass; a.k2 = (char*)k_out; a.v2 = (char*)v_out;
  a.mass2 = mass_out;
  a.sb = kv_batch_stride * e; a.st = kv_token_stride * e; a.sh = kv_head_stride * e;
  a.o_sb = out_batch_stride * e; a.o_st = out_token_stride * e; a.o_sh = out_head_stride * e;
  a.m_sb = mass_batch_stride; a.m_sh = mass_head_stride; a.mo_sb = mass_out_batch_stride; a.mo_sh = mass_out_head_stride;
  a.kept = kept; a.T = T; a.G = shared ? 1 : Hkv; a.Hkv = Hkv; a.budget = budget;
  a.segs = (int)(D * e / 16); a.zero = zero_tail ? 1 : 0;
  int rows = 1;  // about 1024 segments a workgroup
  while (rows < 64 && rows * Hkv * a.segs < 1024) rows *= 2;
  const dim3 grid((unsigned)((budget + rows - 1) / rows), (unsigned)B);
  keep_rows_kernel<<<grid, LSA_BLOCK, 0, (hipStream_t)stream>>>(a, rows);
  LSA_LAUNCHED("lsa_evict_rows");
  return LSA_OK;
}
