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
constexpr int kSlabRun = 32, kSlab = kSlabRun * kKeepThreads;

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

// grid (chunks of T, B). A paged cache's weights are gathered, one 64-byte sector a page and head: 32 rows
// of 32768 positions over 8 kv-heads in 10 us (34 MB, 3.4 TB/s).
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
// The threshold, the budget's last key, comes from three histograms (10, 11 and 11 bits from the
// top), each over the keys that share the digits found so far. Weights crowd into few bins (a third
// of a cache may be exactly zero), and lanes that meet in one bin of LDS wait for each other, so there
// are 16 copies of the first histogram and 8 of the others, a lane's by its number, side by side: a bin's
// copies lie in banks of their own.
//
//   keep_kernel       rows of up to 32768 positions: a wave holds R times 64 in a line, a lane every 64th,
//                     so ranks are bit counts of what the wave's comparisons leave and no key moves
//                     between threads. A CU's vector unit is what bounds it (one CU works on
//                     a selection), so a key costs few instructions: the first and last positions
//                     are the largest key, those past the row the least, and no loop asks which is
//                     which; one scan over the waves' counts ranks everything. 8 selections of 8192 from
//                     32768 take 15 us, 128 take 17: in the kernel 2.5 us until the keys are there, 2.0,
//                     2.3 and 1.4 for the digits, 2.5 to rank and write. (With a line of positions a thread,
//                     turned through LDS, and eight copies of 11 bits first: 21 us.)
//   keep_slab_kernel  longer rows, a workgroup a slab of 32768, four launches: a histogram each, then the
//                     ranks. 131072 positions of 8 kv-heads: about 30 us.
constexpr int kBins = 2048, kHist = 8 * kBins;  // bins at most, and ints of a histogram's copies

template <int PASS>
struct KeepDigit {
  static constexpr int BITS = PASS == 0 ? 10 : 11, SHIFT = PASS == 0 ? 22 : (PASS == 1 ? 11 : 0);
  static constexpr int BINS = 1 << BITS, COPIES = kHist / BINS;
  static constexpr int PER = BINS / kKeepThreads;  // bins of a thread: BINS - 1 - PER tid, and the one below
};

struct KeepLds {
  alignas(16) int hist[2][kHist];  // one is cleared while the other counts
  int wave[2][kKeepWaves];
  uint32_t digit;
  int need;
};

// Of a value that each wave has (the same in its lanes): the sum over the waves before this one, and over all.
// Every thread calls them; a barrier lies between two uses of one `slot`.
__device__ __forceinline__ int keep_wave_values(KeepLds& sh, int slot, int value) {
  const int lane = threadIdx.x % LSA_WAVE;
  if (lane == 0) sh.wave[slot][threadIdx.x / LSA_WAVE] = value;
  __syncthreads();
  return lane < kKeepWaves ? sh.wave[slot][lane] : 0;
}
__device__ __forceinline__ int keep_waves_before(KeepLds& sh, int slot, int value) {
  const int x = keep_wave_values(sh, slot, value);
  return wave_sum(threadIdx.x % LSA_WAVE < threadIdx.x / LSA_WAVE ? x : 0);
}
__device__ __forceinline__ int keep_waves_all(KeepLds& sh, int slot, int value) {
  return wave_sum(keep_wave_values(sh, slot, value));
}

// The bin that the `need`-th key from the top is in, given every thread's counts: its digit, and how
// many of its keys are needed. Ends with a barrier.
template <int PASS>
__device__ __forceinline__ void keep_digit(KeepLds& sh, int need, const int (&c)[2]) {
  using D = KeepDigit<PASS>;
  const int own = D::PER == 2 ? c[0] + c[1] : c[0], to = wave_inclusive_sum(own);
  const int mine = keep_waves_before(sh, 0, __builtin_amdgcn_readlane(to, LSA_WAVE - 1)) + to - own;
  if (mine < need && need <= mine + own) {
    const int e = D::PER == 2 && mine + c[0] < need ? 1 : 0;
    sh.digit = (uint32_t)(D::BINS - 1 - D::PER * (int)threadIdx.x - e);
    sh.need = need - mine - (e ? c[0] : 0);
  }
  __syncthreads();
}
__device__ __forceinline__ void keep_clear(int* hist) {  // no barrier
  int4* h = (int4*)hist;
#pragma unroll
  for (int i = 0; i < kHist / 4 / kKeepThreads; ++i) h[i * kKeepThreads + threadIdx.x] = make_int4(0, 0, 0, 0);
}

// The first of the wave's positions, and a lane's e-th.
template <int R>
__device__ __forceinline__ int keep_base(int p0) {
  return p0 + __builtin_amdgcn_readfirstlane(threadIdx.x / LSA_WAVE) * (R * LSA_WAVE);
}
__device__ __forceinline__ int keep_at(int base, int e) { return base + e * LSA_WAVE + (int)(threadIdx.x % LSA_WAVE); }

// The keys of the thread's R positions (keep_at) from p0 on: the first and last of the row are the largest
// key, which no weight equals, positions past it the least. The histograms are cleared while the keys are on
// their way.
template <int R>
__device__ __forceinline__ void keep_load(KeepLds& sh, const KeepArgs& a, int64_t u, int64_t b, int g, int n, int p0,
                                          uint32_t (&x)[R]) {
  const int base = keep_base<R>(p0);
  const uint32_t* src = a.keys ? a.keys + u * a.T : (const uint32_t*)(a.mass + b * a.mass_sb + g * a.mass_sh);
  if ((int64_t)base + R * LSA_WAVE <= a.T) {  // uniform
    src += base;
#pragma unroll
    for (int e = 0; e < R; ++e) x[e] = src[keep_at(0, e)];
  } else {
#pragma unroll
    for (int e = 0; e < R; ++e) x[e] = src[min((int64_t)keep_at(base, e), a.T - 1)];
  }
  keep_clear(sh.hist[0]);
  keep_clear(sh.hist[1]);
  __syncthreads();
  if (!a.keys) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < R; ++e) top = max(top, x[e]);
    if (!__any(top > 0x7F800000u)) {  // neither NaN nor a sign
#pragma unroll
      for (int e = 0; e < R; ++e) x[e] |= 0x80000000u;
    } else {
#pragma unroll
      for (int e = 0; e < R; ++e) x[e] = seen_key(__uint_as_float(x[e]));
    }
  }
  const int last = n - a.window;
  if (base < a.sink || base + R * LSA_WAVE > last) {  // uniform
#pragma unroll
    for (int e = 0; e < R; ++e) {
      const int i = keep_at(base, e);
      x[e] = i < a.sink || i >= last ? 0xFFFFFFFFu : x[e];
      x[e] = i < n ? x[e] : 0u;
    }
  }
}

// Counts digit PASS of the keys that share `thr` in the ones before. Ends with a barrier. Positions past
// the row are counted, as the least key; there are enough of the row's own before they would matter.
template <int R, int PASS>
__device__ __forceinline__ void keep_count(KeepLds& sh, const uint32_t (&x)[R], uint32_t thr) {
  using D = KeepDigit<PASS>;
  int* hist = &sh.hist[PASS % 2][threadIdx.x % D::COPIES];
  constexpr int E = PASS == 2 ? 4 : 1;  // few share two digits: four keys are asked at once
  constexpr uint32_t UP = PASS == 0 ? ~0u : (1u << KeepDigit<PASS == 0 ? 0 : PASS - 1>::SHIFT) - 1;
#pragma unroll
  for (int e0 = 0; e0 < R; e0 += E) {
    uint32_t off = x[e0] ^ thr;
#pragma unroll
    for (int e = 1; e < E; ++e) off = min(off, x[e0 + e] ^ thr);
    if (PASS == 0 || off <= UP) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (E == 1 || (x[e0 + e] ^ thr) <= UP) atomicAdd(&hist[((x[e0 + e] >> D::SHIFT) & (D::BINS - 1)) * D::COPIES], 1);
      }
    }
  }
  __syncthreads();
}

// What the wave holds above and at the threshold.
template <int R>
__device__ __forceinline__ void keep_above(const uint32_t (&x)[R], uint32_t thr, int& gt, int& eq) {
  gt = eq = 0;
#pragma unroll
  for (int e = 0; e < R; ++e) {
    gt += x[e] > thr;
    eq += x[e] == thr;
  }
  const int both = wave_sum(gt | eq << 16);  // of 2048 at most
  gt = both & 0xFFFF;
  eq = both >> 16;
}

// Writes what the wave's positions become, given how many positions before them are above the threshold
// and at it (TIES: some of its own are). Positions past the row tie with NaN alone, and come after every
// position of the row.
template <int R, bool TABLE, bool TIES>
__device__ __forceinline__ void keep_place(const KeepArgs& a, const uint32_t (&x)[R], int base, int n, int keep, uint32_t thr,
                                           int ties, int gt, int eq, int32_t* kept, const int32_t* table,
                                           int32_t* new_table) {
  int first = gt + min(eq, ties);  // kept positions before these
  constexpr int E = R < 8 ? R : 8;
#pragma unroll
  for (int e0 = 0; e0 < R; e0 += E) {
    int32_t y[E];
    if (TABLE) {
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = table[min((int64_t)keep_at(base, e0 + e), a.T - 1)];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t z = x[e0 + e];
      const int i = keep_at(base, e0 + e);
      bool in = z > thr;
      if (TIES) {
        const uint64_t same = __ballot(z == thr);
        const int tie = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, eq));
        in = z >= thr && (z != thr || tie < ties);
        eq += __popcll(same);
      }
      const uint64_t take = __ballot(in);
      const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(take >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)take, first));
      first += __popcll(take);
      if (in) kept[rank] = i;
      if (TABLE && i < a.T) new_table[in ? rank : (i < n ? keep + (i - rank) : i)] = y[e];
    }
  }
}

// Ranks and writes, given how many are above the threshold and at it before the workgroup's positions.
template <int R, bool TABLE>
__device__ __forceinline__ void keep_write(KeepLds& sh, const KeepArgs& a, const uint32_t (&x)[R], int base, int n, int keep,
                                           uint32_t thr, int ties, int gt0, int eq0, int32_t* kept, const int32_t* table,
                                           int32_t* new_table) {
  int gt, eq;
  keep_above<R>(x, thr, gt, eq);
  static_assert(kSlab < 1 << 16, "two counts in a word");
  const uint32_t before = (uint32_t)keep_waves_before(sh, 0, gt | eq << 16);
  gt0 += (int)(before & 0xFFFFu);
  eq0 += (int)(before >> 16);
  if (eq == 0) keep_place<R, TABLE, false>(a, x, base, n, keep, thr, ties, gt0, eq0, kept, table, new_table);  // uniform
  else keep_place<R, TABLE, true>(a, x, base, n, keep, thr, ties, gt0, eq0, kept, table, new_table);
}

// The thread's bins' counts, summed over the copies.
template <int PASS>
__device__ __forceinline__ void keep_bins(const KeepLds& sh, int (&c)[2]) {
  using D = KeepDigit<PASS>;
  c[1] = 0;
#pragma unroll
  for (int e = 0; e < D::PER; ++e) {
    c[e] = 0;
#pragma unroll
    for (int y = 0; y < D::COPIES; y += 4) {
      const int4 z = *(const int4*)&sh.hist[PASS % 2][(D::BINS - 1 - D::PER * (int)threadIdx.x - e) * D::COPIES + y];
      c[e] += z.x + z.y + z.z + z.w;
    }
  }
}

template <int R, int PASS>
__device__ __forceinline__ void keep_pass(KeepLds& sh, const uint32_t (&x)[R], uint32_t& thr, int& ties) {
  if (PASS == 1) keep_clear(sh.hist[0]);
  keep_count<R, PASS>(sh, x, thr);
  int c[2];
  keep_bins<PASS>(sh, c);
  keep_digit<PASS>(sh, ties, c);
  thr |= sh.digit << KeepDigit<PASS>::SHIFT;
  ties = sh.need;
}

template <int R, bool TABLE>
__global__ __launch_bounds__(kKeepThreads) void keep_kernel(KeepArgs a) {
  __shared__ KeepLds sh;
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
  keep_load<R>(sh, a, u, b, g, n, 0, x);
  uint32_t thr = 0;
  int ties = a.budget;
  keep_pass<R, 0>(sh, x, thr, ties);
  keep_pass<R, 1>(sh, x, thr, ties);
  keep_pass<R, 2>(sh, x, thr, ties);
  keep_write<R, TABLE>(sh, a, x, keep_base<R>(0), n, keep, thr, ties, 0, 0, kept, table, new_table);
}

// A row in slabs of 32768 positions, a workgroup a slab; grid (selection, slab). Phases 0, 1 and 2 leave
// each slab's histogram of their digit, and phases 1, 2 and 3 add the slabs' up and find the digit
// (slab 0 keeps it for the phases after the next). Phase 3 ranks: what is kept before a slab follows from
// the earlier slabs' histograms.
struct KeepFound {
  uint32_t thr;  // the digits so far
  int ties;      // keys needed of those that share them
  int gt, eq;    // phase 3: above and at the threshold in the slabs before
};

// Digit Q from the slabs' histograms of it, or as an earlier phase left it.
template <int Q, int PHASE>
__device__ __forceinline__ void keep_found(KeepLds& sh, const int* hist, int slab, int slabs, int2* state, KeepFound& f) {
  using D = KeepDigit<Q>;
  const int tid = threadIdx.x;
  int c[2] = {0, 0}, before[2] = {0, 0};  // of all slabs, and of the ones before
  if (Q == PHASE - 1 || PHASE == 3) {
    const int* h = hist + D::BINS - D::PER * (tid + 1);
#pragma unroll 4
    for (int y = 0; y < slabs; ++y) {
      int x[2] = {0, 0};
      if constexpr (D::PER == 2) {
        const int2 z = *(const int2*)(h + (int64_t)y * kBins);
        x[0] = z.y; x[1] = z.x;
      } else {
        x[0] = h[(int64_t)y * kBins];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        c[e] += x[e];
        before[e] += y < slab ? x[e] : 0;
      }
    }
  }
  if (Q == PHASE - 1) {
    keep_digit<Q>(sh, f.ties, c);
    if (PHASE < 3 && slab == 0 && tid == 0) state[Q] = make_int2((int)sh.digit, sh.need);
  } else {
    if (tid == 0) {
      const int2 x = state[Q];
      sh.digit = (uint32_t)x.x;
      sh.need = x.y;
    }
    __syncthreads();
  }
  const uint32_t digit = sh.digit;
  f.ties = sh.need;
  f.thr |= digit << D::SHIFT;
  if (PHASE == 3) {
    int more = 0, same = 0;
#pragma unroll
    for (int e = 0; e < D::PER; ++e) {
      const uint32_t bin = (uint32_t)(D::BINS - 1 - D::PER * tid - e);
      more += bin > digit ? before[e] : 0;
      same += Q == 2 && bin == digit ? before[e] : 0;
    }
    f.gt += keep_waves_all(sh, 1, wave_sum(more));
    if (Q == 2) {
      __syncthreads();
      f.eq = keep_waves_all(sh, 1, wave_sum(same));
    }
  }
  __syncthreads();  // the digit is read before the next takes its place
}

template <int PHASE, bool TABLE>
__global__ __launch_bounds__(kKeepThreads) void keep_slab_kernel(KeepArgs a) {
  constexpr int R = kSlabRun;
  __shared__ KeepLds sh;
  const int tid = threadIdx.x;
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
    if (n <= a.budget) {  // uniform: all of it
      for (int i = p0 + tid; i < p1; i += kKeepThreads) {
        if (i < n) kept[i] = i;
        if (TABLE) new_table[i] = table[i];
      }
    }
  }
  if (n <= a.budget) return;
  int* hist = a.hist + u * slabs * kBins;             // of phase 0, [slab][bin]
  const int64_t phase_hist = (int64_t)gridDim.x * slabs * kBins;
  int2* state = a.state + u * 2;                      // digits (and what they leave needed) of phases 0, 1
  KeepFound f{0, a.budget, 0, 0};
  if constexpr (PHASE > 0) keep_found<0, PHASE>(sh, hist, slab, slabs, state, f);
  if constexpr (PHASE > 1) keep_found<1, PHASE>(sh, hist + phase_hist, slab, slabs, state, f);
  if constexpr (PHASE > 2) keep_found<2, PHASE>(sh, hist + 2 * phase_hist, slab, slabs, state, f);
  uint32_t x[R];
  keep_load<R>(sh, a, u, b, g, n, p0, x);
  if constexpr (PHASE < 3) {
    using D = KeepDigit<PHASE>;
    keep_count<R, PHASE>(sh, x, f.thr);
    int c[2];
    keep_bins<PHASE>(sh, c);
    int* to = hist + PHASE * phase_hist + (int64_t)slab * kBins + D::BINS - D::PER * (tid + 1);
    if constexpr (D::PER == 2) *(int2*)to = make_int2(c[1], c[0]);
    else *to = c[0];
  } else {
    keep_write<R, TABLE>(sh, a, x, keep_base<R>(p0), n, keep, f.thr, f.ties, f.gt, f.eq, kept, table, new_table);
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

// HBM-bound: each kept row read and written once (16 caches of 32768 cut to 8192, 1.07 GB moved: 222 us,
// 4.8 TB/s; one: 12 us). grid (rows of the new cache a workgroup, B).
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
