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
  for (int h = 0; h < a.Hkv; ++h) sum += (double)m[h * a.mass_sh];
  a.keys_out[b * a.T + i] = ok ? seen_key((float)sum) : 0u;
}

// One workgroup a selection.
__global__ __launch_bounds__(kKeepThreads) void keep_kernel(KeepArgs a) {
  __shared__ int hist[256];
  __shared__ int wave_gt[kKeepWaves], wave_eq[kKeepWaves];
  __shared__ uint32_t sh_prefix;
  __shared__ int sh_need;
  const int tid = threadIdx.x, lane = tid & (LSA_WAVE - 1), w = tid / LSA_WAVE;
  const int64_t u = blockIdx.x;
  const int64_t b = u / a.G;
  const int g = (int)(u % a.G);
  const int n = row_length(a, b);
  const int keep = n < a.budget ? n : a.budget;
  if (g == 0 && tid == 0) a.new_lengths[b] = keep;
  const bool all = n <= a.budget;
  const int lo = min(a.sink, n), hi = all ? lo : n - a.window;  // the positions that compete
  const float* mass = a.mass + b * a.mass_sb + g * a.mass_sh;
  const uint32_t* keys = a.keys + u * a.T;
  auto key = [&](int i) { return a.keys ? keys[i] : seen_key(mass[i]); };

  uint32_t thr = 0xFFFFFFFFu;
  int ties = 0;  // how many of the keys equal to the threshold stay
  if (!all) {    // uniform
    uint32_t prefix = 0, mask = 0;
    int need = a.budget - lo - (n - hi);
    if (need > 0) {
      for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = lo + tid; i < hi; i += kKeepThreads) {
          const uint32_t x = key(i);
          if ((x & mask) == prefix) atomicAdd(&hist[(x >> shift) & 255], 1);
        }
        __syncthreads();
        if (w == 0) {  // lane l owns bins 255 - 4 l .. 252 - 4 l, from the top
          int c[4], mine = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) mine += c[e] = hist[255 - 4 * lane - e];
          const int inc = wave_inclusive_sum(mine);
          int above = inc - mine;
          if (above < need && need <= inc) {
            int e = 0;
            while (above + c[e] < need) above += c[e++];
            sh_prefix = prefix | ((uint32_t)(255 - 4 * lane - e) << shift);
            sh_need = need - above;
          }
        }
        __syncthreads();
        prefix = sh_prefix;
        need = sh_need;
        mask |= 255u << shift;
      }
      thr = prefix;
      ties = need;
    }
  }
  int32_t* kept = a.kept + u * a.budget;
  const int32_t* table = a.table ? a.table + b * a.table_stride : nullptr;
  int32_t* new_table = a.new_table ? a.new_table + b * a.new_stride : nullptr;
  const uint64_t below = lane == 0 ? 0ull : ~0ull >> (LSA_WAVE - lane);
  int base = 0, base_eq = 0;  // kept for their place or weight, and at the threshold, before this chunk
  for (int i0 = 0; i0 < n; i0 += kKeepThreads) {
    const int i = i0 + tid;
    const bool in = i < n;
    const bool middle = in && !all && i >= lo && i < hi;
    const uint32_t x = middle ? key(i) : 0u;
    const bool gt = in && (!middle || x > thr);
    const bool eq = middle && x == thr && ties > 0;
    const uint64_t mg = __ballot(gt), me = __ballot(eq);
    if (lane == 0) {
      wave_gt[w] = __popcll(mg);
      wave_eq[w] = __popcll(me);
    }
    __syncthreads();
    int bg = base, be = base_eq;
#pragma unroll
    for (int y = 0; y < kKeepWaves; ++y) {
      const int cg = wave_gt[y], ce = wave_eq[y];
      bg += y < w ? cg : 0;
      be += y < w ? ce : 0;
      base += cg;
      base_eq += ce;
    }
    __syncthreads();
    bg += __popcll(mg & below);
    be += __popcll(me & below);
    const int rank = bg + min(be, ties);  // kept positions before i
    const bool stays = gt || (eq && be < ties);
    if (stays) kept[rank] = i;
    if (in && new_table) new_table[stays ? rank : keep + (i - rank)] = table[i];
  }
  for (int j = keep + tid; j < a.budget; j += kKeepThreads) kept[j] = -1;
  if (new_table) {
    for (int64_t i = n + tid; i < a.T; i += kKeepThreads) new_table[i] = table[i];
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

int check_keep(const char* who, const void* mass, int64_t B, int32_t Hkv, int64_t T, int64_t mass_sb, int64_t mass_sh,
               int32_t budget, int32_t window, int32_t sink, const void* kept, const void* new_lengths) {
  LSA_REQUIRE(mass && kept && new_lengths, LSA_ERR_NULL, "%s: NULL pointer", who);
  LSA_REQUIRE(B >= 0 && B <= 65535 && Hkv >= 1 && T >= 1 && T <= 0x7FFFFFFF, LSA_ERR_SHAPE,
              "%s: needs 0..65535 rows of 1..2^31-1 positions and a kv-head", who);
  LSA_REQUIRE(mass_sb >= 0 && mass_sh >= 0, LSA_ERR_SHAPE, "%s: weight strides must be >= 0", who);
  LSA_REQUIRE(budget >= 1 && budget <= T, LSA_ERR_SHAPE, "%s: budget %d not in 1..%lld", who, budget, (long long)T);
  LSA_REQUIRE(window >= 0 && sink >= 0 && (int64_t)window + sink <= budget, LSA_ERR_SHAPE,
              "%s: window %d and sink %d must fit the budget %d", who, window, sink, budget);
  LSA_REQUIRE(B * (int64_t)Hkv <= 0x7FFFFFFF, LSA_ERR_SHAPE, "%s: too many rows", who);
  return LSA_OK;
}

}  // namespace

extern "C" size_t lsa_evict_scratch_bytes(int64_t B, int64_t T, int summed) {
  return summed && B > 0 && T > 0 ? (size_t)B * (size_t)T * sizeof(uint32_t) : 0;
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
  const size_t need = lsa_evict_scratch_bytes(B, T, shared);
  LSA_REQUIRE(need == 0 || (scratch && scratch_bytes >= need), LSA_ERR_WORKSPACE,
              "lsa_evict_keep: scratch missing or %zu < %zu bytes", scratch_bytes, need);
  if (B == 0) return LSA_OK;
  KeepArgs a = {};
  a.mass = mass; a.mass_sb = mass_batch_stride; a.mass_sh = mass_head_stride; a.lengths = lengths; a.T = T;
  a.G = shared ? 1 : Hkv; a.Hkv = Hkv; a.budget = budget; a.window = window; a.sink = sink;
  a.kept = kept; a.new_lengths = new_lengths; a.table = table; a.table_stride = table_stride;
  a.new_table = new_table; a.new_stride = new_table_stride; a.pool = pool_rows;
  hipStream_t s = (hipStream_t)stream;
  if (shared) {
    a.keys = a.keys_out = (uint32_t*)scratch;
    const dim3 grid((unsigned)((T + LSA_BLOCK - 1) / LSA_BLOCK), (unsigned)B);
    seen_keys_kernel<<<grid, LSA_BLOCK, 0, s>>>(a);
    LSA_LAUNCHED("lsa_evict_keep");
  }
  keep_kernel<<<dim3((unsigned)(B * a.G)), kKeepThreads, 0, s>>>(a);
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
