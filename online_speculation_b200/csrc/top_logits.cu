// The k largest logits of every row with their columns, and the row's logsumexp, in one pass.
//
// A logit becomes a 64-bit key: its order-preserving 32 bits above the inverted column, so
// that "larger key" means larger logit and, between equal ones, the lower column; every key is
// distinct.
//
// A block streams its columns in ascending order and appends what beats the bar, a k-th largest so
// far, to a shared-memory buffer.  The bar comes from a select after the first 2048 columns and again
// whenever the columns seen have grown six times: about 5 k of random logits pass in between, so
// most groups of eight logits cost their exponentials, one maximum and one compare, and warps run
// free of each other between the selects.  A buffer that runs over (rising rows) marks the row,
// and its columns are gone through again with a select before every chunk that might not fit.  Few
// rows are cut into column ranges whose winners a second launch merges.
#include "common.cuh"
#include "top_logits.h"

#include <algorithm>

namespace osb {
namespace {

// What a select leaves of n candidates for the k largest to be ranked one by one.
__host__ __device__ constexpr int rank_limit(int k) { return k + k / 4 > 192 ? k + k / 4 : 192; }

constexpr int kThreads = 256;
constexpr int kBlocks = 4;                       // per SM
constexpr int kWarps = kThreads / 32;
constexpr int kPer = 8;                          // logits a thread takes at a time
constexpr int kChunk = kThreads * kPer;
constexpr int kCap = 4096;                       // candidates
constexpr int kGrow = 6;                         // columns seen between two selects grow by this
constexpr int kBins = 2048;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.0f;                   // log2 units above its reference at which a thread rescales
constexpr float kSpread = 32.0f;                 // logits below the largest that the first histogram resolves
static_assert(kChunk + rank_limit(kTopLogitsMax) <= kCap, "a chunk fits on top of what a select leaves");

struct Smem {
  unsigned long long cand[kCap + 2];
  int hist[kBins];
  int warp_tot[kWarps];
  int count;                                     // entries of cand
  int keyed;                                     // the first of them are keys, the others (column, logit bits)
  int overflow;
  int bin, above, in_bin;
  unsigned bar;
  float lo[kWarps], hi[kWarps];
  double s[kWarps];
  float m[kWarps];
};

__device__ __forceinline__ unsigned order_key(float x) {
  if (!(x == x)) return 0xFFFFFFFFu;             // NaN sorts above everything
  const unsigned b = __float_as_uint(x + 0.0f);  // -0 equals +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ unsigned long long make_key(float x, int col) {
  return (static_cast<unsigned long long>(order_key(x)) << 32) | (0xFFFFFFFFu - static_cast<unsigned>(col));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Float of an order key (inverse of order_key; the NaN key gives a NaN).
__device__ __forceinline__ float key_float(unsigned k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// Turns the entries appended since the last call into keys.  All threads call it.
__device__ __forceinline__ void make_keys(Smem& sm, int n) {
  for (int i = sm.keyed + threadIdx.x; i < n; i += kThreads) {
    const unsigned long long e = sm.cand[i];
    sm.cand[i] = make_key(__uint_as_float(static_cast<unsigned>(e >> 32)), static_cast<int>(e));
  }
  __syncthreads();
  if (threadIdx.x == 0) sm.keyed = n;
}

// This thread's bins, from the highest down: their entries, and those in higher bins than its first.  All threads
// call it, after a barrier.
constexpr int kMine = kBins / kThreads;

__device__ __forceinline__ int scan_bins(Smem& sm, int (&own)[kMine]) {
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  int tot = 0;
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    own[j] = sm.hist[kBins - 1 - (tid * kMine + j)];
    tot += own[j];
  }
  int incl = tot;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sm.warp_tot[warp] = incl;
  __syncthreads();
  int before = incl - tot;
#pragma unroll
  for (int q = 0; q < kWarps; ++q) before += q < warp ? sm.warp_tot[q] : 0;
  return before;
}

// Finds in sm.hist, from the highest bin down, the bin that holds the need-th entry: sm.bin, its
// entries sm.in_bin and those above it sm.above.  All threads call it, after a barrier; ends in one.
__device__ __forceinline__ void find_bin(Smem& sm, int need) {
  int own[kMine];
  int before = scan_bins(sm, own);
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    if (before < need && before + own[j] >= need) {
      sm.bin = kBins - 1 - (static_cast<int>(threadIdx.x) * kMine + j);
      sm.above = before;
      sm.in_bin = own[j];
    }
    before += own[j];
  }
  if (threadIdx.x == 0) sm.count = 0;
  __syncthreads();
}

__device__ __forceinline__ void clear_bins(Smem& sm) {
  for (int i = threadIdx.x; i < kBins / 4; i += kThreads) reinterpret_cast<int4*>(sm.hist)[i] = make_int4(0, 0, 0, 0);
}

// Bins that rise with the logit, linear over the range of the candidates.
struct LinearBins {
  float lo, scale;
  __device__ __forceinline__ bool usable() const { return scale > 0.0f && scale < INFINITY; }
  // NaN and +inf in the last bin, -inf and everything far below in the first
  __device__ __forceinline__ int of(unsigned long long key) const {
    const float x = key_float(static_cast<unsigned>(key >> 32));
    if (!(x < INFINITY)) return kBins - 1;
    return static_cast<int>(fminf(fmaxf((x - lo) * scale, 0.0f), static_cast<float>(kBins - 1)));
  }
};

// For the keys cand[0 .. n); leaves the histogram cleared.  All threads call it; ends in a barrier.
__device__ __forceinline__ LinearBins linear_bins(Smem& sm, int n) {
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  float lo = INFINITY, hi = -INFINITY;
  for (int i = tid; i < n; i += kThreads) {
    const float x = key_float(static_cast<unsigned>(sm.cand[i] >> 32));
    if (fabsf(x) < INFINITY) {
      lo = fminf(lo, x);
      hi = fmaxf(hi, x);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (lane == 0) {
    sm.lo[warp] = lo;
    sm.hi[warp] = hi;
  }
  clear_bins(sm);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kWarps; ++q) {
    lo = fminf(lo, sm.lo[q]);
    hi = fmaxf(hi, sm.hi[q]);
  }
  lo = fmaxf(lo, hi - kSpread);
  return {lo, (kBins - 1) / (hi - lo)};
}

// Moves the entries that keep(key) holds for to the front, in rounds: a round's entries are read
// before any is written, and written no further than they stood.
template <typename Keep>
__device__ __forceinline__ void compact(Smem& sm, int n, Keep keep) {
  const int lane = threadIdx.x % 32;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    const unsigned long long key = i < n ? sm.cand[i] : 0ull;
    const bool on = i < n && keep(key);
    const unsigned ballot = __ballot_sync(0xffffffffu, on);
    __syncthreads();
    int at = 0;
    if (lane == 0 && ballot != 0) at = atomicAdd(&sm.count, __popc(ballot));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(ballot & ((1u << lane) - 1u));
    if (on) sm.cand[at] = key;
  }
  __syncthreads();
}

// Cuts the keys cand[0 .. n) down to at most `limit` (k <= limit) that hold the k largest; returns how
// many are left, sm.count.  sm.bar is the smallest logit left: there are k at least as large in
// earlier columns, so a later one has to exceed it.  All threads call it.
//
// First a histogram that is linear in the logit, over the range of the candidates (its bins are about
// equally full, where the leading bits of a float crowd into a few); what that leaves too many
// of, many equal logits or far outliers, is cut by radix digits of the key from the top.
__device__ int narrow(Smem& sm, int n, int k, int limit) {
  const int tid = threadIdx.x, lane = tid % 32;
  if (n <= limit) return n;
  if (tid == 0) sm.bar = 0xFFFFFFFFu;
  const LinearBins bins = linear_bins(sm, n);
  if (bins.usable()) {
    for (int i = tid; i < n; i += kThreads) atomicAdd(&sm.hist[bins.of(sm.cand[i])], 1);
    __syncthreads();
    find_bin(sm, k);
    const int edge = sm.bin;
    compact(sm, n, [&](unsigned long long key) { return bins.of(key) >= edge; });
    n = sm.count;
  }
  if (n > limit) {
    unsigned long long prefix = 0, mask = 0;     // keys with (key & mask) == prefix are undecided
    int need = k;                                // of those, how many belong to the k largest
    for (int digit = 0; digit < 6; ++digit) {    // of 11, 11 and 10 bits: three of the logit, three of the column
      const int part = digit % 3;
      const int shift = (digit < 3 ? 32 : 0) + (part == 0 ? 21 : part == 1 ? 10 : 0);
      const unsigned long long field = (part == 2 ? 0x3FFull : 0x7FFull) << shift;
      __syncthreads();
      clear_bins(sm);
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const unsigned long long c = sm.cand[i];
        if ((c & mask) == prefix) atomicAdd(&sm.hist[static_cast<int>((c & field) >> shift)], 1);
      }
      __syncthreads();
      find_bin(sm, need);
      prefix |= static_cast<unsigned long long>(sm.bin) << shift;
      mask |= field;
      need -= sm.above;
      if (k - need + sm.in_bin <= limit) break;  // everything above the bin, and the bin
    }
    compact(sm, n, [&](unsigned long long key) { return (key & mask) >= prefix; });
  }
  const int kept = sm.count;
  unsigned low = 0xFFFFFFFFu;
  for (int i = tid; i < kept; i += kThreads) low = min(low, static_cast<unsigned>(sm.cand[i] >> 32));
  low = __reduce_min_sync(0xffffffffu, low);
  if (lane == 0) atomicMin(&sm.bar, low);
  if (tid == 0) sm.keyed = kept;
  __syncthreads();                               // nothing is appended before everyone has the count
  return kept;
}

// Sorts the keys cand[0 .. n), n at most kCap / 2, descending; ends in a barrier.  A counting sort over linear bins,
// then compares within a bin.
__device__ __noinline__ void sort_keys(int n) {
  extern __shared__ __align__(16) uint8_t raw[];
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  static_assert(2 * rank_limit(kTopLogitsMax) <= kCap, "room for the sorted keys");
  const int tid = threadIdx.x;
  unsigned long long* sorted = sm.cand + kCap / 2;
  __syncthreads();
  LinearBins bins = linear_bins(sm, n);
  if (!bins.usable()) bins = {0.0f, 0.0f};               // no spread: the first bin, infinities and NaN in the last
  for (int i = tid; i < n; i += kThreads) atomicAdd(&sm.hist[bins.of(sm.cand[i])], 1);
  __syncthreads();
  int own[kMine];
  int before = scan_bins(sm, own);
#pragma unroll
  for (int j = 0; j < kMine; ++j) {                      // where a bin's keys begin
    sm.hist[kBins - 1 - (tid * kMine + j)] = before;
    before += own[j];
  }
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    const unsigned long long key = sm.cand[i];
    sorted[atomicAdd(&sm.hist[bins.of(key)], 1)] = key;  // and, when all are placed, where they end
  }
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    const unsigned long long key = sorted[i];
    const int bin = bins.of(key);
    const int first = bin + 1 < kBins ? sm.hist[bin + 1] : 0, end = sm.hist[bin];
    int rank = first;
    for (int j = first; j < end; ++j) rank += sorted[j] > key;
    sm.cand[rank] = key;
  }
  __syncthreads();
}

// Calls put(key, rank) for the k largest of cand[0 .. n), n at most rank_limit(k), n >= k or all of them.
// More of them than threads are sorted: comparing all with all grows with k^2 (1021 rows of 151937, k 256: 142 us for
// 135 us).  Fewer are compared, all with all: the sort's barriers take longer (4 rows of 152064, k 16: 18.5 us
// for 15.8 us).
template <typename Put>
__device__ void rank_top(Smem& sm, int n, int k, Put put) {
  const int tid = threadIdx.x;
  if (n > kThreads) {
    sort_keys(n);
    for (int i = tid; i < min(n, k); i += kThreads) put(sm.cand[i], i);
    return;
  }
  if (tid == 0 && (n & 1)) sm.cand[n] = 0ull;            // below every key
  __syncthreads();
  const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(sm.cand);
  if (tid < n) {
    const unsigned long long key = sm.cand[tid];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < (n + 1) / 2; ++j) {
      const ulonglong2 p = pairs[j];
      rank += (p.x > key) + (p.y > key);
    }
    if (rank < k) put(key, rank);
  }
}

__device__ __forceinline__ float load_one(const void* p, int bf16, long long i) {
  return bf16 ? bf2f(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}

// Eight logits as loaded: 32 bytes of fp32, 16 of bf16.
template <bool kBf16>
struct Raw {
  uint4 v[kBf16 ? 1 : 2];
};

template <bool kBf16>
__device__ __forceinline__ void load_raw(const char* row, int i, Raw<kBf16>& r) {
  const uint4* p = reinterpret_cast<const uint4*>(row + static_cast<long long>(i) * (kBf16 ? 2 : 4));
  r.v[0] = p[0];
  if (!kBf16) r.v[kBf16 ? 0 : 1] = p[1];
}

template <bool kBf16>
__device__ __forceinline__ void fill_raw(Raw<kBf16>& r) {
#pragma unroll
  for (uint4& v : r.v) v = make_uint4(0, 0, 0, 0);
}

template <bool kBf16>
__device__ __forceinline__ void unpack(const Raw<kBf16>& r, float (&x)[kPer]) {
  if (kBf16) {
    const unsigned u[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(u[j] << 16);
      x[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint4 v = r.v[kBf16 ? 0 : q];
      x[4 * q] = __uint_as_float(v.x);
      x[4 * q + 1] = __uint_as_float(v.y);
      x[4 * q + 2] = __uint_as_float(v.z);
      x[4 * q + 3] = __uint_as_float(v.w);
    }
  }
}

// Two fp32 lanes an instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// A thread's sum of exponentials about a reference of its own.  The reference trails the maximum
// by at most kRaise log2 units and starts at the lowest finite number: rows of -inf sum to 0.
struct RunningSum {
  float ref = -3.402823466e38f, raise = -INFINITY, s = 0.0f;
  __device__ __forceinline__ void lift(float top, float c2) {
    if (top > raise) {
      const float now = fminf(top, 3.402823466e38f);   // +inf adds inf about a finite reference
      s *= ex2((ref - now) * c2);
      ref = now;
      raise = top + kRaise / c2;
    }
  }
  __device__ __forceinline__ void add_eight(const float (&x)[kPer], float c2) {
    const float2 r = make_float2(-ref, -ref), c = make_float2(c2, c2);
    float2 t = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < kPer / 2; ++j) {
      const float2 d = mul2(add2(make_float2(x[2 * j], x[2 * j + 1]), r), c);
      t = add2(t, make_float2(ex2(d.x), ex2(d.y)));
    }
    s += t.x + t.y;
  }
};

// Where x[j] is marked in a word of eight: the even ones in the lower half, as packed compares leave them.
__device__ constexpr unsigned mark(int j) { return 1u << (j / 2 + 16 * (j % 2)); }

__device__ __forceinline__ float largest(const Raw<false>&, const float (&x)[kPer]) {
  return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
}

// The logits that are not at or below the bar (a NaN on either side: marked).
__device__ __forceinline__ unsigned beyond(const Raw<false>&, const float (&x)[kPer], float bar) {
  unsigned pass = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (!(x[j] <= bar)) pass |= mark(j);
  return pass;
}

// bf16 two at a time; the bar is one of the logits, so its rounding is exact.
__device__ __forceinline__ __nv_bfloat162 pair_of(unsigned u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); }

__device__ __forceinline__ float largest(const Raw<true>& r, const float (&)[kPer]) {
  const uint4 v = r.v[0];
  const __nv_bfloat162 m = __hmax2(__hmax2(pair_of(v.x), pair_of(v.y)), __hmax2(pair_of(v.z), pair_of(v.w)));
  return fmaxf(__low2float(m), __high2float(m));
}

__device__ __forceinline__ unsigned beyond(const Raw<true>& r, const float (&)[kPer], float bar) {
  const __nv_bfloat162 b = __float2bfloat162_rn(bar);
  const unsigned u[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
  unsigned pass = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) pass |= __hgtu2_mask(pair_of(u[q]), b) & (mark(2 * q) | mark(2 * q + 1));
  return pass;
}

// Appends the logits marked in `pass` (x[j]: column col + j).
__device__ __forceinline__ void append(Smem& sm, const float (&x)[kPer], int col, unsigned pass) {
  if (pass == 0) return;
  const int mine = __popc(pass);
  int at = atomicAdd(&sm.count, mine);
  if (at + mine > kCap) {
    sm.overflow = 1;
    return;
  }
  uint2* dst = reinterpret_cast<uint2*>(sm.cand) + at;
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (pass & mark(j)) *dst++ = make_uint2(col + j, __float_as_uint(x[j]));
}

// A row's outputs; cand holds n keys, the k largest among them.
__device__ void write_row(const TopLogitsArgs& a, Smem& sm, int n, int row) {
  const char* base = static_cast<const char*>(a.logits) + static_cast<long long>(row) * a.ld * (a.bf16 ? 2 : 4);
  rank_top(sm, n, a.k, [&](unsigned long long key, int rank) {
    const int col = static_cast<int>(0xFFFFFFFFu - static_cast<unsigned>(key));
    const long long o = static_cast<long long>(row) * a.k + rank;
    a.ids[o] = col;
    a.values[o] = load_one(base, a.bf16, col);   // the logit itself: its key lost the sign of -0
  });
}

// Combines every thread's (max, sum) of its logits; the result is valid in thread 0.
__device__ void fold(Smem& sm, float m, float s, float c2, float& m_out, double& s_out) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const float wm = warp_max(m);
  double v = (m == -INFINITY && s == 0.0f) ? 0.0 : static_cast<double>(s) * exp2f((m - wm) * c2);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0) {
    sm.m[warp] = wm;
    sm.s[warp] = v;
  }
  __syncthreads();
  if (warp == 0) {
    const float mine = lane < kWarps ? sm.m[lane] : -INFINITY;
    const float top = warp_max(mine);
    double t = lane < kWarps ? sm.s[lane] : 0.0;
    if (!(mine == -INFINITY && t == 0.0)) t *= exp2f((mine - top) * c2);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    m_out = top;
    s_out = t;
  }
}

template <bool kBf16>
__global__ void __launch_bounds__(kThreads, kBlocks) top_logits_kernel(const TopLogitsArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  const int tid = threadIdx.x;
  const int row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  pdl_trigger();
  pdl_wait();
  const int per = (a.V + a.splits - 1) / a.splits;
  const int c0 = min(a.V, split * per), c1 = min(a.V, c0 + per);
  constexpr int kSize = kBf16 ? 2 : 4;
  constexpr int kAhead = kBf16 ? 4 : 2;          // groups of eight in flight: 64 bytes a thread
  const char* base = static_cast<const char*>(a.logits) + static_cast<long long>(row) * a.ld * kSize;
  const float it = a.inv_temp != nullptr ? a.inv_temp[row] : 1.0f;
  const float c2 = it * kLog2e;

  // columns before the first 16-byte boundary, then groups of eight, then the ragged end
  const uintptr_t start = reinterpret_cast<uintptr_t>(base + static_cast<long long>(c0) * kSize);
  const int head = min(c1 - c0, static_cast<int>((16 - (start & 15)) & 15) / kSize);
  const int v0 = c0 + head;
  const int groups = (c1 - v0) / kPer;
  const int tail0 = v0 + groups * kPer;
  const char* body = base + static_cast<long long>(v0) * kSize;
  if (tid == 0) {
    sm.count = 0;
    sm.keyed = 0;
    sm.overflow = 0;
  }
  __syncthreads();
  RunningSum sum;
  float bar = __uint_as_float(0x7FFFFFFFu);      // NaN: no bar yet, everything passes

  auto group = [&](const Raw<kBf16>& r, int col) {      // whole warps
    float x[kPer];
    unpack<kBf16>(r, x);
    const float top = largest(r, x);
    sum.lift(top, c2);
    sum.add_eight(x, c2);
    // a NaN never shows in a maximum, but stays in the sum
    if (__any_sync(0xffffffffu, !(top <= bar) || !(sum.s == sum.s))) append(sm, x, col, beyond(r, x, bar));
  };
  auto single = [&](int col, bool on) {                 // one column a thread
    float x[kPer] = {0.0f};
    if (on) {
      x[0] = load_one(base, kBf16, col);
      sum.lift(x[0], c2);
      sum.s += ex2((x[0] - sum.ref) * c2);
    }
    append(sm, x, col, on && !(x[0] <= bar) ? mark(0) : 0u);
  };
  auto raise = [&]() {                                  // all threads
    __syncthreads();
    const int n = min(sm.count, kCap);
    __syncthreads();
    const int limit = rank_limit(a.k);
    if (n > limit) {
      make_keys(sm, n);
      narrow(sm, n, a.k, limit);
      bar = key_float(sm.bar);
    }
  };
  auto run = [&](int from, int to) {                    // groups [from, to), multiples of kThreads
    const int count = (to - from) / kThreads;
    int g = from + tid;
    Raw<kBf16> next[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (u < count) load_raw<kBf16>(body, (g + u * kThreads) * kPer, next[u]);
    for (int left = count; left > 0; left -= kAhead, g += kAhead * kThreads) {
      Raw<kBf16> now[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        now[u] = next[u];
        if (kAhead + u < left) load_raw<kBf16>(body, (g + (kAhead + u) * kThreads) * kPer, next[u]);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (u >= left) break;
        group(now[u], v0 + (g + u * kThreads) * kPer);
      }
    }
  };
  const int whole = groups / kThreads * kThreads;       // the rest, less than one a thread, comes last
  auto rest = [&]() {
    const int g = whole + tid;
    Raw<kBf16> r;
    fill_raw<kBf16>(r);
    if (g < groups) load_raw<kBf16>(body, g * kPer, r);
    float x[kPer];
    unpack<kBf16>(r, x);
    if (g < groups) {
      sum.lift(largest(r, x), c2);
      sum.add_eight(x, c2);
    }
    append(sm, x, v0 + g * kPer, g < groups ? beyond(r, x, bar) : 0u);
  };
  single(c0 + tid, tid < head);
  int seen = min(groups, kThreads);
  run(0, min(seen, whole));
  if (whole == 0) rest();
  while (seen < groups) {
    raise();
    // no select just before the end
    const long long grown = static_cast<long long>(seen) * kGrow;
    const int next = grown + grown / 2 >= groups ? groups : static_cast<int>(grown);
    run(seen, min(next, whole));
    if (next == groups) rest();
    seen = next;
  }
  single(tail0 + tid, tail0 + tid < c1);
  __syncthreads();
  if (sm.overflow) {
    __syncthreads();
    // the candidates again, with room made before every chunk
    if (tid == 0) sm.count = sm.keyed = 0;
    unsigned bar_key = 0;                        // 0: everything passes
    for (int col0 = c0; col0 < c1; col0 += kChunk) {
      __syncthreads();
      const int held = sm.count;
      __syncthreads();
      if (held > kCap - kChunk) {
        make_keys(sm, held);
        narrow(sm, held, a.k, rank_limit(a.k));
        bar_key = sm.bar;
      }
      float x[kPer];
      unsigned pass = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int col = col0 + tid * kPer + j;
        x[j] = 0.0f;
        if (col < c1) {
          x[j] = load_one(base, kBf16, col);
          if (bar_key == 0 || order_key(x[j]) > bar_key) pass |= mark(j);
        }
      }
      append(sm, x, col0 + tid * kPer, pass);
    }
    __syncthreads();
  }
  int n = min(sm.count, kCap);
  make_keys(sm, n);
  n = narrow(sm, n, a.k, rank_limit(a.k));
  float m_row = 0.0f;
  double s_row = 0.0;
  fold(sm, sum.ref, sum.s, c2, m_row, s_row);
  if (a.splits == 1) {
    write_row(a, sm, n, row);
    if (tid == 0) a.lse[row] = static_cast<float>(static_cast<double>(m_row) * it + log(s_row));
    return;
  }
  unsigned long long* dst = a.keys + (static_cast<long long>(row) * a.splits + split) * a.k;
  rank_top(sm, n, a.k, [&](unsigned long long key, int rank) { dst[rank] = key; });
  if (tid == 0) a.part[static_cast<long long>(row) * a.splits + split] = make_float2(m_row, static_cast<float>(s_row));
}

__global__ void __launch_bounds__(kThreads) top_logits_merge_kernel(const TopLogitsArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  const int tid = threadIdx.x, row = blockIdx.x;
  pdl_trigger();
  pdl_wait();
  int n = a.splits * a.k;
  const unsigned long long* src = a.keys + static_cast<long long>(row) * n;
  for (int i = tid; i < n; i += kThreads) sm.cand[i] = src[i];
  const float it = a.inv_temp != nullptr ? a.inv_temp[row] : 1.0f;
  const float c2 = it * kLog2e;
  float m = -INFINITY, s = 0.0f;
  if (tid < a.splits) {
    const float2 p = a.part[static_cast<long long>(row) * a.splits + tid];
    m = p.x;
    s = p.y;
  }
  __syncthreads();
  n = narrow(sm, n, a.k, rank_limit(a.k));   // the ranges' winners are keys already
  float m_row = 0.0f;
  double s_row = 0.0;
  fold(sm, m, s, c2, m_row, s_row);
  write_row(a, sm, n, row);
  if (tid == 0) a.lse[row] = static_cast<float>(static_cast<double>(m_row) * it + log(s_row));
}

template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, bool (&set)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && set[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(Smem)));
  if (e == cudaSuccess && dev < 64) set[dev] = true;
  return e;
}

}  // namespace

int top_logits_splits(int R, int V, int k) {
  // every SM full; a range is two chunks at least, so that it has k columns, and the merge buffer holds
  // all winners
  static_assert(2 * kChunk - kThreads >= kTopLogitsMax, "the last range has k columns too");
  const int want = (kBlocks * 148 + R - 1) / std::max(R, 1);
  return std::max(1, std::min({want, V / (2 * kChunk), kCap / k, kThreads}));
}

cudaError_t top_logits_launch(const TopLogitsArgs& a, cudaStream_t stream) {
  static bool set_f[64], set_b[64], set_m[64];
  cudaError_t e = a.bf16 ? allow_smem(top_logits_kernel<true>, set_b) : allow_smem(top_logits_kernel<false>, set_f);
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>(a.splits) * a.R);
  e = a.bf16 ? launch_pdl(top_logits_kernel<true>, grid, dim3(kThreads), sizeof(Smem), stream, a)
             : launch_pdl(top_logits_kernel<false>, grid, dim3(kThreads), sizeof(Smem), stream, a);
  if (e != cudaSuccess || a.splits == 1) return e;
  e = allow_smem(top_logits_merge_kernel, set_m);
  if (e != cudaSuccess) return e;
  return launch_pdl(top_logits_merge_kernel, dim3(a.R), dim3(kThreads), sizeof(Smem), stream, a);
}

}  // namespace osb
