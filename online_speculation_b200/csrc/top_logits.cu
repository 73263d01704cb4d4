// The k largest logits of every row with their columns, and the row's logsumexp, in one pass.
//
// A logit becomes a 64-bit key: its order-preserving 32 bits above the inverted column, so
// that "larger key" means larger logit and, between equal ones, the lower column; every key is
// distinct.  A block streams its columns in ascending order and appends what beats the running
// k-th key to a shared-memory buffer; when the buffer could overflow, a radix select keeps the
// k best and raises the bar.  The bar from the first few thousand columns already turns away
// nearly everything behind them (about k ln(V / chunk) of V random logits pass), so the pass
// costs one compare and one exponential a logit; ascending rows, the worst order, pay one
// select a chunk.  Few rows are cut into column ranges whose winners a second launch merges.
#include "common.cuh"
#include "top_logits.h"

#include <algorithm>

namespace osb {
namespace {

constexpr int kThreads = 512;
constexpr int kPer = 8;                          // logits a thread and chunk
constexpr int kChunk = kThreads * kPer;
constexpr int kCap = 2 * kChunk;                 // candidate buffer
constexpr int kBins = 2048;
constexpr float kLog2e = 1.4426950408889634f;

struct Smem {
  unsigned long long cand[kCap];
  int hist[kBins];
  int warp_tot[kThreads / 32];
  int count;
  int bin, above, in_bin;
  unsigned bar;
  double s[kThreads / 32];
  float m[kThreads / 32];
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

// Keeps the k largest keys of cand[0 .. n) in cand[0 .. k) (any order).  All threads call it.
__device__ void select_top(Smem& sm, int n, int k) {
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (n <= k) return;
  unsigned long long prefix = 0, mask = 0;       // keys with (key & mask) == prefix are undecided
  int need = k;                                  // of those, how many are kept
  const int shifts[6] = {53, 42, 32, 21, 10, 0};
  const int widths[6] = {11, 11, 10, 11, 11, 10};
  for (int p = 0; p < 6; ++p) {
    for (int i = tid; i < kBins; i += kThreads) sm.hist[i] = 0;
    __syncthreads();
    const unsigned long long field = ((1ull << widths[p]) - 1ull) << shifts[p];
    for (int i = tid; i < n; i += kThreads) {
      const unsigned long long c = sm.cand[i];
      if ((c & mask) == prefix) atomicAdd(&sm.hist[static_cast<int>((c & field) >> shifts[p])], 1);
    }
    __syncthreads();
    // four bins a thread, the highest bins first
    int own[4], tot = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      own[j] = sm.hist[kBins - 1 - (tid * 4 + j)];
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
    for (int q = 0; q < warp; ++q) before += sm.warp_tot[q];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (before < need && before + own[j] >= need) {
        sm.bin = kBins - 1 - (tid * 4 + j);
        sm.above = before;
        sm.in_bin = own[j];
      }
      before += own[j];
    }
    __syncthreads();
    prefix |= static_cast<unsigned long long>(sm.bin) << shifts[p];
    mask |= field;
    need -= sm.above;
    const bool whole = sm.in_bin == need;
    __syncthreads();
    if (whole) break;
  }
  // kept: every key at or above the prefix
  unsigned long long mine[kCap / kThreads];
#pragma unroll
  for (int j = 0; j < kCap / kThreads; ++j) {
    const int i = tid + j * kThreads;
    mine[j] = i < n ? sm.cand[i] : 0;
  }
  if (tid == 0) {
    sm.count = 0;
    sm.bar = 0xFFFFFFFFu;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kCap / kThreads; ++j) {
    const int i = tid + j * kThreads;
    if (i < n && (mine[j] & mask) >= prefix) {
      sm.cand[atomicAdd(&sm.count, 1)] = mine[j];
      atomicMin(&sm.bar, static_cast<unsigned>(mine[j] >> 32));
    }
  }
  __syncthreads();
}

__device__ __forceinline__ float load_one(const void* p, int bf16, long long i) {
  return bf16 ? bf2f(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}

template <bool kBf16>
__device__ __forceinline__ void load_eight(const void* row, int i, float (&x)[kPer]) {
  if (kBf16) {
    const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(row) + i);
    const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(u[j] << 16);
      x[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
    }
  } else {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(row) + i);
    const float4 a = p[0], b = p[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
}

// Sorts the k kept keys and writes a row's outputs; cand holds exactly k keys.
__device__ void write_row(const TopLogitsArgs& a, const Smem& sm, int row) {
  const char* base = static_cast<const char*>(a.logits) + static_cast<long long>(row) * a.ld * (a.bf16 ? 2 : 4);
  for (int i = threadIdx.x; i < a.k; i += kThreads) {
    const unsigned long long key = sm.cand[i];
    int rank = 0;
    for (int j = 0; j < a.k; ++j) rank += sm.cand[j] > key;
    const int col = static_cast<int>(0xFFFFFFFFu - static_cast<unsigned>(key));
    const long long o = static_cast<long long>(row) * a.k + rank;
    a.ids[o] = col;
    a.values[o] = load_one(base, a.bf16, col);
  }
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
  if (threadIdx.x == 0) {
    float top = -INFINITY;
    for (int q = 0; q < kThreads / 32; ++q) top = fmaxf(top, sm.m[q]);
    double t = 0.0;
    for (int q = 0; q < kThreads / 32; ++q)
      if (!(sm.m[q] == -INFINITY && sm.s[q] == 0.0)) t += sm.s[q] * exp2f((sm.m[q] - top) * c2);
    m_out = top;
    s_out = t;
  }
}

template <bool kBf16>
__global__ void __launch_bounds__(kThreads) top_logits_kernel(const TopLogitsArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  const int tid = threadIdx.x, lane = tid % 32;
  const int row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  pdl_trigger();
  pdl_wait();
  const int per = (a.V + a.splits - 1) / a.splits;
  const int c0 = min(a.V, split * per), c1 = min(a.V, c0 + per);
  constexpr int kSize = kBf16 ? 2 : 4;
  const char* base = static_cast<const char*>(a.logits) + static_cast<long long>(row) * a.ld * kSize;
  const float it = a.inv_temp != nullptr ? a.inv_temp[row] : 1.0f;
  const float c2 = it * kLog2e;
  if (tid == 0) {
    sm.count = 0;
    sm.bar = 0;
  }
  __syncthreads();
  unsigned bar = 0;                     // keys above it pass (0: all)
  float m = -INFINITY, s = 0.0f;

  // columns before the first 16-byte boundary, then chunks of vectors, then the ragged end
  const int head = min(c1 - c0, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(base + static_cast<long long>(c0) * kSize) & 15)) & 15) / kSize);
  const int v0 = c0 + head;
  const int vecs = (c1 - v0) / kPer;    // whole groups of eight
  const int tail0 = v0 + vecs * kPer;
  auto take = [&](const float (&x)[kPer], int col, int n) {
    float top = m;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < n) top = fmaxf(top, x[j]);
    const float ref = top == -INFINITY ? 0.0f : top;
    s *= ex2((m - ref) * c2);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < n) s += ex2((x[j] - ref) * c2);
    m = top;
    unsigned pass = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < n && (bar == 0 || order_key(x[j]) > bar)) pass |= 1u << j;
    if (__any_sync(0xffffffffu, pass != 0)) {
      const int mine = __popc(pass);
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      int at = 0;
      if (lane == 31) at = atomicAdd(&sm.count, incl);
      at = __shfl_sync(0xffffffffu, at, 31) + incl - mine;
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (pass & (1u << j)) sm.cand[at++] = make_key(x[j], col + j);
    }
  };
  {
    float x[kPer] = {0.0f};
    const bool on = tid < head;
    if (on) x[0] = load_one(base, kBf16, c0 + tid);
    take(x, c0 + tid, on ? 1 : 0);
  }
  const int chunks = (vecs + kThreads - 1) / kThreads;
  for (int c = 0; c < chunks; ++c) {
    const int g = c * kThreads + tid;
    const bool on = g < vecs;
    float x[kPer] = {0.0f};
    if (on) load_eight<kBf16>(base, v0 + g * kPer, x);
    // the buffer takes a whole chunk (and the ragged end's few) on top of what it holds
    __syncthreads();
    const int held = sm.count;
    __syncthreads();
    if (held > kCap - kChunk - 2 * kPer || (c == 1 && held > a.k)) {
      select_top(sm, held, a.k);
      bar = sm.bar;
    }
    take(x, v0 + g * kPer, on ? kPer : 0);
  }
  {
    float x[kPer] = {0.0f};
    const bool on = tail0 + tid < c1;
    if (on) x[0] = load_one(base, kBf16, tail0 + tid);
    take(x, tail0 + tid, on ? 1 : 0);
  }
  __syncthreads();
  const int n = sm.count;
  __syncthreads();
  select_top(sm, n, a.k);
  const int kept = min(n, a.k);
  float m_row = 0.0f;
  double s_row = 0.0;
  fold(sm, m, s, c2, m_row, s_row);
  if (a.splits == 1) {
    write_row(a, sm, row);
    if (tid == 0)
      a.lse[row] = static_cast<float>(static_cast<double>(m_row) * it + log(s_row));
    return;
  }
  unsigned long long* dst = a.keys + (static_cast<long long>(row) * a.splits + split) * a.k;
  for (int i = tid; i < a.k; i += kThreads) dst[i] = i < kept ? sm.cand[i] : 0ull;   // no key is 0
  if (tid == 0) a.part[static_cast<long long>(row) * a.splits + split] = make_float2(m_row, static_cast<float>(s_row));
}

__global__ void __launch_bounds__(kThreads) top_logits_merge_kernel(const TopLogitsArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  const int tid = threadIdx.x, row = blockIdx.x;
  pdl_trigger();
  pdl_wait();
  const int n = a.splits * a.k;
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
  select_top(sm, n, a.k);
  float m_row = 0.0f;
  double s_row = 0.0;
  fold(sm, m, s, c2, m_row, s_row);
  write_row(a, sm, row);
  if (tid == 0)
    a.lse[row] = static_cast<float>(static_cast<double>(m_row) * it + log(s_row));
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
  // blocks for every SM twice over; a range is two chunks at least, and the merge buffer holds all winners
  const int want = (2 * 148 + R - 1) / std::max(R, 1);
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
