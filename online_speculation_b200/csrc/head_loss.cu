// Losses on a vocabulary head that never hold its logits in 32 bits but for few rows: softmax cross entropy and the
// divergence from a teacher's listed logits, with the gradients of the hidden rows and of
// the head.
//
//   l = h W^T,  q = softmax(it * l)                       h [R, H], W [V, H], bf16
//   dl[r, v] = A_r q[r, v] - C_r on the unlisted columns (q for a divergence: softmax over those alone), a stored
//   value on the listed ones
//   dh = dl W,  dW = dl^T h
//
// A row's listed columns are its target, or the teacher's columns; everything dense about
// either loss is one row normaliser and two row coefficients.
//
// * Rows that do not count (ignored targets, empty lists) are taken out first: the products
//   run over compact rows, so padding costs nothing and whatever its hidden rows hold never
//   meets a product (0 * NaN would be NaN in dW).  The count stays on the device.
// * Forward: the logits tile stays in tensor memory.  Lanes are rows, so a thread reduces its
//   own row over the tile's columns (running maximum, sum of exponentials) without shuffles,
//   and lifts the listed logits out on the way.  Listed columns are left out of the sum: the
//   mass of the rest comes out of a sum of its own, not of 1 - (something near 1).
// * Backward goes over pieces of the vocabulary.  A piece's logits, from what the forward pass kept of them (fp16
//   exponentials, for few rows fp32 logits: head_loss_kept) or computed again, are turned into
//   dl in bf16 (the type of the matrix instruction; 2^-9 rms against the same rounding of the
//   outputs), and feed two products: dW of the piece is complete at once, dh adds up in fp32.
//   Both read dl and their other operand in the layout they already have (MN-major
//   shared-memory descriptors): nothing is transposed.  What rounding took from the listed entries is added to dh
//   on its way out, where the list is short against the vocabulary (hidden_grad_kernel).
// * Up to 128 rows take the products the other way around, vocabulary columns in the accumulator's
//   lanes and rows in its columns.  A pass over few rows is the reading of the head, and a tile of
//   256 lanes that holds 64 rows would spend four times the matrix instructions (and the clock that
//   their power costs: 93 % tensor-pipe active at 1.5 GHz for 64 rows) on lanes that nobody looks at.
// * They keep dl as the sum of two bf16 numbers.  A row's gradient is mostly its target's
//   entry: with few rows the rounding of single entries shows in the results (0.0027 relative where the
//   rounding of the outputs alone is 0.0017), and the second half is nearly free, as the head is read
//   all the same.  With many rows the errors average out and the products would double.
#include "common.cuh"
#include "head_loss.h"

#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

namespace osb {
namespace {

constexpr int kBM = 256;                  // tile rows: 128 TMEM lanes in each CTA of the pair
constexpr int kBN = 256;                  // tile columns: both CTAs hold all of them for their rows
constexpr int kHalf = 128;                // rows of A, and of B, that one CTA stages
constexpr int kBK = 64;                   // reduction elements a stage: one 128-byte swizzle row
constexpr int kMaxStages = 12;
// Statistics of many rows: the tensor core truncates at every addition, so a reduction of more than kOneSum blocks is cut
// into sums of at most kSumBlocks, which the epilogue adds in fp32.  The first two are the longest: while they are
// multiplied, the exponentials of the tile before are formed.  Divergence losses of 300 rows of 3584, off by 3.8e-6 in
// one sum: 5.3e-7 (6.2e-7 with fp32 products); the pass over 4096 rows of 3584 and 152064 columns 3.65 ms for 3.50 (sums
// of 14 blocks 3.57, of 8 3.83).  300 rows of 896, off by 9.2e-7 in one sum: 4.2e-7 (3.2e-7); the pass over 2048 rows of
// 896 and 65536 columns 0.261 ms for 0.240.  Rows in columns: chains of at most kChainBlocks, 64 rows of 3584 6.9e-7
// (7.3e-7).
constexpr int kSumBlocks = 10, kOneSum = 12, kChainBlocks = 14;
constexpr int kRowBytes = kBK * 2;        // one staged row of either operand
constexpr int kBox = 64 * 64 * 2;         // one MN-major box: 64 reduction rows of 64 elements
constexpr int kOutBytes = 32 * 128;       // one warp's staged output box: 32 rows of 128 bytes
// Epilogue warps: four cover the accumulator's lanes.  Mostly there are two sets, each for half of the columns:
// below about 600 hidden columns, or with few rows to reduce over, a tile's products take less time than
// one set needs for it.  With rows in columns the logits' passes have one set, which holds the rows' state.
constexpr int epilogue_warps(int mode, bool few) { return few && mode != 2 ? 4 : 8; }
constexpr int threads_of(int mode, bool few) { return 64 + 32 * epilogue_warps(mode, few); }   // and TMA, MMA
constexpr int kOutTotal = 8 * kOutBytes;  // two boxes a warp, or one with twice the warps
constexpr int kFewRows = 128;             // rows that go into the accumulator's columns: see few_rows
constexpr int kCountRows = 256;           // rows that one launch numbers and gathers
// Per-row state of the passes with rows in columns, behind the output boxes: running maximum and sum and
// plain sum (one set a warp), list cursors (one set a warp, two of the CTA), coefficients, row numbers, targets' gradients.
constexpr int kStateMax = 0, kStateSum = kStateMax + 4 * kFewRows * 4, kStatePlain = kStateSum + 4 * kFewRows * 4,
              kStateCursor = kStatePlain + 4 * kFewRows * 4, kStateCoef = kStateCursor + 6 * kFewRows * 8,
              kStateRow = kStateCoef + kFewRows * 16, kStateListed = kStateRow + kFewRows * 4,
              kStateBytes = kStateListed + kFewRows * 4;
constexpr int kBarBytes = 256;            // barriers and the TMEM address
constexpr int kSmemMost = 232448 - 1024;               // behind the alignment
constexpr float kLog2e = 1.4426950408889634f;
// Kept exponentials are fp16 of 2^15 exp(it (l - the largest of 128 columns)): off by 2^-11 relative down to e^-20 of the
// largest, by 2^-40 of it below.
constexpr float kKeptOne = 32768.0f;

enum Mode { kStats = 0, kGrad = 1, kProd = 2 };

struct Maps {
  CUtensorMap a0, b0;      // first kind: stats / grad operands, or the hidden gradient's
  CUtensorMap a1, b1;      // second kind: the head gradient's
  CUtensorMap out0, out1;
};

struct GemmArgs {
  const int* count;
  int H, V;
  int v0, cols;            // this piece: first vocabulary row, columns that exist
  int bn;                  // rows in columns: how many columns, a multiple of 16
  int chains, chain;       // rows in columns: sums of that many blocks of the reduction each, side by side in the accumulator
  int sums;                // statistics: sums that the reduction is cut into one after the other, added up in registers, and
  int sum_first, sum_rest; // the blocks of the first two and of the others
  int tiles_n;             // column tiles of the accumulator grid
  int lo;                  // rows in columns: where a row of the logits' gradient holds what rounding to bf16 took
                           // from its first half
  int slot;                // rows in columns: vocabulary columns in the lanes of one CTA (statistics: a multiple of
                           // 8, gradient: of 32)
  int stages;              // of the ring
  int K;
  const int* row_of;
  const int* list_id;
  float* list_logit;       // stats: written
  const float* list_grad;  // grad: read
  const float4* row_coef;  // grad
  HeadLossState s;         // rows in columns, grad: coefficients and listed values are formed on the spot
  const float* g;
  const float* inv_temp;   // stats
  int kept;                // stats: the logits (rows in columns) or their exponentials are stored for the backward pass
  float2* part;
  float* part_sum;
  int part_tiles;
  int rpad, piece;
  int do_dh, do_dw, splits, first_piece;
  int* status;
};

// Rows in columns, hidden gradient: boxes of 64 rows that one CTA stages, all rows of one of the two halves.
__host__ __device__ inline int row_boxes(const GemmArgs& a) { return (a.bn + 63) / 64; }

// Rows in columns: columns of the accumulator, and the most chains of a sum that stand in it side by side.
__host__ __device__ constexpr int row_columns(int R) { return (R + 15) / 16 * 16; }
__host__ __device__ constexpr int most_chains(int bn) { return kBN / bn < 4 ? kBN / bn : 4; }

// The epilogue loads 32 columns at a time, up to the last row's, of every chain.
constexpr bool loads_stay_inside() {
  for (int R = 1; R <= kFewRows; ++R)
    if ((most_chains(row_columns(R)) - 1) * row_columns(R) + (R + 31) / 32 * 32 > kBN) return false;
  return true;
}
static_assert(loads_stay_inside(), "the last chain's loads end inside the accumulator");

struct StageBytes {
  int a, b;
};

// Shared memory of one stage: this CTA's part of either operand.
__host__ __device__ inline StageBytes stage_bytes_of(int mode, bool few, const GemmArgs& a) {
  if (few && mode != kProd) return {a.slot * kRowBytes, a.bn / 2 * kRowBytes};
  if (few && !a.do_dw) return {kHalf * kRowBytes, row_boxes(a) * kBox};
  return {kHalf * kRowBytes, kHalf * kRowBytes};
}

__host__ __device__ inline int out_bytes_of(int mode, bool few, bool kept) {
  if (few && mode == kProd) return 2 * kOutTotal;
  if (!few) return mode == kStats ? (kept ? 2 * kOutTotal : 0) : kOutTotal;
  return (mode == kStats && !kept ? 0 : kOutTotal) + kOutTotal / 2;   // a block for listed logits, behind the boxes
}

// One work item: an accumulator tile and its range of reduction blocks.
struct Item {
  int kind;                // 0: first operand pair, 1: second
  int m0, n0;
  int kb0, kb1;
  int split;
};

// The i-th item of CTA pair `pair`; false behind its last.  FEW: rows in the accumulator's columns.
template <int MODE, bool FEW>
__device__ __forceinline__ bool item_at(const GemmArgs& a, int rows, int pair, int pairs, int i, Item& it) {
  const int tm = (rows + kBM - 1) / kBM;    // row tiles
  it.split = 0;
  it.kind = 0;
  it.kb0 = 0;
  it.n0 = 0;
  if (MODE != kProd) {
    const int w = pair + i * pairs;
    it.kb1 = (a.H + kBK - 1) / kBK;
    if (FEW) {
      it.m0 = w * 2 * a.slot;
      return it.m0 < a.cols && rows > 0;
    }
    // rows fastest: the pairs that run together read few head tiles, and the hidden rows stay in L2
    if (w >= tm * a.tiles_n) return false;
    it.m0 = (w % tm) * kBM;
    it.n0 = (w / tm) * kBN;
    return true;
  }
  // The hidden gradient's items reduce over the piece, the head gradient's over the rows, and cost
  // accordingly: the former go first, dealt around; the pairs that got one less take as many of the
  // latter in its place as weigh the same, and the rest is dealt around.
  const int kb = (a.cols + kBK - 1) / kBK, per = (kb + a.splits - 1) / a.splits, kbw = (rows + kBK - 1) / kBK * (FEW ? 2 : 1);
  const int per_split = FEW ? (rows > 0 ? a.tiles_n : 0) : tm * a.tiles_n;   // a.tiles_n tiles across the hidden width
  const int nh = a.do_dh ? per_split * a.splits : 0;
  const int nw = a.do_dw ? ((a.cols + kBM - 1) / kBM) * a.tiles_n : 0;
  const int extra = nh % pairs, mine = nh / pairs + (pair < extra ? 1 : 0);
  if (i < mine) {
    const int w = pair + i * pairs, t = w % per_split;
    it.split = w / per_split;
    it.m0 = (FEW ? t : t / a.tiles_n) * kBM;
    if (!FEW) it.n0 = (t % a.tiles_n) * kBN;
    it.kb0 = min(kb, it.split * per);
    it.kb1 = min(kb, it.kb0 + per);
    return true;
  }
  int j = i - mine, t;
  const int late = extra > 0 ? pairs - extra : 0;   // pairs with one less
  // in blocks: a head gradient's tile takes as long as eight at least, for its end and its output; a hidden
  // gradient's block over few rows waits for the head, half again as long as its products
  const int weigh = max(kbw, 8), weigh_hidden = FEW ? per + per / 2 : per;
  const int each = late > 0 && kbw > 0 ? min((weigh_hidden + weigh / 2) / weigh, nw / late) : 0;
  if (late > 0 && pair >= extra && j < each) {
    t = pair - extra + j * late;
  } else {
    if (late > 0 && pair >= extra) j -= each;
    t = each * late + pair + j * pairs;
  }
  if (t >= nw) return false;
  it.kind = 1;
  it.m0 = (t / a.tiles_n) * kBM;
  it.n0 = (t % a.tiles_n) * kBN;
  it.kb1 = kbw;
  return true;
}

// ------------------------------------------------------------- CTA pairs ----
// Loads into this CTA's shared memory that complete on a barrier of the pair's first CTA.
__device__ __forceinline__ void pair_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void pair_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrives on the barrier at this offset in both CTAs when the MMAs issued so far are done.
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

__device__ __forceinline__ void remote_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Adds 32 lanes x 16 accumulator columns (half a load at a time: registers are short where it is used).
__device__ __forceinline__ void add_tmem16(uint32_t from, float* x) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(from)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] += __uint_as_float(r[i]);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations an instruction.
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

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}

__device__ __forceinline__ void tma_add_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}

__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// What rounding eight values to bf16 took from them, rounded itself.
__device__ __forceinline__ uint4 rounded_off(const float* x, uint4 hi) {
  const unsigned h[4] = {hi.x, hi.y, hi.z, hi.w};
  unsigned low[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    low[e] = pack2(x[2 * e] - __uint_as_float(h[e] << 16), x[2 * e + 1] - __uint_as_float(h[e] & 0xFFFF0000u));
  return make_uint4(low[0], low[1], low[2], low[3]);
}

// Position of 16-byte chunk c of row r in a 128-byte-swizzled box of 32 rows.
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + (((c ^ r) & 7) << 4); }

// A row's cursor into its ascending list of columns.  The column behind the next one, and the next one's
// value, are on their way before they are needed.
struct ListCursor {
  const int* ids;
  const float* values;       // or null
  int k, K, next, after;
  float value;
  __device__ __forceinline__ int id(int i) const { return i < K ? ids[i] : INT_MAX; }
  __device__ __forceinline__ void load() {
    next = id(k);
    after = id(k + 1);
    value = values != nullptr && k < K ? values[k] : 0.0f;
  }
  // The first column at or behind `col`, not before the `from`-th.
  __device__ __forceinline__ void seek(int from, int col) {
    int lo = from, hi = K;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ids[mid] < col) lo = mid + 1; else hi = mid;
    }
    k = lo;
    load();
  }
  __device__ __forceinline__ void advance() {
    ++k;
    next = after;
    after = id(k + 1);
    value = values != nullptr && k < K ? values[k] : 0.0f;
  }
};

// Where the lists of all rows reach `col`, and the first column there: a row for each of the 128 epilogue threads.
// (Every warp on its own, its lanes one row after the other, took longer than a tile of 64 hidden columns with 256 rows.)
__device__ __forceinline__ void seek_rows(const int* list_id, int K, const int* row_no, int rows, int col, int2* cursors) {
  static_assert(kFewRows == 128, "a thread a row");
  const int t = threadIdx.x - 64;
  if (t >= rows) return;
  const int* ids = list_id + static_cast<long long>(row_no[t]) * K;
  int at = 0, top = 1;
  while (2 * top <= K) top *= 2;
  for (int step = top; step > 0; step /= 2) at += at + step <= K && ids[at + step - 1] < col ? step : 0;
  cursors[t] = make_int2(at, at < K ? ids[at] : INT_MAX);
}

// A row's coefficients of the logits' gradient: {it log2 e, lse log2 e, A, C} of A exp(it l - lse) - C.  A divergence's are
// about the normaliser of the unlisted columns, that of a cross entropy about all.
__device__ __forceinline__ float4 row_coefficients(const HeadLossState& s, const float* g, int r) {
  const float4 st = s.row_stat[r];
  const float it = s.inv_temp != nullptr ? s.inv_temp[r] : 1.0f;
  const float up = g[r] * it;
  const float flat = s.divergence ? 0.0f : s.smoothing / static_cast<float>(s.V);
  return make_float4(it * kLog2e, (s.divergence ? st.y : st.x) * kLog2e, up * st.z, up * flat);
}

// The gradient of the listed logit `at` of row r.  Written so that every kernel gets the same bits: the rest that
// rounding to bf16 takes from it is added on elsewhere.
__device__ __forceinline__ float listed_gradient(const HeadLossState& s, const float* g, int r, long long at) {
  const float4 st = s.row_stat[r];
  const float it = s.inv_temp != nullptr ? s.inv_temp[r] : 1.0f;
  float v;
  if (s.divergence) {
    v = __fmaf_rn(st.w, expf(__fmaf_rn(s.list_logit[at], it, -st.x)), -s.list_mass[at]);
  } else {
    // a p - 1 with p - 1 = -(mass of the rest): no cancellation in sure rows
    const float flat = s.smoothing / static_cast<float>(s.V);
    v = __fsub_rn(__fadd_rn(__fmaf_rn(st.z - 1.0f, 1.0f - st.y, -st.y), s.smoothing), flat);
  }
  return __fmul_rn(__fmul_rn(g[r], it), v);
}

// Reduces 32 columns over the warp's lanes; lane j returns column j's.
template <typename Op>
__device__ __forceinline__ float reduce_columns(float (&x)[32], Op op) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int n = 16; n > 0; n >>= 1) {
    const bool up = (lane & n) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float send = up ? x[i] : x[i + n], keep = up ? x[i + n] : x[i];
      x[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, n));
    }
  }
  return x[0];
}

// A warp's 32 x 32 block in shared memory (4 KB, lane = row), for the rare access to one element of
// another lane's registers.
__device__ __forceinline__ void spill_block(uint8_t* buf, const float (&x)[32]) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int q = 0; q < 8; ++q)
    *reinterpret_cast<float4*>(buf + swizzled(lane, q)) = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
  __syncwarp();
}

__device__ __forceinline__ void reload_block(const uint8_t* buf, float (&x)[32]) {
  const int lane = threadIdx.x % 32;
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float4 v = *reinterpret_cast<const float4*>(buf + swizzled(lane, q));
    x[4 * q] = v.x;
    x[4 * q + 1] = v.y;
    x[4 * q + 2] = v.z;
    x[4 * q + 3] = v.w;
  }
  __syncwarp();
}

__device__ __forceinline__ float* block_at(uint8_t* buf, int row, int col) {
  return reinterpret_cast<float*>(buf + swizzled(row, col >> 2) + (col & 3) * 4);
}

// SUMS: the reduction is cut into several sums (statistics).
template <int MODE, bool FEW, bool SUMS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(threads_of(MODE, FEW), 1)
    head_gemm_kernel(const __grid_constant__ Maps maps, const GemmArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // A stage is this CTA's part of the first operand, then of the second.  The matrix instruction takes 128
  // lanes of the first whatever `slot` is: what it reads behind them (of the second) only reaches
  // accumulator lanes that nobody looks at.
  const StageBytes sb = stage_bytes_of(MODE, FEW, a);
  const int stage_bytes = sb.a + sb.b;
  const int stages = a.stages;
  uint8_t* sOut = smem + stages * stage_bytes;
  uint8_t* state = sOut + out_bytes_of(MODE, FEW, a.kept);
  uint64_t* full = reinterpret_cast<uint64_t*>(state + (FEW && MODE != kProd ? kStateBytes : 0));
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = static_cast<int>(cluster_ctarank());
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2 * epilogue_warps(MODE, FEW));   // of both CTAs
    }
    mbar_init(drain, 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(2 * kBN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();
  const int rows = *a.count;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      Item it;
      for (int i = 0; ok && item_at<MODE, FEW>(a, rows, pair, pairs, i, it); ++i) {
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, a.status, kErrTmaWait)) {
            ok = false;
            break;
          }
          uint8_t* pa = smem + stage * stage_bytes;
          uint8_t* pb = pa + sb.a;
          // the first CTA's barrier counts the bytes of both
          const uint32_t bar = map_shared_rank(smem_u32(&full[stage]), 0);
          const int k0 = kb * kBK;
          const bool hidden = MODE == kProd && it.kind == 0;
          const int rows_box = row_boxes(a);
          if (rank == 0) {
            const int bytes = MODE != kProd ? stage_bytes
                              : FEW && hidden ? kHalf * kRowBytes + rows_box * kBox
                                              : 2 * kHalf * kRowBytes;
            mbar_arrive_expect_tx(&full[stage], 2 * bytes);
          }
          if (FEW && MODE != kProd) {
            pair_load_2d(pa, &maps.a0, k0, a.v0 + it.m0 + rank * a.slot, bar);
            pair_load_2d(pb, &maps.b0, k0, rank * (a.bn / 2), bar);
          } else if (FEW && hidden) {
#pragma unroll
            for (int j = 0; j < kHalf / 64; ++j)
              pair_load_2d(pa + j * kBox, &maps.a0, it.m0 + rank * kHalf + j * 64, a.v0 + k0, bar);
            for (int j = 0; j < rows_box; ++j)
              pair_load_2d(pb + j * kBox, &maps.b0, rank * a.lo + j * 64, k0, bar);
          } else {
            // head gradient in two halves: the second half's blocks meet the same rows again
            const int over = k0 - (FEW ? (rows + kBK - 1) / kBK * kBK : INT_MAX);
            const int ka = over >= 0 ? a.lo + over : k0, kh = over >= 0 ? over : k0;
            const int ma = it.m0 + rank * kHalf, nb = it.n0 + rank * kHalf;
            if (MODE != kProd) {
              pair_load_2d(pa, &maps.a0, k0, ma, bar);
              pair_load_2d(pb, &maps.b0, k0, a.v0 + nb, bar);
            } else if (hidden) {
              pair_load_2d(pa, &maps.a0, k0, ma, bar);
#pragma unroll
              for (int j = 0; j < kHalf / 64; ++j) pair_load_2d(pb + j * kBox, &maps.b0, nb + j * 64, a.v0 + k0, bar);
            } else {
              if (FEW) pair_load_2d(pa, &maps.a1, ka, ma, bar);
#pragma unroll
              for (int j = 0; j < kHalf / 64; ++j) {
                if (!FEW) pair_load_2d(pa + j * kBox, &maps.a1, ma + j * 64, k0, bar);
                pair_load_2d(pb + j * kBox, &maps.b1, nb + j * 64, kh, bar);
              }
            }
          }
          ++issued;
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok && rank == 0) {
        // copies in flight land before the pair may exit
        for (int s = 0; s < stages && s < issued; ++s) {
          const int fills = (issued - s + stages - 1) / stages;
          mbar_wait(&full[s], static_cast<uint32_t>((fills - 1) & 1), nullptr, 0);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer, for both CTAs
    if (lane == 0 && rank == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      const uint32_t base = smem_u32(smem);
      Item it;
      for (int i = 0; ok && item_at<MODE, FEW>(a, rows, pair, pairs, i, it); ++i) {
        for (int n = 0, begin = it.kb0, end; ok && begin < it.kb1; ++n, begin = end) {
          end = SUMS ? min(begin + (n < 2 ? a.sum_first : a.sum_rest), it.kb1) : it.kb1;
          if (!mbar_wait(&tempty[acc], acc_phase ^ 1, a.status, kErrAccumWait)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + acc * kBN;
          const bool mn_a = MODE == kProd && (it.kind == (FEW ? 0 : 1)), mn_b = MODE == kProd;
          const int columns = FEW && it.kind == 0 ? (MODE == kProd ? 2 * a.bn : a.bn) : kBN;
          const uint32_t idesc = idesc_bf16_f32(kBM, columns) | (mn_a ? 1u << 15 : 0u) | (mn_b ? 1u << 16 : 0u);
          constexpr bool kChains = FEW && MODE != kProd;
          uint32_t dk = d;
          int from = begin, turn = begin + a.chain;
          for (int kb = begin; kb < end; ++kb) {
            if (!mbar_wait(&full[stage], phase, a.status, kErrMmaWait)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t pa = base + stage * stage_bytes, pb = pa + sb.a;
            if (kChains && kb == turn) {
              dk += a.bn;
              from = kb;
              turn += a.chain;
            }
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) {
              const uint64_t ad = mn_a ? sdesc_mn_sw128(pa + k * 2048, kBox, 1024) : sdesc_k_sw128(pa + k * 32);
              const uint64_t bd = mn_b ? sdesc_mn_sw128(pb + k * 2048, kBox, 1024) : sdesc_k_sw128(pb + k * 32);
              pair_mma(dk, ad, bd, idesc, (kb > from || k > 0) ? 1u : 0u);
            }
            pair_commit(&empty[stage]);
            if (++stage == stages) {
              stage = 0;
              phase ^= 1;
            }
          }
          if (!ok) break;
          pair_commit(&tfull[acc]);
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1;
        }
      }
      // every issued MMA completes before TMEM is released
      pair_commit(drain);
      mbar_wait(drain, 0, a.status, kErrMmaWait);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp % 4;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    constexpr int kSets = epilogue_warps(MODE, FEW) / 4;
    constexpr int kBoxes = FEW || MODE == kStats ? 2 : 1;                     // output boxes of a warp
    const int set = (warp - 2) / 4;                         // its share of the columns
    uint8_t* out = sOut + (kSets == 1 ? quarter : warp - 2) * kBoxes * kOutBytes;
    auto next_box = [&](int staged) {
      // the box's last store has read it
      if (lane == 0) bulk_wait_read<kBoxes - 1>();
      __syncwarp();
      return out + (staged & (kBoxes - 1)) * kOutBytes;
    };
    int acc = 0, staged = 0;
    uint32_t acc_phase = 0;
    bool gave_up = false;
    if (FEW && MODE != kProd) {
      for (int t = threadIdx.x - 64; t < kFewRows; t += 128) {
        const int o = t < rows ? a.row_of[t] : -1;
        reinterpret_cast<int*>(state + kStateRow)[t] = o;
        float4 c = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (MODE == kGrad && o >= 0) {
          c = row_coefficients(a.s, a.g, o);
          if (!a.s.divergence) reinterpret_cast<float*>(state + kStateListed)[t] = listed_gradient(a.s, a.g, o, o);
        }
        if (MODE == kStats) c.x = (o >= 0 && a.inv_temp != nullptr ? a.inv_temp[o] : 1.0f) * kLog2e;
        reinterpret_cast<float4*>(state + kStateCoef)[t] = c;
      }
      if (MODE == kStats) {
        for (int t = lane; t < kFewRows; t += 32) {
          reinterpret_cast<float*>(state + kStateMax)[quarter * kFewRows + t] = -INFINITY;
          reinterpret_cast<float*>(state + kStateSum)[quarter * kFewRows + t] = 0.0f;
          reinterpret_cast<float*>(state + kStatePlain)[quarter * kFewRows + t] = 0.0f;
        }
      }
      named_barrier(1, 128);
    }
    const int* row_no = reinterpret_cast<const int*>(state + kStateRow);
    const float4* coef_of = reinterpret_cast<const float4*>(state + kStateCoef);
    const float* listed_of = reinterpret_cast<const float*>(state + kStateListed);
    int2* cursors = reinterpret_cast<int2*>(state + kStateCursor) + quarter * kFewRows;
    // Row inputs of the next tile are fetched while this one is worked on: its row, its first listed column (all
    // that a list of one has), its coefficients.
    int next_row = -1, next_id = INT_MAX;
    float4 next_coef = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto fetch_row = [&](const Item& n) {
      const int m = n.m0 + rank * kHalf + quarter * 32 + lane;
      next_row = m < rows ? a.row_of[m] : -1;
      // zero behind the last row, up to its tile's end: another row's normaliser could overflow there, and the head
      // gradient's product reads those rows
      if (MODE == kGrad) next_coef = a.row_coef[m];
    };
    float next_scale = kLog2e;
    auto fetch_id = [&]() {
      next_id = next_row >= 0 ? a.list_id[static_cast<long long>(next_row) * a.K] : INT_MAX;
      if (MODE == kStats && next_row >= 0 && a.inv_temp != nullptr) next_scale = a.inv_temp[next_row] * kLog2e;
    };
    Item it, ahead;
    bool more = item_at<MODE, FEW>(a, rows, pair, pairs, 0, ahead);
    if (!FEW && MODE != kProd && more) {
      fetch_row(ahead);
      fetch_id();
    }
    for (int i = 0; more; ++i) {
      it = ahead;
      more = item_at<MODE, FEW>(a, rows, pair, pairs, i + 1, ahead);
      const int held = FEW && MODE != kProd ? a.slot : kHalf;
      const int m0 = it.m0 + rank * held + quarter * 32;    // first tile row of this warp
      const int m = m0 + lane;
      const bool empty_sum = it.kb0 >= it.kb1;
      if (empty_sum && !(MODE == kProd && it.kind == 1)) continue;
      // row inputs, fetched while the tile is still being multiplied
      ListCursor cur;
      long long list0 = 0;
      float c2 = kLog2e;
      float4 coef = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      bool live = false;
      if (FEW && MODE != kProd) {
        // every row's place in its list, for this warp's vocabulary columns
        const int first = a.v0 + m0;
        if (a.K == 1) {
          for (int t = lane; t < rows; t += 32) {
            const int id = a.list_id[row_no[t]];
            cursors[t] = id < first ? make_int2(1, INT_MAX) : make_int2(0, id);
          }
        } else {
          int2* found = cursors + (4 - quarter + (i & 1)) * kFewRows;   // of this CTA's first column; in turn
          seek_rows(a.list_id, a.K, row_no, rows, a.v0 + it.m0 + rank * held, found);
          named_barrier(1, 128);
          if (gave_up) continue;
          for (int t = lane; t < rows; t += 32) {
            int2 f = found[t];
            while (f.y < first) {
              ++f.x;
              f.y = f.x < a.K ? a.list_id[static_cast<long long>(row_no[t]) * a.K + f.x] : INT_MAX;
            }
            cursors[t] = f;
          }
        }
        __syncwarp();
      } else if (MODE != kProd) {
        live = m < rows;
        coef = next_coef;
        const int o = next_row, col = a.v0 + it.n0 + set * (kBN / 2);
        list0 = static_cast<long long>(o) * a.K;
        cur.ids = a.list_id + list0;
        cur.values = MODE == kGrad ? a.list_grad + list0 : nullptr;
        cur.K = live ? a.K : 0;
        cur.k = 0;
        cur.next = next_id;
        if (next_id >= col) {
          cur.after = cur.id(1);
          cur.value = MODE == kGrad && live ? cur.values[0] : 0.0f;
        } else if (a.K == 1) {
          cur.next = INT_MAX;
        } else {
          cur.seek(1, col);
        }
        c2 = next_scale;
        if (more) fetch_row(ahead);
      }
      auto wait_accumulator = [&]() {
        gave_up = !__all_sync(0xffffffffu, mbar_wait(&tfull[acc], acc_phase, a.status, kErrEpilogueWait));
        if (!gave_up) tc_fence_after();
        return !gave_up;
      };
      if (!empty_sum && !wait_accumulator()) {
        if (FEW && MODE != kProd && a.K > 1) continue;   // the other warps still wait for this one above
        break;
      }
      const uint32_t t_acc = tmem + lane_base + acc * kBN;
      bool released = false;
      auto release = [&]() {                                // the accumulator has been read
        tc_fence_before();
        __syncwarp();
        if (lane == 0) remote_arrive(map_shared_rank(smem_u32(&tempty[acc]), 0));
        released = true;
      };
      auto next_accumulator = [&]() {
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
        released = false;
      };

      if (FEW && MODE != kProd) {
        // lanes are vocabulary columns, this thread's is `col`; chunks of 32 rows
        const int first = a.v0 + m0;
        const int stop = a.v0 + min(a.cols, it.m0 + (rank + 1) * held);   // behind this CTA's last column
        const bool on = first + lane < stop;
        float* maxes = reinterpret_cast<float*>(state + kStateMax) + quarter * kFewRows;
        float* sums = reinterpret_cast<float*>(state + kStateSum) + quarter * kFewRows;
        float* plains = reinterpret_cast<float*>(state + kStatePlain) + quarter * kFewRows;
        // Runs `use(block)` for rows whose list has a column here, on the block in shared memory.
        auto listed = [&](float (&x)[32], int t, uint8_t* buf, auto use) {
          int2 c = t < rows ? cursors[t] : make_int2(0, INT_MAX);
          const int end = min(first + 32, stop);
          if (!__any_sync(0xffffffffu, c.y < end)) return;
          spill_block(buf, x);
          const long long base = t < rows ? static_cast<long long>(row_no[t]) * a.K : 0;
          int after = c.y < end && c.x + 1 < a.K ? a.list_id[base + c.x + 1] : INT_MAX;
          while (c.y < end) {
            const int here = c.y - first, k = c.x;
            ++c.x;
            c.y = after;
            after = c.x + 1 < a.K ? a.list_id[base + c.x + 1] : INT_MAX;
            use(block_at(buf, here, lane), base + k);
          }
          reload_block(buf, x);
        };
        const int chunks = MODE == kStats ? (rows + 31) / 32 : 2 * ((rows + 63) / 64);
        auto work_on = [&](int c, float (&x)[32]) {
          const int t0 = c * 32, t = t0 + lane;
          if (MODE == kStats) {
            if (a.kept) {
              // lanes outside the vocabulary are cut off by the map: a warp's columns are its own (see lane_slot)
              uint8_t* box = next_box(staged);
              spill_block(box, x);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&maps.out0, box, t0, m0);
                bulk_commit();
              }
              ++staged;
            }
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (!on) x[j] = -INFINITY;
            if (a.part_sum != nullptr) {
              float y[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) y[j] = on ? x[j] : 0.0f;
              const float p = reduce_columns(y, [](float u, float v) { return u + v; });
              plains[t] += p;
            }
            listed(x, t, sOut + (a.kept ? kOutTotal : 0) + quarter * kOutBytes, [&](float* at, long long k) {
              a.list_logit[k] = *at;
              *at = -INFINITY;
            });
            float y[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) y[j] = x[j];
            const float top = reduce_columns(y, [](float u, float v) { return fmaxf(u, v); });
            const float before = maxes[t], now = fmaxf(before, top);
            const float kept = before == -INFINITY ? 0.0f : ex2((before - now) * coef_of[t].x);
            maxes[t] = now;
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float ref = maxes[t0 + j];
              y[j] = ex2((x[j] - (ref == -INFINITY ? 0.0f : ref)) * coef_of[t0 + j].x);
            }
            const float s = reduce_columns(y, [](float u, float v) { return u + v; });
            sums[t] = sums[t] * kept + s;
            __syncwarp();
          } else {
            // a box for either half
            uint8_t* box = out;
            if ((c & 1) == 0) {
              if (lane == 0) bulk_wait_read<0>();
              __syncwarp();
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float4 k = coef_of[t0 + j];
              x[j] = k.z * ex2(fmaf(x[j], k.x, -k.y)) - k.w;
            }
            listed(x, t, sOut + kOutTotal + quarter * kOutBytes,
                   [&](float* at, long long k) {
                     *at = a.s.divergence ? listed_gradient(a.s, a.g, row_no[t], k) : listed_of[t];
                   });
            if (t0 + 32 > rows) {
              // columns behind the rows hold what an earlier tile left
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (t0 + j >= rows) x[j] = 0.0f;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint4 v = make_uint4(pack2(x[8 * q], x[8 * q + 1]), pack2(x[8 * q + 2], x[8 * q + 3]),
                                         pack2(x[8 * q + 4], x[8 * q + 5]), pack2(x[8 * q + 6], x[8 * q + 7]));
              *reinterpret_cast<uint4*>(box + swizzled(lane, (c & 1) * 4 + q)) = on ? v : make_uint4(0, 0, 0, 0);
              const uint4 low = rounded_off(x + 8 * q, v);
              *reinterpret_cast<uint4*>(box + kOutBytes + swizzled(lane, (c & 1) * 4 + q)) = on ? low : make_uint4(0, 0, 0, 0);
            }
            if (c & 1) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&maps.out0, box, (c >> 1) * 64, m0);
                tma_store_2d(&maps.out0, box + kOutBytes, a.lo + (c >> 1) * 64, m0);
                bulk_commit();
              }
              ++staged;
            }
          }
        };
        if (SUMS) {
          // all rows' sums first, so that the accumulator is soon let go of
          float x[kFewRows / 32][32];
          for (int n = 0; n < a.sums; ++n) {
            if (n > 0) {
              release();
              next_accumulator();
              if (!wait_accumulator()) break;
            }
            const uint32_t from = tmem + lane_base + acc * kBN;
            const int blocks = min(a.sum_rest, it.kb1 - n * a.sum_rest), chains = (blocks + a.chain - 1) / a.chain;
            for (int k = 0; k < chains; ++k) {
#pragma unroll
              for (int c = 0; c < kFewRows / 32; ++c) {
                if (c * 32 >= rows || first >= stop) break;
                if (n == 0 && k == 0) {
                  tmem_ld32(from + c * 32, x[c]);
                } else {
                  add_tmem16(from + k * a.bn + c * 32, x[c]);
                  add_tmem16(from + k * a.bn + c * 32 + 16, x[c] + 16);
                }
              }
            }
          }
          if (gave_up) {
            if (a.K > 1) continue;   // as above
            break;
          }
          release();
#pragma unroll
          for (int c = 0; c < kFewRows / 32; ++c) {
            if (c * 32 >= rows || first >= stop) break;
            work_on(c, x[c]);
          }
        } else {
          for (int c = 0; c < chunks && first < stop; ++c) {
            const int t0 = c * 32;
            float x[32];
            if (t0 < rows) {
              tmem_ld32(t_acc + t0, x);
              for (int n = 1; n < a.chains; ++n) {
                float y[32];
                tmem_ld32(t_acc + n * a.bn + t0, y);
#pragma unroll
                for (int j = 0; j < 32; ++j) x[j] += y[j];
              }
            } else {
              // the half of the last box behind the rows: the last chain's columns would end behind the accumulator
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = 0.0f;
            }
            work_on(c, x);
          }
        }
        if (MODE == kGrad && first >= stop && quarter * 32 < held && m0 < a.piece) {
          // behind the vocabulary, but inside a block that the hidden gradient's product reads: zeros
          for (int c = 0; c < (rows + 63) / 64; ++c) {
            uint8_t* box = out + (staged & 1) * kOutBytes;
            if (lane == 0) bulk_wait_read<0>();
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4*>(box + swizzled(lane, q)) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&maps.out0, box, c * 64, m0);
              tma_store_2d(&maps.out0, box, a.lo + c * 64, m0);
              bulk_commit();
            }
            ++staged;
          }
        }
      } else if (MODE == kStats && (SUMS || a.kept)) {
        // the warp's half of the tile in registers: sums added up, then exponentials about its maximum
        float x[kBN / 64][32], plain = 0.0f;
        const int first = it.n0 + set * (kBN / 2);
        // the other sums; rows behind the last only let go of them
        auto next_sum = [&]() {
          if (!released) release();
          next_accumulator();
          return wait_accumulator();
        };
        if (m0 >= rows) {
          for (int n = 1; SUMS && n < a.sums; ++n)
            if (!next_sum()) break;
        } else {
#pragma unroll
          for (int c = 0; c < kBN / 64; ++c) tmem_ld32(t_acc + set * (kBN / 2) + c * 32, x[c]);
          release();
          for (int n = 1; SUMS && n < a.sums; ++n) {
            if (!next_sum()) break;
            const uint32_t from = tmem + lane_base + acc * kBN + set * (kBN / 2);
#pragma unroll
            for (int c = 0; c < kBN / 64; ++c) {
              add_tmem16(from + c * 32, x[c]);
              add_tmem16(from + c * 32 + 16, x[c] + 16);
            }
            release();
          }
        }
        if (SUMS && gave_up) break;
        if (m0 < rows) {
          float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < kBN / 64; ++c) {
            const int col = first + c * 32;
            if (col + 32 > a.V) {
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                if (col + j < a.V) plain += x[c][j];
                else x[c][j] = -INFINITY;
              }
            } else if (a.part_sum != nullptr) {
#pragma unroll
              for (int j = 0; j < 32; ++j) plain += x[c][j];
            }
            while (cur.next < min(col + 32, a.V)) {
              const int at = cur.next - col;
              float v = 0.0f;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (j == at) {
                  v = x[c][j];
                  x[c][j] = -INFINITY;
                }
              a.list_logit[list0 + cur.k] = v;
              cur.advance();
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; ++j) tops[j & 3] = fmaxf(tops[j & 3], x[c][j]);
          }
          const float mx = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
          const float ref = mx == -INFINITY ? 0.0f : mx;
          const float2 minus = make_float2(-ref, -ref), scale = make_float2(c2, c2), up = make_float2(kKeptOne, kKeptOne);
          float2 s2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
          if (!SUMS || a.kept) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              uint8_t* box = next_box(staged);
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                unsigned packed[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float* from = &x[2 * b + q / 4][(q % 4) * 8 + 2 * e];
                  float2 d = mul2(add2(make_float2(from[0], from[1]), minus), scale);
                  d = make_float2(ex2(d.x), ex2(d.y));
                  s2[e & 1] = add2(s2[e & 1], d);
                  d = mul2(d, up);
                  const __half2 h = __floats2half2_rn(d.x, d.y);
                  packed[e] = *reinterpret_cast<const unsigned*>(&h);
                }
                *reinterpret_cast<uint4*>(box + swizzled(lane, q)) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
              }
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&maps.out0, box, first + b * 64, m0);
                bulk_commit();
              }
              ++staged;
            }
          } else {
#pragma unroll
            for (int c = 0; c < kBN / 64; ++c)
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float2 d = mul2(add2(make_float2(x[c][2 * j], x[c][2 * j + 1]), minus), scale);
                s2[j & 1] = add2(s2[j & 1], make_float2(ex2(d.x), ex2(d.y)));
              }
          }
          if (live) {
            const long long p = static_cast<long long>(m) * a.part_tiles + 2 * (it.n0 / kBN) + set;
            a.part[p] = make_float2(mx, (s2[0].x + s2[1].x) + (s2[0].y + s2[1].y));
            if (a.part_sum != nullptr) a.part_sum[p] = plain;
          }
        }
      } else if (MODE == kStats) {
        float mx = -INFINITY, sum = 0.0f, plain = 0.0f;
        const int end = min(a.V, it.n0 + kBN);         // behind the tile's last column
        for (int c = set * (kBN / 64); c < (set + 1) * (kBN / 64); ++c) {
          const int col = it.n0 + c * 32;              // vocabulary column of x[0]
          if (col >= end || m0 >= rows) break;
          float x[32];
          tmem_ld32(t_acc + c * 32, x);
          if (col + 32 > end) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (col + j < end) plain += x[j];
              else x[j] = -INFINITY;
            }
          } else if (a.part_sum != nullptr) {
#pragma unroll
            for (int j = 0; j < 32; ++j) plain += x[j];
          }
          while (cur.next < min(col + 32, end)) {
            const int at = cur.next - col;
            float v = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j == at) {
                v = x[j];
                x[j] = -INFINITY;
              }
            a.list_logit[list0 + cur.k] = v;
            cur.advance();
          }
          __syncwarp();
          float tops[4] = {mx, x[1], x[2], x[3]};
#pragma unroll
          for (int j = 0; j < 32; ++j) tops[j & 3] = fmaxf(tops[j & 3], x[j]);
          const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
          const float ref = top == -INFINITY ? 0.0f : top;
          sum *= ex2((mx - ref) * c2);
          const float2 minus = make_float2(-ref, -ref), scale = make_float2(c2, c2);
          float2 s2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 d = mul2(add2(make_float2(x[2 * j], x[2 * j + 1]), minus), scale);
            s2[j & 1] = add2(s2[j & 1], make_float2(ex2(d.x), ex2(d.y)));
          }
          sum += (s2[0].x + s2[1].x) + (s2[0].y + s2[1].y);
          mx = top;
        }
        if (live) {
          const long long p = static_cast<long long>(m) * a.part_tiles + 2 * (it.n0 / kBN) + set;
          a.part[p] = make_float2(mx, sum);
          if (a.part_sum != nullptr) a.part_sum[p] = plain;
        }
      } else if (MODE == kGrad) {
        // the whole tile is written: the products read its rows up to the tile's end
        for (int c = set * (kBN / 128); c < (set + 1) * (kBN / 128); ++c) {
          uint8_t* box = next_box(staged);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float x[32];
            tmem_ld32(t_acc + c * 64 + half * 32, x);
            const int col = a.v0 + it.n0 + c * 64 + half * 32;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float2 d = fma2(make_float2(x[2 * j], x[2 * j + 1]), make_float2(coef.x, coef.x), make_float2(-coef.y, -coef.y));
              d = fma2(make_float2(ex2(d.x), ex2(d.y)), make_float2(coef.z, coef.z), make_float2(-coef.w, -coef.w));
              x[2 * j] = d.x;
              x[2 * j + 1] = d.y;
            }
            while (cur.next < col + 32) {
              const int at = cur.next - col;
              const float v = cur.value;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (j == at) x[j] = v;
              cur.advance();
            }
            __syncwarp();
            if (col + 32 > a.V) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (col + j >= a.V) x[j] = 0.0f;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint4 v = make_uint4(pack2(x[8 * q], x[8 * q + 1]), pack2(x[8 * q + 2], x[8 * q + 3]),
                                         pack2(x[8 * q + 4], x[8 * q + 5]), pack2(x[8 * q + 6], x[8 * q + 7]));
              *reinterpret_cast<uint4*>(box + swizzled(lane, half * 4 + q)) = v;
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&maps.out0, box, it.n0 + c * 64, m0);
            bulk_commit();
          }
          ++staged;
        }
      } else if (FEW && it.kind == 0) {
        // hidden gradient with hidden columns in the lanes: turned around on the way into the box
        for (int c = set; c < (rows + 31) / 32 && m0 < a.H; c += kSets) {
          float x[32];
          tmem_ld32(t_acc + c * 32, x);
          float y[32];
          tmem_ld32(t_acc + a.bn + c * 32, y);
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] += y[j];
          uint8_t* box = next_box(staged);
#pragma unroll
          for (int j = 0; j < 32; ++j) *block_at(box, j, lane) = x[j];
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            const int y = it.split * a.rpad + c * 32;
            if (a.first_piece)
              tma_store_2d(&maps.out0, box, m0, y);
            else
              tma_add_2d(&maps.out0, box, m0, y);
            bulk_commit();
          }
          ++staged;
        }
      } else if (it.kind == 0) {
        // hidden gradient: fp32, added to what earlier pieces left
        for (int c = set * (kBN / 64); c < (set + 1) * (kBN / 64); ++c) {
          if (it.n0 + c * 32 >= a.H) break;
          float x[32];
          tmem_ld32(t_acc + c * 32, x);
          uint8_t* box = next_box(staged);
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *reinterpret_cast<float4*>(box + swizzled(lane, q)) =
                make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            const int y = it.split * a.rpad + m0;
            if (a.first_piece)
              tma_store_2d(&maps.out0, box, it.n0 + c * 32, y);
            else
              tma_add_2d(&maps.out0, box, it.n0 + c * 32, y);
            bulk_commit();
          }
          ++staged;
        }
      } else {
        // head gradient of the piece: complete, rounded once
        const bool in_rows = a.v0 + m0 < a.V;
        constexpr int kSpan = kBN / 64 / kSets;
        for (int c = set * kSpan; c < (set + 1) * kSpan; ++c) {
          if (it.n0 + c * 64 >= a.H) break;
          uint8_t* box = next_box(staged);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float x[32];
            if (empty_sum) {
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = 0.0f;
            } else {
              tmem_ld32(t_acc + c * 64 + half * 32, x);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint4 v = make_uint4(pack2(x[8 * q], x[8 * q + 1]), pack2(x[8 * q + 2], x[8 * q + 3]),
                                         pack2(x[8 * q + 4], x[8 * q + 5]), pack2(x[8 * q + 6], x[8 * q + 7]));
              *reinterpret_cast<uint4*>(box + swizzled(lane, half * 4 + q)) = v;
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            // a group for every box, stored or not: the waits above count groups
            if (in_rows) tma_store_2d(&maps.out1, box, it.n0 + c * 64, a.v0 + m0);
            bulk_commit();
          }
          ++staged;
        }
      }
      if (!FEW && MODE != kProd && more) fetch_id();
      if (!empty_sum) {
        if (!released) release();
        next_accumulator();
      }
    }
    if (FEW && MODE == kStats) {
      const int column = blockIdx.x * 4 + quarter;
      for (int t = lane; t < rows; t += 32) {
        const long long p = static_cast<long long>(t) * a.part_tiles + column;
        a.part[p] = make_float2(reinterpret_cast<float*>(state + kStateMax)[quarter * kFewRows + t],
                                reinterpret_cast<float*>(state + kStateSum)[quarter * kFewRows + t]);
        if (a.part_sum != nullptr) a.part_sum[p] = reinterpret_cast<float*>(state + kStatePlain)[quarter * kFewRows + t];
      }
    }
    if (lane == 0) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // neither CTA leaves while the other may still signal its barriers
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kBN) : "memory");
  }
}

// ------------------------------------------------------------------ rows ----
__device__ __forceinline__ long long load_id(const void* p, int i64, long long i) {
  return i64 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
}

// Block-wide combinations of one value a thread (128 threads); `buf` holds four values.
template <typename T, typename Op>
__device__ __forceinline__ T block_combine(T v, T* buf, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = v;
  __syncthreads();
  return op(op(buf[0], buf[1]), op(buf[2], buf[3]));
}

// The teacher's list of one row (one block): empty slots dropped, a column listed twice merged, ascending by
// column (a bitonic sort; comparing all with all took 135 us for 3957 rows of 241); its masses in fp64,
// rounded to fp32.
__global__ void __launch_bounds__(128) teacher_rows_kernel(const HeadLossState s, const HeadTargets t) {
  __shared__ unsigned long long key[kHeadMaxListed];   // column above slot; empty slots above all
  __shared__ double mass[kHeadMaxListed];
  __shared__ double buf[4];
  __shared__ int found[4];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, K = s.K, r = blockIdx.x;
  int size = 32;
  while (size < K) size *= 2;
  const long long base = static_cast<long long>(r) * K;
  const double it = s.inv_temp != nullptr ? static_cast<double>(s.inv_temp[r]) : 1.0;
  const auto add = [](double u, double v) { return u + v; };
  const auto larger = [](double u, double v) { return fmax(u, v); };
  double top = -INFINITY;
  bool any = false, nan = false;
  for (int k = tid; k < size; k += 128) {
    key[k] = ~0ull;
    if (k >= K) continue;
    long long v = load_id(t.ids, t.ids_i64, base + k);
    const float x = t.teacher_bf16 ? bf2f(static_cast<const __nv_bfloat16*>(t.teacher)[base + k])
                                   : static_cast<const float*>(t.teacher)[base + k];
    if (v >= s.V) {
      record_error(s.status, kErrBadIndex);
      v = -1;
    }
    mass[k] = -INFINITY;
    if (v < 0 || x == -INFINITY) continue;
    key[k] = (static_cast<unsigned long long>(v) << 32) | static_cast<unsigned>(k);
    const double z = static_cast<double>(x) * it;
    mass[k] = z;
    any = true;
    nan |= !(z == z);
    top = fmax(top, z);
  }
  any = __syncthreads_or(any);
  nan = __syncthreads_or(nan);
  top = block_combine(top, buf, larger);
  const double shift = t.teacher_lse != nullptr ? static_cast<double>(t.teacher_lse[r]) : top;
  double sum = 0.0;
  for (int k = tid; k < K; k += 128) {
    const double e = key[k] == ~0ull ? 0.0 : exp(mass[k] - shift);
    mass[k] = e;
    sum += e;
  }
  sum = block_combine(sum, buf, add);
  const double inv = t.teacher_lse != nullptr ? 1.0 : 1.0 / sum;
  for (int span = 2; span <= size; span *= 2) {
    for (int step = span / 2; step > 0; step /= 2) {
      __syncthreads();
      for (int i = tid; i < size / 2; i += 128) {
        const int at = 2 * i - (i & (step - 1)), other = at + step;
        const unsigned long long u = key[at], v = key[other];
        if ((u > v) == ((at & span) == 0)) {
          key[at] = v;
          key[other] = u;
        }
      }
    }
  }
  __syncthreads();
  int before = 0;
  for (int i0 = 0; i0 < size; i0 += 128) {
    const int i = i0 + tid;
    const unsigned long long mine = i < size ? key[i] : ~0ull;
    const unsigned column = static_cast<unsigned>(mine >> 32);
    // the first of a column takes the masses of its later ones
    const bool first = mine != ~0ull && (i == 0 || static_cast<unsigned>(key[i - 1] >> 32) != column);
    const unsigned ballot = __ballot_sync(0xffffffffu, first);
    __syncthreads();
    if (lane == 0) found[warp] = __popc(ballot);
    __syncthreads();
    int at = before + __popc(ballot & ((1u << lane) - 1u));
    for (int q = 0; q < warp; ++q) at += found[q];
    if (first) {
      double m = mass[static_cast<unsigned>(mine)];
      for (int j = i + 1; j < size && static_cast<unsigned>(key[j] >> 32) == column; ++j)
        m += mass[static_cast<unsigned>(key[j])];
      s.list_id[base + at] = static_cast<int>(column);
      s.list_mass[base + at] = static_cast<float>(m * inv);
    }
    before += found[0] + found[1] + found[2] + found[3];
  }
  for (int k = before + tid; k < K; k += 128) s.list_id[base + k] = INT_MAX;
  if (tid == 0) {
    t.active[r] = any ? 1 : 0;
    // a list of all columns (`before` of them) leaves no rest
    const double rest = t.teacher_lse != nullptr && before < s.V ? (nan ? sum : fmax(1.0 - sum, 0.0)) : 0.0;
    s.rest_mass[r] = static_cast<float>(rest);
    s.all_mass[r] = t.teacher_lse != nullptr ? static_cast<float>(sum + rest) : 1.0f;
  }
}

// Numbers the rows that count (one block); a target outside the vocabulary is recorded and
// its row left out.
__global__ void __launch_bounds__(1024) compact_rows_kernel(const HeadLossState s, const HeadTargets t) {
  __shared__ int warp_sums[32];
  __shared__ int carry;
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int r0 = 0; r0 < s.R; r0 += 1024) {
    const int r = r0 + threadIdx.x;
    bool on = false;
    if (r < s.R) {
      if (s.divergence) {
        on = t.active[r] != 0;
      } else {
        const long long v = load_id(t.ids, t.ids_i64, r);
        on = v != t.ignore_index;
        if (on && (v < 0 || v >= s.V)) {
          record_error(s.status, kErrBadIndex);
          on = false;
        }
        s.list_id[r] = on ? static_cast<int>(v) : INT_MAX;
      }
    }
    const unsigned ballot = __ballot_sync(0xffffffffu, on);
    if (lane == 0) warp_sums[warp] = __popc(ballot);
    __syncthreads();
    int before = carry;
    for (int q = 0; q < warp; ++q) before += warp_sums[q];
    const int m = before + __popc(ballot & ((1u << lane) - 1u));
    if (r < s.R) {
      s.compact_of[r] = on ? m : -1;
      if (on) s.row_of[m] = r;
      else s.loss[r] = 0.0f;
    }
    __syncthreads();
    if (threadIdx.x == 1023) carry = before + __popc(ballot);
    __syncthreads();
  }
  const int n = carry;
  for (int m = n + threadIdx.x; m < s.rpad; m += 1024) s.row_of[m] = -1;
  if (threadIdx.x == 0) *s.count = n;
}

// Both at once for few rows: every block counts the rows before its own.
__global__ void __launch_bounds__(128) few_rows_kernel(const HeadLossState s, const HeadTargets t) {
  __shared__ int before_of[4], total_of[4];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, b = blockIdx.x;
  auto counts = [&](int r) {
    if (r >= s.R) return false;
    if (s.divergence) return t.active[r] != 0;
    const long long v = load_id(t.ids, t.ids_i64, r);
    return v != t.ignore_index && v >= 0 && v < s.V;
  };
  int before = 0, total = 0;
  for (int r0 = warp * 32; r0 < kCountRows; r0 += 128) {
    const unsigned on = __ballot_sync(0xffffffffu, counts(r0 + lane));
    total += __popc(on);
    before += r0 + 32 <= b ? __popc(on) : r0 < b ? __popc(on & ((1u << (b - r0)) - 1u)) : 0;
  }
  if (lane == 0) {
    before_of[warp] = before;
    total_of[warp] = total;
  }
  __syncthreads();
  before = before_of[0] + before_of[1] + before_of[2] + before_of[3];
  total = total_of[0] + total_of[1] + total_of[2] + total_of[3];
  const bool on = counts(b);
  if (threadIdx.x == 0) {
    if (b == 0) *s.count = total;
    if (b >= total) s.row_of[b] = -1;
    if (on) s.row_of[before] = b;
    if (b < s.R) {
      s.compact_of[b] = on ? before : -1;
      if (!on) s.loss[b] = 0.0f;
      if (!s.divergence) {
        const long long v = load_id(t.ids, t.ids_i64, b);
        s.list_id[b] = on ? static_cast<int>(v) : INT_MAX;
        if (!on && v != t.ignore_index) record_error(s.status, kErrBadIndex);
      }
    }
  }
  const int vecs = s.H / 8;
  if (b >= total) {
    uint4* dst = reinterpret_cast<uint4*>(s.hc + static_cast<long long>(b) * s.H);
    for (int i = threadIdx.x; i < vecs; i += 128) dst[i] = make_uint4(0, 0, 0, 0);
  }
  if (on) {
    const uint4* src = reinterpret_cast<const uint4*>(s.h + static_cast<long long>(b) * s.ldh);
    uint4* dst = reinterpret_cast<uint4*>(s.hc + static_cast<long long>(before) * s.H);
    for (int i = threadIdx.x; i < vecs; i += 128) dst[i] = src[i];
  }
}

__global__ void __launch_bounds__(128) gather_rows_kernel(const HeadLossState s) {
  pdl_trigger();
  pdl_wait();
  const int m = blockIdx.x;
  const int n = *s.count;
  if (m >= (n + kHeadRowPad - 1) / kHeadRowPad * kHeadRowPad) return;
  const int vecs = s.H / 8;
  uint4* dst = reinterpret_cast<uint4*>(s.hc + static_cast<long long>(m) * s.H);
  if (m >= n) {
    for (int i = threadIdx.x; i < vecs; i += 128) dst[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const uint4* src = reinterpret_cast<const uint4*>(s.h + static_cast<long long>(s.row_of[m]) * s.ldh);
  for (int i = threadIdx.x; i < vecs; i += 128) dst[i] = src[i];
}

// Folds the tiles of a row and forms its loss (one block a row).  The normaliser and the loss are formed
// in fp64 from fp32 sums: a divergence is a small difference of logarithms.
//
// The tensor core's sums of H products come out a little short (its additions truncate: about 2e-6 of a
// logit at H = 3584 in one chain).  Listed logits and normaliser share that, so most of it cancels in a loss; listed
// logits summed again in fp32 made the losses worse (1.2e-6 for 0.9e-6 relative, 64 rows of 152064).  Up to 128
// rows have room for several chains (2.0e-7, at no time); more are summed in parts (kSumBlocks).
__global__ void __launch_bounds__(128) finish_rows_kernel(const HeadLossState s, const HeadStatsScratch p) {
  __shared__ double buf_d[4];
  __shared__ float buf_f[4];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x;
  const int m = blockIdx.x;
  if (m >= *s.count) return;
  const auto add = [](double u, double v) { return u + v; };
  const auto larger = [](float u, float v) { return fmaxf(u, v); };
  const int r = s.row_of[m];
  const float itf = s.inv_temp != nullptr ? s.inv_temp[r] : 1.0f;
  const double it = itf;
  const float c2 = itf * kLog2e;
  const float2* part = p.part + static_cast<long long>(m) * p.tiles;
  float mx = -INFINITY;
#pragma unroll 4
  for (int i = tid; i < p.tiles; i += 128) mx = fmaxf(mx, part[i].x);
  mx = block_combine(mx, buf_f, larger);
  double part_rest = 0.0, plain = 0.0;
#pragma unroll 4
  for (int i = tid; i < p.tiles; i += 128) {
    const float2 v = part[i];
    if (v.x != -INFINITY || !(v.y == 0.0f)) part_rest += static_cast<double>(v.y) * exp2f((v.x - mx) * c2);
    if (p.part_sum != nullptr) plain += p.part_sum[static_cast<long long>(m) * p.tiles + i];
  }
  part_rest = block_combine(part_rest, buf_d, add);
  if (p.part_sum != nullptr) plain = block_combine(plain, buf_d, add);
  const long long base = static_cast<long long>(r) * s.K;
  float top = mx;
  for (int k = tid; k < s.K; k += 128)
    if (s.list_id[base + k] != INT_MAX) top = fmaxf(top, s.list_logit[base + k]);
  top = block_combine(top, buf_f, larger);
  double listed = 0.0;
  for (int k = tid; k < s.K; k += 128)
    if (s.list_id[base + k] != INT_MAX)
      listed += exp((static_cast<double>(s.list_logit[base + k]) - static_cast<double>(top)) * it);
  listed = block_combine(listed, buf_d, add);
  const double rest =
      mx != -INFINITY ? part_rest * exp((static_cast<double>(mx) - static_cast<double>(top)) * it) : part_rest;
  const double lse = static_cast<double>(top) * it + log(rest + listed);
  const double q_rest = rest / (rest + listed);
  double loss, factor, second = q_rest, listed_factor = 0.0;
  if (!s.divergence) {
    const double target = s.list_logit[base];
    const double hot = listed > 0.0 ? log1p(rest / listed) : lse - target;
    const double eps = s.smoothing;
    loss = (1.0 - eps) * hot + s.z_loss * lse * lse;
    if (p.part_sum != nullptr) loss += eps * (lse - plain / s.V);
    factor = 1.0 + 2.0 * s.z_loss * lse;
  } else {
    double sum = 0.0;
    for (int k = tid; k < s.K; k += 128) {
      if (s.list_id[base + k] == INT_MAX) continue;
      const double mass = s.list_mass[base + k];
      if (mass == 0.0) continue;
      sum += mass * (log(mass) - (static_cast<double>(s.list_logit[base + k]) * it - lse));
    }
    loss = block_combine(sum, buf_d, add);
    // Every log q of the loss brings its mass times q_v to the gradient: all masses, whose sum is above one where a
    // teacher's logits were rounded and its normaliser was not (bf16 logits near 20: up to 6 %).
    //
    // On the unlisted columns q_v = q_rest r_v, with r their own softmax, and the rest takes rest_mass r_v off.  r is
    // at most one however little mass the student leaves there; q_v and rest_mass / q_rest leave fp32 where listed logits
    // lead by 88, and rest leaves fp64 where they lead by 745.
    listed_factor = s.all_mass[r];
    const double lse_rest = part_rest == 0.0 ? -INFINITY : static_cast<double>(mx) * it + log(part_rest);
    const double rest_mass = s.rest_bucket ? static_cast<double>(s.rest_mass[r]) : 0.0;
    if (rest_mass != 0.0) loss += rest_mass * (log(rest_mass) - (lse_rest - lse));
    factor = listed_factor * q_rest - rest_mass;
    second = part_rest == 0.0 ? lse : lse_rest;   // no unlisted column
  }
  if (tid == 0) {
    s.loss[r] = static_cast<float>(loss);
    s.row_stat[r] = make_float4(static_cast<float>(lse), static_cast<float>(second), static_cast<float>(factor),
                                static_cast<float>(listed_factor));
  }
}

// Row coefficients and listed values of the logits' gradient (one warp a compact row).
__global__ void __launch_bounds__(128) grad_rows_kernel(const HeadLossState s, const HeadGradArgs g) {
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int m = blockIdx.x * 4 + warp;
  if (m >= s.rpad) return;
  if (m >= *s.count) {
    // rows behind the last of its tile: zero whatever the tile holds there
    if (lane == 0) g.row_coef[m] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    return;
  }
  const int r = s.row_of[m];
  if (lane == 0) g.row_coef[m] = row_coefficients(s, g.g, r);
  const long long base = static_cast<long long>(r) * s.K;
  for (int k = lane; k < s.K; k += 32)
    if (s.list_id[base + k] != INT_MAX) g.list_grad[base + k] = listed_gradient(s, g.g, r, base + k);
}

// The logits' gradient of a piece from kept logits: [V, kept pitch] fp32 to [piece, pitch] bf16 (with its second
// half).  A thread has eight rows, whose inputs it holds, and goes over the vocabulary.  One pass of
// memory: 6 bytes a logit, 8 with the second half.
constexpr int kKeptAhead = 4;                       // logits of a row in flight a thread

__global__ void __launch_bounds__(256, 2) kept_grad_kernel(const HeadLossState s, const HeadGradArgs g, int kept_pitch, int pitch,
                                                        int lo, int v0, int cols) {
  pdl_trigger();
  pdl_wait();
  const int rows = *s.count;
  const int groups = (rows + 63) / 64 * 8;          // of eight rows; the products read whole blocks of 64
  if (groups == 0) return;
  const int per = 256 / groups, group = threadIdx.x % groups, first = threadIdx.x / groups;
  if (first >= per) return;
  const int t0 = group * 8;
  float4 coef[8];
  int id[8];
  float value[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int r = t0 + e < rows ? s.row_of[t0 + e] : -1;
    coef[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    id[e] = -1;
    value[e] = 0.0f;
    if (r >= 0) {
      coef[e] = row_coefficients(s, g.g, r);
      if (s.K == 1) {
        id[e] = s.list_id[r] - v0;
        value[e] = listed_gradient(s, g.g, r, r);
      }
    }
  }
  const int end = min((cols + kBK - 1) / kBK * kBK, g.piece);   // zeros behind the vocabulary, up to its last block
  const int step = gridDim.x * per;
  for (int at = blockIdx.x * per + first; at < end; at += kKeptAhead * step) {
    float4 in[kKeptAhead][2];
#pragma unroll
    for (int u = 0; u < kKeptAhead; ++u) {
      const int v = at + u * step;
      if (v < cols && t0 < rows) {
        const float4* src = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(g.kept) + static_cast<long long>(v0 + v) * kept_pitch + t0);
        in[u][0] = __ldcs(src);
        in[u][1] = __ldcs(src + 1);
      }
    }
#pragma unroll
    for (int u = 0; u < kKeptAhead; ++u) {
      const int v = at + u * step;
      if (v >= end) break;
      float x[8] = {in[u][0].x, in[u][0].y, in[u][0].z, in[u][0].w, in[u][1].x, in[u][1].y, in[u][1].z, in[u][1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // rows behind the last: whatever the memory held
        x[e] = v < cols && t0 + e < rows ? coef[e].z * ex2(fmaf(x[e], coef[e].x, -coef[e].y)) - coef[e].w : 0.0f;
        if (v == id[e]) x[e] = value[e];
      }
      const uint4 hi = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
      __nv_bfloat16* dst = g.dl + static_cast<long long>(v) * pitch + t0;
      *reinterpret_cast<uint4*>(dst) = hi;
      *reinterpret_cast<uint4*>(dst + lo) = rounded_off(x, hi);
    }
  }
}

// The same from kept exponentials of many rows: [rpad, pitch] fp16 about the maxima of 128 columns to [rpad, piece] bf16.
// A block takes 8192 columns of a row.
__global__ void __launch_bounds__(256) kept_scale_kernel(const HeadLossState s, const HeadGradArgs g, const HeadKept k, int v0,
                                                         int cols) {
  pdl_trigger();
  pdl_wait();
  constexpr int kVecs = 4;
  const int m = blockIdx.x, rows = *s.count;
  if (m >= (rows + kBK - 1) / kBK * kBK) return;           // the head gradient's product reads whole blocks of 64
  const int end = min((cols + kBK - 1) / kBK * kBK, g.piece), begin = blockIdx.y * kVecs * 2048;
  __nv_bfloat16* dst = g.dl + static_cast<long long>(m) * g.piece;
  if (m >= rows) {
    for (int v = begin + threadIdx.x * 8; v < min(end, begin + kVecs * 2048); v += 2048)
      *reinterpret_cast<uint4*>(dst + v) = make_uint4(0, 0, 0, 0);
    return;
  }
  const __half* src = reinterpret_cast<const __half*>(g.kept) + static_cast<long long>(m) * k.pitch + v0;
  const float2* part = reinterpret_cast<const float2*>(g.kept + k.part_at) + static_cast<long long>(m) * k.tiles + v0 / 128;
  uint4 in[kVecs];
  float ref[kVecs];
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int v = begin + u * 2048 + threadIdx.x * 8;
    if (v < cols) {
      in[u] = __ldcs(reinterpret_cast<const uint4*>(src + v));
      ref[u] = part[v / 128].x;
    }
  }
  const float4 coef = g.row_coef[m];
  const long long base = static_cast<long long>(s.row_of[m]) * s.K;
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int v = begin + u * 2048 + threadIdx.x * 8;
    if (begin + u * 2048 >= end) break;
    const float scale = coef.z * ex2(fmaf(ref[u], coef.x, -coef.y)) * (1.0f / kKeptOne);
    const unsigned w[4] = {in[u].x, in[u].y, in[u].z, in[u].w};
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
      x[2 * e] = fmaf(f.x, scale, -coef.w);
      x[2 * e + 1] = fmaf(f.y, scale, -coef.w);
    }
    if (v + 8 > cols) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v + e >= cols) x[e] = 0.0f;
    }
    if (v < end)
      *reinterpret_cast<uint4*>(dst + v) = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
  }
  // listed columns of this block, over what it wrote there
  __syncthreads();
  for (int i = threadIdx.x; i < s.K; i += 256) {
    const int at = s.list_id[base + i] - v0;
    if (at >= begin && at < min(cols, begin + kVecs * 2048)) dst[at] = __float2bfloat16_rn(g.list_grad[base + i]);
  }
}

// Lists of several columns: their gradients, in place of what the pass above left there (one warp a row).
__global__ void __launch_bounds__(128) kept_listed_kernel(const HeadLossState s, const HeadGradArgs g, int pitch, int lo, int v0,
                                                          int cols) {
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, m = blockIdx.x * 4 + warp;
  if (m >= *s.count) return;
  const int r = s.row_of[m];
  const long long base = static_cast<long long>(r) * s.K;
  for (int k = lane; k < s.K; k += 32) {
    const int id = s.list_id[base + k];
    if (id < v0 || id >= v0 + cols) continue;
    const float x = listed_gradient(s, g.g, r, base + k);
    const __nv_bfloat16 hi = __float2bfloat16_rn(x);
    __nv_bfloat16* dst = g.dl + static_cast<long long>(id - v0) * pitch + m;
    *dst = hi;
    dst[lo] = __float2bfloat16_rn(x - __bfloat162float(hi));
  }
}

// Sums the parts of the hidden gradient.  `mend`: dl had its listed entries, which are most of a row's gradient, in
// one bf16 number; what rounding took from them times their head rows comes on top here.  (Relative error
// of dh for a loss with one target 0.0024 without, 0.0017 with it: that of rounding dh itself.)  Few rows have
// those entries in dl's second half.
constexpr int kMendAhead = 16;   // 192 rows of 3584, lists of 64: 40 us; 8 left to the compiler 64 us

__global__ void __launch_bounds__(128) hidden_grad_kernel(const HeadLossState s, const HeadGradArgs g, int mend) {
  __shared__ float lost[kHeadMaxListed];
  __shared__ int column[kHeadMaxListed];
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x;
  const int m = s.compact_of[r];
  int listed = 0;
  if (mend && m >= 0) {
    for (int k = threadIdx.x; k < s.K; k += 128) {
      const long long at = static_cast<long long>(r) * s.K + k;
      column[k] = s.list_id[at];
      const float x = column[k] != INT_MAX ? listed_gradient(s, g.g, r, at) : 0.0f;
      lost[k] = x - __bfloat162float(__float2bfloat16_rn(x));
    }
    __syncthreads();
    listed = s.K;
    while (listed > 0 && column[listed - 1] == INT_MAX) --listed;   // the list's end is empty
  }
  const int i = blockIdx.y * 128 + threadIdx.x;
  if (i >= s.H / 8) return;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (m >= 0) {
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < listed; k0 += kMendAhead) {
      uint4 w[kMendAhead];
#pragma unroll
      for (int a = 0; a < kMendAhead; ++a)
        if (k0 + a < listed)
          w[a] = __ldg(reinterpret_cast<const uint4*>(s.w + static_cast<long long>(column[k0 + a]) * s.ldw) + i);
#pragma unroll
      for (int a = 0; a < kMendAhead; ++a) {
        if (k0 + a >= listed) break;
        const unsigned u[4] = {w[a].x, w[a].y, w[a].z, w[a].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = fmaf(lost[k0 + a], __uint_as_float(u[e] << 16), x[2 * e]);
          x[2 * e + 1] = fmaf(lost[k0 + a], __uint_as_float(u[e] & 0xFFFF0000u), x[2 * e + 1]);
        }
      }
    }
#pragma unroll 4
    for (int q = 0; q < g.splits; ++q) {
      const float4* src = reinterpret_cast<const float4*>(
          g.dh_part + (static_cast<long long>(q) * s.rpad + m) * s.H + i * 8);
      const float4 lo = __ldcg(src), hi = __ldcg(src + 1);
      x[0] += lo.x; x[1] += lo.y; x[2] += lo.z; x[3] += lo.w;
      x[4] += hi.x; x[5] += hi.y; x[6] += hi.z; x[7] += hi.w;
    }
    v = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
  }
  reinterpret_cast<uint4*>(g.dh + static_cast<long long>(r) * s.H)[i] = v;
}

// ------------------------------------------------------------------ host ----
bool encode(CUtensorMap* map, CUtensorMapDataType type, int size, const void* ptr, long long rows, long long cols,
            long long ld, int box_cols, int box_rows) {
  EncodeTiledFn fn = tensor_map_encoder();
  if (!fn) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * size};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool map_bf16(CUtensorMap* map, const void* ptr, long long rows, long long cols, long long ld, int box_cols,
              int box_rows) {
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ptr, rows, cols, ld, box_cols, box_rows);
}

int device_sms() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!cached[dev]) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    cached[dev] = n > 0 ? n : 148;
  }
  return cached[dev];
}

int ceil_div(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

// CTA pairs of a launch.
int pairs_for(int items) { return std::max(1, std::min(items, device_sms() / 2)); }

// Rows in columns, and two such sums in chains, fit up to 128 rows.  More would fit in one chain, three times as far off, and
// without a second half of dl.  In columns / with the many rows, forward pass and with hidden gradient: 129 rows of 3584 and
// 152064 columns 239 / 251, 502 / 516 us; 192 rows 278 / 282, 625 / 602; 256 rows 303 / 286, 692 / 625; 136 rows of
// 896 and 65536 columns 46 / 41, 119 / 99; 192 rows of 512 and 2048 columns 20 / 18, 74 / 78.
bool few_rows(int R) { return R <= kFewRows; }

// Rows in columns: how many vocabulary columns one CTA's lanes hold, a multiple of `step`.  As many tiles as
// fill the rounds: with 152064 columns on 74 pairs, 256 a tile make 594 tiles, two more than eight
// rounds; 240 make nine nearly full ones.
int lane_slot(int cols, int step) {
  const int pairs = device_sms() / 2;
  int best = kHalf;
  long long cost = LLONG_MAX;
  for (int w = kHalf; w >= 96; w -= step) {
    const long long c = static_cast<long long>(ceil_div(ceil_div(cols, 2 * w), pairs)) * (w + 4);
    if (c < cost) {
      cost = c;
      best = w;
    }
  }
  return best;
}

template <int MODE, bool FEW, bool SUMS = false>
cudaError_t launch_gemm(const Maps& maps, GemmArgs a, int max_items, cudaStream_t stream) {
  static bool set[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !set[dev]) {
    e = cudaFuncSetAttribute(head_gemm_kernel<MODE, FEW, SUMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost + 1024);
    if (e != cudaSuccess) return e;
    if (dev < 64) set[dev] = true;
  }
  const int rest = out_bytes_of(MODE, FEW, a.kept) + (FEW && MODE != kProd ? kStateBytes : 0) + kBarBytes;
  const StageBytes sb = stage_bytes_of(MODE, FEW, a);
  a.stages = std::min(kMaxStages, (kSmemMost - rest) / (sb.a + sb.b));
  const int smem = 1024 + a.stages * (sb.a + sb.b) + rest;
  return launch_pdl(head_gemm_kernel<MODE, FEW, SUMS>, dim3(2 * pairs_for(max_items)), dim3(threads_of(MODE, FEW)), smem, stream, maps, a);
}

// Cuts the reduction of the statistics into sums (GemmArgs::sums): as many as the issuer makes of these numbers, none
// empty.  With rows in columns a sum is as long as its chains allow.
void cut_sums(GemmArgs& a, bool few) {
  const int blocks = ceil_div(a.H, kBK);
  a.sums = 1;
  a.sum_first = a.sum_rest = blocks;
  if (few) {
    if (a.chain <= kChainBlocks) return;
    const int chains = most_chains(a.bn);
    a.sum_first = a.sum_rest = ceil_div(blocks, ceil_div(blocks, chains * kChainBlocks));
    a.sums = ceil_div(blocks, a.sum_rest);
    a.chain = ceil_div(a.sum_rest, chains);
  } else if (blocks > kOneSum) {
    a.sum_first = std::min(kSumBlocks, ceil_div(blocks, 2));
    const int rest = blocks - 2 * a.sum_first, others = ceil_div(std::max(rest, 0), kSumBlocks);
    a.sum_rest = others > 0 ? ceil_div(rest, others) : 1;
    a.sums = 2 + others;
  }
}

GemmArgs base_args(const HeadLossState& s) {
  GemmArgs a{};
  a.count = s.count;
  a.H = s.H;
  a.V = s.V;
  a.K = s.K;
  a.row_of = s.row_of;
  a.list_id = s.list_id;
  a.rpad = s.rpad;
  a.slot = kHalf;
  a.bn = few_rows(s.R) ? row_columns(s.R) : kBN;
  // the tensor core truncates at every addition: shorter chains, added in fp32, are off by less.  Blocks in turn took 251
  // us where chains of neighbours take 226 (64 rows of 3584 on 152064 columns).
  a.chain = ceil_div(ceil_div(s.H, kBK), most_chains(a.bn));
  a.chains = ceil_div(ceil_div(s.H, kBK), a.chain);
  a.lo = ceil_div(s.R, 64) * 64;
  a.status = s.status;
  return a;
}

}  // namespace

// What a forward pass keeps for its backward pass.  Few rows: a logit kept is 8 bytes, written and read, and saves the
// second reading of the head with its products.  Forward and hidden gradient, kept against computed again: 16 rows
// of 3584 and 152064 columns 426 / 582 us, 128 rows of 512 174 / 185 us; 128 rows of 896 and 32768 columns
// 75 / 80 us, 64 rows of 512 and 20000 columns 74 / 72 us (one more launch and allocation).  At most 256 MB, and at most
// twice the head.
//
// Many rows: 4 bytes a logit for 2 H operations.  Both gradients: 4096 rows of 3584 and 152064 columns 9.6 / 11.9 ms, 300
// rows of 3584 1449 / 1832 us, 1024 rows of 512 and 50000 columns 214 / 228 us, 4096 rows of 256 and 152064
// columns 1749 / 1695 us, 4096 rows of 64 and 32768 columns 385 / 335 us.  At most 2 GB.
HeadKept head_loss_kept(int R, int H, int V) {
  HeadKept k{};
  if (few_rows(R)) {
    k.pitch = ceil_div(R, 32) * 32;
    k.bytes = 4ll * k.pitch * V;
    if (R > H || V < 32768 || k.bytes > (256ll << 20)) return HeadKept{};
    return k;
  }
  const long long rpad = static_cast<long long>(ceil_div(R, kHeadRowPad)) * kHeadRowPad;
  k.pitch = ceil_div(V, kBN) * kBN;
  k.tiles = 2 * ceil_div(V, kBN);
  k.part_at = 2 * rpad * k.pitch;
  k.bytes = k.part_at + rpad * k.tiles * static_cast<long long>(sizeof(float2));
  return H >= 384 && k.part_at <= (2ll << 30) ? k : HeadKept{};
}

// Partial statistics per row: one a warp of the launch, or two a tile of columns.
int head_loss_vocab_tiles(int R, int V, bool kept) {
  return few_rows(R) ? 8 * pairs_for(ceil_div(V, 2 * lane_slot(V, kept ? 32 : 8))) : 2 * ceil_div(V, kBN);
}

// Row pitch or row count of the logits' gradient: [piece][few rows, in two halves] or
// [rows][piece].
int head_loss_grad_rows(int R) {
  return few_rows(R) ? 2 * ceil_div(R, 64) * 64 : ceil_div(R, kHeadRowPad) * kHeadRowPad;
}

// Columns of the logits that the backward pass works on at a time.  Their gradient takes two bytes a row and
// column: 256 MB of it, so that a pass over a piece is long against the ends of its two launches.
int head_loss_piece(int R, int V) {
  long long piece = (256ll << 20) / (2ll * head_loss_grad_rows(R)) / kBN * kBN;
  piece = std::max<long long>(piece, 4096);
  return static_cast<int>(std::min<long long>(piece, static_cast<long long>(ceil_div(V, kBN)) * kBN));
}

// Parts of the hidden gradient's reduction over a piece.  Next to the head gradient's items, which fill
// the pairs that it leaves idle, as few as keep one part from being longer than a pair's share of
// everything; alone, as many as give every pair the same work.
int head_loss_splits(int R, int H, int piece, int V, bool with_dw) {
  const int pairs = device_sms() / 2, cols = std::min(piece, V), kb = ceil_div(cols, kBK);
  const bool few = few_rows(R);
  const long long tiles = static_cast<long long>(few ? 1 : ceil_div(R, kBM)) * ceil_div(H, kBN);
  const long long kbw = std::max(ceil_div(R, kBK) * (few ? 2 : 1), 8);     // weights: see item_at
  const long long other = static_cast<long long>(ceil_div(cols, kBM)) * ceil_div(H, kBN) * kbw;
  const long long bytes = 4ll * ceil_div(R, kHeadRowPad) * kHeadRowPad * H;             // of one partial sum
  int best = 1;
  long long cost = LLONG_MAX;
  for (int want = 1; want <= pairs && want * 4 <= std::max(kb, 4) && (want == 1 || want * bytes <= (256ll << 20)); ++want) {
    if (want > 1 && tiles >= 2 * pairs) break;          // enough tiles as they are
    const int per = ceil_div(kb, want), splits = ceil_div(kb, per), weigh = few ? per + per / 2 : per;
    if (with_dw && weigh <= (tiles * weigh * splits + other) / pairs) return splits;
    // a tile's end weighs about four blocks, and a partial sum's way through memory a block per MB (few rows, whose blocks
    // wait for the head, per 3 MB): nearly equal rounds would otherwise take 21 parts for 5 of 192 x 3584
    const long long c = static_cast<long long>(ceil_div(tiles * splits, pairs)) * (per + 4) + splits * bytes / ((few ? 3ll : 1ll) << 20);
    if (c < cost) {
      cost = c;
      best = splits;
    }
  }
  return best;
}

cudaError_t head_loss_rows_launch(const HeadLossState& s, const HeadTargets& t, cudaStream_t stream) {
  cudaError_t e;
  if (s.divergence) {
    e = launch_pdl(teacher_rows_kernel, dim3(s.R), dim3(128), 0, stream, s, t);
    if (e != cudaSuccess) return e;
  }
  if (s.R <= kCountRows) return launch_pdl(few_rows_kernel, dim3(s.rpad), dim3(128), 0, stream, s, t);
  e = launch_pdl(compact_rows_kernel, dim3(1), dim3(1024), 0, stream, s, t);
  if (e != cudaSuccess) return e;
  return launch_pdl(gather_rows_kernel, dim3(s.rpad), dim3(128), 0, stream, s);
}

cudaError_t head_loss_forward_launch(const HeadLossState& s, const HeadStatsScratch& p, cudaStream_t stream) {
  Maps maps{};
  const bool few = few_rows(s.R);
  GemmArgs a = base_args(s);
  a.v0 = 0;
  a.cols = s.V;
  a.tiles_n = ceil_div(s.V, kBN);
  a.list_logit = s.list_logit;
  a.inv_temp = s.inv_temp;
  a.part = p.part;
  a.part_sum = p.part_sum;
  a.part_tiles = p.tiles;
  cut_sums(a, few);
  cudaError_t e;
  if (few) {
    a.kept = p.kept != nullptr;
    a.slot = lane_slot(s.V, a.kept ? 32 : 8);
    const int pitch = head_loss_kept(s.R, s.H, s.V).pitch;
    if (a.kept && !encode(&maps.out0, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, p.kept, s.V, pitch, pitch, 32, 32))
      return cudaErrorInvalidValue;
    if (!map_bf16(&maps.a0, s.w, s.V, s.H, s.ldw, kBK, a.slot) ||
        !map_bf16(&maps.b0, s.hc, s.rpad, s.H, s.H, kBK, a.bn / 2))
      return cudaErrorInvalidValue;
    const int items = ceil_div(s.V, 2 * a.slot);
    e = a.sums > 1 ? launch_gemm<kStats, true, true>(maps, a, items, stream) : launch_gemm<kStats, true>(maps, a, items, stream);
  } else {
    if (!map_bf16(&maps.a0, s.hc, s.rpad, s.H, s.H, kBK, kHalf) || !map_bf16(&maps.b0, s.w, s.V, s.H, s.ldw, kBK, kHalf))
      return cudaErrorInvalidValue;
    a.kept = p.kept != nullptr;
    const int pitch = head_loss_kept(s.R, s.H, s.V).pitch;
    if (a.kept && !map_bf16(&maps.out0, p.kept, s.rpad, pitch, pitch, 64, 32)) return cudaErrorInvalidValue;   // fp16
    const int items = ceil_div(s.R, kBM) * a.tiles_n;
    e = a.sums > 1 ? launch_gemm<kStats, false, true>(maps, a, items, stream) : launch_gemm<kStats, false>(maps, a, items, stream);
  }
  if (e != cudaSuccess) return e;
  return launch_pdl(finish_rows_kernel, dim3(s.R), dim3(128), 0, stream, s, p);
}

cudaError_t head_loss_backward_launch(const HeadLossState& s, const HeadGradArgs& g, cudaStream_t stream) {
  const bool dh = g.dh != nullptr, dw = g.dw != nullptr, few = few_rows(s.R);
  cudaError_t e = cudaSuccess;
  if (!few) e = launch_pdl(grad_rows_kernel, dim3(ceil_div(s.rpad, 4)), dim3(128), 0, stream, s, g);
  if (e != cudaSuccess) return e;
  Maps gm{}, pm{};
  GemmArgs base = base_args(s);
  base.piece = g.piece;
  base.list_grad = g.list_grad;
  base.row_coef = g.row_coef;
  base.s = s;
  base.g = g.g;
  base.do_dh = dh;
  base.do_dw = dw;
  base.splits = g.splits;
  const int slot = lane_slot(std::min(g.piece, s.V), 32), pitch = head_loss_grad_rows(s.R);
  bool ok = true;
  if (few) {
    if (g.kept == nullptr)
      ok = map_bf16(&gm.a0, s.w, s.V, s.H, s.ldw, kBK, slot) && map_bf16(&gm.b0, s.hc, s.rpad, s.H, s.H, kBK, base.bn / 2) &&
           map_bf16(&gm.out0, g.dl, g.piece, pitch, pitch, 64, 32);
    if (dh)
      ok = ok && map_bf16(&pm.a0, s.w, s.V, s.H, s.ldw, 64, kBK) &&
           map_bf16(&pm.b0, g.dl, g.piece, pitch, pitch, 64, kBK);
    if (dw) ok = ok && map_bf16(&pm.a1, g.dl, g.piece, pitch, pitch, kBK, kHalf);
  } else {
    if (g.kept == nullptr)
      ok = map_bf16(&gm.a0, s.hc, s.rpad, s.H, s.H, kBK, kHalf) && map_bf16(&gm.b0, s.w, s.V, s.H, s.ldw, kBK, kHalf) &&
           map_bf16(&gm.out0, g.dl, s.rpad, g.piece, g.piece, 64, 32);
    if (dh)
      ok = ok && map_bf16(&pm.a0, g.dl, s.rpad, g.piece, g.piece, kBK, kHalf) &&
           map_bf16(&pm.b0, s.w, s.V, s.H, s.ldw, 64, kBK);
    if (dw) ok = ok && map_bf16(&pm.a1, g.dl, s.rpad, g.piece, g.piece, 64, kBK);
  }
  if (dh)
    ok = ok && encode(&pm.out0, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, g.dh_part, static_cast<long long>(g.splits) * s.rpad,
                      s.H, s.H, 32, 32);
  if (dw)
    ok = ok && map_bf16(&pm.b1, s.hc, s.rpad, s.H, s.H, 64, kBK) && map_bf16(&pm.out1, g.dw, s.V, s.H, s.H, 64, 32);
  if (!ok) return cudaErrorInvalidValue;
  for (int v0 = 0; v0 < s.V; v0 += g.piece) {
    GemmArgs a = base;
    a.v0 = v0;
    a.cols = std::min(g.piece, s.V - v0);
    if (g.kept != nullptr && !few) {
      e = launch_pdl(kept_scale_kernel, dim3(s.rpad, ceil_div(a.cols, 8192)), dim3(256), 0, stream, s, g,
                     head_loss_kept(s.R, s.H, s.V), v0, a.cols);
    } else if (g.kept != nullptr) {
      const int blocks = std::min(2 * device_sms(), ceil_div(a.cols, 8));
      e = launch_pdl(kept_grad_kernel, dim3(blocks), dim3(256), 0, stream, s, g, head_loss_kept(s.R, s.H, s.V).pitch, pitch, a.lo, v0, a.cols);
      if (e == cudaSuccess && s.K > 1)
        e = launch_pdl(kept_listed_kernel, dim3(ceil_div(s.R, 4)), dim3(128), 0, stream, s, g, pitch, a.lo, v0, a.cols);
    } else if (few) {
      a.slot = slot;
      e = launch_gemm<kGrad, true>(gm, a, ceil_div(a.cols, 2 * slot), stream);
      a.slot = kHalf;
    } else {
      a.tiles_n = ceil_div(a.cols, kBN);
      e = launch_gemm<kGrad, false>(gm, a, ceil_div(s.R, kBM) * a.tiles_n, stream);
    }
    if (e != cudaSuccess) return e;
    a.tiles_n = ceil_div(s.H, kBN);
    a.first_piece = v0 == 0;
    const int items = (dh ? (few ? 1 : ceil_div(s.R, kBM)) * a.tiles_n * g.splits : 0) +
                      (dw ? ceil_div(a.cols, kBM) * a.tiles_n : 0);
    e = few ? launch_gemm<kProd, true>(pm, a, items, stream) : launch_gemm<kProd, false>(pm, a, items, stream);
    if (e != cudaSuccess) return e;
  }
  if (dh) {
    // reading the listed head rows again: 2 K H bytes a row, next to 4 or 6 H V operations at least; up to 256 rows the
    // products take as long as one row tile's
    const int mend = !few && s.K <= std::max(1, s.V / (s.R <= 256 ? 1024 : 4096));
    return launch_pdl(hidden_grad_kernel, dim3(s.R, ceil_div(s.H, 1024)), dim3(128), 0, stream, s, g, mend);
  }
  return cudaSuccess;
}

}  // namespace osb
