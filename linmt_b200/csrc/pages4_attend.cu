// pages4_attend.cu -- attention of a few query rows per sentence over a pool of 4-bit pages (linmt_attend_pages4).
//
//   out = sum_t softmax_t(f(scale q . k_t)) v_t,   k_t = sk (codes - 8), v_t = sv (codes - 8) by groups of 32 components
//
// A sentence's beams, and the query heads that share a head of the pool, read the same positions: up to 16 rows are the left
// operand of mma.m16n8k16, so every code is loaded and unpacked once for all of them.  (tcgen05.mma could have 128 positions on the left and the
// 16 rows as its N, but wants the codes unpacked and stored first, into shared memory or TMEM; the unpacking, not the product, is what takes the time.  Not built.)
//   Scales stay out of the products: a key's is multiplied onto its group's sum, a value's into the weight on the left.
//   A word's codes become matrix operands with one AND each: an integer in the low bits of an
//   fp16 number is a subnormal one, that integer times 2^-24, and stays so up to 2047, so every second
//   code may be left four bits up and its 16 taken out elsewhere (of the queries before, of the output's columns after).  What is then too much, 8 for each
//   code, goes off by a product of its own: the queries' sums with the keys' scales, and the weights' sums.  That is 5
//   instructions for 8 codes where a code minus 8 in normal form takes 11, in a kernel bound by what it can issue.  Queries are scaled to
//   fp16's upper range by a power of 2 for each row.  Weights are multiplied by their values' scales and rounded to fp16 (2^-11 each at most), with a power of 2
//   for each row that follows its largest such product, as the maximum follows the scores: what lies far below is rounded to 2^-26 of the largest (2^-21 where that has
//   fallen and the power has not followed yet).  A row's power follows from what it sees itself.  (One power for a warp's 16 rows that followed the largest scale and never
//   came back was quicker with windows, 78 not 83 us for 64 paragraphs of 1 to 4001 positions, and lost rows whose values are 2^20 below those of another row, or of
//   positions without weight.)
//   32-bit queries are two fp16 terms, and so are their weights: 2^-22 of each, or 2^-34 (2^-31) of the largest.  Their codes are made normal numbers less 8 (9
//   instructions for 8 codes): the matrix unit cuts addends off at a place that goes by their exponents, and subnormal operands lose up to 10 bits there, which
//   an output rounded to 16 bits does not see but one of 32 does (2^-14 of a scale was seen).  (Three bf16 terms of each, exact to 2^-24: 18 sentences of
//   6068 to 8725 positions with 10 beams and 28 heads of 64 in 168 us, not 155.)
// Every warp has a ring of tiles of its own (cp.async, no barrier among warps) and its own maximum and sums; the CTA's four are
// joined through shared memory at the end of a piece of work, and where a sentence's positions are shared by CTAs a second kernel joins those.
#include <cmath>

#include "device_ops.h"
#include "pages4.h"

namespace linmt {
namespace ops {
namespace {

constexpr int kWarps = 4;
constexpr int kPairStages = 2;     // pairs of tiles in a warp's ring (three: 2 % longer)
constexpr int kRows = 16;
constexpr float kLog2e = 1.4426950408889634f;

template <class T> constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;           // fp16 terms of a query and of a weight
template <class T> constexpr float kSlack = sizeof(T) == 4 ? 2.f : 8.f;     // the reference maximum follows the true one only when it lags by 2^8 (2^2): few tiles rescale the sums
template <class T> constexpr int kAbove = sizeof(T) == 4 ? 9 : 1;           // the largest weight times scale, in powers of 2 above 1
template <class T> constexpr int kRoom = sizeof(T) == 4 ? 3 : 5;            // and what a scale may be beside it, with a weight of up to 2^kSlack: 2^14 in all
template <class T> constexpr int kFall = sizeof(T) == 4 ? 3 : 5;            // and how far it falls before the power of 2 follows
template <class T> constexpr float kFallen = sizeof(T) == 4 ? 64.f : 0.0625f;      // 2^(kAbove - kFall)

struct AttendParams {
  const unsigned char* data;
  int64_t stride_page, stride_head;
  int32_t n_pages, pool_heads, page;
  const void* q;
  int64_t q_n, q_g, q_h;
  void* out;
  int64_t o_n, o_g, o_h;
  float* lse;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* len;
  const float* slope;
  const float* centre;
  const int32_t* first;
  const int32_t* last;
  float* ws;
  int32_t n, g, heads, rep, width, row_tiles, by_window;
  float scale, cap;
  float mul;                 // mul 2^mul_up = |scale| log2(e); with a cap times 2 / cap, and with one above kHugeCap times kHugeUp
  int32_t mul_up;
  int32_t q_wide, o_wide;    // the rows of q are 16-byte aligned; fours of components of out are aligned to their size
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// The products onto nothing.
__device__ __forceinline__ void mma_bf16_first(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ __nv_bfloat162 bf16_pair(uint32_t x) { return *reinterpret_cast<const __nv_bfloat162*>(&x); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Every second code of a word as matrix operands: `odd`, those four bits up.  16-bit queries: 0 .. 15 (odd: times 16) times 2^-24.  32-bit: less 8, in normal form.
template <class T>
__device__ __forceinline__ uint32_t operand(uint32_t word, bool odd) {
  const uint32_t v = word & (odd ? 0x00f000f0u : 0x000f000fu);
  if constexpr (sizeof(T) == 2) return v;
  const uint32_t up = v | 0x64006400u;      // 1024 more
  const __half2 x = *reinterpret_cast<const __half2*>(&up), y = odd ? __hfma2(x, __float2half2_rn(0.0625f), __float2half2_rn(-72.f)) : __hsub2(x, __float2half2_rn(1032.f));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ float bf16_low(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_high(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// cap tanh(x) as cap - 2 cap / (2^y + 1), y = 2 x log2(e): good to 3e-7 of the cap.  With a cap of up to kQuickCap that is 2e-5 of a score, which a 16-bit result does not
// see (2^-11 of a weight is rounded away besides); the difference of two such numbers has nothing left of scores that are small beside a cap of millions.
constexpr float kQuickCap = 64.f, kHugeCap = 1e30f, kHugeUp = 1.2676506002282294e30f;      // (the last: 2^100)
__device__ __forceinline__ float capped(float y, float cap) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(exp2_of(y) + 1.f));
  return fmaf(-2.f * cap, r, cap);
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The kernel behind this one may be launched now; it waits for this one's end before it reads (join's wait_for_last).
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Four components of row `at` of a sentence's head of the pool, and with the first the log of its weight.  A weight of 0:
// nothing was seen; of NaN (a query that is not finite): so are the row and the log.
template <class T>
__device__ __forceinline__ void write_row(const AttendParams& a, int sent, int kvh, int at, int d, const float4& sum, float top, float weight) {
  const int g = at / a.rep, h = kvh * a.rep + at - g * a.rep;
  const float f = weight == 0.f ? 0.f : 1.f / weight;
  T* const to = static_cast<T*>(a.out) + sent * a.o_n + g * a.o_g + h * a.o_h + d;
  struct alignas(4 * sizeof(T)) Four { T v[4]; };
  const Four v{{from_float<T>(sum.x * f), from_float<T>(sum.y * f), from_float<T>(sum.z * f), from_float<T>(sum.w * f)}};
  if (a.o_wide) {
    *reinterpret_cast<Four*>(to) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = v.v[i];
  }
  if (d == 0 && a.lse) a.lse[((int64_t)sent * a.g + g) * a.heads + h] = weight == 0.f ? -INFINITY : (top + log2f(weight)) * 0.69314718055994531f;
}

// ---- who does what
//
// The work is a list of pairs of tiles (32 positions): sentence by sentence, in each by head of the pool and row tile (a segment), a segment's
// pairs in order, from the first that a row of the sentence sees to the last (where there are windows, and not so many that looking at them takes
// longer than the pairs that they leave out).  It is cut into as many equal parts as CTAs fit on the GPU at once, each of at least kLeast pairs: a segment
// longer than a part is then shared by several CTAs, whose parts the join kernel adds up, and a CTA may have several short ones.  Lengths
// are known on the device only, so every CTA adds them up itself.  A segment counts as kFixed units more than it has pairs, its fixed costs being as large,
// and as kLeast at least; one of up to kLeast + kFixed units or an eighth of a part is not cut: the CTA that has its first unit takes it whole.
constexpr int kLeast = 8;
constexpr int kFixed = 12;      // (64 paragraphs of 1 to 4001 positions: 91, 87, 83, 84, 85, 87 us with 8, 10, 12, 14, 16, 20)
struct Share {
  int64_t begin, end;      // the CTA's units
  int64_t first;           // number of the first unit of sentence `sent`
  int64_t per;             // units of a part
  int sent, whole;         // sentence of `begin`; segments of up to `whole` units are not cut
};
__device__ __forceinline__ int length_of(const AttendParams& a, int sent) {
  return min(max(__ldg(a.len + sent), 0), (int)min((int64_t)a.width * a.page, (int64_t)0x7fffffff - 64));
}
// The pairs of a sentence that any of its rows sees, from pair `from` on, and the units that they count; `a.by_window`: its rows are few enough to look at.
struct Seen { int from, pairs, units; };
__device__ __forceinline__ Seen seen_between(int lo, int hi) {
  if (lo >= hi) return {0, 0, kLeast};
  const int pairs = (hi + 31) / 32 - lo / 32;
  return {lo / 32, pairs, max(kLeast, pairs + kFixed)};
}
__device__ __forceinline__ Seen seen_of(const AttendParams& a, int sent) {             // by one thread
  const int len = length_of(a, sent);
  if (!a.by_window) return seen_between(0, len);
  int lo = 0x7fffffff, hi = 0;
#pragma unroll 4
  for (int g = 0; g < a.g; ++g) {
    const int f = max(__ldg(a.first + (int64_t)sent * a.g + g), 0), l = min(__ldg(a.last + (int64_t)sent * a.g + g), len);
    if (f < l) { lo = min(lo, f); hi = max(hi, l); }
  }
  return seen_between(lo, hi);
}
__device__ __forceinline__ Seen seen_by_warp(const AttendParams& a, int sent) {        // by a warp
  const int len = length_of(a, sent);
  if (!a.by_window) return seen_between(0, len);
  int lo = 0x7fffffff, hi = 0;
  for (int g = threadIdx.x & 31; g < a.g; g += 32) {
    const int f = max(__ldg(a.first + (int64_t)sent * a.g + g), 0), l = min(__ldg(a.last + (int64_t)sent * a.g + g), len);
    if (f < l) { lo = min(lo, f); hi = max(hi, l); }
  }
  return seen_between(__reduce_min_sync(~0u, lo), __reduce_max_sync(~0u, hi));
}

// Share of block `blockIdx.x` of `blocks`; all threads of the CTA (a multiple of 32, at most 512) call it.  The sentences are added up by all
// threads, then those of the thread that has the first pair, until one is left.
__device__ __forceinline__ Share share_of(const AttendParams& a, int blocks) {
  __shared__ int64_t sums[16], found_first;
  __shared__ int found_lo, found_hi;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, segments = a.pool_heads * a.row_tiles;
  Share s{};
  int lo = 0, hi = a.n;
  bool all = true;
  for (;;) {
    const int each = (hi - lo + threads - 1) / threads, i0 = min(hi, lo + tid * each), i1 = min(hi, i0 + each);
    int64_t mine = 0;
#pragma unroll 8
    for (int i = i0; i < i1; ++i) mine += seen_of(a, i).units;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int64_t total = 0;
    for (int w = 0; w < threads / 32; ++w) {
      if (w == warp) upto += total;
      total += sums[w];
    }
    if (all) {
      all = false;
      total *= segments;
      s.per = max((int64_t)kLeast, (total + blocks - 1) / blocks);
      s.begin = min(total, blockIdx.x * s.per);
      s.end = min(total, s.begin + s.per);
      s.whole = (int)min((int64_t)0x7fffffff, max((int64_t)(kLeast + kFixed), s.per / 8));
    }
    if (s.begin >= s.end) return s;
    const int64_t before = s.first + (upto - mine) * segments;
    if (s.begin >= before && s.begin < s.first + upto * segments) {
      found_first = before;
      found_lo = i0;
      found_hi = i1;
    }
    __syncthreads();
    s.first = found_first;
    lo = found_lo;
    hi = found_hi;
    if (hi - lo == 1) break;
    __syncthreads();                     // (before these are written again)
  }
  s.sent = lo;
  return s;
}

// One CTA's piece of a segment.
struct Piece {
  int sent, kvh, rt;
  int u0, u1, units;       // units u0 .. u1 - 1 of the segment's
  int64_t start;           // number of the segment's first unit
  int from, fixed;         // unit u >= fixed is the pair of positions 32 (from + u - fixed) on
  __device__ __forceinline__ bool whole() const { return u0 == 0 && u1 == units; }
};
// The piece that begins at s.begin; false where the CTA has none left.  Moves s on behind it.  All lanes of a warp call it.
__device__ __forceinline__ bool next_piece(const AttendParams& a, Share& s, Piece& p) {
  const int segments = a.pool_heads * a.row_tiles;
  while (s.begin < s.end) {
    const Seen seen = seen_by_warp(a, s.sent);
    p.units = seen.units;
    p.from = seen.from;
    p.fixed = seen.units - seen.pairs;
    const int64_t in = s.begin - s.first, seg = in >> 32 ? in / p.units : (int64_t)((uint32_t)in / (uint32_t)p.units);
    if (seg >= segments) {
      s.first += (int64_t)p.units * segments;
      ++s.sent;
      continue;
    }
    p.sent = s.sent;
    p.kvh = (int)seg / a.row_tiles;
    p.rt = (int)seg - p.kvh * a.row_tiles;
    p.start = s.first + seg * p.units;
    p.u0 = (int)(s.begin - p.start);
    p.u1 = (int)min((int64_t)p.units, s.end - p.start);
    s.begin = p.start + p.u1;
    if (p.units <= s.whole) {
      s.begin = p.start + p.units;
      if (p.u0 > 0) continue;            // the CTA before has all of it
      p.u1 = p.units;
    }
    return true;
  }
  return false;
}

template <class T, int D>
constexpr int attend_smem() {
  return kWarps * kPairStages * 2 * 18 * D + kTerms<T> * (D / 16) * 512;
}

// What a piece's rows see.
struct Job {
  int n_rows;
  int lo[2], hi[2];            // the lane's rows gid and gid + 8
  float slope[2], centre[2];   // their bias, in powers of 2
  int all_lo, all_hi;          // what all of them see
  int t0, t1;                  // the piece's tiles
};

template <class T>
__device__ __forceinline__ Job job_of(const AttendParams& a, const Piece& p, const T* (&q_row)[2]) {
  Job j;
  const int gid = (threadIdx.x & 31) >> 2, len = length_of(a, p.sent);
  j.n_rows = min(kRows, a.g * a.rep - p.rt * kRows);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = gid + 8 * i, at = p.rt * kRows + r, g = at / a.rep, h = p.kvh * a.rep + at - g * a.rep;
    const bool have = r < j.n_rows;
    q_row[i] = have ? static_cast<const T*>(a.q) + p.sent * a.q_n + g * a.q_g + h * a.q_h : nullptr;
    j.lo[i] = have ? (a.first ? max(__ldg(a.first + (int64_t)p.sent * a.g + g), 0) : 0) : 0x7fffffff;
    j.hi[i] = have ? (a.last ? min(__ldg(a.last + (int64_t)p.sent * a.g + g), len) : len) : 0;
    j.slope[i] = have && a.slope ? __ldg(a.slope + h) * kLog2e : 0.f;
    j.centre[i] = have && a.slope ? __ldg(a.centre + (int64_t)p.sent * a.g + g) : 0.f;
  }
  int any_lo = j.lo[0] < j.hi[0] ? j.lo[0] : 0x7fffffff, any_hi = j.lo[0] < j.hi[0] ? j.hi[0] : 0;
  if (j.lo[1] < j.hi[1]) { any_lo = min(any_lo, j.lo[1]); any_hi = max(any_hi, j.hi[1]); }
  j.all_lo = gid < j.n_rows ? j.lo[0] : 0;
  j.all_hi = gid < j.n_rows ? j.hi[0] : 0x7fffffff;
  if (gid + 8 < j.n_rows) { j.all_lo = max(j.all_lo, j.lo[1]); j.all_hi = min(j.all_hi, j.hi[1]); }
  any_lo = __reduce_min_sync(~0u, any_lo);
  any_hi = __reduce_max_sync(~0u, any_hi);
  j.all_lo = __reduce_max_sync(~0u, j.all_lo);
  j.all_hi = __reduce_min_sync(~0u, j.all_hi);
  const bool any = any_lo < any_hi;
  j.t0 = max(2 * (p.from + max(p.u0 - p.fixed, 0)), any ? any_lo / pages4::kTile & ~1 : 0);
  j.t1 = max(j.t0, min(2 * (p.from + max(p.u1 - p.fixed, 0)), any ? (any_hi - 1) / pages4::kTile + 1 : 0));
  return j;
}

// The CTA's warps' parts, joined and written: sums o (o[group][e][2 r + i] = row gid + 8 r, component 32 group + 8 c + 4 i + e), relative to 2^m, and weights l.
template <class T, int D>
__device__ __forceinline__ void join_warps(const AttendParams& a, const Piece& p, const Job& job, unsigned char* smem, const float (&o)[D / 32][4][4], const float (&m)[2], float (&l)[2]) {
  constexpr int NG = D / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, c = lane & 3;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(~0u, l[e], 1);
    l[e] += __shfl_xor_sync(~0u, l[e], 2);
  }
  copy_wait<0>();
  __syncthreads();                    // the rings are free
  float* const part = reinterpret_cast<float*>(smem);              // [warp][row][D]
  __shared__ float part_m[kWarps][kRows], part_l[kWarps][kRows];
  if (c == 0) {
    part_m[warp][gid] = m[0]; part_m[warp][gid + 8] = m[1];
    part_l[warp][gid] = l[0]; part_l[warp][gid + 8] = l[1];
  }
#pragma unroll
  for (int gr = 0; gr < NG; ++gr)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float4* const to = reinterpret_cast<float4*>(part + (warp * kRows + gid + 8 * r) * D + 32 * gr + 8 * c);
      to[0] = make_float4(o[gr][0][2 * r], o[gr][1][2 * r], o[gr][2][2 * r], o[gr][3][2 * r]);
      to[1] = make_float4(o[gr][0][2 * r + 1], o[gr][1][2 * r + 1], o[gr][2][2 * r + 1], o[gr][3][2 * r + 1]);
    }
  __syncthreads();
  const bool whole = p.whole();
  // a part of the workspace: [row][D] sums, [row] maximum, [row] weight.  A CTA's first is of the segment that it has from the CTA before, its second
  // of the one that the next CTA goes on with.
  float* const ws = a.ws + ((int64_t)blockIdx.x * 2 + (p.u0 == 0)) * (kRows * (D + 2));
  const int d = tid % (D / 4) * 4;
  for (int r = tid / (D / 4); r < job.n_rows; r += kWarps * 32 / (D / 4)) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part_m[w][r]);
    const float base = top == -INFINITY ? 0.f : top;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float weight = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2_of(part_m[w][r] - base);
      const float4 v = *reinterpret_cast<const float4*>(part + (w * kRows + r) * D + d);
      sum.x += f * v.x; sum.y += f * v.y; sum.z += f * v.z; sum.w += f * v.w;
      weight += f * part_l[w][r];
    }
    if (whole) {
      write_row<T>(a, p.sent, p.kvh, p.rt * kRows + r, d, sum, top, weight);
    } else {
      *reinterpret_cast<float4*>(ws + r * D + d) = sum;
      if (d == 0) { ws[kRows * D + r] = top; ws[kRows * D + kRows + r] = weight; }
    }
  }
  __syncthreads();                    // (before the next piece's tiles come in)
}

// What is done to scores.  kPlain: no cap, no bias, and a scale: they are products times mul.  kQuick: caps of up to kQuickCap for 16-bit queries.  kExact: tanhf.
enum Scores { kPlain, kQuick, kExact };
template <class T, int D, Scores HOW>
__global__ void __launch_bounds__(kWarps * 32, D == 64 ? 4 : 3) attend_kernel(const __grid_constant__ AttendParams a) {
  constexpr int NG = D / 32, kTileBytes = pages4::tile_bytes(D), QT = kTerms<T>, PT = kTerms<T>;
  constexpr bool kOver = sizeof(T) == 2;      // codes are operands as they are: 8 for each, and every second's 16, come off apart
  extern __shared__ __align__(16) unsigned char smem[];
  launch_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, c = lane & 3;
  Share share = share_of(a, gridDim.x);
  Piece piece;
  int4 ends = make_int4(-1, 0, 0, 0);      // for the join: the segment that ends here and began in a CTA before, and which
  while (next_piece(a, share, piece)) {
    if (piece.u0 > 0 && piece.u1 == piece.units) ends = make_int4(piece.sent, piece.kvh, piece.rt, (int)(piece.start / share.per));
    const T* q_row[2];
    const Job job = job_of<T>(a, piece, q_row);

    unsigned char* const ring = smem + warp * kPairStages * 2 * kTileBytes;
    uint4* const q_smem = reinterpret_cast<uint4*>(smem + kWarps * kPairStages * 2 * kTileBytes);
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    const int32_t* const table = a.table + piece.sent * a.table_stride;
    const unsigned char* const head = a.data + piece.kvh * a.stride_head;
    const int tiles_per_page = a.page / pages4::kTile;
    const int pairs = (job.t1 - job.t0 + 1) / 2, mine = pairs > warp ? (pairs - warp + kWarps - 1) / kWarps : 0;      // this warp's: warp + kWarps i

    // Where this warp's tiles are: looked up 32 at a time, one by each lane.
    int64_t where = -1;
    uint32_t bad = 0;                // bits of a stage: no tile of the pool
    int fetch_stage = 0;
    auto fetch = [&](int i) {
      if ((i & 15) == 0) {
        const int t = job.t0 + 2 * (warp + kWarps * (i + (lane >> 1))) + (lane & 1);
        where = i + (lane >> 1) < mine && t < job.t1 ? pages4::tile_offset(table, t, tiles_per_page, a.n_pages, a.stride_page, D) : -1;
      }
      const int64_t at0 = __shfl_sync(~0u, where, 2 * (i & 15)), at1 = __shfl_sync(~0u, where, 2 * (i & 15) + 1);
      const int stage = fetch_stage;
      fetch_stage = fetch_stage + 1 == kPairStages ? 0 : fetch_stage + 1;
      bad &= ~(3u << (2 * stage));
      if (i >= mine || at0 < 0) bad |= 1u << (2 * stage);
      if (i >= mine || at1 < 0) bad |= 2u << (2 * stage);
      if (i < mine) {
        const uint32_t to = ring_at + stage * 2 * kTileBytes + lane * 16;
        const unsigned char *const from0 = head + at0 + lane * 16, *const from1 = head + at1 + lane * 16;
        constexpr int kWhole = kTileBytes / 512, kRest = (kTileBytes % 512) / 16;      // D = 128: four of 32 lanes and one of 16 for each tile; 64: two and one of 8
        if (at0 >= 0) {
#pragma unroll
          for (int b = 0; b < kWhole; ++b) copy16(to + b * 512, from0 + b * 512);
          if (lane < kRest) copy16(to + kWhole * 512, from0 + kWhole * 512);
        }
        if (at1 >= 0) {
#pragma unroll
          for (int b = 0; b < kWhole; ++b) copy16(to + kTileBytes + b * 512, from1 + b * 512);
          if (lane < kRest) copy16(to + kTileBytes + kWhole * 512, from1 + kWhole * 512);
        }
      }
      copy_commit();
    };
    float x[2][8];                   // the lane's part of two rows of queries: on its way while the table is looked at
    if (warp < NG) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (q_row[r] && a.q_wide) {
          uint4 v[sizeof(T) / 2];
#pragma unroll
          for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(q_row[r] + 32 * warp + 8 * c) + i);
          const T* e = reinterpret_cast<const T*>(v);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[r][i] = to_float(e[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[r][i] = q_row[r] ? to_float(q_row[r][32 * warp + 8 * c + i]) : 0.f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kPairStages - 1; ++i) fetch(i);

    // Queries as left operands in fp16: step (group, half) takes components 32 group + 8 c + 2 half + {0, 4 | 1, 5}, the latter over 16.  A row is scaled
    // so that its largest component is 2^9 to 2^10; what a group's codes carry too much, 8 times the sum of its components, in three bf16
    // terms for a product with the keys' scales: place k of it belongs to group k % 4, term k / 4.  A warp prepares one group.
    uint4 over;
    float mul[2];                  // from a sum of products to a power of 2 (or, with a cap, to what capped() takes)
    {
      __shared__ float s_most[NG][kRows], s_sum[4][kRows];
      if (warp < NG) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float most = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[r][i]));
          most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
          most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
          if (c == 0) s_most[warp][gid + 8 * r] = most;
        }
      } else if (c == 0) {         // (64 components: groups 2 and 3 are none)
        s_sum[warp][gid] = s_sum[warp][gid + 8] = 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float most = s_most[0][gid + 8 * r];
#pragma unroll
        for (int gr = 1; gr < NG; ++gr) most = fmaxf(most, s_most[gr][gid + 8 * r]);
        const int up = most > 0.f && most < INFINITY ? 9 - max(-100, ilogbf(most)) : 0;      // -118 .. 109
        const float by = ldexpf(a.scale < 0.f ? -1.f : 1.f, up);
        mul[r] = ldexpf(a.mul, a.mul_up + (kOver ? 24 : 0) - up);
        if (HOW == kPlain) mul[r] = fmaxf(mul[r], 1.4e-45f);      // (not 0: what is not seen is -inf times this)
        if (warp < NG) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float lo = x[r][i] * by * (kOver && (i & 1) ? 0.0625f : 1.f), hi = x[r][i + 4] * by * (kOver && (i & 1) ? 0.0625f : 1.f);
#pragma unroll
            for (int term = 0; term < QT; ++term) {
              const __half2 h = __floats2half2_rn(lo, hi);
              reinterpret_cast<uint32_t*>(q_smem + (term * NG * 2 + 2 * warp + (i >> 1)) * 32 + lane)[2 * (i & 1) + r] = *reinterpret_cast<const uint32_t*>(&h);
              const float2 back = __half22float2(h);
              sum += (back.x + back.y) * (i & 1 ? 16.f : 1.f);
              lo -= back.x;
              hi -= back.y;
            }
          }
          if constexpr (kOver) {
            sum += __shfl_xor_sync(~0u, sum, 1);
            sum += __shfl_xor_sync(~0u, sum, 2);
            if (c == 0) s_sum[warp][gid + 8 * r] = sum * (-8.f / 16777216.f);
          }
        }
      }
      __syncthreads();
      if constexpr (kOver) {
        uint32_t ov[2][2];
  #pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float s0 = s_sum[2 * (c & 1)][gid + 8 * r], s1 = s_sum[2 * (c & 1) + 1][gid + 8 * r];
  #pragma unroll
          for (int h = 0; h < 2; ++h) {          // terms c / 2 and 2 + c / 2
            float u0 = s0, u1 = s1;
            const int term = 2 * h + (c >> 1);
  #pragma unroll
            for (int i = 0; i < 2; ++i)
              if (i < term) {
                u0 -= __bfloat162float(__float2bfloat16_rn(u0));
                u1 -= __bfloat162float(__float2bfloat16_rn(u1));
              }
            ov[r][h] = term < 3 ? pack_bf16(u0, u1) : 0u;
          }
        }
        over = make_uint4(ov[0][0], ov[1][0], ov[0][1], ov[1][1]);
      }
    }
    // A cap near the largest 32-bit number: its product with log2(e), and one over it, are kept within the normal ones by a power of 2 each.
    const bool huge = HOW == kExact && a.cap > kHugeCap;
    const float cap_by = huge ? 256.f : 1.f, cap_log2 = a.cap / cap_by * kLog2e, tanh_by = 0.5f / kLog2e * (huge ? 1.f / kHugeUp : 1.f);

    // The values' sums are kept times 2^-24 where the codes are, and times a power of 2 for each row that brings its weights times scales into fp16's range.
    float o[NG][4][4] = {}, extra[4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, size[2] = {0.f, 0.f};   // size: that power; 0: the row has none yet
    uint32_t limit = 0xffffu;        // bits of the bf16 that no scale reaches whose weights are in range for certain, whatever they are
    int stage = 0;
    for (int i = 0; i < mine; ++i) {
      copy_wait<kPairStages - 2>();
      __syncwarp();                       // every lane's part of pair i is there, and pair i - 1 has been read by all
      fetch(i + kPairStages - 1);
      const unsigned char* const pair = ring + stage * 2 * kTileBytes;
      const uint32_t gone = (bad >> (2 * stage)) & 3;
      stage = stage + 1 == kPairStages ? 0 : stage + 1;
      if (gone == 3) continue;
      const int pos = (job.t0 + 2 * (warp + kWarps * i)) * pages4::kTile;

      // scores: x[j][0..3] = rows gid, gid, gid + 8, gid + 8 at positions pos + 8 j + 2 c + {0, 1, 0, 1}
      float x[4][4];
      uint32_t w[4][NG], sc[4][NG];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned char* const tile = pair + (j >> 1) * kTileBytes;
        const int j1 = j & 1;
        const unsigned char* const kw = tile + (8 * j1 + gid) * (D / 2) + c * (4 * NG);
        const unsigned char* const ks = tile + pages4::key_scales(D) + (8 * j1 + 2 * c) * (2 * NG);
        if constexpr (NG == 4) {
          *reinterpret_cast<uint4*>(w[j]) = *reinterpret_cast<const uint4*>(kw);
          *reinterpret_cast<uint4*>(sc[j]) = *reinterpret_cast<const uint4*>(ks);
        } else {
          *reinterpret_cast<uint2*>(w[j]) = *reinterpret_cast<const uint2*>(kw);
          *reinterpret_cast<uint2*>(sc[j]) = *reinterpret_cast<const uint2*>(ks);
        }
        if constexpr (kOver) {
          const uint32_t own = *reinterpret_cast<const uint32_t*>(tile + pages4::key_scales(D) + (8 * j1 + gid) * (2 * NG) + (NG == 4 ? 4 * (c & 1) : 0));
          mma_bf16_first(x[j], over, own, own);
        } else {
          x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
        }
      }
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        uint4 qa[QT], qb[QT];
#pragma unroll
        for (int term = 0; term < QT; ++term) {
          qa[term] = q_smem[(term * NG * 2 + 2 * gr) * 32 + lane];
          qb[term] = q_smem[(term * NG * 2 + 2 * gr + 1) * 32 + lane];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float s[4];
          const uint32_t even0 = operand<T>(w[j][gr], false), odd0 = operand<T>(w[j][gr], true), even1 = operand<T>(w[j][gr] >> 8, false), odd1 = operand<T>(w[j][gr] >> 8, true);
          mma_f16_first(s, qa[QT - 1], even0, odd0);         // small terms first
          mma_f16(s, qb[QT - 1], even1, odd1);
          if constexpr (QT == 2) {
            mma_f16(s, qa[0], even0, odd0);
            mma_f16(s, qb[0], even1, odd1);
          }
          // scales of position 2 c: halves gr of the first NG, of 2 c + 1: of the second
          const float s0 = gr & 1 ? bf16_high(sc[j][gr >> 1]) : bf16_low(sc[j][gr >> 1]);
          const float s1 = gr & 1 ? bf16_high(sc[j][NG / 2 + (gr >> 1)]) : bf16_low(sc[j][NG / 2 + (gr >> 1)]);
          x[j][0] = fmaf(s[0], s0, x[j][0]);
          x[j][1] = fmaf(s[1], s1, x[j][1]);
          x[j][2] = fmaf(s[2], s0, x[j][2]);
          x[j][3] = fmaf(s[3], s1, x[j][3]);
        }
      }
      float r0 = mul[0], r1 = mul[1];
      if constexpr (HOW != kPlain) {
        const float at0 = (float)(pos + 2 * c) - job.centre[0], at1 = (float)(pos + 2 * c) - job.centre[1];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = x[j][e] * (e < 2 ? r0 : r1);
            if (a.cap > 0.f) v = HOW == kExact ? cap_log2 * tanhf(v * tanh_by) * cap_by : capped(v, cap_log2);
            if (a.slope) v = fmaf(-job.slope[e >> 1], fabsf((e < 2 ? at0 : at1) + (float)(8 * j + (e & 1))), v);
            x[j][e] = v;
          }
        r0 = r1 = 1.f;
      }
      const bool edge = gone || pos < job.all_lo || pos + 2 * pages4::kTile > job.all_hi;
      if (edge) {
        const int from0 = pos + 2 * c - job.lo[0], from1 = pos + 2 * c - job.lo[1];
        const uint32_t n0 = job.lo[0] < job.hi[0] ? job.hi[0] - job.lo[0] : 0, n1 = job.lo[1] < job.hi[1] ? job.hi[1] - job.lo[1] : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((uint32_t)((e < 2 ? from0 : from1) + 8 * j + (e & 1)) >= (e < 2 ? n0 : n1)) x[j][e] = -INFINITY;
        if (gone) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if ((gone >> (j >> 1)) & 1) x[j][e] = -INFINITY;
        }
      }
      float top[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[e] = fmaxf(fmaxf(fmaxf(x[0][2 * e], x[0][2 * e + 1]), fmaxf(x[1][2 * e], x[1][2 * e + 1])), fmaxf(fmaxf(x[2][2 * e], x[2][2 * e + 1]), fmaxf(x[3][2 * e], x[3][2 * e + 1])));
        top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], 1));
        top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], 2));
        top[e] *= e ? r1 : r0;
      }
      const bool up0 = top[0] > m[0] + kSlack<T> || (m[0] == -INFINITY && top[0] > -INFINITY), up1 = top[1] > m[1] + kSlack<T> || (m[1] == -INFINITY && top[1] > -INFINITY);
      float down[2] = {1.f, 1.f};           // what a row's sums are to be multiplied by (the first positions find sums of 0)
      if (__any_sync(~0u, up0 || up1)) {
        if (up0) { down[0] = m[0] == -INFINITY ? 1.f : exp2_of(m[0] - top[0]); m[0] = top[0]; }
        if (up1) { down[1] = m[1] == -INFINITY ? 1.f : exp2_of(m[1] - top[1]); m[1] = top[1]; }
        l[0] *= down[0];
        l[1] *= down[1];
      }

      // values' scales of the lane's positions, two words for each of the four
      uint32_t vs[4][NG];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned char* const at = pair + (j >> 1) * kTileBytes + pages4::value_scales(D) + (8 * (j & 1) + 2 * c) * (2 * NG);
        if constexpr (NG == 4) *reinterpret_cast<uint4*>(vs[j]) = *reinterpret_cast<const uint4*>(at);
        else *reinterpret_cast<uint2*>(vs[j]) = *reinterpret_cast<const uint2*>(at);
      }
      // A row's power of 2 takes the largest weight times scale that it sees to 2^kAbove and up to twice that.  It goes down when one would come to 2^15, which a scale of
      // 2^kRoom times the largest may, and up with the maximum (by no more than that takes off the sums) when the largest has fallen to 2^-kFall of that: large values of
      // positions that hardly count, or no longer, and of such as another row sees, take nothing from it.  It follows from the row's own weights and scales alone; the
      // scales' extremes, of all that the lane's rows may see, only tell when to look.
      bool look = false;
      if (__any_sync(~0u, up0 || up1)) {
        const int smaller = (int)(min(up0 ? __float_as_uint(size[0]) : ~0u, up1 ? __float_as_uint(size[1]) : ~0u) >> 23);      // (0: a row's first positions)
        look = __any_sync(~0u, smaller == 0);
        if (!look) {
          __nv_bfloat162 least2 = __habs2(bf16_pair(vs[0][0]));
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i2 = 0; i2 < NG; ++i2) least2 = __hmin2(least2, __habs2(bf16_pair(vs[j][i2])));
          const uint32_t least = min(*reinterpret_cast<const uint32_t*>(&least2) & 0xffffu, *reinterpret_cast<const uint32_t*>(&least2) >> 16);
          look = (int)(least >> 7) <= 254 + kAbove<T> - kFall<T> - smaller;
        }
      }
      if (edge) {            // a position that the lane's rows do not see may hold anything: 0 times its scale has to be 0
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (x[j][e] == -INFINITY && x[j][e + 2] == -INFINITY) {
#pragma unroll
              for (int i2 = 0; i2 < NG / 2; ++i2) vs[j][e * (NG / 2) + i2] = 0u;
            }
      }
      __nv_bfloat162 most2 = __habs2(bf16_pair(vs[0][0]));
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i2 = 0; i2 < NG; ++i2) most2 = __hmax2(most2, __habs2(bf16_pair(vs[j][i2])));
      const uint32_t most = max(*reinterpret_cast<const uint32_t*>(&most2) & 0xffffu, *reinterpret_cast<const uint32_t*>(&most2) >> 16);
      const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j][0] = exp2_of(fmaf(x[j][0], r0, -m0));
        x[j][1] = exp2_of(fmaf(x[j][1], r0, -m0));
        x[j][2] = exp2_of(fmaf(x[j][2], r1, -m1));
        x[j][3] = exp2_of(fmaf(x[j][3], r1, -m1));
        l[0] += x[j][0] + x[j][1];
        l[1] += x[j][2] + x[j][3];
      }
      if (__any_sync(~0u, look || most >= limit)) {
        limit = 0xffffu;
        __nv_bfloat162 product2[2] = {bf16_pair(0u), bf16_pair(0u)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t of[2];                        // largest scales of the two positions, by even and odd groups
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            __nv_bfloat162 at = __habs2(bf16_pair(vs[j][e * (NG / 2)]));
            if constexpr (NG == 4) at = __hmax2(at, __habs2(bf16_pair(vs[j][2 * e + 1])));
            of[e] = *reinterpret_cast<const uint32_t*>(&at);
          }
          const __nv_bfloat162 largest = __hmax2(bf16_pair(__byte_perm(of[0], of[1], 0x5410)), bf16_pair(__byte_perm(of[0], of[1], 0x7632)));
#pragma unroll
          for (int r = 0; r < 2; ++r) product2[r] = __hmax2(product2[r], __hmul2(__floats2bfloat162_rn(x[j][2 * r], x[j][2 * r + 1]), largest));
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const bool up = r ? up1 : up0;
          float product = fmaxf(__low2float(product2[r]), __high2float(product2[r]));
          product = fmaxf(product, __shfl_xor_sync(~0u, product, 1));      // (the row's four lanes)
          product = fmaxf(product, __shfl_xor_sync(~0u, product, 2));
          const float scaled = product * size[r];
          const bool anew = size[r] == 0.f || scaled >= 32768.f;
          const int was = (int)(__float_as_uint(size[r]) >> 23);
          if (product > 0.f && (anew || (up && scaled < kFallen<T>))) {
            int now = kAbove<T> + 254 - min(max((int)(__float_as_uint(product) >> 23), 127 - 97), 127 + 99);
            if (!anew) now = max(was, min(now, was + 126 - (int)(__float_as_uint(down[r]) >> 23)));
            if (was) down[r] *= __uint_as_float((uint32_t)max(127 + now - was, 0) << 23);
            size[r] = __uint_as_float((uint32_t)now << 23);
          }
          // (a row that has seen scales of 0 only waits for another)
          if (size[r] != 0.f) limit = min(limit, (uint32_t)min(254 + kAbove<T> + kRoom<T> - (int)(__float_as_uint(size[r]) >> 23), 255) << 7);
          else if (m[r] != -INFINITY) limit = 1u;
        }
      }
      if (__any_sync(~0u, down[0] != 1.f || down[1] != 1.f)) {
        extra[0] *= down[0]; extra[2] *= down[1];
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[gr][e][0] *= down[0]; o[gr][e][1] *= down[0];
            o[gr][e][2] *= down[1]; o[gr][e][3] *= down[1];
          }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] *= size[e >> 1];

      // out += weights . values, a group of 32 components a time: its scales go into the weights
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
        for (int i2 = 0; i2 < NG / 2; ++i2) {
          const uint4 u = *reinterpret_cast<const uint4*>(pair + tt * kTileBytes + pages4::value_codes(D) + 16 * (i2 * 32 + lane));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int gr = 2 * i2 + h;
            const uint32_t w0 = h ? u.y : u.x, w1 = h ? u.w : u.z;
            uint32_t pa[PT][2][2];   // [term][half of the positions][row gid, row gid + 8]
#pragma unroll
            for (int j1 = 0; j1 < 2; ++j1) {
              const int j = 2 * tt + j1;
              const float s0 = h ? bf16_high(vs[j][i2]) : bf16_low(vs[j][i2]), s1 = h ? bf16_high(vs[j][NG / 2 + i2]) : bf16_low(vs[j][NG / 2 + i2]);
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                float p0 = x[j][2 * r] * s0, p1 = x[j][2 * r + 1] * s1;
#pragma unroll
                for (int term = 0; term < PT; ++term) {
                  pa[term][j1][r] = pack_f16(p0, p1);
                  if (term + 1 < PT) {
                    const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&pa[term][j1][r]));
                    p0 -= back.x;
                    p1 -= back.y;
                  }
                }
              }
            }
            const uint32_t eight = (gid >> 1) == gr ? 0x00080008u : 0u;       // columns 2 gr and 2 gr + 1: 8 times the weights' sum
#pragma unroll
            for (int term = PT - 1; term >= 0; --term) {
              const uint4 weights = make_uint4(pa[term][0][0], pa[term][0][1], pa[term][1][0], pa[term][1][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) mma_f16(o[gr][e], weights, operand<T>(w0 >> (e & 2) * 4, e & 1), operand<T>(w1 >> (e & 2) * 4, e & 1));
              if constexpr (kOver) mma_f16(extra, weights, eight, eight);
            }
          }
        }
      }
    }

    // From the sums as they are kept to sums of values: times 1 / size, and with codes as they are less 8 for each and times 2^24.  (A row without a size has sums of 0.)
    float by[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) by[r] = size[r] == 0.f ? 0.f : (kOver ? 16777216.f : 1.f) / size[r];
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      const float e0 = kOver ? __shfl_sync(~0u, extra[0], (lane & ~3) | gr) : 0.f, e1 = kOver ? __shfl_sync(~0u, extra[2], (lane & ~3) | gr) : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[gr][e][i] = fmaf(o[gr][e][i], kOver && (e & 1) ? 0.0625f : 1.f, -(i < 2 ? e0 : e1)) * by[i >> 1];
    }
    join_warps<T, D>(a, piece, job, smem, o, m, l);
  }
  if (a.ws && threadIdx.x == 0) reinterpret_cast<int4*>(a.ws + (int64_t)gridDim.x * 2 * (kRows * (D + 2)))[blockIdx.x] = ends;
}

// Joins the parts of the segment that ends in a CTA's share and began in one before: a CTA for each of attend's.  A thread has four components of a row, in one of kBy
// parts in turn.  (Four CTAs with four rows each: 64 paragraphs of 1 to 4001 positions took 8 us longer.)
constexpr int kJoinThreads = 512;
template <class T, int D>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(const __grid_constant__ AttendParams a, int blocks) {
  constexpr int kPart = kRows * (D + 2), kBy = kJoinThreads / (kRows * D / 4);
  __shared__ float s_top[kBy][kRows], s_weight[kBy][kRows];
  __shared__ float4 s_sum[kBy][kRows * D / 4];
  const int at = threadIdx.x % (kRows * D / 4), by = threadIdx.x / (kRows * D / 4), r = at / (D / 4), d = at % (D / 4) * 4;
  wait_for_last();
  const int4 ends = reinterpret_cast<const int4*>(a.ws + (int64_t)blocks * 2 * kPart)[blockIdx.x];
  if (ends.x < 0) return;
  const int from = ends.w, n_parts = (int)blockIdx.x - from + 1;
  auto part = [&](int i) { return a.ws + ((int64_t)(from + i) * 2 + (i == 0)) * kPart; };
  // The maximum so far goes along, so that every part is waited for once: eight of them at a time are on their way.
  float top = -INFINITY, weight = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = by; i0 < n_parts; i0 += 8 * kBy) {
    float m[8], l[8];
    float4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = -INFINITY;
      if (i0 + j * kBy < n_parts) {
        const float* const w = part(i0 + j * kBy);
        m[j] = w[kRows * D + r];
        l[j] = w[kRows * D + kRows + r];
        v[j] = *reinterpret_cast<const float4*>(w + r * D + d);
      }
    }
    float now = top;
#pragma unroll
    for (int j = 0; j < 8; ++j) now = fmaxf(now, m[j]);
    const float base = now == -INFINITY ? 0.f : now;      // (a part without a maximum has a weight of 0, or of NaN, which stays one)
    const float f0 = exp2_of(top - base);
    top = now;
    weight *= f0;
    sum.x *= f0; sum.y *= f0; sum.z *= f0; sum.w *= f0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (i0 + j * kBy >= n_parts) break;
      const float f = exp2_of(m[j] - base);
      sum.x += f * v[j].x; sum.y += f * v[j].y; sum.z += f * v[j].z; sum.w += f * v[j].w;
      weight += f * l[j];
    }
  }
  s_sum[by][at] = sum;
  if (d == 0) { s_top[by][r] = top; s_weight[by][r] = weight; }
  __syncthreads();
  if (by || r >= a.g * a.rep - ends.z * kRows) return;
#pragma unroll
  for (int i = 1; i < kBy; ++i) top = fmaxf(top, s_top[i][r]);
  const float base = top == -INFINITY ? 0.f : top;
  sum = make_float4(0.f, 0.f, 0.f, 0.f);
  weight = 0.f;
#pragma unroll
  for (int i = 0; i < kBy; ++i) {
    const float f = exp2_of(s_top[i][r] - base);
    const float4 v = s_sum[i][at];
    sum.x += f * v.x; sum.y += f * v.y; sum.z += f * v.z; sum.w += f * v.w;
    weight += f * s_weight[i][r];
  }
  write_row<T>(a, ends.x, ends.y, ends.z * kRows + r, d, sum, top, weight);
}

template <class T, int D>
cudaError_t launch_attend(const AttendParams& p, int blocks, cudaStream_t st) {
  constexpr int smem = attend_smem<T, D>();
  const Scores how = p.cap == 0.f && !p.slope && p.scale != 0.f ? kPlain : sizeof(T) == 4 || p.cap > kQuickCap ? kExact : kQuick;
  void (*kernel)(AttendParams) = how == kPlain ? attend_kernel<T, D, kPlain> : attend_kernel<T, D, kExact>;
  if constexpr (sizeof(T) == 2) {
    if (how == kQuick) kernel = attend_kernel<T, D, kQuick>;
  }
  static_assert(smem + 2048 <= 48 << 10, "more shared memory has to be asked for");
  kernel<<<(unsigned)blocks, kWarps * 32, smem, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !p.ws) return e;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, attend_join_kernel<T, D>, p, blocks);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

int row_tiles_of(const linmt_attend_pages4_args* g) { return (int)(((int64_t)g->g * (g->heads / g->pages.heads) + kRows - 1) / kRows); }

int64_t pairs_at_most(const linmt_attend_pages4_args* g) { const int64_t p = ((int64_t)g->width * g->pages.page + 31) / 32; return p < 1 ? 1 : p; }
// CTAs: as many as fit on the GPU at once (three on an SM with 128 components, four with 64), or as the longest possible sentences
// give kLeast pairs each.
int blocks_of(const linmt_attend_pages4_args* g) {
  const int64_t segments = (int64_t)g->n * g->pages.heads * row_tiles_of(g), most = segments * ((pairs_at_most(g) + kFixed + kLeast - 1) / kLeast), fit = 148 * (g->pages.dim == 64 ? 4 : 3);
  return (int)(most < fit ? most : fit);
}

int check(const linmt_attend_pages4_args* g) {
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "attend_pages4: not this library's argument struct");
  if (int rc = check_pages4(g->pages, "attend_pages4")) return rc;
  if (g->n < 0 || g->g < 0 || g->heads < 1 || g->heads % g->pages.heads || g->width < 0 || !dtype_ok(g->dtype))
    return op_fail(LINMT_EINVAL, "attend_pages4: n = %d, g = %d, heads = %d (a multiple of the pool's %d), width = %d, dtype = %d", g->n, g->g, g->heads, g->pages.heads, g->width, g->dtype);
  if (!(g->scale - g->scale == 0.f) || !(g->cap >= 0.f) || !(g->cap - g->cap == 0.f)) return op_fail(LINMT_EINVAL, "attend_pages4: scale and cap have to be finite, cap not negative");
  if (g->cap > 0.f && (g->cap < 1e-18f || !(g->scale / g->cap - g->scale / g->cap == 0.f))) return op_fail(LINMT_EINVAL, "attend_pages4: cap = %g is too small (0: none)", (double)g->cap);
  if (g->n == 0 || g->g == 0) return LINMT_OK;
  if (!g->q || !g->out || !g->len || (g->width && !g->table)) return op_fail(LINMT_EINVAL, "attend_pages4: an array is missing");
  if (!g->slope != !g->centre || !g->first != !g->last) return op_fail(LINMT_EINVAL, "attend_pages4: slope goes with centre, first with last");
  const int size = dtype_bytes(g->dtype);
  if (!aligned(g->q, size) || !aligned(g->out, size) || !aligned(g->lse, 4) || !aligned(g->table, 4) || !aligned(g->len, 4) || !aligned(g->slope, 4) || !aligned(g->centre, 4) || !aligned(g->first, 4) || !aligned(g->last, 4))
    return op_fail(LINMT_EINVAL, "attend_pages4: an array is not aligned to its type");
  if ((int64_t)g->g * g->heads > INT32_MAX / 2 || (int64_t)g->n * g->pages.heads * row_tiles_of(g) > (1 << 24))
    return op_fail(LINMT_ELIMIT, "attend_pages4: %d sentences of %d rows and %d heads are too many for one call", g->n, g->g, g->heads);
  return LINMT_OK;
}

// Two parts for each CTA, of the segments that it shares with the CTAs before and behind it, and what the join has to know.  None where no segment can be long enough to be cut.
int64_t workspace_of(const linmt_attend_pages4_args* g) {
  return pairs_at_most(g) <= kLeast ? 0 : (int64_t)blocks_of(g) * (2 * (kRows * (g->pages.dim + 2)) * 4 + 16);
}

}  // namespace
}  // namespace ops
}  // namespace linmt

extern "C" {

int64_t linmt_attend_pages4_workspace(const linmt_attend_pages4_args* g) {
  using namespace linmt::ops;
  if (check(g)) return -1;
  return g->n == 0 || g->g == 0 ? 0 : workspace_of(g);
}

int linmt_attend_pages4(const linmt_attend_pages4_args* g) {
  using namespace linmt::ops;
  if (int rc = check(g)) return rc;
  if (g->n == 0 || g->g == 0) return LINMT_OK;
  const int64_t need = workspace_of(g);
  if (need && (!g->workspace || g->workspace_bytes < need || !aligned(g->workspace, 16)))
    return op_fail(LINMT_EINVAL, "attend_pages4: a workspace of %lld bytes is needed, 16-byte aligned", (long long)need);
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "attend_pages4");
  AttendParams p{static_cast<const unsigned char*>(g->pages.data), g->pages.stride_page, g->pages.stride_head, g->pages.n_pages, g->pages.heads, g->pages.page,
                 g->q, g->q_stride_n, g->q_stride_g, g->q_stride_h, g->out, g->out_stride_n, g->out_stride_g, g->out_stride_h, g->lse, g->table, g->table_stride, g->len,
                 g->slope, g->centre, g->first, g->last, need ? static_cast<float*>(g->workspace) : nullptr, g->n, g->g, g->heads, g->heads / g->pages.heads, g->width, row_tiles_of(g), g->first && g->g <= 32 && (int64_t)g->n * g->g <= 65536,
                 g->scale, g->cap, std::fabs(g->scale) * kLog2e * (g->cap > 0.f ? 2.f / g->cap : 1.f), 0, aligned(g->q, 16) && (g->q_stride_n | g->q_stride_g | g->q_stride_h) % (16 / dtype_bytes(g->dtype)) == 0,
                 aligned(g->out, 4 * dtype_bytes(g->dtype)) && (g->out_stride_n | g->out_stride_g | g->out_stride_h) % 4 == 0};
  if (g->cap > kQuickCap) p.mul = (float)std::frexp(std::fabs((double)g->scale) * 1.4426950408889634 * 2 / g->cap, &p.mul_up);
  if (g->cap > kHugeCap) p.mul_up += 100;
  const int blocks = blocks_of(g);
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  cudaError_t e;
  if (g->pages.dim == 64)
    e = g->dtype == LINMT_F32 ? launch_attend<float, 64>(p, blocks, st) : g->dtype == LINMT_BF16 ? launch_attend<__nv_bfloat16, 64>(p, blocks, st) : launch_attend<__half, 64>(p, blocks, st);
  else
    e = g->dtype == LINMT_F32 ? launch_attend<float, 128>(p, blocks, st) : g->dtype == LINMT_BF16 ? launch_attend<__nv_bfloat16, 128>(p, blocks, st) : launch_attend<__half, 128>(p, blocks, st);
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "attend_pages4");
}

}  // extern "C"
