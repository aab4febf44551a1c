// pages8_attend.cu -- attention of a few query rows per sentence over a pool of 8-bit pages (linmt_attend_pages8).
//
//   out = sum_t softmax_t(f(scale q . k_t)) v_t,   k_t = ks code, v_t = vs code, a scale for each block of 16 positions
//
// Both products are tcgen05.mma of bytes into 32-bit integers, with codes as they lie in the pool as the left operand: nothing is unpacked, and no sum is rounded.
//   S[128 positions x 48] = keys . queries: a query of a row is a whole number of 23 bits (to 2^-23 of the row's largest component), cut into three
//   signed bytes, one column each for 16 rows.  s = (65536 S2 + 256 S1 + S0) ks times the row's power of 2.
//   O[dim x 64] += values^T . weights: a weight times its block's scale is a whole number of 32 bits (to 2^-31 of about the row's largest), whose four bytes are a
//   column each.  O = sum over the four of 256^i O_i.
// 16 rows (beams, and the query heads that share a head of the pool) are the right operand, which may be narrow: with 128 positions (or components) on the left a
// product of 32 KB of pages takes some 300 cycles, a fifth of the time that HBM needs for them.
// Weights are relative to 2^M, M a whole number for each row not below the largest exponent of weight times scale less 1; the sum of weights alone is relative to
// 2^L, 40 above such a number.  (One for both would lose rows whose values differ by more than 32 bits hold.)  Both follow when something exceeds them; only
// then, every 256 chunks and at the end are O's integers taken out of TMEM, into 32-bit sums.
// A CTA has 128 threads that turn S into weights, a position each; one warp that copies blocks (bulk copies, two rings) and one that issues the products.  Two CTAs
// share an SM.  The work is cut into equal shares over the CTAs that fit on the GPU at once, and a second kernel joins the parts of what several of them share.
#include <cmath>

#include "device_ops.h"
#include "pages8.h"

namespace linmt {
namespace ops {
namespace {

constexpr int kRows = 16;
constexpr int kChunk = 128;                  // positions of a product
constexpr int kBlocks = kChunk / pages8::kBlock;
constexpr int kWeightWarps = 4, kCopyWarp = 4, kIssueWarp = 5;
constexpr int kThreads = 192;
constexpr int kQueryDigits = 3, kWeightDigits = 4;
constexpr int kQueryCols = kRows * kQueryDigits, kWeightCols = kRows * kWeightDigits;
constexpr int kTmemCols = 256, kTmemS = 64, kTmemO = 128;      // S twice, 64 columns apart, then O
constexpr int kDrain = 256;                  // chunks between two drains: 127 * 255 * 128 * 256 < 2^31
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kAbove = 40.f;               // of L above the exponents so far
constexpr unsigned long long kWaitCycles = 2000000000ull;      // about a second
template <int D> constexpr int kStages = D == 128 ? 3 : 5;

enum Scores { kPlain, kQuick, kExact };      // neither cap nor bias; caps to 3e-7 of the cap; caps by tanhf

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
  int32_t n, g, heads, rep, width, row_tiles, sinks, by_window, dtype, q_wide;
  float cap, mul;            // mul: scale, times what the form of the scores takes it by
};

// ---- PTX
__device__ __forceinline__ uint32_t shared(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// Waits for the barrier's phase, about a second at most.  Where that runs out, *gave_up is raised: all further waits end at once, nothing more is issued, and
// results are NaN.
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
  if (bar_try(bar, parity)) return;
  const unsigned long long t0 = clock64();
  while (!bar_try(bar, parity)) {
    if (*gave_up) return;
    if ((unsigned long long)clock64() - t0 > kWaitCycles) { *gave_up = 1; return; }
  }
}
__device__ __forceinline__ void copy_bulk(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void tmem_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mma_bytes(uint32_t d, uint64_t a, uint64_t b, uint32_t form, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(form), "r"(add) : "memory");
}
// An operand in shared memory without a swizzle: cores of eight rows of 16 bytes, `along` bytes from one to the next along the sum, `across` to the next eight rows.
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t along, uint32_t across) {
  return (uint64_t)(at >> 4 & 0x3fff) | (uint64_t)(along >> 4) << 16 | (uint64_t)(across >> 4) << 32 | (uint64_t)1 << 46;
}
// 32-bit integers of signed bytes times signed (or unsigned) ones, both along the sum; 128 rows, n columns.
__host__ __device__ constexpr uint32_t form_of(int n, bool is_signed) { return 2u << 4 | 1u << 7 | (is_signed ? 1u : 0u) << 10 | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24; }

#define LINMT_OUT16(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7]), \
    "=r"(v[o + 8]), "=r"(v[o + 9]), "=r"(v[o + 10]), "=r"(v[o + 11]), "=r"(v[o + 12]), "=r"(v[o + 13]), "=r"(v[o + 14]), "=r"(v[o + 15])
// 16 columns of the lane's row of TMEM.
__device__ __forceinline__ void tmem_load16(uint32_t at, int (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LINMT_OUT16(v, 0) : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_load48(uint32_t at, int (&v)[48]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%48];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%49];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47}, [%50];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LINMT_OUT16(v, 0), LINMT_OUT16(v, 16), LINMT_OUT16(v, 32) : "r"(at), "r"(at + 16), "r"(at + 32) : "memory");
}
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
// cap tanh(x) as cap - 2 cap / (2^y + 1), y = 2 x log2(e): good to 3e-7 of the cap, 2e-5 of a score with a cap of up to kQuickCap, which a 16-bit result does not see.
constexpr float kQuickCap = 64.f;
__device__ __forceinline__ float capped(float y, float cap) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(exp2_of(y) + 1.f));
  return fmaf(-2.f * cap, r, cap);
}
// The 128 threads of the weights: wait for each other; whether one of them says so.
__device__ __forceinline__ void weights_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool weights_any(bool x) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 128, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(r) : "r"((int)x) : "memory");
  return r != 0;
}
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- who does what
//
// The work is a list of units: sentence by sentence, in each by head of the pool and row tile (a segment), a segment's chunks in order, those that a row of the
// sentence sees (where there are windows, and not so many that looking at them takes longer than the chunks that they leave out).  It is cut into as
// many equal parts as CTAs fit on the GPU at once: a segment longer than a part is then shared by several CTAs, whose parts the join kernel adds up, and a
// CTA may have several short ones.  Lengths are known on the device only, so every CTA adds them up itself.  A segment counts as kFixed units more than it has chunks, its fixed costs
// being as large; one of up to kWhole units or an eighth of a part is not cut: the CTA that has its first unit takes it whole.
constexpr int kFixed = 3;
constexpr int kWhole = kFixed + 3;
struct Share {
  int64_t begin, end;      // the CTA's units
  int64_t first;           // number of the first unit of sentence `sent`
  int64_t per;             // units of a part
  int sent, whole;         // sentence of `begin`; segments of up to `whole` units are not cut
};
__device__ __forceinline__ int length_of(const AttendParams& a, int sent) {
  return min(max(__ldg(a.len + sent), 0), (int)min((int64_t)a.width * a.page, (int64_t)0x7fffffff - 2 * kChunk));
}
// The chunks that any row of a sentence sees: the first n1, and n2 from chunk b0 on.
struct Seen {
  int n1, b0, n2;
  __device__ __forceinline__ int units() const { return n1 + n2 + kFixed; }
  __device__ __forceinline__ int chunk(int i) const { return i < n1 ? i : b0 + i - n1; }
};
__device__ __forceinline__ int chunks_of(int positions) { return (positions + kChunk - 1) / kChunk; }
__device__ __forceinline__ Seen seen_between(int lo, int hi, int sinks) {
  const int first = chunks_of(sinks);
  if (lo >= hi) return {first, 0, 0};
  const int from = lo / kChunk, to = chunks_of(hi);
  return first < from ? Seen{first, from, to - from} : Seen{0, 0, max(to, first)};
}
__device__ __forceinline__ Seen seen_of(const AttendParams& a, int sent) {             // by one thread
  const int len = length_of(a, sent);
  if (!a.by_window) return seen_between(0, len, 0);
  int lo = 0x7fffffff, hi = 0;
#pragma unroll 4
  for (int g = 0; g < a.g; ++g) {
    const int f = max(__ldg(a.first + (int64_t)sent * a.g + g), 0), l = min(__ldg(a.last + (int64_t)sent * a.g + g), len);
    if (f < l) { lo = min(lo, f); hi = max(hi, l); }
  }
  return seen_between(lo, hi, min(a.sinks, len));
}
__device__ __forceinline__ Seen seen_by_warp(const AttendParams& a, int sent) {        // by a warp
  const int len = length_of(a, sent);
  if (!a.by_window) return seen_between(0, len, 0);
  int lo = 0x7fffffff, hi = 0;
  for (int g = threadIdx.x & 31; g < a.g; g += 32) {
    const int f = max(__ldg(a.first + (int64_t)sent * a.g + g), 0), l = min(__ldg(a.last + (int64_t)sent * a.g + g), len);
    if (f < l) { lo = min(lo, f); hi = max(hi, l); }
  }
  return seen_between(__reduce_min_sync(~0u, lo), __reduce_max_sync(~0u, hi), min(a.sinks, len));
}

// Share of block `blockIdx.x` of `blocks`; all threads of the CTA call it.  The sentences are added up by all threads, then those of the thread that has the first
// unit, until one is left.
__device__ __forceinline__ Share share_of(const AttendParams& a, int blocks) {
  __shared__ int64_t sums[kThreads / 32], found_first;
  __shared__ int found_lo, found_hi;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, segments = a.pool_heads * a.row_tiles;
  Share s{};
  int lo = 0, hi = a.n;
  bool all = true;
  for (;;) {
    const int each = (hi - lo + kThreads - 1) / kThreads, i0 = min(hi, lo + tid * each), i1 = min(hi, i0 + each);
    int64_t mine = 0;
#pragma unroll 8
    for (int i = i0; i < i1; ++i) mine += seen_of(a, i).units();
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int64_t total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w == warp) upto += total;
      total += sums[w];
    }
    if (all) {
      all = false;
      total *= segments;
      s.per = max((int64_t)kWhole, (total + blocks - 1) / blocks);
      s.begin = min(total, blockIdx.x * s.per);
      s.end = min(total, s.begin + s.per);
      s.whole = (int)min((int64_t)0x7fffffff, max((int64_t)kWhole, s.per / 8));
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

// One CTA's piece of a segment: chunks c0 .. c1 - 1 of those seen.
struct Piece {
  int sent, kvh, rt, len;
  int u0, u1, units;       // units u0 .. u1 - 1 of the segment's
  int64_t start;           // number of the segment's first unit
  int c0, c1;
  Seen seen;
  __device__ __forceinline__ bool whole() const { return u0 == 0 && u1 == units; }
};
// The piece that begins at s.begin; false where the CTA has none left.  Moves s on behind it.  All lanes of a warp call it.
__device__ __forceinline__ bool next_piece(const AttendParams& a, Share& s, Piece& p) {
  const int segments = a.pool_heads * a.row_tiles;
  while (s.begin < s.end) {
    p.seen = seen_by_warp(a, s.sent);
    p.units = p.seen.units();
    const int64_t in = s.begin - s.first, seg = in >> 32 ? in / p.units : (int64_t)((uint32_t)in / (uint32_t)p.units);
    if (seg >= segments) {
      s.first += (int64_t)p.units * segments;
      ++s.sent;
      continue;
    }
    p.sent = s.sent;
    p.len = length_of(a, s.sent);
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
    p.c0 = max(p.u0 - kFixed, 0);
    p.c1 = max(p.u1 - kFixed, 0);
    return true;
  }
  return false;
}

// ---- shared memory
template <int D>
struct Shared {
  static constexpr int S = kStages<D>, kPart = kChunk * D;
  static constexpr int kAcross = 8 * 16 * kBlocks;                 // bytes from eight columns of the weights to the next
  alignas(128) unsigned char keys[S][kPart];
  alignas(128) unsigned char values[S][kPart];
  alignas(128) unsigned char queries[kQueryCols * D];              // (behind the values: with 64 components a product's lower half reads a block further, into rows of O that nobody looks at)
  alignas(128) unsigned char weights[kWeightCols / 8 * kAcross];
  alignas(16) float scales[S][kBlocks][4];
  float m[kRows], l[kRows], by[kRows], slope[kRows], centre[kRows];
  int lo[kRows], span[kRows], bad[kRows];
  float most[2][kWeightWarps][kRows];
  unsigned valid[S];
  int add, gave_up;
  uint32_t tmem;
  alignas(8) unsigned long long k_full[S], k_empty[S], v_full[S], v_empty[S], s_full[2], s_empty[2], p_full, o_full, q_full;
};

// A component's number of rows: where row `at` of a sentence's head of the pool is in q and out.
struct Place { int g, h; };
__device__ __forceinline__ Place place_of(const AttendParams& a, const Piece& p, int r) {
  const int at = p.rt * kRows + r, g = at / a.rep;
  return {g, p.kvh * a.rep + at - g * a.rep};
}

__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dtype) {
  return dtype == LINMT_F32 ? __ldg(static_cast<const float*>(p) + i) : dtype == LINMT_BF16 ? to_float(__ldg(static_cast<const __nv_bfloat16*>(p) + i)) : to_float(__ldg(static_cast<const __half*>(p) + i));
}
__device__ __forceinline__ void store_as(void* p, int64_t i, int dtype, float x) {
  if (dtype == LINMT_F32) static_cast<float*>(p)[i] = x;
  else if (dtype == LINMT_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

// N neighbouring components of a row, 16-byte aligned (q_wide) or not.
template <int N>
__device__ __forceinline__ void load_row(const AttendParams& a, int64_t at, float (&x)[N]) {
  if (!a.q_wide) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = load_as_float(a.q, at + i, a.dtype);
  } else if (a.dtype == LINMT_F32) {
    const float4* const p = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 v = __ldg(p + i);
      x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
    }
  } else {
    const uint4* const p = reinterpret_cast<const uint4*>(static_cast<const __half*>(a.q) + at);
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      const uint4 v = __ldg(p + i);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 two = a.dtype == LINMT_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j])) : __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        x[8 * i + 2 * j] = two.x;
        x[8 * i + 2 * j + 1] = two.y;
      }
    }
  }
}

__device__ __forceinline__ float power_of_2(int e) { return __int_as_float((127 + e) << 23); }      // -126 .. 127

// The piece's queries as bytes, and what its rows see; by the 128 threads of the weights, eight for a row.
template <int D>
__device__ __forceinline__ void take_queries(const AttendParams& a, const Piece& p, Shared<D>& sh) {
  constexpr int N = D / 8;
  const int tid = threadIdx.x, r = tid / 8, part = tid % 8, n_rows = min(kRows, a.g * a.rep - p.rt * kRows);
  const bool have = r < n_rows;
  const Place at = place_of(a, p, have ? r : 0);
  float x[N], most = 0.f;
  if (have) {
    load_row<N>(a, p.sent * a.q_n + at.g * a.q_g + at.h * a.q_h + part * N, x);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) most = max_nan(most, fabsf(x[i]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) most = max_nan(most, __shfl_xor_sync(~0u, most, o));
  const bool bad = !(most < INFINITY);
  const int e = most > 0.f && !bad ? ilogbf(most) : 0;              // 2^e <= most < 2^(e + 1); components times 2^(21 - e) are below 2^22
  const float up0 = power_of_2((21 - e) / 2), up1 = power_of_2(21 - e - (21 - e) / 2);
  uint32_t d[kQueryDigits][N / 4];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int v = bad ? 0 : __float2int_rn(x[i] * up0 * up1);
#pragma unroll
    for (int k = 0; k < kQueryDigits; ++k) {
      const int low = (int)(int8_t)v;
      v = (v - low) >> 8;
      if (i % 4 == 0) d[k][i / 4] = 0;
      d[k][i / 4] |= (uint32_t)(low & 255) << (8 * (i % 4));
    }
  }
#pragma unroll
  for (int k = 0; k < kQueryDigits; ++k) {
    const int n = k * kRows + r, c = part * N;
    uint32_t* const to = reinterpret_cast<uint32_t*>(sh.queries + n / 8 * 8 * D + c / 16 * 128 + n % 8 * 16 + c % 16);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) to[i] = d[k][i];
  }
  if (part == 0) {
    sh.m[r] = sh.l[r] = kLowest;
    sh.by[r] = have ? ldexpf(a.mul, e - 21) : 0.f;
    sh.bad[r] = bad;
    sh.slope[r] = have && a.slope ? __ldg(a.slope + at.h) * kLog2e : 0.f;
    sh.centre[r] = have && a.slope ? __ldg(a.centre + (int64_t)p.sent * a.g + at.g) : 0.f;
    const int lo = a.first && have ? max(__ldg(a.first + (int64_t)p.sent * a.g + at.g), 0) : 0, hi = a.first && have ? min(__ldg(a.last + (int64_t)p.sent * a.g + at.g), p.len) : p.len;
    sh.lo[r] = lo;
    sh.span[r] = max(hi - lo, 0);
  }
}

// What a row's weights are relative to behind a chunk, from the warps' largest exponents: `was` as long as none exceeds it by more than 1.
template <int D>
__device__ __forceinline__ float raised(const Shared<D>& sh, int which, int r, float was, float above) {
  const float most = fmaxf(fmaxf(sh.most[which][0][r], sh.most[which][1][r]), fmaxf(sh.most[which][2][r], sh.most[which][3][r]));
  return most - was > 1.f ? ceilf(most) + above : was;
}

template <int D, int HOW>
__global__ void __launch_bounds__(kThreads, 2) attend_kernel(const __grid_constant__ AttendParams a) {
  extern __shared__ __align__(128) unsigned char attend_smem[];
  Shared<D>& sh = *reinterpret_cast<Shared<D>*>(attend_smem);
  constexpr int S = kStages<D>;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(~0u, tid >> 5, 0);
  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      bar_init(shared(&sh.k_full[i]), 1);
      bar_init(shared(&sh.k_empty[i]), 1);
      bar_init(shared(&sh.v_full[i]), 1);
      bar_init(shared(&sh.v_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(shared(&sh.s_full[i]), 1);
      bar_init(shared(&sh.s_empty[i]), kWeightWarps);
    }
    bar_init(shared(&sh.p_full), kWeightWarps);
    bar_init(shared(&sh.o_full), 1);
    bar_init(shared(&sh.q_full), kWeightWarps);
    sh.gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared(&sh.tmem)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  launch_next();
  Share share = share_of(a, gridDim.x);
  tmem_before();
  __syncthreads();
  tmem_after();
  const uint32_t tmem = sh.tmem;
  volatile int* const gave_up = &sh.gave_up;
  Piece p;
  int4 ends = make_int4(-1, 0, 0, 0);                 // the segment that ends in this share and began before it: sentence, head, row tile, first CTA

  if (warp == kCopyWarp) {
    // ---- blocks into the rings, a lane for each of a chunk's
    int it = 0;
    while (next_piece(a, share, p)) {
      const unsigned char* const head = a.data + p.kvh * a.stride_head;
      const int32_t* const table = a.table + p.sent * a.table_stride;
      const int blocks = (p.len + pages8::kBlock - 1) / pages8::kBlock, per_page = a.page / pages8::kBlock;
      for (int c = p.c0; c < p.c1; ++c, ++it) {
        const int stage = it % S, block = p.seen.chunk(c) * kBlocks + lane;
        const uint32_t parity = (uint32_t)(it / S & 1) ^ 1;
        const int64_t at = lane < kBlocks && block < blocks ? pages8::block_offset(table, block, per_page, a.n_pages, a.stride_page, D) : -1;
        const unsigned valid = __ballot_sync(~0u, at >= 0);
        const int count = __popc(valid);
        bar_wait(shared(&sh.k_empty[stage]), parity, gave_up);
        __syncwarp();
        if (!*gave_up) {
          if (lane == 0) bar_expect(shared(&sh.k_full[stage]), count * 16 * D);
          __syncwarp();
          if (at >= 0) copy_bulk(shared(sh.keys[stage] + lane * 16 * D), head + at, 16 * D, shared(&sh.k_full[stage]));
        }
        bar_wait(shared(&sh.v_empty[stage]), parity, gave_up);
        __syncwarp();
        if (!*gave_up) {
          if (lane == 0) {
            sh.valid[stage] = valid;
            bar_expect(shared(&sh.v_full[stage]), count * (16 * D + 16));
          }
          __syncwarp();
          if (at >= 0) {
            copy_bulk(shared(sh.values[stage] + lane * 16 * D), head + at + pages8::value_codes(D), 16 * D, shared(&sh.v_full[stage]));
            copy_bulk(shared(sh.scales[stage][lane]), head + at + pages8::scales(D), 16, shared(&sh.v_full[stage]));
          }
        }
      }
    }
    if (*gave_up) {                                   // what is on its way still lands in this CTA's memory
      const unsigned long long t0 = clock64();
      while ((unsigned long long)clock64() - t0 < kWaitCycles / 100) {}
    }
  } else if (warp == kIssueWarp) {
    // ---- the products
    const bool elected = elect_one();
    int it = 0, queries = 0;
    auto weights_times_values = [&](int i) {
      const int stage = i % S;
      bar_wait(shared(&sh.p_full), i & 1, gave_up);
      bar_wait(shared(&sh.v_full[stage]), i / S & 1, gave_up);
      __syncwarp();
      tmem_after();
      if (elected && !*gave_up) {
        const uint32_t add = *(volatile int*)&sh.add;
        const uint64_t left = operand(shared(sh.values[stage]), 16 * D, 128), right = operand(shared(sh.weights), 128, Shared<D>::kAcross);
#pragma unroll
        for (int k = 0; k < kChunk / 32; ++k)
          mma_bytes(tmem + kTmemO, left + (uint64_t)(k * 2 * 16 * D >> 4), right + (uint64_t)(k * 2 * 128 >> 4), form_of(kWeightCols, false), k ? 1u : add);
        commit(shared(&sh.v_empty[stage]));
        commit(shared(&sh.o_full));
      }
      __syncwarp();
    };
    while (next_piece(a, share, p)) {
      if (p.c0 == p.c1) continue;
      bar_wait(shared(&sh.q_full), queries++ & 1, gave_up);
      for (int c = p.c0; c < p.c1; ++c, ++it) {
        const int stage = it % S, half = it & 1;
        bar_wait(shared(&sh.k_full[stage]), it / S & 1, gave_up);
        bar_wait(shared(&sh.s_empty[half]), (it >> 1 & 1) ^ 1, gave_up);
        __syncwarp();
        tmem_after();
        if (elected && !*gave_up) {
          const uint64_t left = operand(shared(sh.keys[stage]), 128, 8 * D), right = operand(shared(sh.queries), 128, 8 * D);
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
            mma_bytes(tmem + half * kTmemS, left + (uint64_t)(k * 2 * 128 >> 4), right + (uint64_t)(k * 2 * 128 >> 4), form_of(kQueryCols, true), k ? 1u : 0u);
          commit(shared(&sh.k_empty[stage]));
          commit(shared(&sh.s_full[half]));
        }
        __syncwarp();
        if (c > p.c0) weights_times_values(it - 1);
      }
      weights_times_values(it - 1);
    }
  } else {
    // ---- scores to weights, a position for each thread; then a component for each thread
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    int it = 0;
    while (next_piece(a, share, p)) {
      const int n_rows = min(kRows, a.g * a.rep - p.rt * kRows);
      float sum[kRows], acc[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) sum[r] = acc[r] = 0.f;
      weights_sync();                                 // (the piece before is written: its rows' numbers are free)
      if (p.c0 < p.c1) {
        take_queries<D>(a, p, sh);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        weights_sync();
        if (lane == 0) bar_arrive(shared(&sh.q_full));
      }
      int since = 0;                                  // chunks in O
      // O's integers into sums, which are relative to 2^m then.
      auto drain = [&](const float (&down)[kRows]) {
        tmem_after();
#pragma unroll
        for (int i = 0; i < kRows / 4; ++i) {
          int o[16];
          tmem_load16(lanes + kTmemO + 16 * i, o);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = 4 * i + j;
            const float v = fmaf((float)o[4 * j + 3], 16777216.f, fmaf((float)o[4 * j + 2], 65536.f, fmaf((float)o[4 * j + 1], 256.f, (float)o[4 * j])));
            acc[r] = fmaf(v, 9.3132257461547852e-10f, acc[r]) * down[r];       // 2^-30
          }
        }
        tmem_before();
        since = 0;
      };
      for (int c = p.c0; c < p.c1; ++c, ++it) {
        const int stage = it % S, half = it & 1;
        bar_wait(shared(&sh.v_full[stage]), it / S & 1, gave_up);
        bar_wait(shared(&sh.s_full[half]), it >> 1 & 1, gave_up);
        tmem_after();
        int t[kQueryCols];
        tmem_load48(lanes + half * kTmemS, t);
        tmem_before();
        __syncwarp();
        if (lane == 0) bar_arrive(shared(&sh.s_empty[half]));

        const int at = tid / pages8::kBlock, pos = p.seen.chunk(c) * kChunk + tid;
        // A block that is not there has left whatever was in its place before; what lies behind a sentence's end may be anything.
        const bool there = pos < p.len && (sh.valid[stage] >> at & 1);
        const float ks = there ? sh.scales[stage][at][0] : 0.f, none = there ? 0.f : -INFINITY;
        const uint32_t vs = there ? __float_as_uint(sh.scales[stage][at][1]) : 0;
        // the values' scale as 2^ve times 2^-30 vf
        const float ve = vs ? (float)((int)(vs >> 23 & 255) - 127) : -1000.f, vf = vs ? __uint_as_float((vs & 0x7fffff) | (127 + 30) << 23) : 0.f;
        float s[kRows], most = -INFINITY;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float whole = fmaf((float)t[2 * kRows + r], 65536.f, (float)(t[kRows + r] * 256 + t[r])), by = sh.by[r] * ks;
          if constexpr (HOW == kPlain) {
            s[r] = fmaf(whole, by, none);
          } else {
            float x = whole * by;
            if constexpr (HOW == kQuick) {
              if (a.cap > 0.f) x = capped(x, a.cap * kLog2e);
            } else {
              if (a.cap > 0.f) x = a.cap * kLog2e * tanhf(x);
            }
            s[r] = x - sh.slope[r] * fabsf((float)pos - sh.centre[r]) + none;
          }
          if (a.first) s[r] = (unsigned)(pos - sh.lo[r]) < (unsigned)sh.span[r] || pos < a.sinks ? s[r] : -INFINITY;
          most = fmaxf(most, fmaxf(s[r] + (ve - sh.m[r]), s[r] - sh.l[r]));
        }
        // Something exceeds what the rows' weights are relative to: that follows.
        if (weights_any(most > 1.f) || since == kDrain) {
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            const float both = warp_max(s[r] + ve), alone = warp_max(s[r]);
            if (lane == 0) {
              sh.most[0][warp][r] = both;
              sh.most[1][warp][r] = alone;
            }
          }
          weights_sync();
          float down[kRows];
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            down[r] = exp2_of(sh.m[r] - raised(sh, 0, r, sh.m[r], 0.f));
            sum[r] *= exp2_of(sh.l[r] - raised(sh, 1, r, sh.l[r], kAbove));
          }
          weights_sync();
          if (tid < kRows) {
            sh.m[tid] = raised(sh, 0, tid, sh.m[tid], 0.f);
            sh.l[tid] = raised(sh, 1, tid, sh.l[tid], kAbove);
          }
          if (c > p.c0) bar_wait(shared(&sh.o_full), it - 1 & 1, gave_up);
          if (since) drain(down);
          else {
#pragma unroll
            for (int r = 0; r < kRows; ++r) acc[r] *= down[r];
          }
          weights_sync();
        } else if (c > p.c0) {
          bar_wait(shared(&sh.o_full), it - 1 & 1, gave_up);
        }
        unsigned char* const to = sh.weights + at * 128 + tid % 16;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          sum[r] += exp2_of(s[r] - sh.l[r]);
          const uint32_t w = __float2uint_rn(exp2_of(s[r] + (ve - sh.m[r])) * vf);
#pragma unroll
          for (int d = 0; d < kWeightDigits; ++d) to[(r * kWeightDigits + d) / 8 * Shared<D>::kAcross + (r * kWeightDigits + d) % 8 * 16] = (unsigned char)(w >> (8 * d));
        }
        if (tid == 0) sh.add = since > 0;
        ++since;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(shared(&sh.p_full));
      }
      if (p.c0 < p.c1) bar_wait(shared(&sh.o_full), it - 1 & 1, gave_up);
      if (since) {
        float as_is[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) as_is[r] = 1.f;
        drain(as_is);
      }
      // The rows' sums of weights, and out with it.
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) sum[r] += __shfl_xor_sync(~0u, sum[r], o);
        if (lane == 0) sh.most[0][warp][r] = sum[r];
      }
      weights_sync();
      const bool whole = p.whole();
      if (tid == 0 && !whole && p.u0 > 0 && p.u1 == p.units) ends = make_int4(p.sent, p.kvh, p.rt, (int)(p.start / share.per));
      // a part of the workspace: [row][D] values, [row] exponent, [row] weight.  A CTA's first is of the segment that it has from the CTA before, its second of the one that the next goes on with.
      float* const ws = a.ws + ((int64_t)blockIdx.x * 2 + (p.u0 == 0)) * (kRows * (D + 2));
      const bool empty = p.c0 == p.c1;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (r >= n_rows) break;
        float weight = empty ? 0.f : (sh.most[0][0][r] + sh.most[0][1][r] + sh.most[0][2][r] + sh.most[0][3][r]) * 1099511627776.f;      // 2^40
        const float m = empty ? 0.f : sh.m[r], l = empty ? kLowest : sh.l[r] - kAbove;
        float value = weight > 0.f ? acc[r] / weight * exp2_of(m - l) : 0.f;
        if (!empty && ((sh.bad[r] && weight > 0.f) || *gave_up)) value = weight = NAN;
        if (whole) {
          const Place at = place_of(a, p, r);
          if (tid < D) store_as(a.out, p.sent * a.o_n + at.g * a.o_g + at.h * a.o_h + tid, a.dtype, value);
          if (tid == 0 && a.lse) a.lse[((int64_t)p.sent * a.g + at.g) * a.heads + at.h] = weight == 0.f ? -INFINITY : (l + log2f(weight)) * kLn2;
        } else {
          if (tid < D) ws[r * D + tid] = value;
          if (tid == 0) { ws[kRows * D + r] = l; ws[kRows * D + kRows + r] = weight; }
        }
      }
    }
    if (a.ws && tid == 0) reinterpret_cast<int4*>(a.ws + (int64_t)gridDim.x * 2 * (kRows * (D + 2)))[blockIdx.x] = ends;
  }
  tmem_before();
  __syncthreads();
  if (warp == kIssueWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// Joins the parts of the segment that ends in a CTA's share and began in one before: a CTA for each of attend's.  A thread has four components of a row, in one of kBy
// parts in turn.
constexpr int kJoinThreads = 512;
template <int D>
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
  // The largest exponent so far goes along, so that every part is waited for once: eight of them at a time are on their way.
  float top = kLowest, weight = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = by; i0 < n_parts; i0 += 8 * kBy) {
    float m[8], l[8];
    float4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = kLowest;
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
    const float f0 = exp2_of(top - now);
    top = now;
    weight *= f0;
    sum.x *= f0; sum.y *= f0; sum.z *= f0; sum.w *= f0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (i0 + j * kBy >= n_parts) break;
      const float f = exp2_of(m[j] - now) * l[j];
      sum.x += f * v[j].x; sum.y += f * v[j].y; sum.z += f * v[j].z; sum.w += f * v[j].w;
      weight += f;
    }
  }
  s_sum[by][at] = sum;
  if (d == 0) { s_top[by][r] = top; s_weight[by][r] = weight; }
  __syncthreads();
  if (by || r >= a.g * a.rep - ends.z * kRows) return;
#pragma unroll
  for (int i = 1; i < kBy; ++i) top = fmaxf(top, s_top[i][r]);
  sum = make_float4(0.f, 0.f, 0.f, 0.f);
  weight = 0.f;
#pragma unroll
  for (int i = 0; i < kBy; ++i) {
    const float f = exp2_of(s_top[i][r] - top);
    const float4 v = s_sum[i][at];
    sum.x += f * v.x; sum.y += f * v.y; sum.z += f * v.z; sum.w += f * v.w;
    weight += f * s_weight[i][r];
  }
  const int row = ends.z * kRows + r, g = row / a.rep, h = ends.y * a.rep + row - g * a.rep;
  const float f = weight == 0.f ? 0.f : 1.f / weight;
  const int64_t to = ends.x * a.o_n + g * a.o_g + h * a.o_h + d;
  store_as(a.out, to, a.dtype, sum.x * f);
  store_as(a.out, to + 1, a.dtype, sum.y * f);
  store_as(a.out, to + 2, a.dtype, sum.z * f);
  store_as(a.out, to + 3, a.dtype, sum.w * f);
  if (d == 0 && a.lse) a.lse[((int64_t)ends.x * a.g + g) * a.heads + h] = weight == 0.f ? -INFINITY : (top + log2f(weight)) * kLn2;
}

template <int D>
cudaError_t launch_attend(AttendParams p, float scale, int blocks, cudaStream_t st) {
  constexpr int smem = (int)sizeof(Shared<D>);
  static_assert(smem <= 113 << 10, "two CTAs have to fit on an SM");
  const Scores how = p.cap == 0.f && !p.slope ? kPlain : p.dtype == LINMT_F32 || p.cap > kQuickCap ? kExact : kQuick;
  void (*const kernel)(AttendParams) = how == kPlain ? attend_kernel<D, kPlain> : how == kQuick ? attend_kernel<D, kQuick> : attend_kernel<D, kExact>;
  p.mul = (float)(p.cap == 0.f ? scale * 1.4426950408889634 : how == kQuick ? scale * 2.8853900817779268 / p.cap : (double)scale / p.cap);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)blocks, kThreads, smem, st>>>(p);
  e = cudaGetLastError();
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
  e = cudaLaunchKernelEx(&cfg, attend_join_kernel<D>, p, blocks);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

int row_tiles_of(const linmt_attend_pages8_args* g) { return (int)(((int64_t)g->g * (g->heads / g->pages.heads) + kRows - 1) / kRows); }

int64_t chunks_at_most(const linmt_attend_pages8_args* g) { return ((int64_t)g->width * g->pages.page + kChunk - 1) / kChunk; }
// CTAs: as many as fit on the GPU at once, or as the longest possible sentences give kWhole units each.
int blocks_of(const linmt_attend_pages8_args* g) {
  const int64_t segments = (int64_t)g->n * g->pages.heads * row_tiles_of(g), most = segments * ((chunks_at_most(g) + kFixed + kWhole - 1) / kWhole), fit = 148 * 2;
  return (int)(most < fit ? most : fit);
}
// Two parts for each CTA, of the segments that it shares with the CTAs before and behind it, and what the join has to know.  None where no segment can be long enough to be cut.
int64_t workspace_of(const linmt_attend_pages8_args* g) {
  return chunks_at_most(g) + kFixed <= kWhole ? 0 : (int64_t)blocks_of(g) * (2 * (kRows * (g->pages.dim + 2)) * 4 + 16);
}

int check(const linmt_attend_pages8_args* g) {
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "attend_pages8: not this library's argument struct");
  if (int rc = check_pages8(g->pages, "attend_pages8")) return rc;
  if (g->n < 0 || g->g < 0 || g->heads < 1 || g->heads % g->pages.heads || g->width < 0 || g->sinks < 0 || !dtype_ok(g->dtype))
    return op_fail(LINMT_EINVAL, "attend_pages8: n = %d, g = %d, heads = %d (a multiple of the pool's %d), width = %d, sinks = %d, dtype = %d", g->n, g->g, g->heads, g->pages.heads, g->width, g->sinks, g->dtype);
  if (!(g->scale - g->scale == 0.f) || !(g->cap >= 0.f) || !(g->cap - g->cap == 0.f)) return op_fail(LINMT_EINVAL, "attend_pages8: scale and cap have to be finite, cap not negative");
  if (g->cap > 0.f && (g->cap < 1e-18f || !(g->scale / g->cap - g->scale / g->cap == 0.f))) return op_fail(LINMT_EINVAL, "attend_pages8: cap = %g is too small (0: none)", (double)g->cap);
  if (g->n == 0 || g->g == 0) return LINMT_OK;
  if (!g->q || !g->out || !g->len || (g->width && !g->table)) return op_fail(LINMT_EINVAL, "attend_pages8: an array is missing");
  if (!g->slope != !g->centre || !g->first != !g->last) return op_fail(LINMT_EINVAL, "attend_pages8: slope goes with centre, first with last");
  const int size = dtype_bytes(g->dtype);
  if (!aligned(g->q, size) || !aligned(g->out, size) || !aligned(g->lse, 4) || !aligned(g->table, 4) || !aligned(g->len, 4) || !aligned(g->slope, 4) || !aligned(g->centre, 4) || !aligned(g->first, 4) || !aligned(g->last, 4))
    return op_fail(LINMT_EINVAL, "attend_pages8: an array is not aligned to its type");
  if ((int64_t)g->g * g->heads > INT32_MAX / 2 || (int64_t)g->n * g->pages.heads * row_tiles_of(g) > (1 << 24))
    return op_fail(LINMT_ELIMIT, "attend_pages8: %d sentences of %d rows and %d heads are too many for one call", g->n, g->g, g->heads);
  return LINMT_OK;
}

}  // namespace
}  // namespace ops
}  // namespace linmt

extern "C" {

int64_t linmt_attend_pages8_workspace(const linmt_attend_pages8_args* g) {
  using namespace linmt::ops;
  if (check(g)) return -1;
  return g->n == 0 || g->g == 0 ? 0 : workspace_of(g);
}

int linmt_attend_pages8(const linmt_attend_pages8_args* g) {
  using namespace linmt::ops;
  if (int rc = check(g)) return rc;
  if (g->n == 0 || g->g == 0) return LINMT_OK;
  const int64_t need = workspace_of(g);
  if (need && (!g->workspace || g->workspace_bytes < need || !aligned(g->workspace, 16)))
    return op_fail(LINMT_EINVAL, "attend_pages8: a workspace of %lld bytes is needed, 16-byte aligned", (long long)need);
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "attend_pages8");
  const AttendParams p{static_cast<const unsigned char*>(g->pages.data), g->pages.stride_page, g->pages.stride_head, g->pages.n_pages, g->pages.heads, g->pages.page,
                       g->q, g->q_stride_n, g->q_stride_g, g->q_stride_h, g->out, g->out_stride_n, g->out_stride_g, g->out_stride_h, g->lse, g->table, g->table_stride, g->len,
                       g->slope, g->centre, g->first, g->last, need ? static_cast<float*>(g->workspace) : nullptr, g->n, g->g, g->heads, g->heads / g->pages.heads, g->width, row_tiles_of(g),
                       g->sinks, g->first && g->g <= 32 && (int64_t)g->n * g->g <= 65536, g->dtype,
                       aligned(g->q, 16) && (g->q_stride_n | g->q_stride_g | g->q_stride_h) % (16 / dtype_bytes(g->dtype)) == 0, g->cap, 0.f};
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  const cudaError_t e = g->pages.dim == 64 ? launch_attend<64>(p, g->scale, blocks_of(g), st) : launch_attend<128>(p, g->scale, blocks_of(g), st);
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "attend_pages8");
}

}  // extern "C"
