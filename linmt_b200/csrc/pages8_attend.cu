// pages8_attend.cu -- attention of a few query rows per sentence over a pool of 8-bit pages (linmt_attend_pages8).
//
//   out = sum_t softmax_t(f(scale q . k_t)) v_t,   k_t = ks code, v_t = vs code, a scale for each block of 16 positions
//
// Both products are tcgen05.mma of bytes into 32-bit integers, with codes as they lie in the pool as the left operand: nothing is unpacked, and no sum is rounded.
//   S[128 positions x 3 R] = keys . queries: a query of a row is a whole number of 23 bits (to 2^-22 of the row's largest component), cut into three
//   signed bytes, a column each for R rows.  s = (65536 S2 + 256 S1 + S0) ks times the row's power of 2.
//   O[dim x 4 R] += values^T . weights: a weight times its block's scale is a whole number of 32 bits, whose four bytes are a column each.  O = sum over the
//   four of 256^i O_i.
// R rows (4, 8 or 16 of a sentence's beams and of the query heads that share a head of the pool) are the right operand, which may be narrow: with 128 positions (or components) on
// the left a product of 32 KB of pages takes some 300 cycles, a fifth of the time that HBM needs for them.
// Scores s are taken relative to X, a whole number for each row next to the largest so far, before anything else is added to them: weights are 2^(s - X), and times their scales they are relative to 2^M, M
// a whole number that is a power of 2 at most above the row's largest weight times scale so far, and at most one below it with 32-bit queries (weights
// are good to 2^-30 of the largest then), four with 16-bit ones (2^-27, and M follows less often).  (M relative to 0, and X and M each rounded by itself, lost scores of 2^24 and more; one number for both
// would lose rows whose values differ by more than 32 bits hold.)  M follows when something exceeds it, X when a score exceeds it by 40 more; only then, every 256 chunks and at the end are O's integers taken out of TMEM, into 32-bit sums.
// A CTA has 128 threads (256 with 16 rows) that turn S into weights, a position and up to eight rows each; one warp that copies blocks and makes queries ready, two pieces ahead, and one that
// issues the products.  Two CTAs share an SM, three with four rows.  The work is cut into equal shares over the CTAs that fit on the GPU at once, and a second kernel joins the parts of what
// several of them share.
// What bounds it: long sentences HBM (8 documents of 20-32k, 16 rows of 128: 84 us, 5.2 TB/s, of which 6 us until the first weights and 4 for the join) and, as much, the weights' latencies:
// 2700 cycles a chunk of a CTA's, of which the conversions and exponentials take 640.  Where scores rise from chunk to chunk (a bias that falls with the distance) taking O out each time is another 1600.
// Tried: weights stored byte by byte, positions as neighbours: 129 us where columns as neighbours took 105.  A bulk copy for each block's keys, values and scales: 110 us where four blocks a copy took
// 83.  Single rows that see nothing of a chunk left out: 92 us, and no faster with windows, as what is saved in work is lost in order.  Two rows an instruction: no difference.

#include <cuda.h>

#include <cmath>

#include "device_ops.h"
#include "pages8.h"

namespace linmt {
namespace ops {
namespace {

constexpr int kChunk = 128;                  // positions of a product
constexpr int kBlocks = kChunk / pages8::kBlock;
constexpr int kQueryDigits = 3, kWeightDigits = 4;
// R rows: 4, 8 or 16 of a head of the pool at once.
template <int R> constexpr int kQueryCols = (R * kQueryDigits + 15) / 16 * 16;
template <int R> constexpr int kWeightCols = R * kWeightDigits;
template <int R> constexpr int kTmemCols = R == 16 ? 256 : R == 8 ? 128 : 64;      // S twice, then O
template <int R> constexpr int kTmemO = 2 * kQueryCols<R>;
template <int R> constexpr int kCtas = R == 4 ? 3 : 2;                             // of an SM
// A thread of the weights has a position and kRows rows: with 16, two groups of four warps (the products' rows are 32 to a warp) share them.
template <int R> constexpr int kRows = R == 16 ? 8 : R;
template <int R> constexpr int kWeightWarps = 4 * (R / kRows<R>);
template <int R> constexpr int kThreads = 32 * (kWeightWarps<R> + 2);              // and a warp that copies, one that issues
constexpr int kDrain = 256;                  // chunks between two drains: 127 * 255 * 128 * 256 < 2^31
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kAbove = 40.f;               // by how much more a score may exceed X than a weight what it is relative to
constexpr unsigned long long kWaitCycles = 2000000000ull;      // about a second
template <int D, int R> constexpr int kKeyStages = (R == 8 ? 3 : 2) * 128 / D;
template <int D, int R> constexpr int kValueStages = (R == 4 ? 2 : 3) * 128 / D;

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
  int32_t row_page, row_head, rows;      // the pool as rows of blocks: from a page, a head to the next, and all (0: its strides are none of whole blocks)
  int32_t slack;             // by how many powers of 2 a weight may exceed what it is relative to
  int32_t give_up;           // every so many-th CTA gives up before its first wait; 0: none
};

// The pool's rows of blocks: codes of a block (keys, or values), and its scales.
struct alignas(64) AttendMaps { CUtensorMap codes, scales; };

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
// Columns from x on of four rows of a tensor, one behind the other.
__device__ __forceinline__ void copy_rows(uint32_t to, const CUtensorMap* map, int x, int r0, int r1, int r2, int r3, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
               ::"r"(to), "l"(map), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar) : "memory");
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
// 32-bit integers of signed bytes times bytes; 128 rows, n columns.  Queries: signed, 16 neighbouring bytes lie along the sum.  Weights: not signed, 16 neighbouring bytes are columns.
constexpr uint32_t kForm = 2u << 4 | 1u << 7 | (128u >> 4) << 24;
template <int R> constexpr uint32_t kQueryForm = kForm | 1u << 10 | (uint32_t)(kQueryCols<R> >> 3) << 17;
template <int R> constexpr uint32_t kWeightForm = kForm | 1u << 16 | (uint32_t)(kWeightCols<R> >> 3) << 17;

#define LINMT_OUT4(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3])
#define LINMT_OUT8(v, o) LINMT_OUT4(v, o), LINMT_OUT4(v, o + 4)
// Columns of the lane's row of TMEM: three times N, `apart` from each other.
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t apart, int (&v)[3][8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%24];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%25];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%16,%17,%18,%19,%20,%21,%22,%23}, [%26];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LINMT_OUT8(v[0], 0), LINMT_OUT8(v[1], 0), LINMT_OUT8(v[2], 0) : "r"(at), "r"(at + apart), "r"(at + 2 * apart) : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t apart, int (&v)[3][4]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%12];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x4.b32 {%4,%5,%6,%7}, [%13];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x4.b32 {%8,%9,%10,%11}, [%14];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LINMT_OUT4(v[0], 0), LINMT_OUT4(v[1], 0), LINMT_OUT4(v[2], 0) : "r"(at), "r"(at + apart), "r"(at + 2 * apart) : "memory");
}
// N neighbouring ones.
__device__ __forceinline__ void tmem_load(uint32_t at, int (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LINMT_OUT8(v, 0), LINMT_OUT8(v, 8), LINMT_OUT8(v, 16), LINMT_OUT8(v, 24) : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t at, int (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : LINMT_OUT8(v, 0), LINMT_OUT8(v, 8) : "r"(at) : "memory");
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
// cap tanh(x) as cap - 2 cap / (2^y + 1), y = 2 x log2(e): good to 3e-7 of the cap, 2e-5 of a score with a cap of up to kQuickCap, which a 16-bit result does not see.
constexpr float kQuickCap = 64.f;
__device__ __forceinline__ float capped(float y, float cap) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(exp2_of(y) + 1.f));
  return fmaf(-2.f * cap, r, cap);
}
// The N threads of the weights: wait for each other; whether one of them says so.
template <int N>
__device__ __forceinline__ void weights_sync() { asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory"); }
template <int N>
__device__ __forceinline__ bool weights_any(bool x) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, %2, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(r) : "r"((int)x), "n"(N) : "memory");
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
  int begin, end;          // the CTA's units
  int first;               // number of the first unit of sentence `sent`
  int per;                 // units of a part
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
template <int kThreads>
__device__ __forceinline__ Share share_of(const AttendParams& a, int blocks) {
  __shared__ int sums[kThreads / 32], found_first;
  __shared__ int found_lo, found_hi;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, segments = a.pool_heads * a.row_tiles;
  Share s{};
  int lo = 0, hi = a.n;
  bool all = true;
  for (;;) {
    const int each = (hi - lo + kThreads - 1) / kThreads, i0 = min(hi, lo + tid * each), i1 = min(hi, i0 + each);
    int mine = 0;
#pragma unroll 4
    for (int i = i0; i < i1; ++i) mine += seen_of(a, i).units();
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w == warp) upto += total;
      total += sums[w];
    }
    if (all) {
      all = false;
      total *= segments;
      s.per = max(kWhole, (int)(((unsigned)total + blocks - 1) / blocks));
      s.begin = (int)min((int64_t)total, (int64_t)blockIdx.x * s.per);
      s.end = (int)min((int64_t)total, (int64_t)s.begin + s.per);
      s.whole = max(kWhole, s.per / 8);
    }
    if (s.begin >= s.end) return s;
    const int before = s.first + (upto - mine) * segments;
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
  int start;               // number of the segment's first unit
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
    const int in = s.begin - s.first, seg = (int)((uint32_t)in / (uint32_t)p.units);
    if (seg >= segments) {
      s.first += p.units * segments;
      ++s.sent;
      continue;
    }
    p.sent = s.sent;
    p.len = length_of(a, s.sent);
    p.kvh = a.row_tiles == 1 ? seg : seg / a.row_tiles;
    p.rt = seg - p.kvh * a.row_tiles;
    p.start = s.first + seg * p.units;
    p.u0 = s.begin - p.start;
    p.u1 = min(p.units, s.end - p.start);
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
// A piece that is ready to be worked on: its queries and rows are in place.
struct Ready {
  int sent, kvh, rt, len;
  int chunks;              // -1: there are no more pieces
  int c0, n1, b0;          // chunk i is chunk_at(c0 + i) of the sentence
  int whole, part, from;   // part: which of the CTA's two places in the workspace it has; from: first CTA of the segment that ends with it, -1: it ends with another
  __device__ __forceinline__ int position(int i) const { return (c0 + i < n1 ? c0 + i : b0 + c0 + i - n1) * kChunk; }
};
constexpr int kQueryAlong = 128 + 16;        // bytes between cores of the queries along the sum: a lane's four (two) components of them meet different banks
template <int D, int R>
struct Shared {
  static constexpr int KS = kKeyStages<D, R>, VS = kValueStages<D, R>;
  alignas(128) unsigned char keys[KS][kChunk * D];
  alignas(128) unsigned char values[VS][kChunk * D];
  alignas(128) unsigned char queries[2][kQueryCols<R> / 8 * D / 16 * kQueryAlong];      // (behind the values: with 64 components a product's lower half reads a block further, into rows of O that nobody looks at)
  alignas(128) uint4 weights[R / 4][kChunk];                                            // four rows' 32 bits a position
  alignas(128) float scales[VS][2][8][4];                                               // of four blocks, and as much again that is free
  // of the rows of two pieces
  alignas(16) float by[2][R], slope[2][R], centre[2][R];
  alignas(16) int lo[2][R], span[2][R];
  long long out[2][R];
  int bad[2][R];
  Ready ready[2];
  // what the rows' scores, and their weights times scales, are relative to, as it is and as it was before
  alignas(16) float x[2][R], m[2][R], down_x[R], down_m[R], most_x[4][R], most_m[4][R];
  unsigned valid[VS];
  int add, gave_up;
  uint32_t tmem;
  alignas(8) unsigned long long k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], s_full[2], s_empty[2], q_full[2], q_empty[2], p_full, o_full, first;
};

__device__ __forceinline__ void store_as(void* p, int64_t i, int dtype, float x) {
  if (dtype == LINMT_F32) static_cast<float*>(p)[i] = x;
  else if (dtype == LINMT_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dtype) {
  return dtype == LINMT_F32 ? __ldg(static_cast<const float*>(p) + i) : dtype == LINMT_BF16 ? to_float(__ldg(static_cast<const __nv_bfloat16*>(p) + i)) : to_float(__ldg(static_cast<const __half*>(p) + i));
}
// Four neighbouring rows' numbers.
__device__ __forceinline__ void four(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void four(const int* p, int (&x)[4]) {
  const int4 v = *reinterpret_cast<const int4*>(p);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ float power_of_2(int e) { return __int_as_float((127 + e) << 23); }      // -126 .. 127
// A sum of weights, 0 or 2^-1 .. 2^76, as 2^k times something between 1 and 2; NaN goes with k = 0.
__device__ __forceinline__ int exponent_of(float weight) { return weight > 0.f ? (__float_as_int(weight) >> 23) - 127 : 0; }

// What a piece's rows see and where their results go; by a warp, a lane for each row.
template <int D, int R>
__device__ __forceinline__ void take_rows(const AttendParams& a, const Piece& p, Shared<D, R>& sh, int buffer) {
  const int lane = threadIdx.x & 31, row = p.rt * R + lane;
  if (lane >= R) return;
  const bool have = row < a.g * a.rep;
  const int at = have ? row : p.rt * R, g = at / a.rep, h = p.kvh * a.rep + at - g * a.rep;
  const int64_t by_row = (int64_t)p.sent * a.g + g;
  const int lo = a.first && have ? max(__ldg(a.first + by_row), 0) : 0, hi = a.first && have ? min(__ldg(a.last + by_row), p.len) : p.len;
  sh.slope[buffer][lane] = have && a.slope ? __ldg(a.slope + h) * kLog2e : 0.f;
  sh.centre[buffer][lane] = have && a.slope ? __ldg(a.centre + by_row) : 0.f;
  sh.lo[buffer][lane] = lo;
  sh.span[buffer][lane] = max(hi - lo, 0);
  sh.out[buffer][lane] = p.sent * a.o_n + g * a.o_g + h * a.o_h;
}

// A piece's queries from row r0 on as bytes; by a warp, a lane for two or four neighbouring components of each row.
constexpr int kAtOnce = 4;
template <int D, int R>
__device__ __forceinline__ void take_queries(const AttendParams& a, const Piece& p, Shared<D, R>& sh, int buffer, int r0) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31, n_rows = min(R, a.g * a.rep - p.rt * R);
  int64_t from;                                       // of row r0 + lane; rows that are not there have another's queries, and their products are multiplied by 0
  {
    const int at = p.rt * R + min(r0 + lane, n_rows - 1), g = at / a.rep, h = p.kvh * a.rep + at - g * a.rep;
    from = p.sent * a.q_n + g * a.q_g + h * a.q_h;
  }
  float x[kAtOnce][N];
  int64_t at[kAtOnce];
#pragma unroll
  for (int j = 0; j < kAtOnce; ++j) at[j] = __shfl_sync(~0u, (long long)from, j) + lane * N;
  if (!a.q_wide) {
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) x[j][i] = load_as_float(a.q, at[j] + i, a.dtype);
  } else if (a.dtype == LINMT_F32) {
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const float* const q = static_cast<const float*>(a.q) + at[j];
      if constexpr (N == 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(q));
        x[j][0] = v.x; x[j][1] = v.y; x[j][2] = v.z; x[j][3] = v.w;
      } else {
        const float2 v = __ldg(reinterpret_cast<const float2*>(q));
        x[j][0] = v.x; x[j][1] = v.y;
      }
    }
  } else {
    uint32_t raw[kAtOnce][N / 2];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const unsigned short* const q = static_cast<const unsigned short*>(a.q) + at[j];
      if constexpr (N == 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(q));
        raw[j][0] = v.x; raw[j][1] = v.y;
      } else {
        raw[j][0] = __ldg(reinterpret_cast<const uint32_t*>(q));
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float2 v = a.dtype == LINMT_BF16 ? make_float2(__uint_as_float(raw[j][i / 2] << 16), __uint_as_float(raw[j][i / 2] & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&raw[j][i / 2]));
        x[j][i] = v.x;
        x[j][i + 1] = v.y;
      }
  }
  // The rows' largest components, each in a lane, and what it takes to bring them below 2^22: 2^e <= the largest < 2^(e + 1), components times 2^(21 - e).  (Below 2^-106 it stays
  // at that of 2^-106.)
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < kAtOnce; ++j) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(x[j][i]) & 0x7fffffff);
    m = __reduce_max_sync(~0u, m);
    if (lane == j) most = m;
  }
  const bool bad = most >= 0x7f800000;
  const int e = bad ? 0 : max((int)(most >> 23) - 127, -106);
  const float up = bad ? 0.f : power_of_2(21 - e);
  if (lane < kAtOnce) {
    sh.by[buffer][r0 + lane] = r0 + lane < n_rows ? a.mul * power_of_2((e - 21) / 2) * power_of_2(e - 21 - (e - 21) / 2) : 0.f;
    sh.bad[buffer][r0 + lane] = bad;
  }
  // Digits to the base 256, -128 .. 127: with 128 added to each, the bytes of the sum.
#pragma unroll
  for (int j = 0; j < kAtOnce; ++j) {
    const int r = r0 + j;
    const float by = __shfl_sync(~0u, up, j);
    uint32_t u[N];
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = (uint32_t)(__float2int_rn(x[j][i] * by) + 0x808080) ^ 0x808080;
    auto place = [&](int k) { return sh.queries[buffer] + ((k * R + r) / 8 * (D / 16) + lane * N / 16) * kQueryAlong + (k * R + r) % 8 * 16 + lane * N % 16; };
    if constexpr (N == 4) {
      const uint32_t low01 = __byte_perm(u[0], u[1], 0x5140), low23 = __byte_perm(u[2], u[3], 0x5140);
      *reinterpret_cast<uint32_t*>(place(0)) = __byte_perm(low01, low23, 0x5410);
      *reinterpret_cast<uint32_t*>(place(1)) = __byte_perm(low01, low23, 0x7632);
      *reinterpret_cast<uint32_t*>(place(2)) = __byte_perm(__byte_perm(u[0], u[1], 0x0062), __byte_perm(u[2], u[3], 0x0062), 0x5410);
    } else {
      const uint32_t low = __byte_perm(u[0], u[1], 0x5140);
      *reinterpret_cast<uint16_t*>(place(0)) = (uint16_t)low;
      *reinterpret_cast<uint16_t*>(place(1)) = (uint16_t)(low >> 16);
      *reinterpret_cast<uint16_t*>(place(2)) = (uint16_t)__byte_perm(u[0], u[1], 0x0062);
    }
  }
}

template <int D, int R, int HOW>
__global__ void __launch_bounds__(kThreads<R>) __maxnreg__(65536 / (kThreads<R> * kCtas<R>) / 8 * 8) attend_kernel(const __grid_constant__ AttendParams a, const __grid_constant__ AttendMaps maps) {
  extern __shared__ __align__(128) unsigned char attend_smem[];
  Shared<D, R>& sh = *reinterpret_cast<Shared<D, R>*>(attend_smem);
  constexpr int KS = kKeyStages<D, R>, VS = kValueStages<D, R>, kPart = R * (D + 2), RT = kRows<R>, kWeights = 32 * kWeightWarps<R>, kCopyWarp = kWeightWarps<R>, kIssueWarp = kCopyWarp + 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(~0u, tid >> 5, 0);
  if (tid == 0) {
    for (int i = 0; i < KS; ++i) {
      bar_init(shared(&sh.k_full[i]), 1);
      bar_init(shared(&sh.k_empty[i]), 1);
    }
    for (int i = 0; i < VS; ++i) {
      bar_init(shared(&sh.v_full[i]), 1);
      bar_init(shared(&sh.v_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(shared(&sh.s_full[i]), 1);
      bar_init(shared(&sh.s_empty[i]), kWeightWarps<R>);
      bar_init(shared(&sh.q_full[i]), 1);
      bar_init(shared(&sh.q_empty[i]), 1 + kWeightWarps<R>);
    }
    bar_init(shared(&sh.p_full), kWeightWarps<R>);
    bar_init(shared(&sh.o_full), 1);
    bar_init(shared(&sh.first), kWeightWarps<R>);
    sh.gave_up = a.give_up && blockIdx.x % (unsigned)a.give_up == 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared(&sh.tmem)), "r"(kTmemCols<R>) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  launch_next();
  Share share = share_of<kThreads<R>>(a, gridDim.x);
  tmem_before();
  __syncthreads();
  tmem_after();
  const uint32_t tmem = sh.tmem;
  volatile int* const gave_up = &sh.gave_up;

  if (warp == kCopyWarp) {
    // ---- blocks into the rings, four with a copy where the pool is rows of whole blocks (eight documents of 20-32k: 110 us with a bulk copy for each
    // block's keys, values and scales, which a warp issues every 50 to 100 cycles); behind a piece's first chunk its queries
    const bool elected = elect_one();
    Piece p;
    int it = 0, pieces = 0;
    auto announce = [&](int chunks) {
      const int buffer = pieces & 1;
      bar_wait(shared(&sh.q_empty[buffer]), (pieces >> 1 & 1) ^ 1, gave_up);
      __syncwarp();
      if (!*gave_up) {
        if (chunks > 0) {
          take_rows<D, R>(a, p, sh, buffer);
          if (pieces == 0) bar_wait(shared(&sh.first), 0, gave_up);
          else
#pragma unroll 1
            for (int r0 = 0; r0 < R; r0 += kAtOnce) take_queries<D, R>(a, p, sh, buffer, r0);
        }
        if (lane == 0) {
          Ready& r = sh.ready[buffer];
          r.chunks = chunks;
          if (chunks >= 0) {
            r.sent = p.sent; r.kvh = p.kvh; r.rt = p.rt; r.len = p.len;
            r.c0 = p.c0; r.n1 = p.seen.n1; r.b0 = p.seen.b0;
            r.whole = p.whole();
            r.part = p.u0 == 0;
            r.from = !p.whole() && p.u0 > 0 && p.u1 == p.units ? p.start / share.per : -1;
          }
        }
        if (chunks == 0 && lane < R) {                 // (nothing to multiply: only where the zeros go)
          const int at = min(p.rt * R + lane, a.g * a.rep - 1), g = at / a.rep;
          sh.out[buffer][lane] = p.sent * a.o_n + g * a.o_g + (p.kvh * a.rep + at - g * a.rep) * a.o_h;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(shared(&sh.q_full[buffer]));
      }
      ++pieces;
    };
    while (next_piece(a, share, p)) {
      const int32_t* const table = a.table + p.sent * a.table_stride;
      const int blocks = (p.len + pages8::kBlock - 1) / pages8::kBlock, per_page = a.page / pages8::kBlock;
      auto page_at = [&](int c, int& in) {            // page and block of it that the lane has of a chunk, -1: none
        const int block = p.seen.chunk(c) * kBlocks + lane, column = block / per_page;
        in = block - column * per_page;
        const int page = c < p.c1 && lane < kBlocks && block < blocks ? __ldg(table + column) : -1;
        return page < a.n_pages ? page : -1;
      };
      int next_in, next = page_at(p.c0, next_in);
      for (int c = p.c0; c < p.c1; ++c, ++it) {
        const int ks = it % KS, vs = it % VS, page = next, in = next_in;
        const unsigned valid = __ballot_sync(~0u, page >= 0);
        next = page_at(c + 1, next_in);
        const uint32_t k_full = shared(&sh.k_full[ks]), v_full = shared(&sh.v_full[vs]), to_k = shared(sh.keys[ks]), to_v = shared(sh.values[vs]);
        if (a.rows) {
          // A row that is not there reads as zeros.
          const int row = page >= 0 ? page * a.row_page + p.kvh * a.row_head + in : a.rows;
          int r[kBlocks];
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) r[i] = __shfl_sync(~0u, row, i);
          bar_wait(shared(&sh.k_empty[ks]), (it / KS & 1) ^ 1, gave_up);
          __syncwarp();
          if (elected && !*gave_up) {
            bar_expect(k_full, kBlocks * 16 * D);
            copy_rows(to_k, &maps.codes, 0, r[0], r[1], r[2], r[3], k_full);
            copy_rows(to_k + 4 * 16 * D, &maps.codes, 0, r[4], r[5], r[6], r[7], k_full);
          }
          bar_wait(shared(&sh.v_empty[vs]), (it / VS & 1) ^ 1, gave_up);
          __syncwarp();
          if (elected && !*gave_up) {
            sh.valid[vs] = valid;
            bar_expect(v_full, kBlocks * (16 * D + 16));
            copy_rows(shared(sh.scales[vs][0]), &maps.scales, 32 * D / 8, r[0], r[1], r[2], r[3], v_full);
            copy_rows(shared(sh.scales[vs][1]), &maps.scales, 32 * D / 8, r[4], r[5], r[6], r[7], v_full);
            copy_rows(to_v, &maps.codes, 16 * D / 8, r[0], r[1], r[2], r[3], v_full);
            copy_rows(to_v + 4 * 16 * D, &maps.codes, 16 * D / 8, r[4], r[5], r[6], r[7], v_full);
          }
        } else {
          const unsigned char* const block = a.data + page * a.stride_page + p.kvh * a.stride_head + (int64_t)in * pages8::block_bytes(D);
          const int count = __popc(valid);
          bar_wait(shared(&sh.k_empty[ks]), (it / KS & 1) ^ 1, gave_up);
          __syncwarp();
          if (!*gave_up) {
            if (lane == 0) bar_expect(k_full, count * 16 * D);
            __syncwarp();
            if (page >= 0) copy_bulk(to_k + lane * 16 * D, block, 16 * D, k_full);
          }
          bar_wait(shared(&sh.v_empty[vs]), (it / VS & 1) ^ 1, gave_up);
          __syncwarp();
          if (!*gave_up) {
            if (lane == 0) {
              sh.valid[vs] = valid;
              bar_expect(v_full, count * (16 * D + 16));
            }
            __syncwarp();
            if (page >= 0) {
              copy_bulk(shared(sh.scales[vs][lane / 4][lane % 4]), block + pages8::scales(D), 16, v_full);
              copy_bulk(to_v + lane * 16 * D, block + pages8::value_codes(D), 16 * D, v_full);
            }
          }
        }
        if (c == p.c0) announce(p.c1 - p.c0);
      }
      if (p.c0 == p.c1) announce(0);
    }
    announce(-1);
    if (*gave_up) {                                   // what is on its way still lands in this CTA's memory
      const unsigned long long t0 = clock64();
      while ((unsigned long long)clock64() - t0 < kWaitCycles / 100) {}
    }
  } else if (warp == kIssueWarp) {
    // ---- the products
    const bool elected = elect_one();
    int it = 0;
    auto weights_times_values = [&](int i) {
      const int vs = i % VS;
      bar_wait(shared(&sh.p_full), i & 1, gave_up);
      bar_wait(shared(&sh.v_full[vs]), i / VS & 1, gave_up);
      __syncwarp();
      tmem_after();
      if (elected && !*gave_up) {
        const uint32_t add = *(volatile int*)&sh.add;
        const uint64_t left = operand(shared(sh.values[vs]), 16 * D, 128), right = operand(shared(sh.weights), 128, 16 * kChunk);
#pragma unroll
        for (int k = 0; k < kChunk / 32; ++k)
          mma_bytes(tmem + kTmemO<R>, left + (uint64_t)(k * 2 * 16 * D >> 4), right + (uint64_t)(k * 4 * 128 >> 4), kWeightForm<R>, k ? 1u : add);
        commit(shared(&sh.v_empty[vs]));
        commit(shared(&sh.o_full));
      }
      __syncwarp();
    };
    for (int pieces = 0;; ++pieces) {
      const int buffer = pieces & 1;
      bar_wait(shared(&sh.q_full[buffer]), pieces >> 1 & 1, gave_up);
      const int chunks = *(volatile int*)&sh.ready[buffer].chunks;
      if (chunks < 0 || *gave_up) break;
      for (int c = 0; c < chunks; ++c, ++it) {
        const int ks = it % KS, half = it & 1;
        bar_wait(shared(&sh.k_full[ks]), it / KS & 1, gave_up);
        bar_wait(shared(&sh.s_empty[half]), (it >> 1 & 1) ^ 1, gave_up);
        __syncwarp();
        tmem_after();
        if (elected && !*gave_up) {
          const uint64_t left = operand(shared(sh.keys[ks]), 128, 8 * D), right = operand(shared(sh.queries[buffer]), kQueryAlong, D / 16 * kQueryAlong);
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
            mma_bytes(tmem + half * kQueryCols<R>, left + (uint64_t)(k * 2 * 128 >> 4), right + (uint64_t)(k * 2 * kQueryAlong >> 4), kQueryForm<R>, k ? 1u : 0u);
          commit(shared(&sh.k_empty[ks]));
          commit(shared(&sh.s_full[half]));
          if (c + 1 == chunks) commit(shared(&sh.q_empty[buffer]));
        }
        __syncwarp();
        if (c > 0) weights_times_values(it - 1);
      }
      if (chunks) weights_times_values(it - 1);
      else if (lane == 0) bar_arrive(shared(&sh.q_empty[buffer]));
    }
  } else {
    // ---- scores to weights, a position for each thread; then a component for each thread
    const int mine = tid & (kChunk - 1), row0 = warp / 4 * RT;      // the thread's position, or component, and its first row
    const uint32_t lanes = tmem + ((uint32_t)(warp % 4 * 32) << 16);
    const float slack = (float)a.slack, unit = power_of_2(a.slack - 31);
    int it = 0, pieces = 0;
    // The first piece's queries are made ready by these warps, which have nothing else to do yet; later ones by the warp that copies.  (All by that one: 5400 cycles with 16 rows.)
    {
      Piece first;
      Share s = share;
      if (next_piece(a, s, first) && first.c0 < first.c1 && warp * kAtOnce < R) take_queries<D, R>(a, first, sh, 0, warp * kAtOnce);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(shared(&sh.first));
    }
    int4 ends = make_int4(-1, 0, 0, 0);               // the segment that ends in this share and began before it: sentence, head, row tile, first CTA
    for (;; ++pieces) {
      const int buffer = pieces & 1;
      bar_wait(shared(&sh.q_full[buffer]), pieces >> 1 & 1, gave_up);
      if (weights_any<kWeights>(*gave_up)) break;
      const Ready p = sh.ready[buffer];
      if (p.chunks < 0) break;
      const int n_rows = min(R, a.g * a.rep - p.rt * R);
      int now = 0, since = 0;                         // which of x and m; chunks in O
      if (tid < R) {
        sh.x[0][tid] = kLowest;
        sh.m[0][tid] = 0.f;
      }
      weights_sync<kWeights>();
      float sum[RT], acc[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) sum[r] = acc[r] = 0.f;
      for (int c = 0;; ++c, ++it) {
        const bool last = c == p.chunks;
        if (last && since == 0) break;
        float s[RT], ve = 0.f, vf = 0.f;
        bool over = last || since == kDrain;
        if (!last) {
          const int vs = it % VS, half = it & 1;
          bar_wait(shared(&sh.v_full[vs]), it / VS & 1, gave_up);
          bar_wait(shared(&sh.s_full[half]), it >> 1 & 1, gave_up);
          tmem_after();
          int t[kQueryDigits][RT];
          tmem_load(lanes + half * kQueryCols<R> + row0, R, t);
          tmem_before();
          __syncwarp();
          if (lane == 0) bar_arrive(shared(&sh.s_empty[half]));

          const int at = mine / pages8::kBlock, pos = p.position(c) + mine;
          // A block that is not there has left whatever was in its place before; what lies behind a sentence's end may be anything.
          const bool there = pos < p.len && (sh.valid[vs] >> at & 1);
          const float2 scales = *reinterpret_cast<const float2*>(sh.scales[vs][at / 4][at % 4]);
          const float ks = there ? scales.x : 0.f, none = there ? 0.f : -INFINITY;
          const uint32_t scale = there ? __float_as_uint(scales.y) : 0;
          // the values' scale as 2^ve times vf, and in vf 1 / unit
          ve = scale ? (float)((int)(scale >> 23 & 255) - 127) : -1000.f;
          vf = scale ? __uint_as_float((scale & 0x7fffff) | (uint32_t)(127 + 31 - a.slack) << 23) : 0.f;
          float most = -INFINITY;
#pragma unroll
          for (int r4 = 0; r4 < RT; r4 += 4) {
            if (r4 > 0 && row0 + r4 >= n_rows) {       // four rows that are not there
#pragma unroll
              for (int j = 0; j < 4; ++j) s[r4 + j] = -INFINITY;
              break;
            }
            float by[4], x[4], m[4], slope[4], centre[4];
            int lo[4], span[4];
            four(sh.by[buffer] + row0 + r4, by);
            four(sh.x[now] + row0 + r4, x);
            four(sh.m[now] + row0 + r4, m);
            if constexpr (HOW != kPlain) {
              four(sh.slope[buffer] + row0 + r4, slope);
              four(sh.centre[buffer] + row0 + r4, centre);
            }
            if (a.first) {
              four(sh.lo[buffer] + row0 + r4, lo);
              four(sh.span[buffer] + row0 + r4, span);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int r = r4 + j;
              const float whole = fmaf((float)t[2][r], 65536.f, (float)(t[1][r] * 256 + t[0][r]));
              if constexpr (HOW == kPlain) {
                s[r] = fmaf(whole, by[j] * ks, none);
              } else {
                float y = whole * (by[j] * ks);
                if constexpr (HOW == kQuick) {
                  if (a.cap > 0.f) y = capped(y, a.cap * kLog2e);
                } else {
                  if (a.cap > 0.f) y = a.cap * kLog2e * tanhf(y);
                }
                s[r] = y - slope[j] * fabsf((float)pos - centre[j]) + none;
              }
              if (a.first) s[r] = (unsigned)(pos - lo[j]) < (unsigned)span[j] || pos < a.sinks ? s[r] : -INFINITY;
              const float d = s[r] - x[j];
              most = fmaxf(most, fmaxf(d + (ve - m[j]), d - kAbove));
            }
          }
          over = weights_any<kWeights>(most > slack) || over;
          if (c > 0) bar_wait(shared(&sh.o_full), it - 1 & 1, gave_up);
          // Something exceeds what the rows' weights are relative to: that follows.
          if (over) {
            float most_x = kLowest, most_m = kLowest;      // of row row0 + lane: the warp's largest score, and the largest sum of a scale's exponent and a score's distance from that, as a sum with a
                                                           // far score itself has no bits left for it
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              const float x = fmaxf(warp_max(s[r]), kLowest), y = warp_max(s[r] - x + ve);
              if (lane == r) { most_x = x; most_m = y; }
            }
            if (lane < RT) { sh.most_x[warp % 4][row0 + lane] = most_x; sh.most_m[warp % 4][row0 + lane] = most_m; }
            weights_sync<kWeights>();
            if (tid < R) {
              const float was_x = sh.x[now][tid], x0 = sh.most_x[0][tid], x1 = sh.most_x[1][tid], x2 = sh.most_x[2][tid], x3 = sh.most_x[3][tid], top_x = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3));
              const float x = top_x - was_x > kAbove + slack ? ceilf(top_x) : was_x, was = was_x - x + sh.m[now][tid];
              const float top = fmaxf(fmaxf(x0 - x + sh.most_m[0][tid], x1 - x + sh.most_m[1][tid]), fmaxf(x2 - x + sh.most_m[2][tid], x3 - x + sh.most_m[3][tid]));
              const float m = top - was > slack ? ceilf(top) : was;
              sh.x[now ^ 1][tid] = x;
              sh.m[now ^ 1][tid] = m;
              sh.down_x[tid] = exp2_of(was_x - x);
              sh.down_m[tid] = exp2_of(was - m);
            }
            weights_sync<kWeights>();
            now ^= 1;
          }
        } else {
          bar_wait(shared(&sh.o_full), it - 1 & 1, gave_up);
        }
        if (over) {
          // O's integers into sums, which are relative to 2^M then.
          tmem_after();
          int o[kWeightDigits * RT];
          if (since) tmem_load(lanes + kTmemO<R> + kWeightDigits * row0, o);
#pragma unroll
          for (int r4 = 0; r4 < RT; r4 += 4) {
            float down_x[4], down_m[4];
            four(sh.down_x + row0 + r4, down_x);
            four(sh.down_m + row0 + r4, down_m);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int* const x = o + 4 * (r4 + j);
              const float v = fmaf((float)x[3], 16777216.f, fmaf((float)x[2], 65536.f, fmaf((float)x[1], 256.f, (float)x[0])));
              if (since) acc[r4 + j] = fmaf(v, unit, acc[r4 + j]);
              if (!last) {
                acc[r4 + j] *= down_m[j];
                sum[r4 + j] *= down_x[j];
              }
            }
          }
          tmem_before();
          since = 0;
        }
        if (last) break;
#pragma unroll
        for (int r4 = 0; r4 < RT; r4 += 4) {
          float x[4], m[4];
          uint32_t w[4];
          if (r4 > 0 && row0 + r4 >= n_rows) {
            sh.weights[(row0 + r4) / 4][mine] = make_uint4(0, 0, 0, 0);
            break;
          }
          four(sh.x[now] + row0 + r4, x);
          four(sh.m[now] + row0 + r4, m);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float d = s[r4 + j] - x[j];
            sum[r4 + j] += exp2_of(d);
            w[j] = __float2uint_rn(exp2_of(d + (ve - m[j])) * vf);
          }
          sh.weights[(row0 + r4) / 4][mine] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (tid == 0) sh.add = since > 0;
        ++since;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(shared(&sh.p_full));
      }
      // The rows' sums of weights, and out with it.
      if (p.chunks) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) sum[r] += __shfl_xor_sync(~0u, sum[r], o);
          if (lane == r) sh.most_m[warp % 4][row0 + r] = sum[r];
        }
      }
      weights_sync<kWeights>();
      // a part of the workspace: [row][D] values, [row] exponent, [row] weight.  A CTA's first is of the segment that it has from the CTA before, its second of the one that the next goes on with.
      float* const ws = a.ws + ((int64_t)blockIdx.x * 2 + p.part) * kPart;
      if (tid < R) {
        // 2^M / weight, as values of up to 2^127 ask for it, is no number of 32 bits: two factors, the first a power of 2.
        float weight = 0.f, x = kLowest, f = 0.f;
        int e = 0;
        if (p.chunks) {
          weight = sh.most_m[0][tid] + sh.most_m[1][tid] + sh.most_m[2][tid] + sh.most_m[3][tid];
          x = sh.x[now][tid];
          const int k = exponent_of(weight);
          e = min(max((int)fmaxf(sh.m[now][tid], -1000.f) - k, -250), 250);
          const float one = weight * power_of_2(-k);
          f = weight == 0.f ? 0.f : power_of_2(e - e / 2) / one;
          if (x + (float)k - x == (float)k) { x += (float)k; weight = one; }      // between 1 and 2 then, where x has a place for k's last bits
          if ((sh.bad[buffer][tid] && weight > 0.f) || *gave_up) f = weight = NAN;
        }
        sh.down_x[tid] = power_of_2(e / 2);
        sh.down_m[tid] = f;
        if (tid < n_rows) {
          if (p.whole) {
            const int row = p.rt * R + tid, g = row / a.rep;
            if (a.lse) a.lse[((int64_t)p.sent * a.g + g) * a.heads + p.kvh * a.rep + row - g * a.rep] = weight == 0.f ? -INFINITY : (x + log2f(weight)) * kLn2;
          } else {
            ws[R * D + tid] = x;
            ws[R * D + R + tid] = weight;
          }
        }
      }
      weights_sync<kWeights>();
      if (mine < D) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float value = acc[r] * sh.down_x[row0 + r] * sh.down_m[row0 + r];
          if (row0 + r < n_rows) {
            if (p.whole) store_as(a.out, sh.out[buffer][row0 + r] + mine, a.dtype, value);
            else ws[(row0 + r) * D + mine] = value;
          }
        }
      }
      if (p.from >= 0) ends = make_int4(p.sent, p.kvh, p.rt, p.from);
      __syncwarp();
      if (lane == 0) bar_arrive(shared(&sh.q_empty[buffer]));
    }
    if (*gave_up) {                                   // what there is from here on is NaN
      Piece p;
      for (Share s = share; next_piece(a, s, p);) {
        for (int r = 0; r < min(R, a.g * a.rep - p.rt * R); ++r) {
          const int row = p.rt * R + r, g = row / a.rep, h = p.kvh * a.rep + row - g * a.rep;
          if (p.whole()) {
            if (tid < D) store_as(a.out, p.sent * a.o_n + g * a.o_g + h * a.o_h + tid, a.dtype, NAN);
            if (tid == 0 && a.lse) a.lse[((int64_t)p.sent * a.g + g) * a.heads + h] = NAN;
          } else if (tid == 0) {
            float* const ws = a.ws + ((int64_t)blockIdx.x * 2 + (p.u0 == 0)) * kPart;
            ws[R * D + r] = 0.f;
            ws[R * D + R + r] = NAN;
          }
        }
        if (!p.whole() && p.u0 > 0 && p.u1 == p.units) ends = make_int4(p.sent, p.kvh, p.rt, p.start / s.per);
      }
    }
    if (a.ws && tid == 0) reinterpret_cast<int4*>(a.ws + (int64_t)gridDim.x * 2 * kPart)[blockIdx.x] = ends;
  }
  tmem_before();
  __syncthreads();
  if (warp == kIssueWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols<R>) : "memory");
}

// Joins the parts of the segment that ends in a CTA's share and began in one before: a CTA for each of attend's.  A thread has four components of a row, in one of kBy
// parts in turn.
constexpr int kJoinThreads = 512;
template <int D, int R>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(const __grid_constant__ AttendParams a, int blocks) {
  constexpr int kPart = R * (D + 2), kBy = kJoinThreads / (R * D / 4);
  __shared__ float s_x[kBy][R], s_k[kBy][R], s_weight[kBy][R];
  __shared__ float4 s_sum[kBy][R * D / 4];
  const int at = threadIdx.x % (R * D / 4), by = threadIdx.x / (R * D / 4), r = at / (D / 4), d = at % (D / 4) * 4;
  wait_for_last();
  const int4 ends = reinterpret_cast<const int4*>(a.ws + (int64_t)blocks * 2 * kPart)[blockIdx.x];
  if (ends.x < 0) return;
  const int from = ends.w, n_parts = (int)blockIdx.x - from + 1;
  auto part = [&](int i) { return a.ws + ((int64_t)(from + i) * 2 + (i == 0)) * kPart; };
  // The largest exponent so far goes along, and the largest sum of weights, so that every part is waited for once: eight of them at a time are on their way.  A part's share is relative
  // to 2^(x + k), k that sum's exponent, and 2^fewer times smaller, so that values of up to 2^127 have room; x may have no place for k's last bits.
  const float fewer = (float)(33 - __clz(n_parts));
  float x = kLowest, most = 0.f, k = 0.f, weight = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = by; i0 < n_parts; i0 += 8 * kBy) {
    float m[8], l[8];
    float4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = kLowest;
      l[j] = 0.f;
      if (i0 + j * kBy < n_parts) {
        const float* const w = part(i0 + j * kBy);
        m[j] = w[R * D + r];
        l[j] = w[R * D + R + r];
        v[j] = *reinterpret_cast<const float4*>(w + r * D + d);
      }
    }
    const float was_x = x, was_k = k;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x = fmaxf(x, m[j]);
      most = fmaxf(most, l[j]);
    }
    k = (float)exponent_of(most);
    const float f0 = exp2_of(was_x - x + (was_k - k));
    weight *= f0;
    sum.x *= f0; sum.y *= f0; sum.z *= f0; sum.w *= f0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (i0 + j * kBy >= n_parts) break;
      const float f = exp2_of(m[j] - x - k - fewer) * l[j];
      sum.x += f * v[j].x; sum.y += f * v[j].y; sum.z += f * v[j].z; sum.w += f * v[j].w;
      weight += f;
    }
  }
  s_sum[by][at] = sum;
  if (d == 0) { s_x[by][r] = x; s_k[by][r] = k; s_weight[by][r] = weight; }
  __syncthreads();
  if (by || r >= a.g * a.rep - ends.z * R) return;
#pragma unroll
  for (int i = 1; i < kBy; ++i) {
    x = fmaxf(x, s_x[i][r]);
    k = fmaxf(k, s_k[i][r]);
  }
  sum = make_float4(0.f, 0.f, 0.f, 0.f);
  weight = 0.f;
#pragma unroll
  for (int i = 0; i < kBy; ++i) {
    const float f = exp2_of(s_x[i][r] - x + (s_k[i][r] - k));
    const float4 v = s_sum[i][at];
    sum.x += f * v.x; sum.y += f * v.y; sum.z += f * v.z; sum.w += f * v.w;
    weight += f * s_weight[i][r];
  }
  const int row = ends.z * R + r, g = row / a.rep, h = ends.y * a.rep + row - g * a.rep;
  const float f = weight == 0.f ? 0.f : 1.f / weight;
  const int64_t to = ends.x * a.o_n + g * a.o_g + h * a.o_h + d;
  store_as(a.out, to, a.dtype, sum.x * f);
  store_as(a.out, to + 1, a.dtype, sum.y * f);
  store_as(a.out, to + 2, a.dtype, sum.z * f);
  store_as(a.out, to + 3, a.dtype, sum.w * f);
  if (d == 0 && a.lse) a.lse[((int64_t)ends.x * a.g + g) * a.heads + h] = weight == 0.f ? -INFINITY : (x + (k + fewer + log2f(weight))) * kLn2;
}

template <int D, int R>
cudaError_t launch_attend(AttendParams p, const AttendMaps& maps, float scale, int blocks, cudaStream_t st) {
  constexpr int smem = (int)sizeof(Shared<D, R>);
  static_assert((smem + 1280) * kCtas<R> <= 228 << 10, "so many CTAs have to fit on an SM");
  const Scores how = p.cap == 0.f && !p.slope ? kPlain : p.dtype == LINMT_F32 || p.cap > kQuickCap ? kExact : kQuick;
  void (*const kernel)(AttendParams, AttendMaps) = how == kPlain ? attend_kernel<D, R, kPlain> : how == kQuick ? attend_kernel<D, R, kQuick> : attend_kernel<D, R, kExact>;
  p.mul = (float)(p.cap == 0.f ? scale * 1.4426950408889634 : how == kQuick ? scale * 2.8853900817779268 / p.cap : (double)scale / p.cap);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)blocks, kThreads<R>, smem, st>>>(p, maps);
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
  e = cudaLaunchKernelEx(&cfg, attend_join_kernel<D, R>, p, blocks);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}
// The pool as a tensor of rows of blocks, where its strides are whole blocks; false where they are not.
bool rows_of_blocks(const linmt_pages8& pool, AttendParams& p, AttendMaps& maps) {
  const int64_t block = pages8::block_bytes(pool.dim);
  const int64_t page = pool.n_pages > 1 ? pool.stride_page : 0, head = pool.heads > 1 ? pool.stride_head : 0;
  if (page < 0 || head < 0 || page % block || head % block) return false;
  const int64_t rows = (pool.n_pages - 1) * (page / block) + (pool.heads - 1) * (head / block) + pool.page / pages8::kBlock;
  if (rows >= INT32_MAX || !encoder()) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)block / 8, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)block};
  const cuuint32_t codes[2] = {(cuuint32_t)(2 * pool.dim), 1}, scales[2] = {2, 1}, step[2] = {1, 1};
  auto encode = [&](CUtensorMap* map, const cuuint32_t* box) {
    return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 2, pool.data, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (!encode(&maps.codes, codes) || !encode(&maps.scales, scales)) return false;
  p.row_page = (int)(page / block);
  p.row_head = (int)(head / block);
  p.rows = (int)rows;
  return true;
}

// Rows of a head of the pool that go together: what there are, up to 16.
int rows_of(const linmt_attend_pages8_args* g) { const int64_t all = (int64_t)g->g * (g->heads / g->pages.heads); return all <= 4 ? 4 : all <= 8 ? 8 : 16; }
int row_tiles_of(const linmt_attend_pages8_args* g) { return (int)(((int64_t)g->g * (g->heads / g->pages.heads) + rows_of(g) - 1) / rows_of(g)); }
template <int D>
cudaError_t launch_rows(const AttendParams& p, const AttendMaps& maps, const linmt_attend_pages8_args* g, int blocks, cudaStream_t st) {
  const int rows = rows_of(g);
  return rows == 4 ? launch_attend<D, 4>(p, maps, g->scale, blocks, st) : rows == 8 ? launch_attend<D, 8>(p, maps, g->scale, blocks, st) : launch_attend<D, 16>(p, maps, g->scale, blocks, st);
}

int64_t chunks_at_most(const linmt_attend_pages8_args* g) { return ((int64_t)g->width * g->pages.page + kChunk - 1) / kChunk; }
// CTAs: as many as fit on the GPU at once, or as the longest possible sentences give kWhole units each.
int blocks_of(const linmt_attend_pages8_args* g) {
  const int64_t segments = (int64_t)g->n * g->pages.heads * row_tiles_of(g), most = segments * ((chunks_at_most(g) + kFixed + kWhole - 1) / kWhole), fit = 148 * (rows_of(g) == 4 ? kCtas<4> : kCtas<16>);
  return (int)(most < fit ? most : fit);
}
// Two parts for each CTA, of the segments that it shares with the CTAs before and behind it, and what the join has to know.  None where no segment can be long enough to be cut.
int64_t workspace_of(const linmt_attend_pages8_args* g) {
  return chunks_at_most(g) + kFixed <= kWhole ? 0 : (int64_t)blocks_of(g) * (2 * (rows_of(g) * (g->pages.dim + 2)) * 4 + 16);
}

thread_local int give_up_each = 0;

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
  if ((int64_t)g->g * g->heads > INT32_MAX / 2 || (int64_t)g->n * g->pages.heads * row_tiles_of(g) > (1 << 24) || (int64_t)g->n * g->pages.heads * row_tiles_of(g) * (chunks_at_most(g) + kFixed) > INT32_MAX / 2)
    return op_fail(LINMT_ELIMIT, "attend_pages8: %d sentences of %d rows, %d heads and %d columns of pages are too many for one call", g->n, g->g, g->heads, g->width);
  return LINMT_OK;
}

}  // namespace
}  // namespace ops
}  // namespace linmt

extern "C" {

int linmt_k_attend8_give_up(int32_t each) {
  if (each < 0) return LINMT_EINVAL;
  linmt::ops::give_up_each = each;
  return LINMT_OK;
}

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
  AttendParams p{static_cast<const unsigned char*>(g->pages.data), g->pages.stride_page, g->pages.stride_head, g->pages.n_pages, g->pages.heads, g->pages.page,
                       g->q, g->q_stride_n, g->q_stride_g, g->q_stride_h, g->out, g->out_stride_n, g->out_stride_g, g->out_stride_h, g->lse, g->table, g->table_stride, g->len,
                       g->slope, g->centre, g->first, g->last, need ? static_cast<float*>(g->workspace) : nullptr, g->n, g->g, g->heads, g->heads / g->pages.heads, g->width, row_tiles_of(g),
                       g->sinks, g->first && g->g <= 32 && (int64_t)g->n * g->g <= 65536, g->dtype,
                       aligned(g->q, 16) && (g->q_stride_n | g->q_stride_g | g->q_stride_h) % (16 / dtype_bytes(g->dtype)) == 0, g->cap, 0.f, 0, 0, 0, g->dtype == LINMT_F32 ? 1 : 4, give_up_each};
  AttendMaps maps{};
  rows_of_blocks(g->pages, p, maps);
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  const cudaError_t e = g->pages.dim == 64 ? launch_rows<64>(p, maps, g, blocks_of(g), st) : launch_rows<128>(p, maps, g, blocks_of(g), st);
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "attend_pages8");
}

}  // extern "C"
