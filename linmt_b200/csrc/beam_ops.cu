// beam_ops.cu -- beam selection and reordering on device tensors (linmt_beam_select, linmt_beam_reorder).
#include <cooperative_groups.h>

#include <type_traits>

#include "device_ops.h"

namespace cg = cooperative_groups;

namespace linmt {
namespace ops {

char* op_error_text() {
  static thread_local char text[kOpErrorBytes] = "";
  return text;
}

namespace {

// ---- selection ---------------------------------------------------------------------------------
//
// One cluster of C CTAs per sentence.  The work of a sentence is its live rows, each cut into as many stretches as there are warps for
// it; the cluster's CTAs exchange what they find through distributed shared memory, so a step is one launch without a workspace.
//   1  A warp reads its stretch once: per lane the running maximum and the sum of exponentials relative to it, and where
//      the lane's maximum lies; per chunk of 128 vectors the maximum.
//   2  Every CTA has the normalisers of all rows.  A lane's best is a bid, a candidate's sum with an upper bound of its index; the
//      `need`-th best bid of the cluster is a bar that at least need = k + kBeyond candidates reach.
//   3  Only the chunks whose maximum can reach the bar are read again (some `need` of hundreds, from L2).
//   4  The candidates found, some dozens, are ranked by counting.
// Sums are compared in 64 bits (as integers of the same order: a comparison of two doubles costs several times one of two integers), but
// exponentials cost five instructions in 32 bits and twenty in 64, and the logits arrive at a rate that allows for the former.  So the
// normaliser is summed in 32 bits with a bound on its error (row_error); where two neighbours of the final order come from different rows and
// lie closer than twice that, their rows' normalisers are summed once more to 2^-36 (PairSum) and the steps from 2 on repeat.
constexpr int kMaxC = 8;
constexpr int kMaxK = 32;
constexpr int kWarps = 12;                       // 96 of a cluster of 8: 12 beams leave none without a stretch, 5, 7, 16, 31 few
constexpr int kBeyond = 8;                       // candidates past the k-th that the order is checked on
constexpr int kChunkVecs = 128;                  // a warp's step: four 16-byte vectors a lane
constexpr int kMaxima = 64;                      // maxima that a warp keeps: of one chunk each, of more where its stretch has more
constexpr int kMany = 128;                       // candidates of a CTA that are listed as they are found; of more the best `need`:
constexpr int kFound = 512;                      // of up to so many by ranking them, of more one by one
constexpr int kMaxList = kMaxC * kMany + kMaxK;  // kMany places for each CTA; finished rows add one each
constexpr int kSorted = 64;                      // of them that are put in order (>= need)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLeastRef = -92.f;               // -64 log2 e, rounded
typedef long long Key;                           // a sum, as an integer that is ordered alike
constexpr Key kNone = -0x7fffffffffffffffll - 1; // below every sum

__device__ __forceinline__ Key key_of(double sum) {
  const long long b = __double_as_longlong(sum + 0.0);      // (-0 counts as 0)
  return b ^ ((b >> 63) & 0x7fffffffffffffffll);
}
__device__ __forceinline__ double sum_of_key(Key k) { return __longlong_as_double(k ^ ((k >> 63) & 0x7fffffffffffffffll)); }
// A candidate is its key and `at` = row * vocab + word.
__device__ __forceinline__ bool before(Key s, int32_t at, Key s2, int32_t at2) { return (s > s2) | ((s == s2) & (at < at2)); }
// The same among bids, whose index is a bound that two may share: those go by their place in the list, so that ranks are distinct.
__device__ __forceinline__ bool bid_before(Key s, int32_t at, int i, Key s2, int32_t at2, int i2) {
  return (s > s2) | ((s == s2) & ((at < at2) | ((at == at2) & (i < i2))));
}

// ---- a sum of exponentials in pairs of 32-bit numbers
//
// Near ties are settled with sums that are good to 2^-36, which 64-bit arithmetic would give too, but at an eighth of the rate: exp(d) = 2^(j / 64) exp(r) with j the
// nearest integer of 64 d / ln 2 and |r| <= ln 2 / 128 (the table-driven method of P. T. P. Tang, ACM TOMS 15, 1989), the reduction, the table's value and the sum
// each as a number and its rest.
constexpr double kStep = 0.6931471805599453094 / 64;
struct ExpTable { float hi[64], lo[64]; };
struct PairSum {
  float hi = 0.f, lo = 0.f;
  // Adds exp(x - m).
  __device__ __forceinline__ void add(const ExpTable& table, float x, float m) {
    constexpr float step_hi = (float)kStep, step_lo = (float)(kStep - (double)step_hi);
    const float d = x - m;
    if (!(d > -86.f)) return;                                          // (below 2^-124 of the largest; -inf)
    const float back = d + m, d_lo = (x - back) - (m + (d - back));    // d + d_lo = x - m
    const float jf = rintf(d * (float)(1.0 / kStep));
    const int j = (int)jf;
    const float p = jf * step_hi, p_lo = fmaf(jf, step_hi, -p);
    const float a = d - p, r = a - p_lo, r_lo = ((a - r) - p_lo) + fmaf(-jf, step_lo, d_lo);
    const float rest = fmaf(r * r, fmaf(r, fmaf(r, 1.f / 24, 1.f / 6), 0.5f), fmaf(r, r_lo, r_lo));      // exp(r) = 1 + r + rest
    const float t = table.hi[j & 63], t_lo = table.lo[j & 63];
    const float b = t * r, b_lo = fmaf(t, r, -b);
    const float h = t + b, l = (b - (h - t)) + (b_lo + fmaf(t, rest, fmaf(t_lo, r, t_lo)));
    const float scale = __int_as_float(((j >> 6) + 127) << 23);
    const float y = h * scale, s = hi + y, z = s - hi;
    lo += ((hi - (s - z)) + (y - z)) + l * scale;
    hi = s;
  }
};

struct SelectSmem {
  float unit_max[kMaxC * kWarps], unit_sum[kMaxC * kWarps];
  int32_t unit_changes[kMaxC * kWarps];      // how often its sum was scaled by other than a power of 2
  double row_lse[kMaxK];         // log of the row's sum, relative to row_max
  float row_max[kMaxK];
  int32_t row_changes[kMaxK];
  float row_floor[kMaxK];        // what an element has to be to come near the bar
  float score[kMaxK];
  int32_t live[kMaxK];           // rows that are read, in order
  uint32_t done_bits, finite_bits, exact_bits, ask_bits;   // per row: finished; score is finite; summed exactly; to be summed so
  int32_t n_live;
  Key bid[kWarps * 32];                      // each warp's, in order
  int32_t bid_at[kWarps * 32];
  float chunk_max[kWarps][kMaxima];
  Key top[kMaxC * 32];                       // each CTA's best bids, in order
  int32_t top_at[kMaxC * 32];
  Key bar;
  int32_t bar_at;
  int32_t n_listed[kMaxC];       // candidates that each CTA has put into the list
  int32_t n_had[kMaxC];          // candidates that it had: of more than it has put there only the best `need`
  int32_t n_todo, n_found;
  uint16_t todo[kWarps * kMaxima];           // chunks to be read again: warp * kMaxima + kept maximum
  Key found[kFound];
  int32_t found_at[kFound];
  Key most[kWarps];
  int32_t most_at[kWarps];
  Key list[kMaxC * kMany], packed[kMaxList];
  int32_t list_at[kMaxC * kMany], packed_at[kMaxList];
  Key sorted[kSorted];
  int32_t sorted_at[kSorted];
  ExpTable exps;
};

template <class T>
struct SelectParams {
  const T* logits;
  int64_t stride_n, stride_k;
  const float* scores;
  const uint8_t* done;
  const uint32_t* allowed;
  int64_t allowed_stride;
  int32_t* out_tokens;
  int32_t* out_parents;
  float* out_scores;
  uint8_t* out_done;
  int k, vocab, eos;
};

// Bytes of x picked by the four digits of `which`; a digit with its 8 set gives eight copies of the byte's top bit.
__device__ __forceinline__ uint32_t top_bits(uint32_t x, uint32_t which) {
  uint32_t r;
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(x), "r"(which));
  return r;
}

template <class T> struct Packed;      // elements in the 32-bit words of a 16-byte vector
template <> struct Packed<float> {
  static constexpr uint32_t kNegInf = 0xff800000u;
  static constexpr int kPer = 1;
  static __device__ __forceinline__ void get(uint32_t w, float (&x)[1]) { x[0] = __uint_as_float(w); }
  static __device__ __forceinline__ float max4(uint4 r) { return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w))); }
  static __device__ __forceinline__ uint32_t bits(float x) { return __float_as_uint(x); }
};
template <> struct Packed<__nv_bfloat16> {
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static constexpr int kPer = 2;
  static __device__ __forceinline__ void get(uint32_t w, float (&x)[2]) { x[0] = __uint_as_float(w << 16); x[1] = __uint_as_float(w & 0xffff0000u); }
  static __device__ __forceinline__ float max4(uint4 r) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint32_t bits(__nv_bfloat16 x) { return __bfloat16_as_ushort(x); }
};
template <> struct Packed<__half> {
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static constexpr int kPer = 2;
  static __device__ __forceinline__ void get(uint32_t w, float (&x)[2]) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    x[0] = f.x;
    x[1] = f.y;
  }
  static __device__ __forceinline__ float max4(uint4 r) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint32_t bits(__half x) { return __half_as_ushort(x); }
};

// A row as 16-byte vectors counted from the boundary at or before its first element.
template <class T>
struct Row {
  static constexpr int E = 16 / sizeof(T), P = Packed<T>::kPer;
  const T* p;
  const uint32_t* allowed;
  int vocab, shift, n_vecs, whole0, whole1;      // vectors whole0 .. whole1 - 1 lie in the row from end to end

  __device__ Row(const T* p_, int vocab_, const uint32_t* allowed_) : p(p_), allowed(allowed_), vocab(vocab_) {
    shift = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    n_vecs = (int)(((int64_t)vocab + shift + E - 1) / E);
    whole0 = shift != 0;
    whole1 = (int)(((int64_t)vocab + shift) / E);
  }
  __device__ bool whole(int v) const { return v >= whole0 && v < whole1; }
  __device__ bool may(int at) const { return !allowed || ((__ldg(allowed + (at >> 5)) >> (at & 31)) & 1); }
  __device__ static uint4 nothing() { return make_uint4(Packed<T>::kNegInf, Packed<T>::kNegInf, Packed<T>::kNegInf, Packed<T>::kNegInf); }
  // Vector v as it lies there, if all of it belongs to the row.
  __device__ uint4 raw(int v) const { return __ldg(reinterpret_cast<const uint4*>(p + ((int64_t)v * E - shift))); }
  // Bits of a whole vector's elements that are allowed.
  __device__ uint32_t bits_of(int v) const {
    const int first = v * E - shift;
    if (shift == 0) return __ldg(reinterpret_cast<const uint8_t*>(allowed) + (first >> 3)) >> (first & 7);
    const int at = first >> 5;
    return __funnelshift_r(__ldg(allowed + at), (first & 31) + E > 32 ? __ldg(allowed + at + 1) : 0u, first & 31);
  }
  // -inf for the elements whose bit is not set.
  __device__ static uint4 keep(uint32_t bits, uint4 r) {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int h = 0; h < E / 4; ++h) {
      // four bits to the tops of four bytes, and those over the elements' width
      const uint32_t tops = ((bits >> (4 * h)) & 15) * 0x10204080u;
#pragma unroll
      for (int i = 0; i < 4 / P; ++i) {
        const uint32_t all = top_bits(tops, P == 1 ? 0x8888 + 0x1111 * i : 0x9988 + 0x2222 * i);
        uint32_t& x = w[h * (4 / P) + i];
        x = (x & all) | (Packed<T>::kNegInf & ~all);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // Vector v with -inf for what lies outside the row or is not allowed.
  __device__ uint4 clean(int v, bool is_whole, uint4 r) const {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
    const int first = v * E - shift;
    if (is_whole) {
      if (!allowed) return r;
      return keep(bits_of(v), r);
    }
    {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = Packed<T>::kNegInf;
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const int at = first + i * P + e;
          if (at >= 0 && at < vocab && may(at)) {
            const uint32_t b = Packed<T>::bits(p[at]);
            w[i] = P == 1 ? b : e == 0 ? (w[i] & 0xffff0000u) | b : (w[i] & 0xffffu) | b << 16;
          }
        }
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Where part `part` of `parts` equal ones begins (the first n % parts are one longer).
__device__ __forceinline__ int cut(int n, int part, int parts) { return part * (int)((uint32_t)n / (uint32_t)parts) + min(part, (int)((uint32_t)n % (uint32_t)parts)); }

// A float as an integer that is ordered alike.
__device__ __forceinline__ int ordered(float x) {
  const int b = __float_as_int(x + 0.f);
  return b ^ ((b >> 31) & 0x7fffffff);
}

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bound on the error of a row's log of its sum, where a lane adds it up in `chunks` steps and scales it by other than a power of 2 `changes` times: two roundings
// of an exponent's argument (2^-24 of it, on average at most log2(vocab) + 1 in size: 1.5e-6 below a vocabulary of 2^17; or one, and log2 e's of logits
// below 64), exp2's own 2^-22, 20 additions deep inside and across lanes, the same where stretches are joined, the logarithm's last place (2^-20 below
// 16); an addition for each chunk, and an exp2 and a product for each change.
__device__ __forceinline__ double row_error(int chunks, int changes) { return 6e-6 + 6e-8 * chunks + 4.5e-7 * changes; }

template <class T, int C>
__global__ void __launch_bounds__(kWarps * 32, 2) select_kernel(const SelectParams<T> a) {
  constexpr int E = Row<T>::E, kUnits = C * kWarps;
  __shared__ SelectSmem s;
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = (int)cluster.block_rank(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int sent = blockIdx.x / C, k = a.k, need = k + kBeyond;

  cluster.barrier_arrive();        // (waited for before the first write into another CTA's memory: all of them run by then)
  if (warp == 0) {
    const float sc = lane < k ? a.scores[(int64_t)sent * k + lane] : -INFINITY;
    const bool fin = isfinite(sc), dn = lane < k && a.done && a.done[(int64_t)sent * k + lane] != 0;
    const uint32_t finite = __ballot_sync(~0u, fin), done = __ballot_sync(~0u, dn), live = finite & ~done;
    if (lane < k) s.score[lane] = sc;
    if ((live >> lane) & 1) s.live[__popc(live & ((1u << lane) - 1))] = lane;
    if (lane == 0) {
      s.finite_bits = finite; s.done_bits = done; s.exact_bits = done; s.ask_bits = 0;
      s.n_live = __popc(live);
    }
  }
  __syncthreads();

  // Units: (live row, stretch), dealt to the cluster's CTAs in turn so that every CTA has a part of every row.
  const int n_live = s.n_live, per_row = n_live ? kUnits / n_live : 1;
  const int unit = warp * C + cta;
  const bool busy = unit < per_row * n_live;
  const int row = busy ? s.live[unit / per_row] : 0, part = busy ? unit % per_row : 0;
  const Row<T> r(a.logits + sent * a.stride_n + row * a.stride_k, a.vocab, a.allowed ? a.allowed + sent * a.allowed_stride : nullptr);
  const int v0 = cut(r.n_vecs, part, per_row), v1 = busy ? cut(r.n_vecs, part + 1, per_row) : v0;

  // 1. the stretch, once
  float top = -INFINITY;                 // the lane's maximum
  float wtop = -INFINITY, sum = 0.f, ref = 0.f;      // the warp's; the lane's sum, relative to it
  int changes = 0, top_vec = 0;          // top_vec: first vector of the warp's chunk that the lane's maximum is in
  const int n_chunks = (v1 - v0 + kChunkVecs - 1) / kChunkVecs;
  const int most_chunks = ((a.vocab / E + 2) / per_row + kChunkVecs) / kChunkVecs;      // of any stretch of the sentence
  int group = 0;                         // chunks of a kept maximum, as a power of 2
  while ((most_chunks - 1) >> group >= kMaxima) ++group;
  // (The next chunk is on its way while one is added up, where it lies in the row from end to end.)
  uint4 ahead[4];
  uint32_t ahead_bits[4];
  auto inside = [&](int vb) { return vb >= r.whole0 && vb + kChunkVecs <= min(v1, r.whole1); };
  auto fetch = [&](int vb) {
    if (!inside(vb)) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ahead[j] = r.raw(vb + lane + 32 * j);
      if (r.allowed) ahead_bits[j] = r.bits_of(vb + lane + 32 * j);
    }
  };
  // Terms are exp2(x log2 e - ref), ref the whole number next to the warp's maximum in these units: one instruction for the exponent, and a new maximum
  // scales the sum by an exact power of 2.  A maximum below -64 (words masked by a finite value, before the ordinary ones) counts as -64: what lies far below makes terms
  // of 0, and the factors stay within 1.  FAR: the stretch's maximum is 64 or more in size, where log2 e's own rounding (1.4e-8 of x) would tell:
  // the stretch is read again with differences to the maximum itself.
  auto scan = [&](auto is_far) {
    constexpr bool FAR = decltype(is_far)::value;
    top = wtop = -INFINITY;
    sum = 0.f;
    ref = kLeastRef;
    fetch(v0);
    for (int c = 0; c < n_chunks; ++c) {
      const int vb = v0 + c * kChunkVecs;
      uint4 raw[4];
      if (inside(vb)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[j] = r.allowed ? r.keep(ahead_bits[j], ahead[j]) : ahead[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int v = vb + lane + 32 * j;
          const bool whole = v < v1 && r.whole(v);
          raw[j] = whole ? r.raw(v) : r.nothing();
          if (v < v1) raw[j] = r.clean(v, whole, raw[j]);
        }
      }
      fetch(vb + kChunkVecs);
      const float m = fmaxf(fmaxf(Packed<T>::max4(raw[0]), Packed<T>::max4(raw[1])), fmaxf(Packed<T>::max4(raw[2]), Packed<T>::max4(raw[3])));
      if (m > top) {
        top = m;
        top_vec = vb;
      }
      const int most = __reduce_max_sync(~0u, ordered(m));
      const float chunk_max = __int_as_float(most ^ ((most >> 31) & 0x7fffffff));
      if (lane == 0) {
        float* const slot = &s.chunk_max[warp][c >> group];
        *slot = c & ((1 << group) - 1) ? fmaxf(*slot, chunk_max) : chunk_max;
      }
      if (chunk_max > wtop) {
        if (FAR) {
          sum *= exp2_of((wtop - chunk_max) * kLog2e);
          ++changes;
        } else {
          const float now = fmaxf(rintf(chunk_max * kLog2e), kLeastRef);
          sum *= ref - now < -126.f ? 0.f : __int_as_float((127 + (int)(ref - now)) << 23);
          ref = now;
        }
        wtop = chunk_max;
      }
      const float base = wtop == -INFINITY ? 0.f : wtop;     // (nothing allowed yet: every term is exp2(-inf), or a NaN, which stays one)
      float part_sum[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
        part_sum[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[Packed<T>::kPer];
          Packed<T>::get(w[i], x);
#pragma unroll
          for (int e = 0; e < Packed<T>::kPer; ++e) part_sum[j] += exp2_of(FAR ? (x[e] - base) * kLog2e : fmaf(x[e], kLog2e, -ref));
        }
      }
      sum += (part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]);
    }
    if (!FAR && wtop > -INFINITY) sum *= exp2_of(fmaf(-wtop, kLog2e, ref));      // relative to exp(wtop)
  };
  scan(std::false_type{});
  if (wtop > -INFINITY && !(fabsf(wtop) < 64.f)) scan(std::true_type{});
  // (Maxima pass over NaN: the sum has it.  +inf: its own term is a NaN.)
  float wsum = sum;
#pragma unroll
  for (int o = 16; o; o >>= 1) wsum += __shfl_xor_sync(~0u, wsum, o);
  cluster.barrier_wait();
  if (busy && lane < C) {
    SelectSmem* to = cluster.map_shared_rank(&s, lane);
    to->unit_max[unit] = wtop;
    to->unit_sum[unit] = wsum;
    to->unit_changes[unit] = changes;
  }
  cluster.sync();

  // The lanes' bids, best first: by the largest logit, of equal ones by the bound of its index.  All of a warp's are of one row, so that
  // their order holds whatever the normaliser.
  const int row_base = row * a.vocab;
  uint64_t lane_bid = (uint64_t)((uint32_t)ordered(top) ^ 0x80000000u) << 32 | (uint32_t)~(row_base + min(a.vocab - 1, (top_vec + lane + 96) * E + E - 1 - r.shift));
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(~0u, lane_bid, o);
      const bool larger_first = ((lane & size) == 0) == ((lane & o) == 0);
      lane_bid = (lane_bid > other) == larger_first ? lane_bid : other;
    }
  const int best_bits = (int)((uint32_t)(lane_bid >> 32) ^ 0x80000000u), best_at = (int)~(uint32_t)lane_bid;
  const float best = __int_as_float(best_bits ^ ((best_bits >> 31) & 0x7fffffff));
  SelectSmem* const lead = cluster.map_shared_rank(&s, 0);

  // The rows' normalisers from the units' sums, a warp for each.
  for (int i = warp; i < n_live; i += kWarps) {
    float m = -INFINITY;
    for (int u = lane; u < per_row; u += 32) m = fmaxf(m, s.unit_max[i * per_row + u]);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    float t = 0.f;
    int most = 0;
    for (int u = i * per_row + lane; u < (i + 1) * per_row; u += 32) {
      t += s.unit_max[u] == -INFINITY ? s.unit_sum[u] : s.unit_sum[u] * exp2_of((s.unit_max[u] - m) * kLog2e);
      most = max(most, s.unit_changes[u]);
    }
    most = __reduce_max_sync(~0u, most);
#pragma unroll
    for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
    if (lane == 0) {
      s.row_max[s.live[i]] = m;
      s.row_lse[s.live[i]] = m == -INFINITY ? (double)NAN : (double)logf(t);
      s.row_changes[i] = most;
    }
  }
  __syncthreads();

  for (;;) {
    // 2. bids and the bar
    const double score = busy ? s.score[row] : 0.0, base = busy ? s.row_max[row] : 0.0, lse = busy ? s.row_lse[row] : 0.0;
    auto sum_of = [&](float x) { return score + (((double)x - base) - lse); };
    const double best_sum = busy && best != -INFINITY ? sum_of(best) : (double)NAN;
    const Key bid = best_sum == best_sum ? key_of(best_sum) : kNone;       // a row without a normaliser (NaN, +inf, nothing allowed) bids nothing
    int bid_at = bid == kNone ? 0x7fffffff : best_at;
    {
      // Logits that differ may give equal sums (1e-20 and 2e-20): among those the bounds have to rise too, and a larger bound is one as well.
      const Key prev = __shfl_up_sync(~0u, bid, 1);
      const int prev_at = __shfl_up_sync(~0u, bid_at, 1);
      if (__any_sync(~0u, lane && prev == bid && prev_at > bid_at)) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const Key k2 = __shfl_up_sync(~0u, bid, o);
          const int a2 = __shfl_up_sync(~0u, bid_at, o);
          if (lane >= o && k2 == bid) bid_at = max(bid_at, a2);
        }
      }
    }
    // The CTA's 32 best: two sorted lists' are the larger of each pair from opposite ends, put in order by five exchanges.
    Key mine = bid;
    int mine_at = bid_at;
    for (int left = kWarps; left > 1; left = (left + 1) / 2) {
      const int half = (left + 1) / 2;
      if (warp >= half && warp < left) { s.bid[tid] = mine; s.bid_at[tid] = mine_at; }
      __syncthreads();
      if (warp + half < left) {
        const int j = (warp + half) * 32 + 31 - lane;
        const Key k2 = s.bid[j];
        const int a2 = s.bid_at[j];
        if (before(k2, a2, mine, mine_at)) { mine = k2; mine_at = a2; }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const Key k3 = __shfl_xor_sync(~0u, mine, o);
          const int a3 = __shfl_xor_sync(~0u, mine_at, o);
          if (before(k3, a3, mine, mine_at) == ((lane & o) == 0)) { mine = k3; mine_at = a3; }
        }
      }
    }
    if (tid == 0) s.n_todo = s.n_found = 0;
    if (warp == 0) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        SelectSmem* to = cluster.map_shared_rank(&s, c);
        to->top[cta * 32 + lane] = mine;
        to->top_at[cta * 32 + lane] = mine_at;
      }
    }
    cluster.sync();
    // A thread counts, by bisection, what one CTA's list has before one bid of all.
    const int len = min(need, 32);
    for (int t0 = 0; t0 < C * C * len; t0 += kWarps * 32) {
      const int n = min(t0 + tid, C * C * len - 1) / C, b = n / len * 32 + n % len, in = tid % C;
      const Key bk = s.top[b];
      const int ba = s.top_at[b];
      int lo = 0, hi = len;                  // entries before lo are before the bid, those from hi on are not
      while (lo < hi) {
        const int mid = (lo + hi) >> 1, j = in * 32 + mid;
        if (bid_before(s.top[j], s.top_at[j], j, bk, ba, b)) lo = mid + 1; else hi = mid;
      }
#pragma unroll
      for (int o = 1; o < C; o <<= 1) lo += __shfl_xor_sync(~0u, lo, o);
      if (lo == need - 1) { s.bar = bk; s.bar_at = ba; }
    }
    __syncthreads();

    // 3. the chunks whose maximum can reach the bar, shared out among the CTA's warps: most are of one or two rows
    const Key bar = s.bar;
    const int bar_at = s.bar_at;
    // What an element of a row has to be to come near the bar, with room for the roundings on the way: spares the others the 64-bit sum.
    auto floor_of = [&](double sc, double ls, double bs) {
      if (bar == kNone) return -INFINITY;
      const double lowest = sum_of_key(bar) - sc + ls + bs;
      return (float)(lowest - 1e-6 * (1.0 + fabs(lowest) + fabs(sc) + fabs(ls) + fabs(bs)));
    };
    if (__shfl_sync(~0u, bid, 0) != kNone) {           // (a warp's best bid is its best candidate's sum)
      const float floor_x = floor_of(score, lse, base);
      if (lane == 0) s.row_floor[row] = floor_x;         // (all its warps say the same)
#pragma unroll
      for (int h = 0; h < kMaxima / 32; ++h) {
        const int g = lane + 32 * h;
        const float cm = g << group < n_chunks ? s.chunk_max[warp][g] : -INFINITY;
        if (cm >= floor_x && cm != -INFINITY) s.todo[atomicAdd(&s.n_todo, 1)] = (uint16_t)(warp * kMaxima + g);
      }
    }
    __syncthreads();
    const int n_todo = s.n_todo;
    // Calls found(hit, key, at) for the elements of the warp's share that come near, every lane together.
    auto sweep = [&](auto&& found) {
      for (int i = warp; i < n_todo; i += kWarps) {
        const int w = s.todo[i] / kMaxima, g = s.todo[i] % kMaxima, u = w * C + cta, rw = s.live[u / per_row], pt = u % per_row;
        const Row<T> q(a.logits + sent * a.stride_n + rw * a.stride_k, a.vocab, r.allowed);
        const int q0 = cut(q.n_vecs, pt, per_row), q1 = cut(q.n_vecs, pt + 1, per_row);
        const double sc = s.score[rw], bs = s.row_max[rw], ls = s.row_lse[rw];
        const float floor_x = s.row_floor[rw];
        const int c1 = min((g + 1) << group, (q1 - q0 + kChunkVecs - 1) / kChunkVecs);
        for (int c = g << group; c < c1; ++c) {
          const int vb = q0 + c * kChunkVecs + lane;
          uint4 raw[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) raw[j] = vb + 32 * j < q1 && q.whole(vb + 32 * j) ? q.raw(vb + 32 * j) : q.nothing();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int v = vb + 32 * j;
            if (v < q1) raw[j] = q.clean(v, q.whole(v), raw[j]);
            if (!__any_sync(~0u, Packed<T>::max4(raw[j]) >= floor_x)) continue;
            const uint32_t word[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
              float x[Packed<T>::kPer];
              Packed<T>::get(word[i4], x);
#pragma unroll
              for (int e = 0; e < Packed<T>::kPer; ++e) {
                const bool close = x[e] >= floor_x && x[e] != -INFINITY;
                const int at = rw * a.vocab + v * E - q.shift + i4 * Packed<T>::kPer + e;
                const Key key = close ? key_of(sc + (((double)x[e] - bs) - ls)) : kNone;
                if (close && !before(bar, bar_at, key, at)) found(key, at);
              }
            }
          }
        }
      }
    };
    sweep([&](Key key, int at) {
      const int slot = atomicAdd(&s.n_found, 1);
      if (slot < kFound) { s.found[slot] = key; s.found_at[slot] = at; }
    });
    __syncthreads();
    const int n_found = s.n_found;
    Key* const list = lead->list + cta * kMany;
    int32_t* const list_at = lead->list_at + cta * kMany;
    if (tid == 0) {
      lead->n_listed[cta] = min(n_found, n_found <= kMany ? kMany : need);
      lead->n_had[cta] = n_found;
    }
    if (n_found <= kMany) {
      for (int i = tid; i < n_found; i += kWarps * 32) { list[i] = s.found[i]; list_at[i] = s.found_at[i]; }
    } else if (n_found <= kFound) {
      for (int i = tid; i < n_found; i += kWarps * 32) {
        const Key fk = s.found[i];
        const int fa = s.found_at[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n_found; ++j) rank += before(s.found[j], s.found_at[j], fk, fa);
        if (rank < need) { list[rank] = fk; list_at[rank] = fa; }
      }
    } else {
      Key prev = kNone;                      // many (equal or sorted logits): the best `need` of them, one by one
      int prev_at = 0;
      for (int turn = 0; turn < need; ++turn) {
        Key most = kNone;
        int most_at = 0x7fffffff;
        sweep([&](Key key, int at) {
          if ((turn == 0 || before(prev, prev_at, key, at)) && before(key, at, most, most_at)) { most = key; most_at = at; }
        });
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const Key k2 = __shfl_xor_sync(~0u, most, o);
          const int a2 = __shfl_xor_sync(~0u, most_at, o);
          if (before(k2, a2, most, most_at)) { most = k2; most_at = a2; }
        }
        if (lane == 0) { s.most[warp] = most; s.most_at[warp] = most_at; }
        __syncthreads();
        for (int w = 0; w < kWarps; ++w)
          if (before(s.most[w], s.most_at[w], most, most_at)) { most = s.most[w]; most_at = s.most_at[w]; }
        if (tid == 0) { list[turn] = most; list_at[turn] = most_at; }
        prev = most;
        prev_at = most_at;
        __syncthreads();
      }
    }
    cluster.sync();

    // 4. the order
    int n_sorted = 0;
    if (cta == 0) {
      // the CTAs' candidates one after the other, then one for each finished beam
      const uint32_t ended = s.done_bits & s.finite_bits;
      Key rest = bar;              // no candidate that is not in order at the end has a larger key
      int before_cta = 0;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int m = s.n_listed[c];
        for (int i = tid; i < m; i += kWarps * 32) { s.packed[before_cta + i] = s.list[c * kMany + i]; s.packed_at[before_cta + i] = s.list_at[c * kMany + i]; }
        if (s.n_had[c] > m) rest = max(rest, s.list[c * kMany + m - 1]);
        before_cta += m;
      }
      const int n = before_cta + __popc(ended);
      if (warp == 0 && ((ended >> lane) & 1)) {
        const int slot = before_cta + __popc(ended & ((1u << lane) - 1));
        s.packed[slot] = key_of((double)s.score[lane]);
        s.packed_at[slot] = lane * a.vocab + a.eos;
      }
      __syncthreads();
      n_sorted = min(n, kSorted);
      for (int i = tid; i < n; i += kWarps * 32) {
        const Key ck = s.packed[i];
        const int ca = s.packed_at[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += before(s.packed[j], s.packed_at[j], ck, ca);
        if (rank < kSorted) { s.sorted[rank] = ck; s.sorted_at[rank] = ca; }
      }
      __syncthreads();
      if (warp == 0) {
        // Pair i = sorted i and i + 1.  It is open where i + 1, or what is not in order, is near: the first from the k-th on that is not closes the order, and what comes
        // behind it cannot be among the k best.  A near pair of two rows before that, one of them summed in 32 bits, has to be settled.
        const int changes_most = __reduce_max_sync(~0u, lane < n_live ? s.row_changes[lane] : 0);
        const double near = 2 * row_error(most_chunks, changes_most);
        if (n > kSorted) rest = max(rest, s.sorted[kSorted - 1]);
        uint32_t open_bits[2], unsure_bits[2], ask = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = lane + 32 * h;
          bool is_open = false, unsure = false;
          if (i < n_sorted) {
            const double sum = sum_of_key(s.sorted[i]);
            is_open = rest != kNone && sum - sum_of_key(rest) < near;
            if (i + 1 < n_sorted && sum - sum_of_key(s.sorted[i + 1]) < near) {
              const uint32_t r1 = s.sorted_at[i] / a.vocab, r2 = s.sorted_at[i + 1] / a.vocab;
              is_open = true;
              unsure = r1 != r2 && !((s.exact_bits >> r1) & (s.exact_bits >> r2) & 1);
            }
          }
          open_bits[h] = __ballot_sync(~0u, is_open);
          unsure_bits[h] = __ballot_sync(~0u, unsure);
        }
        const uint64_t is_open = open_bits[0] | (uint64_t)open_bits[1] << 32, unsure = unsure_bits[0] | (uint64_t)unsure_bits[1] << 32;
        const uint64_t from_k = ~is_open & ~((1ull << (k - 1)) - 1);
        const int close = from_k ? __ffsll((long long)from_k) - 1 : kSorted - 1;
        const uint64_t matter = unsure & ((2ull << close) - 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = lane + 32 * h;
          if ((matter >> i) & 1) ask |= (1u << (s.sorted_at[i] / a.vocab)) | (1u << (s.sorted_at[i + 1] / a.vocab));
        }
        ask = __reduce_or_sync(~0u, ask);
        if (!from_k || close >= n_sorted) ask = rest == kNone ? ask : ~0u;      // the list ends before the order is closed
        // (a row whose sum is NaN offers nothing, and the sums in pairs pass over NaN)
        ask &= s.finite_bits & ~s.exact_bits & __ballot_sync(~0u, ((s.finite_bits & ~s.done_bits) >> lane) & 1 && !isnan(s.row_lse[lane]));
        if (lane < C) cluster.map_shared_rank(&s, lane)->ask_bits = ask;
      }
    }
    cluster.sync();
    const uint32_t ask = s.ask_bits;
    if (!ask) {
      if (cta == 0 && tid < k) {
        const int64_t o = (int64_t)sent * k + tid;
        const bool some = tid < n_sorted;
        const int at = some ? s.sorted_at[tid] : 0, parent = some ? at / a.vocab : tid, token = some ? at - parent * a.vocab : a.eos;
        a.out_tokens[o] = token;
        a.out_parents[o] = parent;
        a.out_scores[o] = some ? (float)sum_of_key(s.sorted[tid]) : -INFINITY;
        if (a.out_done) a.out_done[o] = !some || ((s.done_bits >> parent) & 1) || token == a.eos;
      }
      return;
    }
    // The rows that are asked for once more, exactly, a part by each of the cluster's warps: cut and added up by the words' own numbers, wherever
    // the row begins, so that equal rows get equal sums and their ties stay ties.  (The list's place is free.)
    constexpr int kRowsAtOnce = kMany / kWarps;
    if (tid < 64) {
      const double e = exp2(tid / 64.0);
      s.exps.hi[tid] = (float)e;
      s.exps.lo[tid] = (float)(e - (double)(float)e);
    }
    __syncthreads();
    for (uint32_t left = ask; left;) {
      uint32_t now = 0;
      for (int i = 0; i < kRowsAtOnce && left; ++i) { now |= left & (0u - left); left &= left - 1; }
      int i = 0;
      for (uint32_t rows = now; rows; rows &= rows - 1, ++i) {
        const int rw = __ffs(rows) - 1;
        const T* const p = a.logits + sent * a.stride_n + rw * a.stride_k;
        const float m = s.row_max[rw];
        PairSum sums;
        const int e1 = cut(a.vocab, unit + 1, kUnits);
        for (int at = cut(a.vocab, unit, kUnits) + lane; at < e1; at += 8 * 32) {
          T x[8];                          // (eight on their way at once: loaded whether they count or not)
          uint32_t word[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int i = min(at + 32 * j, e1 - 1);
            x[j] = p[i];
            word[j] = r.allowed ? __ldg(r.allowed + (i >> 5)) >> (i & 31) : 1u;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) sums.add(s.exps, at + 32 * j < e1 && (word[j] & 1) ? to_float(x[j]) : -INFINITY, m);
        }
        double t = (double)sums.hi + (double)sums.lo;
#pragma unroll
        for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
        if (lane < C) reinterpret_cast<double*>(cluster.map_shared_rank(&s, lane)->list)[i * kUnits + unit] = t;
      }
      cluster.sync();
      i = 0;
      for (uint32_t rows = now; rows; rows &= rows - 1, ++i) {
        if (i % kWarps != warp) continue;
        double t = 0.0;
        for (int u = lane; u < kUnits; u += 32) t += reinterpret_cast<const double*>(s.list)[i * kUnits + u];
#pragma unroll
        for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
        if (lane == 0) s.row_lse[__ffs(rows) - 1] = log(t);
      }
      cluster.sync();              // (before the next rows' parts are written, or the next list)
    }
    if (tid == 0) s.exact_bits |= ask;
    __syncthreads();
  }
}

template <class T>
cudaError_t launch_select(const linmt_beam_select_args& g) {
  SelectParams<T> p{static_cast<const T*>(g.logits), g.stride_n, g.stride_k, g.scores, g.done, g.allowed, g.allowed_stride,
                    g.out_tokens, g.out_parents, g.out_scores, g.out_done, g.k, g.vocab, g.eos};
  // As many CTAs for a sentence as leave all of them on the GPU at once (two on an SM; clusters of 8 only reach 33), since a second round of
  // clusters costs its latencies again, and as have 16k logits each: exchanges among more take longer (64 x 12 x 30k fp32: 40, 30 and 51 us
  // with 2, 4 and 8; 128 x 12 x 80k bf16: 82, 95 and 141; 1 x 4 x 1000: 10.2, 10.6 and 12.4).  A row has a warp at
  // least, and as many as have 8 / 7 of `need` lanes, or the bar falls below what its best candidates are when one beam is ahead (139 x 30 x 5.9k fp16
  // with one warp a row: 480 us; 300 x 20 x 4000 with two a row, not one: 77, not 50).  A row so short that all of it can be ranked needs no more than one
  // (300 x 27 x 300: 81 us; 208 with three).
  const int64_t logits = (int64_t)g.k * g.vocab;
  int c = g.n <= 33 ? 8 : g.n <= 74 ? 4 : g.n <= 148 ? 2 : 1;
  while (c > 1 && logits < (int64_t)(c / 2 + 1) * 16384) c /= 2;
  const int need = g.k + kBeyond;
  while (c * kWarps < g.k || (need > 28 * (c * kWarps / g.k) && g.vocab + need > kFound)) c *= 2;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = c;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)g.n * c);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = static_cast<cudaStream_t>(g.stream);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, c == 8 ? select_kernel<T, 8> : c == 4 ? select_kernel<T, 4> : c == 2 ? select_kernel<T, 2> : select_kernel<T, 1>, p);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

// ---- reordering --------------------------------------------------------------------------------
//
// A thread owns one column (a vector of 1 to 16 bytes) of one sentence's k rows of a state: it loads the k parents' values, then stores them, so a
// state can be reordered in place without a copy or a barrier, and k loads are in flight.  Bound by the bytes moved.
struct ReorderState {
  const unsigned char* src;
  unsigned char* dst;
  int64_t src_l, src_n, src_k, dst_l, dst_n, dst_k;
  int64_t cols, first_block;      // vectors of a row; first block of the state
  int64_t layers;
  int32_t vec_bytes;
};
struct ReorderParams {
  const int32_t* parents;
  int32_t n, k, n_states, narrow;        // narrow: every state's columns can be counted in 32 bits
  ReorderState state[16];
};
constexpr int kReorderThreads = 128;

template <class V, int K>
__device__ __forceinline__ void move_column(const ReorderState& st, const int32_t* parents, int k, int64_t l, int64_t n, int64_t col) {
  const unsigned char* src = st.src + l * st.src_l + n * st.src_n + col * (int64_t)sizeof(V);
  unsigned char* dst = st.dst + l * st.dst_l + n * st.dst_n + col * (int64_t)sizeof(V);
  V v[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (j < k) {
      const uint32_t p = (uint32_t)__ldg(parents + n * k + j);
      v[j] = *reinterpret_cast<const V*>(src + (p < (uint32_t)k ? (int64_t)p : (int64_t)j) * st.src_k);
    }
  }
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (j < k) *reinterpret_cast<V*>(dst + j * st.dst_k) = v[j];
}

template <int K>
__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const __grid_constant__ ReorderParams a) {
  int i = 0;
  while (i + 1 < a.n_states && (int64_t)blockIdx.x >= a.state[i + 1].first_block) ++i;
  const ReorderState& st = a.state[i];
  const int64_t at = ((int64_t)blockIdx.x - st.first_block) * kReorderThreads + threadIdx.x;
  const int64_t ln = a.narrow ? (int64_t)((uint32_t)at / (uint32_t)st.cols) : at / st.cols, col = at - ln * st.cols;
  const int64_t l = a.narrow ? (int64_t)((uint32_t)ln / (uint32_t)a.n) : ln / a.n, n = ln - l * a.n;
  if (l >= st.layers) return;
  switch (st.vec_bytes) {
    case 16: move_column<uint4, K>(st, a.parents, a.k, l, n, col); break;
    case 8: move_column<uint2, K>(st, a.parents, a.k, l, n, col); break;
    case 4: move_column<uint32_t, K>(st, a.parents, a.k, l, n, col); break;
    case 2: move_column<uint16_t, K>(st, a.parents, a.k, l, n, col); break;
    default: move_column<uint8_t, K>(st, a.parents, a.k, l, n, col); break;
  }
}

}  // namespace
}  // namespace ops
}  // namespace linmt

extern "C" {

const char* linmt_op_error(void) { return linmt::ops::op_error_text(); }

int linmt_beam_select(const linmt_beam_select_args* g) {
  using namespace linmt::ops;
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "beam_select: not this library's argument struct");
  if (!g->logits || !g->scores || !g->out_tokens || !g->out_parents || !g->out_scores) return op_fail(LINMT_EINVAL, "beam_select: an array is missing");
  if (g->n < 0 || g->k < 1 || g->vocab < 1 || !dtype_ok(g->dtype)) return op_fail(LINMT_EINVAL, "beam_select: n = %d, k = %d, vocab = %d, dtype = %d", g->n, g->k, g->vocab, g->dtype);
  if (g->eos < 0 || g->eos >= g->vocab) return op_fail(LINMT_EINVAL, "beam_select: eos = %d is not in a vocabulary of %d", g->eos, g->vocab);
  if (!aligned(g->logits, dtype_bytes(g->dtype)) || !aligned(g->scores, 4) || !aligned(g->allowed, 4) || !aligned(g->out_tokens, 4) || !aligned(g->out_parents, 4) || !aligned(g->out_scores, 4))
    return op_fail(LINMT_EINVAL, "beam_select: an array is not aligned to its type");
  if (g->k > kMaxK || (int64_t)g->k * g->vocab > INT32_MAX - 4095 || g->n > (1 << 27))
    return op_fail(LINMT_ELIMIT, "beam_select: k = %d (at most %d), k * vocab = %lld (at most 2^31 - 4096), n = %d", g->k, kMaxK, (long long)g->k * g->vocab, g->n);
  if (g->n == 0) return LINMT_OK;
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "beam_select");
  const cudaError_t e = g->dtype == LINMT_F32 ? launch_select<float>(*g) : g->dtype == LINMT_BF16 ? launch_select<__nv_bfloat16>(*g) : launch_select<__half>(*g);
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "beam_select");
}

int linmt_beam_reorder(const linmt_beam_reorder_args* g) {
  using namespace linmt::ops;
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "beam_reorder: not this library's argument struct");
  if (!g->parents || !aligned(g->parents, 4) || g->n < 0 || g->k < 1 || g->n_states < 0 || g->n_states > 16)
    return op_fail(LINMT_EINVAL, "beam_reorder: n = %d, k = %d, %d states (at most 16), parents %p", g->n, g->k, g->n_states, (const void*)g->parents);
  if (g->k > kMaxK) return op_fail(LINMT_ELIMIT, "beam_reorder: k = %d (at most %d)", g->k, kMaxK);
  ReorderParams p{};
  p.parents = g->parents; p.n = g->n; p.k = g->k; p.narrow = 1;
  int64_t blocks = 0;
  for (int i = 0; i < g->n_states; ++i) {
    const linmt_beam_state& s = g->state[i];
    if (s.layers < 0 || s.row_bytes < 0) return op_fail(LINMT_EINVAL, "beam_reorder: state %d has %lld layers of %lld bytes a row", i, (long long)s.layers, (long long)s.row_bytes);
    if (!s.layers || !s.row_bytes || !g->n) continue;
    if (!s.src || !s.dst) return op_fail(LINMT_EINVAL, "beam_reorder: state %d is missing", i);
    if (s.src == s.dst && (s.src_stride_l != s.dst_stride_l || s.src_stride_n != s.dst_stride_n || s.src_stride_k != s.dst_stride_k))
      return op_fail(LINMT_EINVAL, "beam_reorder: state %d is moved within one buffer between two sets of strides", i);
    uint64_t bits = reinterpret_cast<uintptr_t>(s.src) | reinterpret_cast<uintptr_t>(s.dst) | (uint64_t)s.row_bytes | (uint64_t)s.src_stride_k | (uint64_t)s.dst_stride_k |
                    (g->n > 1 ? (uint64_t)s.src_stride_n | (uint64_t)s.dst_stride_n : 0) | (s.layers > 1 ? (uint64_t)s.src_stride_l | (uint64_t)s.dst_stride_l : 0);
    int vec = 16;
    while (bits % vec) vec /= 2;
    ReorderState& d = p.state[p.n_states++];
    d = ReorderState{static_cast<const unsigned char*>(s.src), static_cast<unsigned char*>(s.dst), s.src_stride_l, s.src_stride_n, s.src_stride_k,
                     s.dst_stride_l, s.dst_stride_n, s.dst_stride_k, s.row_bytes / vec, blocks, s.layers, vec};
    if (s.layers * g->n * d.cols > INT32_MAX - kReorderThreads) p.narrow = 0;
    blocks += (s.layers * g->n * d.cols + kReorderThreads - 1) / kReorderThreads;
  }
  if (!blocks) return LINMT_OK;
  if (blocks > INT32_MAX) return op_fail(LINMT_ELIMIT, "beam_reorder: %lld blocks of columns in one call", (long long)blocks);
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "beam_reorder");
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  const dim3 grid((unsigned)blocks), block(kReorderThreads);
  if (g->k <= 4) reorder_kernel<4><<<grid, block, 0, st>>>(p);
  else if (g->k <= 8) reorder_kernel<8><<<grid, block, 0, st>>>(p);
  else if (g->k <= 16) reorder_kernel<16><<<grid, block, 0, st>>>(p);
  else reorder_kernel<32><<<grid, block, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "beam_reorder");
}

}  // extern "C"
