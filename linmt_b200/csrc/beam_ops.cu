// beam_ops.cu -- beam selection and reordering on device tensors (linmt_beam_select, linmt_beam_reorder).
#include <cooperative_groups.h>

#include <atomic>

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
// One cluster of 8 CTAs per sentence.  The work of a sentence is its live rows, each cut into as many stretches as there are warps for
// it; the clusters' CTAs exchange what they find through distributed shared memory, so a step is one launch without a workspace.
//   1  A warp reads its stretch once: per lane the running maximum and the sum of exponentials relative to it, and where
//      the lane's maximum lies.
//   2  Every CTA has the normalisers of all rows.  The best of each four lanes is a bid, a candidate's sum with an upper bound of
//      its index; the kNeed-th best bid of the cluster is a bar that at least kNeed = k + kBeyond candidates reach.
//   3  Only the stretches of lanes whose bid reaches the bar are read again (some kNeed of 1000, from L2).
//   4  The candidates found, some dozens, are ranked by counting.
// Sums are compared in 64 bits, but exponentials cost four to five instructions in 32 bits and twenty in 64, and the logits arrive at a rate that
// allows for the former.  So the normaliser is summed in 32 bits with a bound on its error (row_error); where two
// neighbours of the final order come from different rows and lie closer than twice that, their rows' normalisers are summed once more in 64 bits
// and the steps from 2 on repeat.  Some 1 sentence in 500 needs it, for 2 us.
constexpr int kClusterCtas = 8;
constexpr int kMaxK = 32;
constexpr int kMaxWarps = 16;
constexpr int kUnits = kClusterCtas * kMaxWarps;
constexpr int kBeyond = 8;                       // candidates past the k-th that the order is checked on
constexpr int kChunkVecs = 128;                  // a warp's step: four 16-byte vectors a lane
// Lanes that reach the bar: kNeed fours, and at most 7 more of the bar's own chunk whose index bounds overlap its.  Each gives up to
// max(32, kNeed) candidates; finished rows add one each.
constexpr int kMaxList = (kMaxK + kBeyond + 7) * (kMaxK + kBeyond) + kMaxK;
constexpr int kSorted = 64;                      // of them that are put in order (>= kNeed)
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kNone = -1.7976931348623157e308;   // below every candidate (sums of finite numbers below 1e39 in size)

// A candidate is its sum and `at` = row * vocab + word.
__device__ __forceinline__ bool before(double s, int32_t at, double s2, int32_t at2) { return s > s2 || (s == s2 && at < at2); }
// The same among bids, whose index is a bound that two may share: those go by their place in the list, so that ranks are distinct.
__device__ __forceinline__ bool bid_before(double s, int32_t at, int i, double s2, int32_t at2, int i2) {
  return s > s2 || (s == s2 && (at < at2 || (at == at2 && i < i2)));
}

struct SelectSmem {
  float unit_max[kUnits];
  double unit_sum[kUnits];
  double row_lse[kMaxK];         // log of the row's sum, relative to row_max
  float row_max[kMaxK];
  float score[kMaxK];
  int32_t live[kMaxK];           // rows that are read, in order
  uint32_t done_bits, finite_bits, exact_bits, ask_bits;   // per row: finished; score is finite; summed in 64 bits; to be summed so
  int32_t n_live;
  double bid_sum[kMaxWarps * 8];
  int32_t bid_at[kMaxWarps * 8];
  double top_sum[kClusterCtas * (kMaxK + kBeyond)];
  int32_t top_at[kClusterCtas * (kMaxK + kBeyond)];
  double bar_sum;
  int32_t bar_at;
  int32_t n_list;
  double list_sum[kMaxList];
  int32_t list_at[kMaxList];
  double sorted_sum[kSorted];
  int32_t sorted_at[kSorted];
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

// A row as 16-byte vectors counted from the boundary at or before its first element.
template <class T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* p;
  const uint32_t* allowed;
  int vocab, shift, n_vecs, n_words;

  __device__ Row(const T* p_, int vocab_, const uint32_t* allowed_) : p(p_), allowed(allowed_), vocab(vocab_) {
    shift = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    n_vecs = (int)(((int64_t)vocab + shift + E - 1) / E);
    n_words = (vocab + 31) / 32;
  }
  __device__ bool whole(int v) const { return v * (int64_t)E >= shift && (v + 1) * (int64_t)E <= (int64_t)vocab + shift; }
  __device__ bool may(int at) const { return !allowed || ((__ldg(allowed + (at >> 5)) >> (at & 31)) & 1); }
  __device__ uint4 raw(int v) const { return __ldg(reinterpret_cast<const uint4*>(p + ((int64_t)v * E - shift))); }
  // Elements of vector v, -inf for what lies outside the row or is not allowed.
  __device__ void elements(int v, bool is_whole, uint4 r, float (&x)[E]) const {
    const int first = v * E - shift;
    if (is_whole) {
      const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = to_float(e[i]);
      if (allowed) {
        const int w = first >> 5;
        const uint32_t lo = __ldg(allowed + w), hi = (first & 31) + E > 32 ? __ldg(allowed + w + 1) : 0u;
        const uint32_t bits = __funnelshift_r(lo, hi, first & 31);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = (bits >> i) & 1 ? x[i] : -INFINITY;
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int at = first + i;
        x[i] = at >= 0 && at < vocab && may(at) ? to_float(p[at]) : -INFINITY;
      }
    }
  }
};

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bound on the error of a row's log of its sum as a lane adds it up in `chunks` steps: two roundings of an exponent's argument
// (2^-24 of it, on average at most log2(vocab) + 1), exp2's own 2^-22, 20 additions deep inside and across lanes, and for each chunk one
// addition and one change of the maximum.
__device__ __forceinline__ double row_error(int chunks) { return 4.2e-6 + 4.5e-7 * chunks; }

template <class T>
__global__ void __cluster_dims__(kClusterCtas, 1, 1) __launch_bounds__(kMaxWarps * 32, 1) select_kernel(const SelectParams<T> a) {
  constexpr int E = Row<T>::E;
  __shared__ SelectSmem s;
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = (int)cluster.block_rank(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  const int sent = blockIdx.x / kClusterCtas, k = a.k, need = k + kBeyond;

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
  const int n_live = s.n_live, per_row = n_live ? kClusterCtas * warps / n_live : 1;
  const int unit = warp * kClusterCtas + cta;
  const bool busy = unit < per_row * n_live;
  const int row = busy ? s.live[unit / per_row] : 0, part = busy ? unit % per_row : 0;
  const Row<T> r(a.logits + sent * a.stride_n + row * a.stride_k, a.vocab, a.allowed ? a.allowed + sent * a.allowed_stride : nullptr);
  const int v0 = (int)((int64_t)r.n_vecs * part / per_row), v1 = busy ? (int)((int64_t)r.n_vecs * (part + 1) / per_row) : v0;

  // 1. the stretch, once
  float top = -INFINITY, sum = 0.f;
  int top_vec = 0;                       // first vector of the warp's chunk that the lane's maximum is in
  for (int vb = v0; vb < v1; vb += kChunkVecs) {
    uint4 raw[4];
    bool whole[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int v = vb + lane + 32 * j;
      whole[j] = v < v1 && r.whole(v);
      raw[j] = whole[j] ? r.raw(v) : make_uint4(0, 0, 0, 0);
    }
    float x[4][E], m = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int v = vb + lane + 32 * j;
      if (v < v1) {
        r.elements(v, whole[j], raw[j], x[j]);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[j][i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < E; ++i) m = fmaxf(m, x[j][i]);
    }
    if (m > top) {
      sum *= exp2_of((top - m) * kLog2e);
      top = m;
      top_vec = vb;
    }
    const float base = top == -INFINITY ? 0.f : top;     // (nothing allowed yet: every term is exp2(-inf), or a NaN, which stays one)
    float part_sum[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      part_sum[j] = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) part_sum[j] += exp2_of((x[j][i] - base) * kLog2e);
    }
    sum += (part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]);
  }
  // (fmaxf passes over NaN: the sum has it.  +inf: its own term is a NaN.)
  float wtop = top;
#pragma unroll
  for (int o = 16; o; o >>= 1) wtop = fmaxf(wtop, __shfl_xor_sync(~0u, wtop, o));
  float wsum = top == -INFINITY ? sum : sum * exp2_of((top - wtop) * kLog2e);
#pragma unroll
  for (int o = 16; o; o >>= 1) wsum += __shfl_xor_sync(~0u, wsum, o);
  cluster.barrier_wait();
  if (busy && lane < kClusterCtas) {
    SelectSmem* to = cluster.map_shared_rank(&s, lane);
    to->unit_max[unit] = wtop;
    to->unit_sum[unit] = (double)wsum;
  }
  cluster.sync();

  // The four lanes' bid: the largest maximum, and of equal ones the first chunk.
  float bid = top;
  int bid_vec = top_vec;
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const float b2 = __shfl_xor_sync(~0u, bid, o);
    const int v2 = __shfl_xor_sync(~0u, bid_vec, o);
    if (b2 > bid || (b2 == bid && v2 < bid_vec)) { bid = b2; bid_vec = v2; }
  }
  const int four = lane >> 2, four_lane = lane & 3;
  const int row_base = row * a.vocab;
  const int bid_first = row_base + max(0, (bid_vec + 4 * four) * E - r.shift);
  const int bid_last = row_base + min(a.vocab - 1, (bid_vec + 4 * four + 3 + 96) * E + E - 1 - r.shift);
  const double near = 2 * row_error((a.vocab / E + 2) / (per_row * kChunkVecs) + 2);
  SelectSmem* const lead = cluster.map_shared_rank(&s, 0);

  // Normalisers of the rows that this CTA's thread `tid` looks after, from the units' sums.
  if (tid < n_live) {
    float m = -INFINITY;
    for (int i = 0; i < per_row; ++i) m = fmaxf(m, s.unit_max[tid * per_row + i]);
    double t = 0.0;
    for (int i = 0; i < per_row; ++i) {
      const int u = tid * per_row + i;
      t += s.unit_max[u] == -INFINITY ? s.unit_sum[u] : s.unit_sum[u] * exp((double)s.unit_max[u] - (double)m);
    }
    s.row_max[s.live[tid]] = m;
    s.row_lse[s.live[tid]] = m == -INFINITY ? (double)NAN : log(t);
  }
  __syncthreads();

  for (;;) {
    // 2. bids and the bar
    const double score = busy ? s.score[row] : 0.0, base = busy ? s.row_max[row] : 0.0, lse = busy ? s.row_lse[row] : 0.0;
    auto sum_of = [&](float x) { return score + (((double)x - base) - lse); };
    double bid_sum = busy && bid != -INFINITY ? sum_of(bid) : kNone;
    if (!(bid_sum > kNone)) bid_sum = kNone;              // a row without a normaliser (NaN, +inf, nothing allowed) bids nothing
    const int bid_at = bid_sum == kNone ? 0x7fffffff : bid_last;
    if (four_lane == 0) { s.bid_sum[warp * 8 + four] = bid_sum; s.bid_at[warp * 8 + four] = bid_at; }
    if (tid == 0) s.n_list = 0;
    __syncthreads();
    {
      int rank = 0;
      for (int i = four_lane; i < warps * 8; i += 4) rank += bid_before(s.bid_sum[i], s.bid_at[i], i, bid_sum, bid_at, warp * 8 + four);
      rank += __shfl_xor_sync(~0u, rank, 1);
      rank += __shfl_xor_sync(~0u, rank, 2);
      if (rank < need) {
        for (int c = four_lane; c < kClusterCtas; c += 4) {
          SelectSmem* to = cluster.map_shared_rank(&s, c);
          to->top_sum[cta * need + rank] = bid_sum;
          to->top_at[cta * need + rank] = bid_at;
        }
      }
    }
    cluster.sync();
    const int n_top = kClusterCtas * need;
    for (int b0 = 0; b0 < n_top; b0 += blockDim.x / 2) {        // two threads a bid
      const int b = min(b0 + (tid >> 1), n_top - 1);
      const double bs = s.top_sum[b];
      const int ba = s.top_at[b];
      int rank = 0;
      for (int j = tid & 1; j < n_top; j += 2) rank += bid_before(s.top_sum[j], s.top_at[j], j, bs, ba, b);
      rank += __shfl_xor_sync(~0u, rank, 1);
      if (rank == need - 1) { s.bar_sum = bs; s.bar_at = ba; }
    }
    __syncthreads();

    // 3. the stretches whose bid reaches the bar
    const double bar_sum = s.bar_sum;
    const int bar_at = s.bar_at;
    // Calls found(sum, at) for what the lane holds of four f's candidates that reach the bar: of two chunks a turn, a vector a lane.
    auto sweep = [&](int f, auto&& found) {
      for (int vb = v0; vb < v1; vb += 2 * kChunkVecs) {
        const int c = lane & 15, v = vb + (lane >> 4) * kChunkVecs + 4 * f + (c & 3) + 32 * (c >> 2);
        if (v >= v1) continue;
        float x[E];
        const bool whole = r.whole(v);
        r.elements(v, whole, whole ? r.raw(v) : make_uint4(0, 0, 0, 0), x);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          if (x[i] == -INFINITY) continue;
          const int at = row_base + v * E - r.shift + i;
          const double c_sum = sum_of(x[i]);
          if (!before(bar_sum, bar_at, c_sum, at)) found(c_sum, at);
        }
      }
    };
    auto put = [&](double c_sum, int at) {
      const int slot = atomicAdd(&lead->n_list, 1);
      if (slot < kMaxList - kMaxK) { lead->list_sum[slot] = c_sum; lead->list_at[slot] = at; }
    };
    uint32_t todo = __ballot_sync(~0u, four_lane == 0 && bid_sum > kNone && !before(bar_sum, bar_at, bid_sum, bid_first));
    while (todo) {
      const int f = (__ffs(todo) - 1) >> 2;
      todo &= todo - 1;
      int n = 0;
      sweep(f, [&](double, int) { ++n; });
      n = __reduce_add_sync(~0u, n);
      if (n <= 32) {
        sweep(f, put);
        continue;
      }
      double prev_sum = 0.0;                 // many (equal or sorted logits): the best `need` of them, one by one
      int prev_at = 0;
      for (int turn = 0; turn < need; ++turn) {
        double best_sum = kNone;
        int best_at = 0x7fffffff;
        sweep(f, [&](double c_sum, int at) {
          if ((turn == 0 || before(prev_sum, prev_at, c_sum, at)) && before(c_sum, at, best_sum, best_at)) { best_sum = c_sum; best_at = at; }
        });
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const double s2 = __shfl_xor_sync(~0u, best_sum, o);
          const int a2 = __shfl_xor_sync(~0u, best_at, o);
          if (before(s2, a2, best_sum, best_at)) { best_sum = s2; best_at = a2; }
        }
        if (best_sum == kNone) break;
        if (lane == 0) put(best_sum, best_at);
        prev_sum = best_sum;
        prev_at = best_at;
      }
    }
    cluster.sync();

    // 4. the order
    int n_sorted = 0;
    if (cta == 0) {
      if (warp == 0) {
        const int n = min(s.n_list, kMaxList - kMaxK);
        const uint32_t ended = s.done_bits & s.finite_bits;
        __syncwarp();
        if ((ended >> lane) & 1) {
          const int slot = n + __popc(ended & ((1u << lane) - 1));
          s.list_sum[slot] = s.score[lane];
          s.list_at[slot] = lane * a.vocab + a.eos;
        }
        if (lane == 0) s.n_list = n + __popc(ended);
      }
      __syncthreads();
      const int n = s.n_list;
      n_sorted = min(n, kSorted);
      for (int i = tid; i < n; i += blockDim.x) {
        const double cs = s.list_sum[i];
        const int ca = s.list_at[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += before(s.list_sum[j], s.list_at[j], cs, ca);
        if (rank < kSorted) { s.sorted_sum[rank] = cs; s.sorted_at[rank] = ca; }
      }
      __syncthreads();
      if (warp == 0) {
        // Pair i = sorted i and i + 1.  The first pair from the k-th on that is not near closes the order: what comes behind it cannot be
        // among the k best.  A near pair of two rows before that, one of them summed in 32 bits, has to be settled.
        uint32_t near_bits[2], ask = 0;
        uint32_t unsure_bits[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = lane + 32 * h;
          bool is_near = false, unsure = false;
          if (i + 1 < n_sorted) {
            const uint32_t r1 = s.sorted_at[i] / a.vocab, r2 = s.sorted_at[i + 1] / a.vocab;
            is_near = s.sorted_sum[i] - s.sorted_sum[i + 1] < near;
            unsure = is_near && r1 != r2 && !((s.exact_bits >> r1) & (s.exact_bits >> r2) & 1);
          }
          near_bits[h] = __ballot_sync(~0u, is_near);
          unsure_bits[h] = __ballot_sync(~0u, unsure);
        }
        const uint64_t is_near = near_bits[0] | (uint64_t)near_bits[1] << 32, unsure = unsure_bits[0] | (uint64_t)unsure_bits[1] << 32;
        const uint64_t from_k = ~is_near & ~((1ull << (k - 1)) - 1);
        const int close = __ffsll((long long)from_k) - 1;                     // (pair kSorted - 1 is never near)
        const uint64_t matter = unsure & ((2ull << close) - 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = lane + 32 * h;
          if ((matter >> i) & 1) ask |= (1u << (s.sorted_at[i] / a.vocab)) | (1u << (s.sorted_at[i + 1] / a.vocab));
        }
        ask = __reduce_or_sync(~0u, ask);
        if (close >= n_sorted - 1 && n_sorted >= k && bar_sum > kNone) ask = ~0u;      // the list ends before the order is closed
        ask &= s.finite_bits & ~s.exact_bits;
        if (lane < kClusterCtas) cluster.map_shared_rank(&s, lane)->ask_bits = ask;
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
        a.out_scores[o] = some ? (float)s.sorted_sum[tid] : -INFINITY;
        if (a.out_done) a.out_done[o] = !some || ((s.done_bits >> parent) & 1) || token == a.eos;
      }
      return;
    }
    // The rows that are asked for, in 64 bits: cut and added up by the words' own numbers, wherever the row begins, so that equal rows get
    // equal sums and their ties stay ties.
    if (busy && ((ask >> row) & 1)) {
      double t = 0.0;
      const int e1 = (int)((int64_t)a.vocab * (part + 1) / per_row);
      for (int at = (int)((int64_t)a.vocab * part / per_row) + lane; at < e1; at += 32)
        if (r.may(at)) t += exp((double)to_float(r.p[at]) - base);
#pragma unroll
      for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
      if (lane < kClusterCtas) cluster.map_shared_rank(&s, lane)->unit_sum[unit] = t;
    }
    cluster.sync();
    if (tid < n_live && ((ask >> s.live[tid]) & 1)) {
      double t = 0.0;
      for (int i = 0; i < per_row; ++i) t += s.unit_sum[tid * per_row + i];
      s.row_lse[s.live[tid]] = log(t);
    }
    if (tid == 0) s.exact_bits |= ask;
    __syncthreads();
  }
}

template <class T>
cudaError_t launch_select(const linmt_beam_select_args& g, int warps) {
  SelectParams<T> p{static_cast<const T*>(g.logits), g.stride_n, g.stride_k, g.scores, g.done, g.allowed, g.allowed_stride,
                    g.out_tokens, g.out_parents, g.out_scores, g.out_done, g.k, g.vocab, g.eos};
  select_kernel<T><<<dim3((unsigned)g.n * kClusterCtas), dim3(warps * 32), 0, static_cast<cudaStream_t>(g.stream)>>>(p);
  return cudaGetLastError();
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
  int32_t n, k, n_states;
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
  const int64_t at = ((int64_t)blockIdx.x - st.first_block) * kReorderThreads + threadIdx.x, ln = at / st.cols, col = at - ln * st.cols;
  const int64_t l = ln / a.n, n = ln - l * a.n;
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
  if (g->k > kMaxK || (int64_t)g->k * g->vocab >= INT32_MAX || g->n > (1 << 27))
    return op_fail(LINMT_ELIMIT, "beam_select: k = %d (at most %d), k * vocab = %lld (below 2^31), n = %d", g->k, kMaxK, (long long)g->k * g->vocab, g->n);
  if (g->n == 0) return LINMT_OK;
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "beam_select");
  // Warps of a CTA: as many as leave the fewest without a stretch when every beam is live (12 beams: 96 of 8 x 12).
  int warps = kMaxWarps, most = 0;
  for (int w = kMaxWarps; w >= kMaxWarps / 2; --w) {
    const int used = kClusterCtas * w / g->k * g->k * 1000 / (kClusterCtas * w);
    if (used > most) { most = used; warps = w; }
  }
  const cudaError_t e = g->dtype == LINMT_F32 ? launch_select<float>(*g, warps) : g->dtype == LINMT_BF16 ? launch_select<__nv_bfloat16>(*g, warps) : launch_select<__half>(*g, warps);
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "beam_select");
}

int linmt_beam_reorder(const linmt_beam_reorder_args* g) {
  using namespace linmt::ops;
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "beam_reorder: not this library's argument struct");
  if (!g->parents || !aligned(g->parents, 4) || g->n < 0 || g->k < 1 || g->n_states < 0 || g->n_states > 16)
    return op_fail(LINMT_EINVAL, "beam_reorder: n = %d, k = %d, %d states (at most 16), parents %p", g->n, g->k, g->n_states, (const void*)g->parents);
  if (g->k > kMaxK) return op_fail(LINMT_ELIMIT, "beam_reorder: k = %d (at most %d)", g->k, kMaxK);
  ReorderParams p{};
  p.parents = g->parents; p.n = g->n; p.k = g->k;
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
