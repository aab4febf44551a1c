// token_ops.cu -- scores of given tokens (linmt_score_tokens): log probability, entropy and the best alternatives of rows of logits.
//
//   d = x log2 e - k, S = sum 2^d, T = sum 2^d d:   log sum exp x = (k + log2 S) ln 2,   entropy = ln 2 (log2 S - T / S)
// with a whole number k, at most 8 below the largest x log2 e, so that d is rounded once.  (Of an entropy next to 0 some 1e-6 are left: log2 S and T / S may both be about 8 then, and what they were rounded by is.)  One pass over a row, each thread
// with a k of its own, two logits an instruction where there is one for two.  A row whose largest logit is beyond 65536 in size is added up once more relative to e^m, m that logit itself:
// k and x log2 e have no place left behind the point from 2^23 on, and logits that far apart are told apart by x - m alone.  Bound by HBM in 32 bits, by instructions (unpacking 1, list 2, the rest 6 an element) in 16.
// The k-th largest of 32 groups' maxima is reached by k words at least: only the words of threads whose own maximum reaches it are looked at again (from L2), by their whole warp, and what
// reaches it goes on a list in shared memory, which is ranked by counting.  (Each such thread by itself, its warp waiting: 1968 rows of 80,000 words in 16 bits took 189 us.)  Equal logits
// may overfill the list; then the best are found one by one, in a pass over the row for each.  Long rows where there are few go to a cluster of CTAs, joined through its shared memory.
#include <cooperative_groups.h>

#include "device_ops.h"

namespace linmt {
namespace ops {
namespace {

namespace cg = cooperative_groups;

constexpr int kGroups = 32;                                // a group: the same lane of all warps
constexpr int kTop = 32;
constexpr int kList = 1024;
constexpr int kMaxCluster = 8;
constexpr int kAhead = 4;                                  // vectors of a thread on their way
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

struct ScoreParams {
  const void* logits;
  int64_t stride_n, stride_t;
  const int32_t* tokens;
  const uint32_t* allowed;
  int64_t allowed_stride;
  float* logprob;
  float* entropy;
  int32_t* top_tokens;
  float* top_logprobs;
  int32_t t, vocab, top;
};

__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float exp2_of(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__device__ __forceinline__ float max_nan(float a, float b, float c) { return max_nan(max_nan(a, b), c); }
// Two numbers at a time.
__device__ __forceinline__ unsigned long long bits_of(float2 a) { unsigned long long r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y)); return r; }
__device__ __forceinline__ float2 pair_of(unsigned long long a) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a)); return r; }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { unsigned long long r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c))); return pair_of(r); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { unsigned long long r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b))); return pair_of(r); }

// m the largest logit (NaN once one was met), s and t the sums relative to 2^k.  Nothing so far: -inf and sums of 0.  Where m is beyond kFar the sums of a CTA are relative to e^m, and k is not used.
constexpr float kFar = 65536.f, kLost = 4194304.f, kNone = -1e30f, kSlack = 8.f;
struct Sums { float m, k, s, t; };
__device__ __forceinline__ bool far(const Sums& a) { return fabsf(a.m) > kFar; }
// The sums relative to something 2^-d times as large.
__device__ __forceinline__ void lower(Sums& a, float d) {
  d = fmaxf(d, -150.f);
  const float f = exp2_of(d);
  a.t = f * fmaf(a.s, d, a.t);
  a.s *= f;
}
// Of two threads: both relative to 2^k.  One's beyond kLost (2^22, where k is no longer exact) count nothing beside another's, or the row is added up again.
__device__ __forceinline__ Sums join_threads(Sums a, Sums b) {
  Sums r{max_nan(a.m, b.m), fmaxf(a.k, b.k), 0.f, 0.f};
  if (fabsf(a.m) <= kLost) { lower(a, a.k - r.k); r.s += a.s; r.t += a.t; }
  if (fabsf(b.m) <= kLost) { lower(b, b.k - r.k); r.s += b.s; r.t += b.t; }
  return r;
}
// Of two threads or CTAs whose sums are relative to e^m, m far or not and the same for all; and of two CTAs, each by its own largest logit.
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  Sums r{max_nan(a.m, b.m), fmaxf(a.k, b.k), 0.f, 0.f};
  auto above = [&](const Sums& x) {              // of what x is relative to, above what r is
    return far(r) ? far(x) ? (x.m - r.m) * kLog2e : -fmaf(r.m, kLog2e, -x.k) : far(x) ? fmaf(x.m, kLog2e, -r.k) : x.k - r.k;
  };
  lower(a, above(a));
  lower(b, above(b));
  r.s = a.s + b.s;
  r.t = a.t + b.t;
  return r;
}

// A word with its logit; of two the better has the larger logit, or the lower number.
struct Word { float x; int32_t v; };
__device__ __forceinline__ bool better(const Word& a, const Word& b) { return a.x > b.x || (a.x == b.x && a.v < b.v); }

template <class T, bool LISTS>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  const T* x;
  const uint32_t* allowed;
  int vocab, lead, vectors;          // words before the first 16-byte boundary; whole vectors behind it

  __device__ __forceinline__ float at(int v) const {
    const float y = to_float(x[v]);
    return !LISTS || (__ldg(allowed + (v >> 5)) >> (v & 31) & 1) ? y : -INFINITY;
  }
  // Which of words first .. first + kVec - 1 are allowed, and a vector of them as numbers, -inf where they are not.
  __device__ __forceinline__ uint32_t list(int first) const {
    if (!LISTS) return ~0u;
    const int w = first >> 5, s = first & 31;
    return __funnelshift_r(__ldg(allowed + w), s + kVec > 32 ? __ldg(allowed + w + 1) : 0, s);
  }
  __device__ __forceinline__ void open(const uint4& raw, uint32_t bits, float (&y)[kVec]) const {
    const T* const e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < kVec; ++i) y[i] = !LISTS || (bits >> i & 1) ? to_float(e[i]) : -INFINITY;
  }
  __device__ __forceinline__ const uint4* vector(int i) const { return reinterpret_cast<const uint4*>(x + lead) + i; }
  // The words outside the vectors: fewer than 2 kVec.
  __device__ __forceinline__ int odd(int i) const { return i < lead ? i : vectors * kVec + i; }
  __device__ __forceinline__ int odds() const { return vocab - vectors * kVec; }
};

// A thread's sums as it goes: two of each.
struct Running {
  float m = -INFINITY, k = kNone;
  float2 s = {0.f, 0.f}, t = {0.f, 0.f};
  __device__ __forceinline__ void follow() {           // k follows a maximum that exceeds it
    float now = ceilf(m * kLog2e);
    if (fabsf(now) > kLost) now += fabsf(now) * 4.76837158203125e-7f;      // (rounded: no term may exceed it, as sums that go into nothing still have to be numbers)
    const float d = fmaxf(k - now, -150.f), f = exp2_of(d);
    t.x = f * fmaf(s.x, d, t.x);
    t.y = f * fmaf(s.y, d, t.y);
    s.x *= f;
    s.y *= f;
    k = now;
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&y)[N]) {
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) m = max_nan(m, y[i], y[i + 1]);
    if (N & 1) m = max_nan(m, y[N - 1]);
    if (fmaf(m, kLog2e, -k) > kSlack) follow();
    const float2 up = make_float2(kLog2e, kLog2e), down = make_float2(-k, -k);
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) {
      float2 d = fma2(make_float2(y[i], y[i + 1]), up, down);
      d.x = fmaxf(d.x, -150.f);                        // (-inf; NaN, too: the maximum has it)
      d.y = fmaxf(d.y, -150.f);
      const float2 e = make_float2(exp2_of(d.x), exp2_of(d.y));
      s = add2(s, e);
      t = fma2(e, d, t);
    }
    if (N & 1) {
      const float d = fmaxf(fmaf(y[N - 1], kLog2e, -k), -150.f), e = exp2_of(d);
      s.x += e;
      t.x = fmaf(e, d, t.x);
    }
  }
  __device__ __forceinline__ Sums sums() const { return {m, k, s.x + s.y, t.x + t.y}; }
};

template <class T, bool LISTS, int kThreads>
__global__ void __launch_bounds__(kThreads, (sizeof(T) == 4 && !LISTS ? 1536 : 1280) / kThreads) score_kernel(const ScoreParams a) {
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row_at = blockIdx.x / ctas, i_n = row_at / a.t, i_t = row_at - i_n * a.t;
  constexpr int kVec = Row<T, LISTS>::kVec;
  __shared__ Sums warp_sums[kThreads / 32], cta_sums;
  __shared__ float most[kThreads / 32][kGroups], group_most[kGroups], bar;
  __shared__ int listed;
  __shared__ Word list[kList], best[kTop], found[kThreads / 32];

  Row<T, LISTS> row;
  row.x = static_cast<const T*>(a.logits) + i_n * a.stride_n + i_t * a.stride_t;
  row.allowed = LISTS ? a.allowed + i_n * a.allowed_stride : nullptr;
  row.vocab = a.vocab;
  row.lead = min(a.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row.x) & 15)) & 15) / (int)sizeof(T));
  row.vectors = (a.vocab - row.lead) / kVec;
  const int at = rank * kThreads + tid, all = ctas * kThreads;

  // Each of the thread's words: f(logits, first word's number) for its vectors, and for the one outside them that it may have.
  auto each = [&](auto f) {
    for (int i0 = at; i0 < row.vectors; i0 += kAhead * all) {
      uint4 raw[kAhead];
      uint32_t bits[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (i0 + j * all < row.vectors) {
          raw[j] = __ldg(row.vector(i0 + j * all));
          bits[j] = row.list(row.lead + (i0 + j * all) * kVec);
        }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (i0 + j * all >= row.vectors) break;
        float y[kVec];
        row.open(raw[j], bits[j], y);
        f(y);
      }
    }
    if (at < row.odds()) {
      const float y[1] = {row.at(row.odd(at))};
      f(y);
    }
  };
  auto join_lanes = [](Sums x, int lanes, auto two) {
    for (int o = 1; o < lanes; o <<= 1) x = two(x, {__shfl_xor_sync(~0u, x.m, o), __shfl_xor_sync(~0u, x.k, o), __shfl_xor_sync(~0u, x.s, o), __shfl_xor_sync(~0u, x.t, o)});
    return x;
  };
  auto near = [](const Sums& a, const Sums& b) { return join_threads(a, b); };
  const Sums nothing{-INFINITY, kNone, 0.f, 0.f};
  Running running;
  each([&](const auto& y) { running.add(y); });
  const float own = running.m;

  // The row's sums, and a bar that `top` words reach.
  if (a.top) most[warp][lane] = own;
  Sums sums = join_lanes(running.sums(), 32, near);
  if (lane == 0) warp_sums[warp] = sums;
  if (tid == 0) {
    listed = 0;
    bar = INFINITY;                                 // (stays where there is a NaN, and nothing is listed)
  }
  __syncthreads();
  if (warp == 0) {
    sums = join_lanes(lane < kThreads / 32 ? warp_sums[lane] : nothing, kThreads / 32, near);
    if (lane == 0) cta_sums = sums;
  } else if (warp == 1 && a.top) {
    float m = most[0][lane];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) m = max_nan(m, most[w][lane]);
    group_most[lane] = m;
    __syncwarp();
    int above = 0;                                  // groups before this one, by their maximum and number
    for (int i = 0; i < kGroups; ++i) {
      const float x = group_most[i];
      above += x > m || (x == m && i < lane);
    }
    if (above == a.top - 1) bar = m;
  }
  __syncthreads();
  if (far(cta_sums) && fabsf(cta_sums.m) < INFINITY) {
    const float m = cta_sums.m;
    Sums mine{m, kNone, 0.f, 0.f};
    each([&](const auto& y) {
      for (float x : y) {
        const float d = fmaxf((x - m) * kLog2e, -150.f), e = exp2_of(d);
        mine.s += e;
        mine.t = fmaf(e, d, mine.t);
      }
    });
    mine = join_lanes(mine, 32, join);
    if (lane == 0) warp_sums[warp] = mine;
    __syncthreads();
    if (warp == 0) {
      mine = join_lanes(lane < kThreads / 32 ? warp_sums[lane] : nothing, kThreads / 32, join);
      if (lane == 0) cta_sums = mine;
    }
  }
  if (ctas > 1) cluster.sync();
  else __syncthreads();

  if (a.top) {
    // The CTA's own best.
    const float reach = bar;
    const bool nan = !(cta_sums.m == cta_sums.m) || cta_sums.m == INFINITY;
    auto put = [&](float x, int v) {
      if (!(x >= reach) || x == -INFINITY) return;
      const int i = atomicAdd(&listed, 1);
      if (i < kList) list[i] = {x, v};
    };
    if (!nan) {
      // The words of the warp's threads that reach the bar, each thread's by all lanes.
      for (uint32_t left = __ballot_sync(~0u, own >= reach && own > -INFINITY); left; left &= left - 1) {
        const int from = at - lane + __ffs(left) - 1;
        for (int i = from + lane * all; i < row.vectors; i += 32 * all) {
          float y[kVec];
          row.open(__ldg(row.vector(i)), row.list(row.lead + i * kVec), y);
#pragma unroll
          for (int j = 0; j < kVec; ++j) put(y[j], row.lead + i * kVec + j);
        }
      }
      if (at < row.odds()) put(row.at(row.odd(at)), row.odd(at));
    }
    __syncthreads();
    const int n = listed;
    if (tid < a.top) best[tid] = {-INFINITY, -1};
    __syncthreads();
    if (n <= kList) {
      for (int i = tid; i < n; i += kThreads) {
        const Word mine = list[i];
        int before = 0;
        for (int j = 0; j < n; ++j) before += better(list[j], mine);
        if (before < a.top) best[before] = mine;
      }
    } else {
      Word last{INFINITY, -1};                       // (+inf is nowhere in the row)
      for (int k = 0; k < a.top; ++k) {
        Word w{-INFINITY, 0x7fffffff};
        auto look = [&](float x, int v) {
          const Word y{x, v};
          if (better(last, y) && better(y, w)) w = y;
        };
        for (int i = at; i < row.vectors; i += all) {
          float y[kVec];
          row.open(__ldg(row.vector(i)), row.list(row.lead + i * kVec), y);
#pragma unroll
          for (int j = 0; j < kVec; ++j) look(y[j], row.lead + i * kVec + j);
        }
        if (at < row.odds()) look(row.at(row.odd(at)), row.odd(at));
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const Word y{__shfl_xor_sync(~0u, w.x, o), __shfl_xor_sync(~0u, w.v, o)};
          if (better(y, w)) w = y;
        }
        if (lane == 0) found[warp] = w;
        __syncthreads();
        w = found[0];
        for (int i = 1; i < kThreads / 32; ++i)
          if (better(found[i], w)) w = found[i];
        __syncthreads();
        last = w;
        if (w.x == -INFINITY) break;
        if (tid == 0) best[k] = w;
      }
    }
    if (ctas > 1) cluster.sync();
    else __syncthreads();
  }

  if (rank == 0) {
    Sums r = cta_sums;
    for (int i = 1; i < ctas; ++i) r = join(r, *cluster.map_shared_rank(&cta_sums, i));
    const bool nan = !(r.m == r.m) || r.m == INFINITY, none = r.m == -INFINITY;
    const float log_s = log2f(r.s);
    auto logprob = [&](float x) { return far(r) ? (x - r.m) - kLn2 * log_s : fabsf(x) > 1e38f ? x - (r.k + log_s) * kLn2 : (fmaf(x, kLog2e, -r.k) - log_s) * kLn2; };
    if (tid == 0) {
      const int token = __ldg(a.tokens + row_at);
      const float x = token >= 0 && token < a.vocab ? row.at(token) : 0.f;
      a.logprob[row_at] = nan ? NAN : token < 0 || token >= a.vocab ? 0.f : none || x == -INFINITY ? -INFINITY : logprob(x);
      a.entropy[row_at] = nan ? NAN : none ? 0.f : fmaxf(kLn2 * (log_s - r.t / r.s), 0.f);
    }
    if (a.top) {
      for (int i = tid; i < ctas * kTop; i += kThreads) list[i] = i % kTop < a.top ? cluster.map_shared_rank(best, i / kTop)[i % kTop] : Word{-INFINITY, -1};
      __syncthreads();
      static_assert(kMaxCluster * kTop <= 2 * kThreads, "up to two a thread");
      int words = 0;
      for (int i0 = 0; i0 < ctas * kTop; i0 += kThreads) {
        const int i = i0 + tid;
        const Word w = i < ctas * kTop ? list[i] : Word{-INFINITY, -1};
        words += __syncthreads_count(w.v >= 0);
        if (w.v < 0) continue;
        int before = i % kTop;                      // and in each of the others' lists, which are in order, those that are better
        for (int c = 0; c < ctas; ++c) {
          if (c == i / kTop) continue;
          int lo = 0;
#pragma unroll
          for (int step = kTop / 2; step; step /= 2)
            if (better(list[c * kTop + lo + step - 1], w)) lo += step;
          before += lo + better(list[c * kTop + lo], w);
        }
        if (before < a.top && !nan) {
          a.top_tokens[(int64_t)row_at * a.top + before] = w.v;
          a.top_logprobs[(int64_t)row_at * a.top + before] = logprob(w.x);
        }
      }
      for (int i = (nan ? 0 : min(words, a.top)) + tid; i < a.top; i += kThreads) {      // no word is left
        a.top_tokens[(int64_t)row_at * a.top + i] = -1;
        a.top_logprobs[(int64_t)row_at * a.top + i] = nan ? NAN : -INFINITY;
      }
    }
  }
  if (ctas > 1) cluster.sync();
}

template <class T, bool LISTS>
cudaError_t launch_score(const ScoreParams& p, int64_t rows, cudaStream_t st) {
  // A short row (up to eight vectors a thread) needs no more than four warps: 3306 rows of 689 words took 37 us with 16.
  constexpr int kLong = 256, kShort = 128;
  const int64_t vectors = (int64_t)p.vocab * sizeof(T) / 16;
  const bool is_short = vectors <= 8 * kShort;
  // Several CTAs a row as long as the GPU has room for them, and each has a few vectors a thread.
  int ctas = 1;
  while (!is_short && ctas < kMaxCluster && rows * ctas * 2 <= 4 * 148 && vectors >= (int64_t)ctas * 2 * kLong * 4) ctas *= 2;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(is_short ? kShort : kLong);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = is_short ? cudaLaunchKernelEx(&cfg, score_kernel<T, LISTS, kShort>, p) : cudaLaunchKernelEx(&cfg, score_kernel<T, LISTS, kLong>, p);
  return e == cudaSuccess ? cudaGetLastError() : e;
}
template <class T>
cudaError_t launch_score(const ScoreParams& p, int64_t rows, cudaStream_t st) {
  return p.allowed ? launch_score<T, true>(p, rows, st) : launch_score<T, false>(p, rows, st);
}

}  // namespace
}  // namespace ops
}  // namespace linmt

extern "C" {

int linmt_score_tokens(const linmt_score_tokens_args* g) {
  using namespace linmt::ops;
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "score_tokens: not this library's argument struct");
  if (g->n < 0 || g->t < 0 || g->vocab < 1 || g->top < 0 || !dtype_ok(g->dtype)) return op_fail(LINMT_EINVAL, "score_tokens: n = %d, t = %d, vocab = %d, top = %d, dtype = %d", g->n, g->t, g->vocab, g->top, g->dtype);
  if (g->top > kTop || (int64_t)g->n * g->t > INT32_MAX || g->vocab > INT32_MAX - 4095) return op_fail(LINMT_ELIMIT, "score_tokens: top = %d (at most %d), n * t = %lld, vocab = %d (below 2^31)", g->top, kTop, (long long)g->n * g->t, g->vocab);
  if (g->n == 0 || g->t == 0) return LINMT_OK;
  if (!g->logits || !g->tokens || !g->out_logprob || !g->out_entropy || (g->top && (!g->out_top_tokens || !g->out_top_logprobs))) return op_fail(LINMT_EINVAL, "score_tokens: an array is missing");
  if (!aligned(g->logits, dtype_bytes(g->dtype)) || !aligned(g->tokens, 4) || !aligned(g->allowed, 4) || !aligned(g->out_logprob, 4) || !aligned(g->out_entropy, 4) || !aligned(g->out_top_tokens, 4) || !aligned(g->out_top_logprobs, 4))
    return op_fail(LINMT_EINVAL, "score_tokens: an array is not aligned to its type");
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "score_tokens");
  const ScoreParams p{g->logits, g->stride_n, g->stride_t, g->tokens, g->allowed, g->allowed_stride, g->out_logprob, g->out_entropy, g->out_top_tokens, g->out_top_logprobs, g->t, g->vocab, g->top};
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  const int64_t rows = (int64_t)g->n * g->t;
  const cudaError_t e = g->dtype == LINMT_F32 ? launch_score<float>(p, rows, st) : g->dtype == LINMT_BF16 ? launch_score<__nv_bfloat16>(p, rows, st) : launch_score<__half>(p, rows, st);
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "score_tokens");
}

}  // extern "C"
