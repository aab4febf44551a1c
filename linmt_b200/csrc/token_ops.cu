// token_ops.cu -- scores of given tokens (linmt_score_tokens): log probability, entropy and the best alternatives of rows of logits.
//
//   m = max x, d = (x - m) log2 e, S = sum 2^d, T = sum 2^d d:   log sum exp x = m + ln S,   entropy = ln S - ln 2 T / S
// T's terms are all of one sign, so nothing cancels.  One pass over a row, each thread with a maximum of its own so far and sums relative to it.
// The k-th largest of 32 groups' maxima is reached by k words at least: only threads whose own maximum reaches it look at their words again (from L2), and what
// reaches it goes on a list in shared memory, which is ranked by counting.  Equal logits may overfill the list; then the k best are found one by
// one, in k passes over the row.  Long rows where there are few go to a cluster of CTAs, joined through its shared memory.
#include <cooperative_groups.h>

#include "device_ops.h"

namespace linmt {
namespace ops {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kGroups = 32, kGroup = kThreads / kGroups;   // lanes of a group: half a warp
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

// m the largest logit so far (NaN once one was met), sums relative to it.  Nothing so far: -inf, 0, 0.
struct Sums { float m, s, t; };
// The sums relative to a larger maximum.
__device__ __forceinline__ void raise(Sums& a, float m) {
  if (a.s > 0.f) {
    const float d = fmaxf((a.m - m) * kLog2e, -150.f), f = exp2_of(d);
    a.t = f * fmaf(a.s, d, a.t);
    a.s *= f;
  }
  a.m = m;
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = max_nan(a.m, b.m);
  raise(a, m);
  raise(b, m);
  return {m, a.s + b.s, a.t + b.t};
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
  // Words first .. first + kVec - 1 of a vector, -inf where they are not allowed.
  __device__ __forceinline__ void open(const uint4& raw, int first, float (&y)[kVec]) const {
    const T* const e = reinterpret_cast<const T*>(&raw);
    uint32_t bits = ~0u;
    if (LISTS) {
      const int w = first >> 5, s = first & 31;
      bits = __ldg(allowed + w) >> s;
      if (s + kVec > 32) bits |= __ldg(allowed + w + 1) << (32 - s);
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) y[i] = !LISTS || (bits >> i & 1) ? to_float(e[i]) : -INFINITY;
  }
  __device__ __forceinline__ const uint4* vector(int i) const { return reinterpret_cast<const uint4*>(x + lead) + i; }
  // The words outside the vectors: fewer than 2 kVec.
  __device__ __forceinline__ int odd(int i) const { return i < lead ? i : vectors * kVec + i; }
  __device__ __forceinline__ int odds() const { return vocab - vectors * kVec; }
};

template <int N>
__device__ __forceinline__ void add(Sums& a, const float (&y)[N]) {
  float m = y[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = max_nan(m, y[i]);
  if (!(m <= a.m)) raise(a, max_nan(m, a.m));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = fmaxf((y[i] - a.m) * kLog2e, -150.f), e = exp2_of(d);      // (NaN: -150; the maximum has it)
    a.s += e;
    a.t = fmaf(e, d, a.t);
  }
}

template <class T, bool LISTS>
__global__ void __launch_bounds__(kThreads) score_kernel(const ScoreParams a) {
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row_at = blockIdx.x / ctas, i_n = row_at / a.t, i_t = row_at - i_n * a.t;
  constexpr int kVec = Row<T, LISTS>::kVec;
  __shared__ Sums warp_sums[kThreads / 32], cta_sums;
  __shared__ float group_most[kGroups], bar;
  __shared__ int listed;
  __shared__ Word list[kList], best[kTop], found[kThreads / 32];

  Row<T, LISTS> row;
  row.x = static_cast<const T*>(a.logits) + i_n * a.stride_n + i_t * a.stride_t;
  row.allowed = LISTS ? a.allowed + i_n * a.allowed_stride : nullptr;
  row.vocab = a.vocab;
  row.lead = min(a.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row.x) & 15)) & 15) / (int)sizeof(T));
  row.vectors = (a.vocab - row.lead) / kVec;
  const int at = rank * kThreads + tid, all = ctas * kThreads;

  Sums sums{-INFINITY, 0.f, 0.f};
  for (int i0 = at; i0 < row.vectors; i0 += kAhead * all) {
    uint4 raw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + j * all < row.vectors) raw[j] = __ldg(row.vector(i0 + j * all));
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j * all >= row.vectors) break;
      float y[kVec];
      row.open(raw[j], row.lead + (i0 + j * all) * kVec, y);
      add(sums, y);
    }
  }
  if (at < row.odds()) {
    const float y[1] = {row.at(row.odd(at))};
    add(sums, y);
  }
  const float own = sums.m;

  // The row's sums, and a bar that `top` words reach.
  if (a.top) {
    float m = own;
#pragma unroll
    for (int o = 1; o < kGroup; o <<= 1) m = max_nan(m, __shfl_xor_sync(~0u, m, o));
    if (tid % kGroup == 0) group_most[tid / kGroup] = m;
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) sums = join(sums, {__shfl_xor_sync(~0u, sums.m, o), __shfl_xor_sync(~0u, sums.s, o), __shfl_xor_sync(~0u, sums.t, o)});
  if (lane == 0) warp_sums[warp] = sums;
  if (tid == 0) {
    listed = 0;
    bar = INFINITY;                                 // (stays where there is a NaN, and nothing is listed)
  }
  __syncthreads();
  if (warp == 0) {
    sums = lane < kThreads / 32 ? warp_sums[lane] : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = 1; o < kThreads / 32; o <<= 1) sums = join(sums, {__shfl_xor_sync(~0u, sums.m, o), __shfl_xor_sync(~0u, sums.s, o), __shfl_xor_sync(~0u, sums.t, o)});
    if (lane == 0) cta_sums = sums;
  } else if (warp == 1 && a.top) {
    const float m = group_most[lane];
    int above = 0;                                  // groups before this one, by their maximum and number
    for (int i = 0; i < kGroups; ++i) {
      const float x = group_most[i];
      above += x > m || (x == m && i < lane);
    }
    if (above == a.top - 1) bar = m;
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
    if (!nan && own >= reach && own > -INFINITY) {
      for (int i = at; i < row.vectors; i += all) {
        float y[kVec];
        row.open(__ldg(row.vector(i)), row.lead + i * kVec, y);
#pragma unroll
        for (int j = 0; j < kVec; ++j) put(y[j], row.lead + i * kVec + j);
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
          row.open(__ldg(row.vector(i)), row.lead + i * kVec, y);
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
    const float log_s = logf(r.s);
    if (tid == 0) {
      const int token = __ldg(a.tokens + row_at);
      const float x = token >= 0 && token < a.vocab ? row.at(token) : 0.f;
      a.logprob[row_at] = nan ? NAN : token < 0 || token >= a.vocab ? 0.f : none || x == -INFINITY ? -INFINITY : (x - r.m) - log_s;
      a.entropy[row_at] = nan ? NAN : none ? 0.f : fmaxf(log_s - kLn2 * r.t / r.s, 0.f);
    }
    if (a.top) {
      for (int i = tid; i < ctas * kTop; i += kThreads) list[i] = i % kTop < a.top ? cluster.map_shared_rank(best, i / kTop)[i % kTop] : Word{-INFINITY, -1};
      __syncthreads();
      int words = 0;
      for (int i = tid; i < ctas * kTop; i += kThreads) {
        const Word w = list[i];
        if (w.v < 0) continue;
        int before = i % kTop;
        for (int j = 0; j < ctas * kTop; ++j) before += j / kTop != i / kTop && list[j].v >= 0 && better(list[j], w);
        if (before < a.top && !nan) {
          a.top_tokens[(int64_t)row_at * a.top + before] = w.v;
          a.top_logprobs[(int64_t)row_at * a.top + before] = (w.x - r.m) - log_s;
        }
      }
      for (int j = 0; j < ctas * kTop; ++j) words += list[j].v >= 0;
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
  // Several CTAs a row as long as the GPU has room for them, and each has a few vectors a thread.
  const int64_t vectors = (int64_t)p.vocab * sizeof(T) / 16;
  int ctas = 1;
  while (ctas < kMaxCluster && rows * ctas * 2 <= 2 * 148 && vectors >= (int64_t)ctas * 2 * kThreads * 2) ctas *= 2;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, score_kernel<T, LISTS>, p);
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
