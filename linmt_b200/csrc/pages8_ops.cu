// pages8_ops.cu -- keys and values into and out of pages in 8 bits (linmt_write_pages8, linmt_read_pages8).  Attention over them: pages8_attend.cu.
//
// A scale belongs to a block of 16 positions, so positions of a block that are written together have to be looked at together: a CTA
// takes the runs (neighbours in the list that are neighbours in a block) that begin among its positions, one after the other, head by head.  Half of its threads
// have the keys, half the values, a thread 16 components of one position.  Keys go out as they come, 16 bytes a thread.  Values
// lie position by position within a component and are turned round in shared memory.
// A block is written whole: a position's value codes lie in every 32-byte sector of the block's half, so they would all be touched anyway.
#include "device_ops.h"
#include "pages8.h"

namespace linmt {
namespace ops {
namespace {

struct RowsParams {
  unsigned char* data;
  int64_t stride_page, stride_head;
  int32_t n_pages, heads, page;
  const int64_t* slots;
  void* k;
  void* v;
  int64_t k_t, k_h, v_t, v_h;
  int32_t t, heads_each, window;
};

struct Run {
  int64_t at;              // the block's place in the pool (head 0); -1: slots outside it (of a read)
  int first, len, offset;  // positions first .. first + len - 1 of the call are the block's offset ..
};

// The runs that begin at the CTA's positions; of a read those among them alone.  All threads call it.
template <bool WRITE, int D>
__device__ __forceinline__ int runs_of_cta(const RowsParams& a, Run* runs) {
  __shared__ int count;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const int64_t t = (int64_t)blockIdx.x * a.window - 1 + lane;                       // lane 1 has the CTA's first position
    const bool mine = lane >= 1 && lane <= a.window && t < a.t, there = t >= 0 && t < a.t && (WRITE || mine);
    int64_t slot = there ? __ldg(a.slots + t) : -1;
    if (pages8::slot_page(slot, a.n_pages, a.page) < 0) slot = -1;
    const int64_t before = __shfl_up_sync(~0u, (long long)slot, 1);
    const uint32_t goes_on = __ballot_sync(~0u, lane > 0 && there && pages8::follows(before, slot));
    const bool begins = mine && (WRITE ? slot >= 0 : true) && !(goes_on >> lane & 1);
    const uint32_t all = __ballot_sync(~0u, begins);
    if (begins) {
      Run r;
      r.at = pages8::slot_block(slot, a.n_pages, a.page, a.stride_page, D);
      r.first = (int)t;
      r.offset = slot < 0 ? 0 : (int)(slot & (pages8::kBlock - 1));
      r.len = lane == 31 ? 1 : __ffs(~(goes_on >> (lane + 1)));                        // (lane 31 begins a run with a window of 31 only, and there is none)
      runs[__popc(all & ((1u << lane) - 1))] = r;
    }
    if (lane == 0) count = __popc(all);
  }
  __syncthreads();
  return count;
}

// 16 components of a row.
template <class T> struct Raw16 { uint4 r[sizeof(T)]; };
template <class T>
__device__ __forceinline__ Raw16<T> load16(const T* p) {
  Raw16<T> x;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) x.r[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return x;
}
template <class T>
__device__ __forceinline__ void store16(T* p, const float (&x)[16]) {
  uint4 r[sizeof(T)];
  T* e = reinterpret_cast<T*>(r);
#pragma unroll
  for (int i = 0; i < 16; ++i) e[i] = from_float<T>(x[i]);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) reinterpret_cast<uint4*>(p)[i] = r[i];
}

constexpr float kMost = 1.7014118346046923e38f;      // 2^127
constexpr float kMagic = 12582912.f;                 // 1.5 * 2^23: added to a number of a few bits, it leaves the nearest integer in the last ones

// The smallest of 4, 5, 6, 7 times a power of 2 whose 127-fold reaches `big`.  Three bits behind the point of a quotient are enough to find it but
// for its rounding, and 127 times such a number is exact.
__device__ __forceinline__ float scale_of(float big) {
  if (big == 0.f) return 0.f;
  const float least = 1.1754943508222875e-38f;       // 2^-126
  if (big <= 127.f * least) return least;
  uint32_t b = __float_as_uint(__fdiv_rn(big, 127.f)) & ~0x1fffffu;      // at most the scale, and at most one step below it
  if (b < 0x00800000u) b = 0x00800000u;
  // (the quotient may have been rounded up onto a scale that is a step too large: never, as big <= 127 s then)
  if (__uint_as_float(b) * 127.f < big) b += 0x200000u;
  return __uint_as_float(b);
}

// Codes of 16 components, as bytes.  A code is the quotient in 32 bits, rounded.  With the rounded reciprocal y of s, q = x y is one unit off at most and
// q + (x - q s) y, each a fused multiply-add, is the correctly rounded quotient (P. Markstein, IBM J. Res. Dev. 34, 1990), as long as nothing underflows
// on the way.
__device__ __forceinline__ uint4 codes_of(const float (&x)[16], float s) {
  if (s == 0.f) return make_uint4(0, 0, 0, 0);
  uint32_t b[16];
  if (s > 1e-30f && s < 1e30f) {
    const float y = 1.f / s;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float q = x[i] * y;
      b[i] = __float_as_uint(fmaf(fmaf(-q, s, x[i]), y, q) + kMagic);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = __float_as_uint(__fdiv_rn(x[i], s) + kMagic);
  }
  auto four = [&](int i) { return __byte_perm(__byte_perm(b[i], b[i + 1], 0x0040), __byte_perm(b[i + 2], b[i + 3], 0x0040), 0x5410); };
  return make_uint4(four(0), four(4), four(8), four(12));
}
__device__ __forceinline__ float code_at(const uint4& c, int i) {
  const uint32_t w = i < 4 ? c.x : i < 8 ? c.y : i < 12 ? c.z : c.w;
  return (float)(int8_t)(w >> (8 * (i & 3)));
}
// Codes for one scale as codes for another.
__device__ __forceinline__ uint4 again(const uint4& c, float from, float to) {
  if (from == to) return c;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = code_at(c, i) * from;
  return codes_of(x, to);
}
// Bytes lo .. hi - 1 of 16.
__device__ __forceinline__ uint32_t byte_mask(int lo, int hi, int word) {
  auto below = [&](int n) { n -= 4 * word; return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1; };
  return below(hi) & ~below(lo);
}
__device__ __forceinline__ uint4 bytes_between(const uint4& c, int lo, int hi) {
  return make_uint4(c.x & byte_mask(lo, hi, 0), c.y & byte_mask(lo, hi, 1), c.z & byte_mask(lo, hi, 2), c.w & byte_mask(lo, hi, 3));
}

// Where a component's 16 positions lie in shared memory: 16 components, and 16 bytes free, so that the eight threads of a position meet different banks.
__device__ __forceinline__ int turned(int c) { return 16 * c + (c & ~15); }
template <int D> constexpr int kTurned = 17 * D;

template <class T, int D>
__global__ void __launch_bounds__(2 * D) write_kernel(const RowsParams a) {
  constexpr int U = D / 16;
  __shared__ Run runs[32];
  __shared__ float most[2][2 * D / 32];
  __shared__ __align__(16) unsigned char turn[2][kTurned<D>];
  const int tid = threadIdx.x, part = tid / D, in = tid % D, r = in / U, u = in % U, h0 = blockIdx.y * a.heads_each, h1 = min(a.heads, h0 + a.heads_each);
  const int n_runs = runs_of_cta<true, D>(a, runs);
  const T* const rows = static_cast<const T*>(part ? a.v : a.k);
  const int64_t stride_t = part ? a.v_t : a.k_t, stride_h = part ? a.v_h : a.k_h;
  int turns = 0;
  for (int i = 0; i < n_runs; ++i) {
    const Run run = runs[i];
    const bool have = r >= run.offset && r < run.offset + run.len;
    const T* from = rows + (int64_t)(run.first + (have ? r - run.offset : 0)) * stride_t + h0 * stride_h + 16 * u;
    for (int h = h0; h < h1; ++h, from += stride_h, ++turns) {
      unsigned char* const block = a.data + run.at + h * a.stride_head;
      // The block as it was: the thread's key unit, or component `in`'s 16 values.
      const uint4 was = run.offset ? *reinterpret_cast<const uint4*>(block + (part ? pages8::value_unit(in, D) : pages8::key_unit(r, u, D))) : make_uint4(0, 0, 0, 0);
      const float old = run.offset ? *reinterpret_cast<const float*>(block + pages8::scales(D) + 4 * part) : 0.f;
      float x[16], big = 0.f;
      if (have) {
        const Raw16<T> raw = load16(from);
        const T* const e = reinterpret_cast<const T*>(raw.r);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          x[j] = to_float(e[j]);
          x[j] = x[j] != x[j] ? 0.f : fminf(fmaxf(x[j], -kMost), kMost);
          big = fmaxf(big, fabsf(x[j]));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = 0.f;
      }
      big = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(big)));           // (not negative: ordered as integers)
      if ((tid & 31) == 0) most[turns & 1][tid / 32] = big;
      __syncthreads();                                                                // (also: the readers of the turn before last are done with `turn`)
#pragma unroll
      for (int w = 0; w < D / 32; ++w) big = fmaxf(big, most[turns & 1][part * (D / 32) + w]);
      const float s = fmaxf(scale_of(big), old);
      const uint4 c = have ? codes_of(x, s) : make_uint4(0, 0, 0, 0);
      if (part == 0) {
        *reinterpret_cast<uint4*>(block + pages8::key_unit(r, u, D)) = have ? c : r < run.offset ? again(was, old, s) : make_uint4(0, 0, 0, 0);
      } else if (have) {
#pragma unroll
        for (int j = 0; j < 16; ++j) turn[turns & 1][turned(16 * u + j) + r] = (unsigned char)((j < 4 ? c.x : j < 8 ? c.y : j < 12 ? c.z : c.w) >> (8 * (j & 3)));
      }
      __syncthreads();                                                                // (before a scale is written, too: all have read it)
      if (part == 1) {
        const uint4 now = bytes_between(*reinterpret_cast<const uint4*>(&turn[turns & 1][turned(in)]), run.offset, run.offset + run.len);
        const uint4 kept = bytes_between(again(was, old, s), 0, run.offset);
        *reinterpret_cast<uint4*>(block + pages8::value_unit(in, D)) = make_uint4(now.x | kept.x, now.y | kept.y, now.z | kept.z, now.w | kept.w);
      }
      if (in == 0) *reinterpret_cast<float*>(block + pages8::scales(D) + 4 * part) = s;
      if (in == 1) *reinterpret_cast<float*>(block + pages8::scales(D) + 8 + 4 * part) = 0.f;
    }
  }
}

template <class T, int D>
__global__ void __launch_bounds__(2 * D) read_kernel(const RowsParams a) {
  constexpr int U = D / 16;
  __shared__ Run runs[32];
  __shared__ __align__(16) unsigned char turn[2][kTurned<D>];
  const int tid = threadIdx.x, part = tid / D, in = tid % D, r = in / U, u = in % U, h0 = blockIdx.y * a.heads_each, h1 = min(a.heads, h0 + a.heads_each);
  const int n_runs = runs_of_cta<false, D>(a, runs);
  T* const rows = static_cast<T*>(part ? a.v : a.k);
  const int64_t stride_t = part ? a.v_t : a.k_t, stride_h = part ? a.v_h : a.k_h;
  int turns = 0;
  for (int i = 0; i < n_runs; ++i) {
    const Run run = runs[i];
    const bool have = r >= run.offset && r < run.offset + run.len;
    T* to = rows + (int64_t)(run.first + (have ? r - run.offset : 0)) * stride_t + h0 * stride_h + 16 * u;
    for (int h = h0; h < h1; ++h, to += stride_h, ++turns) {
      const unsigned char* const block = a.data + run.at + h * a.stride_head;
      float s = 0.f;
      uint4 c = make_uint4(0, 0, 0, 0);
      if (run.at >= 0) {
        s = __ldg(reinterpret_cast<const float*>(block + pages8::scales(D)) + part);
        c = __ldg(reinterpret_cast<const uint4*>(block + (part ? pages8::value_unit(in, D) : pages8::key_unit(r, u, D))));
      }
      if (part) *reinterpret_cast<uint4*>(&turn[turns & 1][turned(in)]) = c;
      __syncthreads();                                                                // (one a turn: the readers of the turn before last have come here too)
      if (have) {
        float x[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = (part ? (float)(int8_t)turn[turns & 1][turned(16 * u + j) + r] : code_at(c, j)) * s;
        store16(to, x);
      }
    }
  }
}

template <bool WRITE, class T>
void launch_rows(RowsParams p, int dim, cudaStream_t st) {
  // A step's positions each in a block of their own: a CTA for each, and each head.  Texts: 16 positions and, where that leaves some 16 CTAs for each SM all the same, several heads in
  // turn, as looking at the slots takes as long as a head.
  p.window = (int64_t)p.t * p.heads <= 16 * 16 * 148 ? 1 : 16;
  const int64_t windows = ((int64_t)p.t + p.window - 1) / p.window, each = windows * p.heads / (16 * 148);
  p.heads_each = (int)(each < 1 ? 1 : each > p.heads ? p.heads : each);
  const dim3 grid((unsigned)windows, (unsigned)((p.heads + p.heads_each - 1) / p.heads_each));
  if (WRITE) {
    if (dim == 64) write_kernel<T, 64><<<grid, 128, 0, st>>>(p);
    else write_kernel<T, 128><<<grid, 256, 0, st>>>(p);
  } else {
    if (dim == 64) read_kernel<T, 64><<<grid, 128, 0, st>>>(p);
    else read_kernel<T, 128><<<grid, 256, 0, st>>>(p);
  }
}

template <bool WRITE>
int rows(const linmt_pages8_rows_args* g, const char* what) {
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "%s: not this library's argument struct", what);
  if (int rc = check_pages8(g->pages, what)) return rc;
  if (g->t < 0 || !dtype_ok(g->dtype)) return op_fail(LINMT_EINVAL, "%s: t = %d, dtype = %d", what, g->t, g->dtype);
  if (g->t == 0) return LINMT_OK;
  if (!g->slots || !g->k || !g->v) return op_fail(LINMT_EINVAL, "%s: an array is missing", what);
  const int64_t unit = 16 / dtype_bytes(g->dtype);
  if (!aligned(g->slots, 8) || !aligned(g->k, 16) || !aligned(g->v, 16) || g->k_stride_t % unit || g->k_stride_h % unit || g->v_stride_t % unit || g->v_stride_h % unit)
    return op_fail(LINMT_EINVAL, "%s: keys, values and their strides have to be multiples of 16 bytes", what);
  const linmt_pages8& pg = g->pages;
  if (pg.heads > 65535) return op_fail(LINMT_ELIMIT, "%s: %d heads (at most 65535)", what, pg.heads);
  RowsParams p{static_cast<unsigned char*>(pg.data), pg.stride_page, pg.stride_head, pg.n_pages, pg.heads, pg.page, g->slots, g->k, g->v,
               g->k_stride_t, g->k_stride_h, g->v_stride_t, g->v_stride_h, g->t, 1, 1};
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, what);
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  if (g->dtype == LINMT_F32) launch_rows<WRITE, float>(p, pg.dim, st);
  else if (g->dtype == LINMT_BF16) launch_rows<WRITE, __nv_bfloat16>(p, pg.dim, st);
  else launch_rows<WRITE, __half>(p, pg.dim, st);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, what);
}

}  // namespace

int check_pages8(const linmt_pages8& p, const char* what) {
  if (!p.data || p.n_pages < 1 || p.heads < 1 || p.page < pages8::kBlock || p.page % pages8::kBlock)
    return op_fail(LINMT_EINVAL, "%s: a pool of %d pages of %d positions (a multiple of 16), %d heads at %p", what, p.n_pages, p.page, p.heads, p.data);
  if (p.dim != 64 && p.dim != 128) return op_fail(LINMT_ELIMIT, "%s: dim = %d (64 or 128)", what, p.dim);
  if (!aligned(p.data, 16) || p.stride_page % 16 || p.stride_head % 16) return op_fail(LINMT_EINVAL, "%s: the pool and its strides have to be multiples of 16 bytes", what);
  return LINMT_OK;
}

}  // namespace ops
}  // namespace linmt

extern "C" {

int linmt_write_pages8(const linmt_pages8_rows_args* args) { return linmt::ops::rows<true>(args, "write_pages8"); }
int linmt_read_pages8(const linmt_pages8_rows_args* args) { return linmt::ops::rows<false>(args, "read_pages8"); }

}  // extern "C"
