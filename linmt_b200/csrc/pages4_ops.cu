// pages4_ops.cu -- pages for growing sentences, keys and values in them in 4 bits (linmt_plan_pages, linmt_write_pages4,
// linmt_read_pages4).  Attention over them: pages4_attend.cu.
#include <atomic>

#include "device_ops.h"
#include "pages4.h"

namespace linmt {
namespace ops {
namespace {

// ---- pages and slots ---------------------------------------------------------------------------
//
// Every CTA sums the sentences' new positions and pages itself (two numbers a sentence, from L2) and then deals with its part of
// the slots and of the new pages, found by bisection: one launch whose CTAs need nothing from one another, however the
// positions are spread over the sentences.
constexpr int kPlanThreads = 512;
constexpr int kPlanMaxN = 16384;
constexpr int kPlanSlots = 4;          // slots of a thread's turn: two 16-byte stores

struct PlanParams {
  const int32_t* old_len;
  const int32_t* new_len;
  int32_t* table;
  int64_t table_stride;
  const int32_t* free_pages;
  const int32_t* used;
  int32_t* out_used;
  int64_t* out_slots;
  int32_t* out_starts;
  int32_t n, width, page, n_free;
  int64_t total;
};

__device__ __forceinline__ int sat_add(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, 0x7fffffffu); }   // a, b >= 0

// Largest i < n with sums[i] <= x (sums[0] = 0 <= x); with empty sentences the last of equals.
__device__ __forceinline__ int find_row(const int* sums, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams a) {
  extern __shared__ int plan_smem[];
  int* tok = plan_smem;                 // [n + 1] new positions before sentence i
  int* pag = plan_smem + a.n + 1;       // [n + 1] new pages before sentence i
  __shared__ int warp_tok[kPlanThreads / 32], warp_pag[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t most64 = (int64_t)a.width * a.page;
  const int most = (int)min(most64, (int64_t)0x7fffffff);
  auto lengths = [&](int i, int& o, int& w) {
    o = a.old_len ? min(max(__ldg(a.old_len + i), 0), most) : 0;
    w = max(min(max(__ldg(a.new_len + i), 0), most), o);
  };
  auto pages_of = [&](int len) { return len / a.page + (len % a.page != 0); };
  const int each = (a.n + kPlanThreads - 1) / kPlanThreads, i0 = min(tid * each, a.n), i1 = min(i0 + each, a.n);
  int t = 0, p = 0;
  for (int i = i0; i < i1; ++i) {
    int o, w;
    lengths(i, o, w);
    tok[i] = t;
    pag[i] = p;
    t = sat_add(t, w - o);
    p += pages_of(w) - pages_of(o);
  }
  int st = t, sp = p;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int t2 = __shfl_up_sync(~0u, st, d), p2 = __shfl_up_sync(~0u, sp, d);
    if (lane >= d) { st = sat_add(st, t2); sp += p2; }
  }
  if (lane == 31) { warp_tok[warp] = st; warp_pag[warp] = sp; }
  int before_t = __shfl_up_sync(~0u, st, 1), before_p = __shfl_up_sync(~0u, sp, 1);
  if (lane == 0) before_t = before_p = 0;
  __syncthreads();
  int all_t = 0, all_p = 0;
  for (int i = 0; i < kPlanThreads / 32; ++i) {
    if (i == warp) { before_t = sat_add(before_t, all_t); before_p += all_p; }
    all_t = sat_add(all_t, warp_tok[i]);
    all_p += warp_pag[i];
  }
  for (int i = i0; i < i1; ++i) { tok[i] = sat_add(tok[i], before_t); pag[i] += before_p; }
  if (tid == 0) { tok[a.n] = all_t; pag[a.n] = all_p; }
  __syncthreads();

  const int64_t used = *a.used;
  auto fresh = [&](int q) {      // the q-th page that the call wants
    const int64_t at = used + q;
    return at >= 0 && at < a.n_free ? __ldg(a.free_pages + at) : -1;
  };
  if (blockIdx.x == 0) {
    if (tid == 0) *a.out_used = (int)min(used + all_p, (int64_t)0x7fffffff);
    for (int i = tid; i <= a.n; i += kPlanThreads) a.out_starts[i] = tok[i];
  }
  for (int64_t q64 = (int64_t)blockIdx.x * kPlanThreads + tid; q64 < all_p; q64 += (int64_t)gridDim.x * kPlanThreads) {
    const int q = (int)q64;
    const int i = find_row(pag, a.n, q);
    int o, w;
    lengths(i, o, w);
    a.table[i * a.table_stride + pages_of(o) + (q - pag[i])] = fresh(q);
  }
  const bool wide = (reinterpret_cast<uintptr_t>(a.out_slots) & 15) == 0;
  for (int64_t s = ((int64_t)blockIdx.x * kPlanThreads + tid) * kPlanSlots; s < a.total; s += (int64_t)gridDim.x * kPlanThreads * kPlanSlots) {
    long long slot[kPlanSlots];
    int i = -1, o = 0, have = 0, ends = 0;
#pragma unroll
    for (int j = 0; j < kPlanSlots; ++j) {
      slot[j] = -1;
      if (s + j >= all_t) continue;
      const int x = (int)(s + j);
      if (i < 0 || x >= ends) {
        if (i < 0) i = find_row(tok, a.n, x);
        else while (tok[i + 1] <= x) ++i;
        int w;
        lengths(i, o, w);
        have = pages_of(o);
        ends = tok[i + 1];
      }
      const int pos = o + (x - tok[i]), col = pos / a.page;
      const int page = col < have ? a.table[i * a.table_stride + col] : fresh(pag[i] + col - have);
      if (page >= 0) slot[j] = (int64_t)page * a.page + (pos - col * a.page);
    }
    if (wide && s + kPlanSlots <= a.total) {
      reinterpret_cast<longlong2*>(a.out_slots + s)[0] = make_longlong2(slot[0], slot[1]);
      reinterpret_cast<longlong2*>(a.out_slots + s)[1] = make_longlong2(slot[2], slot[3]);
    } else {
#pragma unroll
      for (int j = 0; j < kPlanSlots; ++j)
        if (s + j < a.total) a.out_slots[s + j] = slot[j];
    }
  }
}

// ---- rows in and out of a pool -------------------------------------------------------------------
//
// A thread has eight components of one position and head, four neighbours the 32 of a scale.  Bound by the bytes moved.
constexpr int kRowThreads = 256;

struct RowsParams {
  unsigned char* data;
  int64_t stride_page, stride_head;
  int32_t n_pages, heads, page;
  const int64_t* slots;
  void* k;
  void* v;
  int64_t k_t, k_h, v_t, v_h;
  int64_t words;            // t * heads * dim / 8
};

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  uint4 r[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  const T* e = reinterpret_cast<const T*>(r);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_float(e[i]);
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint4 r[sizeof(T) / 2];
  T* e = reinterpret_cast<T*>(r);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_float<T>(x[i]);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = r[i];
}

// Codes and scale of the thread's eight components, the scale that of 32 in four neighbouring threads.
__device__ __forceinline__ uint32_t quantise(float (&x)[8], __nv_bfloat16& scale) {
  constexpr float kMost = 3.3895313892515355e38f;      // largest finite bf16
  float hi = -INFINITY, lo = INFINITY;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -kMost), kMost);
    hi = fmaxf(hi, x[i]);
    lo = fminf(lo, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, o));
    lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
  }
  scale = __float2bfloat16_rn((hi >= -lo ? hi : lo) * -0.125f);
  const float s = __bfloat162float(scale);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // (a true quotient: a product with 1 / scale would round some components to the other neighbour)
    const float c = s == 0.f ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -8.f), 7.f);
    codes |= (uint32_t)((int)c + 8) << (4 * i);
  }
  return codes;
}

template <class T, int D>
__global__ void __launch_bounds__(kRowThreads) write_kernel(const RowsParams a) {
  constexpr int W = D / 8;
  const int64_t at = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  const int64_t th = min(at, a.words - 1) / W;                 // (the last warp's idle lanes repeat the last word: the shuffles need them)
  const int w = (int)(min(at, a.words - 1) % W), h = (int)(th % a.heads);
  const int64_t t = th / a.heads, slot = __ldg(a.slots + t), page = pages4::slot_page(slot, a.n_pages, a.page);
  float x[8];
  __nv_bfloat16 ks, vs;
  load8(static_cast<const T*>(a.k) + t * a.k_t + h * a.k_h + 8 * w, x);
  const uint32_t kc = quantise(x, ks);
  load8(static_cast<const T*>(a.v) + t * a.v_t + h * a.v_h + 8 * w, x);
  const uint32_t vc = quantise(x, vs);
  if (page < 0 || at >= a.words) return;
  const int pos = (int)(slot - page * a.page), r = pos % pages4::kTile;
  unsigned char* tile = a.data + page * a.stride_page + h * a.stride_head + (int64_t)(pos / pages4::kTile) * pages4::tile_bytes(D);
  *reinterpret_cast<uint32_t*>(tile + pages4::key_word(r, w, D)) = kc;
  *reinterpret_cast<uint16_t*>(tile + pages4::value_four(r, 2 * w, D)) = (uint16_t)vc;
  *reinterpret_cast<uint16_t*>(tile + pages4::value_four(r, 2 * w + 1, D)) = (uint16_t)(vc >> 16);
  if ((w & 3) == 0) {
    *reinterpret_cast<__nv_bfloat16*>(tile + pages4::key_scales(D) + pages4::scale_at(r, w >> 2, D)) = ks;
    *reinterpret_cast<__nv_bfloat16*>(tile + pages4::value_scales(D) + pages4::scale_at(r, w >> 2, D)) = vs;
  }
}

template <class T, int D>
__global__ void __launch_bounds__(kRowThreads) read_kernel(const RowsParams a) {
  constexpr int W = D / 8;
  const int64_t at = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  if (at >= a.words) return;
  const int64_t th = at / W, t = th / a.heads, slot = __ldg(a.slots + t), page = pages4::slot_page(slot, a.n_pages, a.page);
  const int w = (int)(at % W), h = (int)(th % a.heads);
  uint32_t kc = 0, vc = 0;
  float ks = 0.f, vs = 0.f;
  if (page >= 0) {
    const int pos = (int)(slot - page * a.page), r = pos % pages4::kTile;
    const unsigned char* tile = a.data + page * a.stride_page + h * a.stride_head + (int64_t)(pos / pages4::kTile) * pages4::tile_bytes(D);
    kc = *reinterpret_cast<const uint32_t*>(tile + pages4::key_word(r, w, D));
    vc = *reinterpret_cast<const uint16_t*>(tile + pages4::value_four(r, 2 * w, D)) |
         (uint32_t) * reinterpret_cast<const uint16_t*>(tile + pages4::value_four(r, 2 * w + 1, D)) << 16;
    ks = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(tile + pages4::key_scales(D) + pages4::scale_at(r, w >> 2, D)));
    vs = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(tile + pages4::value_scales(D) + pages4::scale_at(r, w >> 2, D)));
  }
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = page < 0 ? 0.f : (float)((int)((kc >> (4 * i)) & 15) - 8) * ks;
  store8(static_cast<T*>(a.k) + t * a.k_t + h * a.k_h + 8 * w, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = page < 0 ? 0.f : (float)((int)((vc >> (4 * i)) & 15) - 8) * vs;
  store8(static_cast<T*>(a.v) + t * a.v_t + h * a.v_h + 8 * w, x);
}

template <bool WRITE, class T>
void launch_rows(const RowsParams& p, int dim, unsigned blocks, cudaStream_t st) {
  if (WRITE) {
    if (dim == 64) write_kernel<T, 64><<<blocks, kRowThreads, 0, st>>>(p);
    else write_kernel<T, 128><<<blocks, kRowThreads, 0, st>>>(p);
  } else {
    if (dim == 64) read_kernel<T, 64><<<blocks, kRowThreads, 0, st>>>(p);
    else read_kernel<T, 128><<<blocks, kRowThreads, 0, st>>>(p);
  }
}

template <bool WRITE>
int rows(const linmt_pages4_rows_args* g, const char* what) {
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "%s: not this library's argument struct", what);
  if (int rc = check_pages4(g->pages, what)) return rc;
  if (g->t < 0 || !dtype_ok(g->dtype)) return op_fail(LINMT_EINVAL, "%s: t = %d, dtype = %d", what, g->t, g->dtype);
  if (g->t == 0) return LINMT_OK;
  if (!g->slots || !g->k || !g->v) return op_fail(LINMT_EINVAL, "%s: an array is missing", what);
  const int64_t unit = 16 / dtype_bytes(g->dtype);
  if (!aligned(g->slots, 8) || !aligned(g->k, 16) || !aligned(g->v, 16) || g->k_stride_t % unit || g->k_stride_h % unit || g->v_stride_t % unit || g->v_stride_h % unit)
    return op_fail(LINMT_EINVAL, "%s: keys, values and their strides have to be multiples of 16 bytes", what);
  const linmt_pages4& pg = g->pages;
  RowsParams p{static_cast<unsigned char*>(pg.data), pg.stride_page, pg.stride_head, pg.n_pages, pg.heads, pg.page, g->slots, g->k, g->v,
               g->k_stride_t, g->k_stride_h, g->v_stride_t, g->v_stride_h, (int64_t)g->t * pg.heads * (pg.dim / 8)};
  const int64_t blocks = (p.words + kRowThreads - 1) / kRowThreads;
  if (blocks > INT32_MAX) return op_fail(LINMT_ELIMIT, "%s: %lld components in one call", what, (long long)p.words * 8);
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, what);
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  if (g->dtype == LINMT_F32) launch_rows<WRITE, float>(p, pg.dim, (unsigned)blocks, st);
  else if (g->dtype == LINMT_BF16) launch_rows<WRITE, __nv_bfloat16>(p, pg.dim, (unsigned)blocks, st);
  else launch_rows<WRITE, __half>(p, pg.dim, (unsigned)blocks, st);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, what);
}

}  // namespace

int check_pages4(const linmt_pages4& p, const char* what) {
  if (!p.data || p.n_pages < 1 || p.heads < 1 || p.page < pages4::kTile || p.page % pages4::kTile)
    return op_fail(LINMT_EINVAL, "%s: a pool of %d pages of %d positions (a multiple of 16), %d heads at %p", what, p.n_pages, p.page, p.heads, p.data);
  if (p.dim != 64 && p.dim != 128) return op_fail(LINMT_ELIMIT, "%s: dim = %d (64 or 128)", what, p.dim);
  if (!aligned(p.data, 16) || p.stride_page % 16 || p.stride_head % 16) return op_fail(LINMT_EINVAL, "%s: the pool and its strides have to be multiples of 16 bytes", what);
  return LINMT_OK;
}

}  // namespace ops
}  // namespace linmt

extern "C" {

int linmt_plan_pages(const linmt_plan_pages_args* g) {
  using namespace linmt::ops;
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "plan_pages: not this library's argument struct");
  if (g->n < 0 || g->width < 0 || g->page < 1 || g->n_free < 0 || g->total < 0)
    return op_fail(LINMT_EINVAL, "plan_pages: n = %d, width = %d, page = %d, n_free = %d, total = %lld", g->n, g->width, g->page, g->n_free, (long long)g->total);
  if (!g->used || !g->out_used || g->used == g->out_used || !g->out_starts || (g->n && !g->new_len) || (g->n && g->width && !g->table) || (g->n_free && !g->free_pages) || (g->total && !g->out_slots))
    return op_fail(LINMT_EINVAL, "plan_pages: an array is missing, or `used` is both read and written");
  if (!aligned(g->old_len, 4) || !aligned(g->new_len, 4) || !aligned(g->table, 4) || !aligned(g->free_pages, 4) || !aligned(g->used, 4) || !aligned(g->out_used, 4) || !aligned(g->out_starts, 4) || !aligned(g->out_slots, 8))
    return op_fail(LINMT_EINVAL, "plan_pages: an array is not aligned to its type");
  if (g->n > kPlanMaxN || (int64_t)g->n * g->width > INT32_MAX || g->total > INT32_MAX)
    return op_fail(LINMT_ELIMIT, "plan_pages: n = %d (at most %d), n * width = %lld, total = %lld (below 2^31)", g->n, kPlanMaxN, (long long)g->n * g->width, (long long)g->total);
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "plan_pages");
  const size_t smem = (size_t)2 * (g->n + 1) * sizeof(int);
  if (smem > 40 << 10) {
    const cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * (kPlanMaxN + 1) * (int)sizeof(int));
    if (e != cudaSuccess) return op_cuda(e, "plan_pages");
  }
  PlanParams p{g->old_len, g->new_len, g->table, g->table_stride, g->free_pages, g->used, g->out_used, g->out_slots, g->out_starts, g->n, g->width, g->page, g->n_free, g->total};
  int64_t blocks = (g->total + kPlanThreads * kPlanSlots - 1) / (kPlanThreads * kPlanSlots);
  blocks = blocks < 1 ? 1 : blocks > 2 * 148 ? 2 * 148 : blocks;
  plan_kernel<<<(unsigned)blocks, kPlanThreads, smem, static_cast<cudaStream_t>(g->stream)>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "plan_pages");
}

int linmt_write_pages4(const linmt_pages4_rows_args* args) { return linmt::ops::rows<true>(args, "write_pages4"); }
int linmt_read_pages4(const linmt_pages4_rows_args* args) { return linmt::ops::rows<false>(args, "read_pages4"); }

}  // extern "C"
