// pages8_attend.cu -- attention of a few query rows per sentence over a pool of 8-bit pages (linmt_attend_pages8).
#include <cmath>

#include "device_ops.h"
#include "pages8.h"

namespace linmt {
namespace ops {
namespace {

constexpr int kRows = 16;
constexpr float kLog2e = 1.4426950408889634f;

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
  int32_t n, g, heads, rep, width, row_tiles, sinks;
  float scale, cap;
};

template <class T, int D>
__global__ void __launch_bounds__(D) attend_kernel(const AttendParams a) {
  __shared__ float q[kRows][D], key[pages8::kBlock][D + 1], value[pages8::kBlock][D], weight[kRows][pages8::kBlock], top[kRows], total[kRows], down[kRows];
  const int tid = threadIdx.x, sent = blockIdx.x / (a.pool_heads * a.row_tiles), kvh = blockIdx.x / a.row_tiles % a.pool_heads, rt = blockIdx.x % a.row_tiles;
  const int rows = min(kRows, a.g * a.rep - rt * kRows), len = (int)min((int64_t)max(a.len[sent], 0), (int64_t)a.width * a.page);
  auto place = [&](int r, int& g, int& h) {
    const int at = rt * kRows + r;
    g = at / a.rep;
    h = kvh * a.rep + at - g * a.rep;
  };
  float acc[kRows] = {};
  for (int r = 0; r < rows; ++r) {
    int g, h;
    place(r, g, h);
    q[r][tid] = to_float(static_cast<const T*>(a.q)[sent * a.q_n + g * a.q_g + h * a.q_h + tid]);
  }
  if (tid < kRows) { top[tid] = -INFINITY; total[tid] = 0.f; }
  for (int b = 0; b * pages8::kBlock < len; ++b) {
    const int64_t at = pages8::block_offset(a.table + sent * a.table_stride, b, a.page / pages8::kBlock, a.n_pages, a.stride_page, D);
    if (at < 0) continue;
    const unsigned char* const block = a.data + at + kvh * a.stride_head;
    const float ks = *reinterpret_cast<const float*>(block + pages8::scales(D)), vs = *reinterpret_cast<const float*>(block + pages8::scales(D) + 4);
    __syncthreads();
    for (int t = 0; t < pages8::kBlock; ++t) {
      key[t][tid] = (float)(int8_t)block[pages8::key_unit(t, tid / 16, D) + tid % 16] * ks;
      value[t][tid] = (float)(int8_t)block[pages8::value_unit(tid, D) + t] * vs;
    }
    __syncthreads();
    for (int i = tid; i < rows * pages8::kBlock; i += D) {
      const int r = i / pages8::kBlock, t = i % pages8::kBlock, pos = b * pages8::kBlock + t;
      int g, h;
      place(r, g, h);
      float s = 0.f;
      for (int d = 0; d < D; ++d) s = fmaf(q[r][d], key[t][d], s);
      s *= a.scale;
      if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
      if (a.slope) s -= a.slope[h] * fabsf((float)pos - a.centre[(int64_t)sent * a.g + g]);
      const bool window = !a.first || pos < a.sinks || (pos >= a.first[(int64_t)sent * a.g + g] && pos < a.last[(int64_t)sent * a.g + g]);
      weight[r][t] = pos < len && window ? s * kLog2e : -INFINITY;
    }
    __syncthreads();
    if (tid < rows) {
      float m = top[tid], sum = 0.f;
      for (int t = 0; t < pages8::kBlock; ++t) m = fmaxf(m, weight[tid][t]);
      const float base = m == -INFINITY ? 0.f : m;
      down[tid] = exp2f(top[tid] - base);
      for (int t = 0; t < pages8::kBlock; ++t) sum += weight[tid][t] = exp2f(weight[tid][t] - base);
      total[tid] = total[tid] * down[tid] + sum;
      top[tid] = m;
    }
    __syncthreads();
    for (int r = 0; r < rows; ++r) {
      acc[r] *= down[r];
      for (int t = 0; t < pages8::kBlock; ++t) acc[r] = fmaf(weight[r][t], value[t][tid], acc[r]);
    }
  }
  __syncthreads();
  for (int r = 0; r < rows; ++r) {
    int g, h;
    place(r, g, h);
    float bad = 0.f;
    for (int d = 0; d < D; ++d) bad += q[r][d] - q[r][d];
    const bool none = top[r] == -INFINITY && !(total[r] != total[r]);
    static_cast<T*>(a.out)[sent * a.o_n + g * a.o_g + h * a.o_h + tid] = from_float<T>(none ? 0.f : acc[r] / total[r]);
    if (tid == 0 && a.lse) a.lse[((int64_t)sent * a.g + g) * a.heads + h] = none ? -INFINITY : (top[r] + log2f(total[r])) / kLog2e + bad;
  }
}

template <class T, int D>
cudaError_t launch_attend(const AttendParams& p, cudaStream_t st) {
  attend_kernel<T, D><<<(unsigned)(p.n * p.pool_heads * p.row_tiles), D, 0, st>>>(p);
  return cudaGetLastError();
}

int row_tiles_of(const linmt_attend_pages8_args* g) { return (int)(((int64_t)g->g * (g->heads / g->pages.heads) + kRows - 1) / kRows); }

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
  return check(g) ? -1 : 0;
}

int linmt_attend_pages8(const linmt_attend_pages8_args* g) {
  using namespace linmt::ops;
  if (int rc = check(g)) return rc;
  if (g->n == 0 || g->g == 0) return LINMT_OK;
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "attend_pages8");
  const AttendParams p{static_cast<const unsigned char*>(g->pages.data), g->pages.stride_page, g->pages.stride_head, g->pages.n_pages, g->pages.heads, g->pages.page,
                       g->q, g->q_stride_n, g->q_stride_g, g->q_stride_h, g->out, g->out_stride_n, g->out_stride_g, g->out_stride_h, g->lse, g->table, g->table_stride, g->len,
                       g->slope, g->centre, g->first, g->last, g->n, g->g, g->heads, g->heads / g->pages.heads, g->width, row_tiles_of(g), g->sinks, g->scale, g->cap};
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  cudaError_t e;
  if (g->pages.dim == 64) e = g->dtype == LINMT_F32 ? launch_attend<float, 64>(p, st) : g->dtype == LINMT_BF16 ? launch_attend<__nv_bfloat16, 64>(p, st) : launch_attend<__half, 64>(p, st);
  else e = g->dtype == LINMT_F32 ? launch_attend<float, 128>(p, st) : g->dtype == LINMT_BF16 ? launch_attend<__nv_bfloat16, 128>(p, st) : launch_attend<__half, 128>(p, st);
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "attend_pages8");
}

}  // extern "C"
