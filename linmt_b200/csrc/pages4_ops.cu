// pages4_ops.cu -- pages for growing sentences, keys and values in them in 4 bits (linmt_plan_pages, linmt_write_pages4,
// linmt_read_pages4).  Attention over them: pages4_attend.cu.
#include "device_ops.h"
#include "pages4.h"

namespace linmt {
namespace ops {
namespace {

// ---- pages and slots ---------------------------------------------------------------------------
//
// Every CTA sums the sentences' new positions and pages itself (two lengths a sentence, from L2) and then deals with its part of
// the slots and of the new pages, found by bisection: one launch whose CTAs need nothing from one another, however the
// positions are spread over the sentences.
constexpr int kPlanThreads = 512;
constexpr int kPlanMaxN = 16384;

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

// Numbers of the sentences, every 32 one place further on: a thread's stretch of them begins in another bank than its neighbours'.
struct Sums {
  int* p;
  __device__ __forceinline__ int& operator[](int i) const { return p[i + (i >> 5)]; }
};
__host__ __device__ constexpr int sums_ints(int n) { return n + n / 32 + 1; }

// Largest i < n with sums[i] <= x (sums[0] = 0 <= x); with empty sentences the last of equals.
__device__ __forceinline__ int find_row(const Sums& sums, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// kPlanSlots: slots of a thread's turn.  One where that gives every thread of two CTAs an SM at most one turn, as the new positions of a step do (64: 5.8 -> 3.9 us);
// four, which look for their sentence once, for texts.
template <int kPlanSlots>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams a) {
  extern __shared__ int plan_smem[];
  const Sums tok{plan_smem};                            // [n + 1] new positions before sentence i
  const Sums pag{plan_smem + sums_ints(a.n + 1)};       // [n + 1] new pages before sentence i
  int* const old = plan_smem + 2 * sums_ints(a.n + 1);  // [n] old lengths
  __shared__ int warp_tok[kPlanThreads / 32], warp_pag[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int most = (int)min((int64_t)a.width * a.page, (int64_t)0x7fffffff);
  const uint32_t page = a.page;
  auto pages_of = [&](int len) { return (int)(((uint32_t)len + page - 1) / page); };       // (both below 2^31)
#pragma unroll 4
  for (int i = tid; i < a.n; i += kPlanThreads) {
    const int o = a.old_len ? min(max(__ldg(a.old_len + i), 0), most) : 0, w = max(min(max(__ldg(a.new_len + i), 0), most), o);
    old[i] = o;
    tok[i] = w - o;
    pag[i] = pages_of(w) - pages_of(o);
  }
  __syncthreads();
  const int each = (a.n + kPlanThreads - 1) / kPlanThreads, i0 = min(tid * each, a.n), i1 = min(i0 + each, a.n);
  int t = 0, p = 0;
  for (int i = i0; i < i1; ++i) {
    const int x = tok[i], y = pag[i];
    tok[i] = t;
    pag[i] = p;
    t = sat_add(t, x);
    p += y;
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
#pragma unroll
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
    a.table[i * a.table_stride + pages_of(old[i]) + (q - pag[i])] = fresh(q);
  }
  const bool wide = (reinterpret_cast<uintptr_t>(a.out_slots) & 15) == 0;
  for (int64_t s = ((int64_t)blockIdx.x * kPlanThreads + tid) * kPlanSlots; s < a.total; s += (int64_t)gridDim.x * kPlanThreads * kPlanSlots) {
    long long slot[kPlanSlots];
    int i = -1, o = 0, have = 0, ends = 0, at = -1, found = -1;
#pragma unroll
    for (int j = 0; j < kPlanSlots; ++j) {
      slot[j] = -1;
      if (s + j >= all_t) continue;
      const int x = (int)(s + j);
      if (i < 0 || x >= ends) {
        if (i < 0) i = find_row(tok, a.n, x);
        else while (tok[i + 1] <= x) ++i;
        o = old[i];
        have = pages_of(o);
        ends = tok[i + 1];
        at = -1;
      }
      const int pos = o + (x - tok[i]), col = (int)((uint32_t)pos / page);
      if (col != at) {                   // (neighbours mostly share a page)
        at = col;
        found = col < have ? a.table[i * a.table_stride + col] : fresh(pag[i] + col - have);
      }
      if (found >= 0) slot[j] = (int64_t)found * a.page + (pos - col * a.page);
    }
    if (kPlanSlots == 4 && wide && s + kPlanSlots <= a.total) {
      reinterpret_cast<longlong2*>(a.out_slots + s)[0] = make_longlong2(slot[0], slot[1 % kPlanSlots]);
      reinterpret_cast<longlong2*>(a.out_slots + s)[1] = make_longlong2(slot[2 % kPlanSlots], slot[3 % kPlanSlots]);
    } else {
#pragma unroll
      for (int j = 0; j < kPlanSlots; ++j)
        if (s + j < a.total) a.out_slots[s + j] = slot[j];
    }
  }
}

// ---- rows in and out of a pool -------------------------------------------------------------------
//
// A CTA has 16 neighbours of the call's positions and some heads in turn, a thread eight components of one position (four neighbours share a scale).  Where positions fill
// a tile one after the other, as in a text that is written at once, the CTA that has the tile's first does all 16 through shared memory: a
// value's codes lie two bytes at a time among those of the positions beside it, and two-byte stores of many CTAs to the same sectors cost four times
// what the bytes do.  Other positions go one by one.  Bound by the bytes moved (a text), by latency (a step's positions).
struct RowsParams {
  unsigned char* data;
  int64_t stride_page, stride_head;
  int32_t n_pages, heads, page;
  const int64_t* slots;
  void* k;
  void* v;
  int64_t k_t, k_h, v_t, v_h;
  int32_t t, heads_each;
};

template <class T> struct Raw8 { uint4 r[sizeof(T) / 2]; };
template <class T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> x;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) x.r[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return x;
}
template <class T>
__device__ __forceinline__ void floats_of(const Raw8<T>& raw, float (&x)[8]) {
  const T* e = reinterpret_cast<const T*>(raw.r);
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

// Largest and smallest of the eight; NaN if one of them is.
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
template <class T, class T2>
__device__ __forceinline__ void extremes16(const uint4& r, float& hi, float& lo) {
  const T2* p = reinterpret_cast<const T2*>(&r);
  const T2 a = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3])), b = __hmin2_nan(__hmin2_nan(p[0], p[1]), __hmin2_nan(p[2], p[3]));
  hi = max_nan(to_float(T(a.x)), to_float(T(a.y)));
  lo = min_nan(to_float(T(b.x)), to_float(T(b.y)));
}
__device__ __forceinline__ void extremes(const Raw8<__nv_bfloat16>& r, const float (&)[8], float& hi, float& lo) { extremes16<__nv_bfloat16, __nv_bfloat162>(r.r[0], hi, lo); }
__device__ __forceinline__ void extremes(const Raw8<__half>& r, const float (&)[8], float& hi, float& lo) { extremes16<__half, __half2>(r.r[0], hi, lo); }
__device__ __forceinline__ void extremes(const Raw8<float>&, const float (&x)[8], float& hi, float& lo) {
  hi = lo = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    hi = max_nan(hi, x[i]);
    lo = min_nan(lo, x[i]);
  }
}

// Codes and scale of the thread's eight components, the scale that of 32 in four neighbouring threads; every lane of the warp calls it.
template <class T>
__device__ __forceinline__ uint32_t quantise(const Raw8<T>& raw, __nv_bfloat16& scale) {
  constexpr float kMost = 3.3895313892515355e38f;      // largest finite bf16
  float x[8], hi, lo;
  floats_of(raw, x);
  extremes(raw, x, hi, lo);
  if (!(hi <= kMost && lo >= -kMost)) {
    hi = -INFINITY;
    lo = INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -kMost), kMost);
      hi = fmaxf(hi, x[i]);
      lo = fminf(lo, x[i]);
    }
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, o));
    lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
  }
  scale = __float2bfloat16_rn((hi >= -lo ? hi : lo) * -0.125f);
  const float s = __bfloat162float(scale);
  if (s == 0.f) return 0x88888888u;
  // A code is the quotient in 32 bits, rounded.  With the rounded reciprocal y of s, q = x y is one unit off at most and q + (x - q s) y, each a
  // fused multiply-add, is the correctly rounded quotient (P. Markstein, IBM J. Res. Dev. 34, 1990), as long as nothing underflows on the way.
  // 1.5 * 2^23 + 8 makes a float's last bits the code; a component is at most 8 (1 + 2^-8) scales in size, so only 8 itself has to be held to 7.
  const float magic = 12582920.f;
  float t[8];
  if (fabsf(s) > 1e-30f && fabsf(s) < 1e30f) {
    const float y = 1.f / s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = x[i] * y;
      t[i] = fminf(fmaf(fmaf(-q, s, x[i]), y, q), 7.f) + magic;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = fminf(fmaxf(__fdiv_rn(x[i], s), -8.f), 7.f) + magic;
  }
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(t[i]);
  const uint32_t even = __byte_perm(__byte_perm(b[0], b[2], 0x0040), __byte_perm(b[4], b[6], 0x0040), 0x5410);
  const uint32_t odds = __byte_perm(__byte_perm(b[1], b[3], 0x0040), __byte_perm(b[5], b[7], 0x0040), 0x5410);
  return even | odds << 4;
}

// Where the CTA's 16 positions go: which are part of a tile that is filled in order (and done by the CTA that has its first), and the tile that begins here.
struct Rows {
  int64_t slot;            // of position threadIdx.x / W; -1 where there is none, or it has nothing to do
  int64_t at;              // its tile's place in the pool (head 0)
  int lead;                // 0..15: the position whose tile the CTA does; -1: none
  int64_t lead_at;
};
template <int W, int BYTES>
__device__ __forceinline__ Rows rows_of_cta(const RowsParams& a) {
  constexpr int kReach = 15, kMine = 16 + kReach;
  __shared__ int64_t slots[16 + 2 * kReach];
  __shared__ int gap[kMine];               // no tile's 16 begin at position first - 15 + i
  __shared__ int lead;
  __shared__ int64_t lead_at;
  const int tid = threadIdx.x;
  const int64_t first = (int64_t)blockIdx.x * 16, most = (int64_t)a.n_pages * a.page;
  auto place = [&](int64_t slot) {
    const int64_t page = pages4::slot_page(slot, a.n_pages, a.page);
    return page * a.stride_page + (int)(slot - page * a.page) / pages4::kTile * (int64_t)BYTES;
  };
  if (tid < 16 + 2 * kReach) {
    const int64_t t = first - kReach + tid;
    const int64_t s = t >= 0 && t < a.t ? __ldg(a.slots + t) : -1;
    slots[tid] = s >= 0 && s < most ? s : -1;
  }
  if (tid < kMine) gap[tid] = 0;
  if (tid == 0) lead = -1;
  __syncthreads();
  for (int i = tid; i < kMine * 16; i += 16 * W) {
    const int64_t s = slots[i / 16];
    if (s < 0 || (s & (pages4::kTile - 1)) || slots[i / 16 + i % 16] != s + i % 16) gap[i / 16] = 1;
  }
  __syncthreads();
  if (tid >= kReach && tid < kMine && !gap[tid]) {     // one at most: two that overlap could not both go on by ones
    lead = tid - kReach;
    lead_at = place(slots[tid]);
  }
  const int j = kReach + tid / W;
  Rows r;
  r.slot = slots[j];
  if (r.slot >= 0 && !gap[j - (int)(r.slot & (pages4::kTile - 1))]) r.slot = -1;
  r.at = r.slot >= 0 ? place(r.slot) : 0;
  __syncthreads();
  r.lead = lead;
  r.lead_at = lead_at;
  return r;
}

template <class T, int D>
__global__ void __launch_bounds__(2 * D) write_kernel(const RowsParams a) {
  constexpr int W = D / 8, kBytes = pages4::tile_bytes(D);
  __shared__ __align__(16) unsigned char tile[2][kBytes];
  const int tid = threadIdx.x, j = tid / W, w = tid % W, h0 = blockIdx.y * a.heads_each, h1 = min(a.heads, h0 + a.heads_each);
  const Rows rows = rows_of_cta<W, kBytes>(a);
  auto put = [&](unsigned char* to, int r, uint32_t kc, uint32_t vc, __nv_bfloat16 ks, __nv_bfloat16 vs) {
    *reinterpret_cast<uint32_t*>(to + pages4::key_word(r, w, D)) = kc;
    *reinterpret_cast<uint16_t*>(to + pages4::value_four(r, 2 * w, D)) = (uint16_t)vc;
    *reinterpret_cast<uint16_t*>(to + pages4::value_four(r, 2 * w + 1, D)) = (uint16_t)(vc >> 16);
    if ((w & 3) == 0) {
      *reinterpret_cast<__nv_bfloat16*>(to + pages4::key_scales(D) + pages4::scale_at(r, w >> 2, D)) = ks;
      *reinterpret_cast<__nv_bfloat16*>(to + pages4::value_scales(D) + pages4::scale_at(r, w >> 2, D)) = vs;
    }
  };
  __nv_bfloat16 ks, vs;
  if (rows.lead >= 0) {
    const int64_t t = (int64_t)blockIdx.x * 16 + rows.lead + j;
    const T *k = static_cast<const T*>(a.k) + t * a.k_t + h0 * a.k_h + 8 * w, *v = static_cast<const T*>(a.v) + t * a.v_t + h0 * a.v_h + 8 * w;
    Raw8<T> rk = load8(k), rv = load8(v);
    for (int h = h0; h < h1; ++h) {
      Raw8<T> nk = rk, nv = rv;
      k += a.k_h;
      v += a.v_h;
      if (h + 1 < h1) { nk = load8(k); nv = load8(v); }
      const uint32_t kc = quantise(rk, ks), vc = quantise(rv, vs);
      unsigned char* const here = tile[h & 1];
      put(here, j, kc, vc, ks, vs);
      __syncthreads();              // (one for each head: the other tile's readers have come here too)
      unsigned char* const to = a.data + rows.lead_at + h * a.stride_head;
      for (int i = tid; i < kBytes / 16; i += 2 * D) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(here)[i];
      rk = nk;
      rv = nv;
    }
  }
  if (__any_sync(~0u, rows.slot >= 0)) {
    const int64_t t = min((int64_t)blockIdx.x * 16 + j, (int64_t)a.t - 1);      // (lanes without a position take part in the scales' exchange)
    for (int h = h0; h < h1; ++h) {
      const Raw8<T> rk = load8(static_cast<const T*>(a.k) + t * a.k_t + h * a.k_h + 8 * w), rv = load8(static_cast<const T*>(a.v) + t * a.v_t + h * a.v_h + 8 * w);
      const uint32_t kc = quantise(rk, ks), vc = quantise(rv, vs);
      if (rows.slot >= 0) put(a.data + rows.at + h * a.stride_head, (int)(rows.slot & (pages4::kTile - 1)), kc, vc, ks, vs);
    }
  }
}

template <class T, int D>
__global__ void __launch_bounds__(2 * D) read_kernel(const RowsParams a) {
  constexpr int W = D / 8, kBytes = pages4::tile_bytes(D);
  static_assert(kBytes / 16 <= 2 * D, "a tile is one vector a thread");
  __shared__ __align__(16) unsigned char tile[2][2][kBytes];
  const int tid = threadIdx.x, j = tid / W, w = tid % W, h0 = blockIdx.y * a.heads_each, h1 = min(a.heads, h0 + a.heads_each);
  const Rows rows = rows_of_cta<W, kBytes>(a);
  auto get = [&](const unsigned char* from, int r, int64_t t, int h) {
    const uint32_t kc = *reinterpret_cast<const uint32_t*>(from + pages4::key_word(r, w, D));
    const uint32_t vc = *reinterpret_cast<const uint16_t*>(from + pages4::value_four(r, 2 * w, D)) |
                        (uint32_t) * reinterpret_cast<const uint16_t*>(from + pages4::value_four(r, 2 * w + 1, D)) << 16;
    const float ks = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(from + pages4::key_scales(D) + pages4::scale_at(r, w >> 2, D)));
    const float vs = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(from + pages4::value_scales(D) + pages4::scale_at(r, w >> 2, D)));
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)((int)((kc >> (4 * i)) & 15) - 8) * ks;
    store8(static_cast<T*>(a.k) + t * a.k_t + h * a.k_h + 8 * w, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)((int)((vc >> (4 * i)) & 15) - 8) * vs;
    store8(static_cast<T*>(a.v) + t * a.v_t + h * a.v_h + 8 * w, x);
  };
  const int64_t own = (int64_t)blockIdx.x * 16 + j;
  if (rows.lead >= 0) {
    const unsigned char* const from = a.data + rows.lead_at + tid * 16;
    const bool has = tid < kBytes / 16;
    auto fetch = [&](int h) { return has && h < h1 ? __ldg(reinterpret_cast<const uint4*>(from + h * a.stride_head)) : make_uint4(0, 0, 0, 0); };
    uint4 r0 = fetch(h0), r1 = fetch(h0 + 1);
    for (int h = h0, at = 0; h < h1; h += 2, at ^= 1) {        // two heads a turn
      if (has) {
        reinterpret_cast<uint4*>(tile[at][0])[tid] = r0;
        reinterpret_cast<uint4*>(tile[at][1])[tid] = r1;
      }
      r0 = fetch(h + 2);
      r1 = fetch(h + 3);
      __syncthreads();
      get(tile[at][0], j, own + rows.lead, h);
      if (h + 1 < h1) get(tile[at][1], j, own + rows.lead, h + 1);
    }
  }
  if (rows.slot >= 0) {
    for (int h = h0; h < h1; ++h) get(a.data + rows.at + h * a.stride_head, (int)(rows.slot & (pages4::kTile - 1)), own, h);
  } else if (own < a.t) {
    const int64_t s = __ldg(a.slots + own);
    if (s < 0 || s >= (int64_t)a.n_pages * a.page) {
      const float none[8] = {};
      for (int h = h0; h < h1; ++h) {
        store8(static_cast<T*>(a.k) + own * a.k_t + h * a.k_h + 8 * w, none);
        store8(static_cast<T*>(a.v) + own * a.v_t + h * a.v_h + 8 * w, none);
      }
    }
  }
}

template <bool WRITE, class T>
void launch_rows(RowsParams p, int dim, cudaStream_t st) {
  // Heads in turn where that leaves some 16 CTAs for each SM all the same: looking at the slots takes as long as a head.
  const int64_t rows = ((int64_t)p.t + 15) / 16, each = rows * p.heads / (16 * 148);
  p.heads_each = (int)(each < 1 ? 1 : each > p.heads ? p.heads : each);
  const dim3 grid((unsigned)rows, (unsigned)((p.heads + p.heads_each - 1) / p.heads_each));
  if (WRITE) {
    if (dim == 64) write_kernel<T, 64><<<grid, 128, 0, st>>>(p);
    else write_kernel<T, 128><<<grid, 256, 0, st>>>(p);
  } else {
    if (dim == 64) read_kernel<T, 64><<<grid, 128, 0, st>>>(p);
    else read_kernel<T, 128><<<grid, 256, 0, st>>>(p);
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
               g->k_stride_t, g->k_stride_h, g->v_stride_t, g->v_stride_h, g->t, 1};
  if (pg.heads > 65535) return op_fail(LINMT_ELIMIT, "%s: %d heads (at most 65535)", what, pg.heads);
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
  const size_t smem = (size_t)(2 * sums_ints(g->n + 1) + g->n) * sizeof(int);
  const int each = g->total <= 2 * 148 * kPlanThreads ? 1 : 4;
  void (*const kernel)(PlanParams) = each == 1 ? plan_kernel<1> : plan_kernel<4>;
  if (smem > 40 << 10) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (2 * sums_ints(kPlanMaxN + 1) + kPlanMaxN) * (int)sizeof(int));
    if (e != cudaSuccess) return op_cuda(e, "plan_pages");
  }
  PlanParams p{g->old_len, g->new_len, g->table, g->table_stride, g->free_pages, g->used, g->out_used, g->out_slots, g->out_starts, g->n, g->width, g->page, g->n_free, g->total};
  int64_t blocks = (g->total + kPlanThreads * each - 1) / (kPlanThreads * each);
  blocks = blocks < 1 ? 1 : blocks > 2 * 148 ? 2 * 148 : blocks;
  kernel<<<(unsigned)blocks, kPlanThreads, smem, static_cast<cudaStream_t>(g->stream)>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "plan_pages");
}

int linmt_write_pages4(const linmt_pages4_rows_args* args) { return linmt::ops::rows<true>(args, "write_pages4"); }
int linmt_read_pages4(const linmt_pages4_rows_args* args) { return linmt::ops::rows<false>(args, "read_pages4"); }

}  // extern "C"
