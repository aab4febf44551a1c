// pages8_ops.cu -- keys and values into and out of pages in 8 bits (linmt_write_pages8, linmt_read_pages8).  Attention over them: pages8_attend.cu.
//
// A scale belongs to a block of 16 positions, so positions of a block that are written together have to be looked at together: a warp
// has a run (neighbours in the list that are neighbours in a block) of one head, its keys or its values, and needs nothing from another.  Of keys a lane has
// 16 components of a position at a time, of values two components of eight positions: two lanes exchange halves then and each has the 16 positions of
// a component, as they lie in the block.  A block is written whole: a position's value codes lie in every 32-byte sector of the block's half, so they would all be touched anyway.
// Bound by the bytes moved (a text), by latency (a step's positions).  (One CTA for a run with the values turned round in shared memory: 100,003 positions of 8 heads of 128 and back in 392 us.)
#include <type_traits>

#include "device_ops.h"
#include "pages8.h"

namespace linmt {
namespace ops {
namespace {

constexpr int kWarps = 8;

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

// The runs that begin among a window's positions, one in each lane that `begins` names; of a read also slots outside the pool, as many of the window's as there are side by side.
struct Runs {
  uint32_t begins;
  long long at;            // the block's place in the pool (head 0); -1: slots outside it
  int offset, len;         // the run is the block's positions offset ..
};
template <bool WRITE, int D>
__device__ __forceinline__ Runs runs_of_window(const RowsParams& a, int window) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)window * a.window - 1 + lane;                           // lane 1 has the window's first position
  const bool mine = lane >= 1 && lane <= a.window && t < a.t;
  long long slot = t >= 0 && t < a.t ? __ldg(a.slots + t) : -1;
  if (pages8::slot_page(slot, a.n_pages, a.page) < 0) slot = -1;
  const long long before = __shfl_up_sync(~0u, slot, 1);
  const bool outside = !WRITE && mine && slot < 0;
  const uint32_t goes_on = __ballot_sync(~0u, lane > 0 && (pages8::follows(before, slot) || (outside && lane > 1 && before < 0)));
  Runs r;
  r.begins = __ballot_sync(~0u, (mine && slot >= 0 || outside) && !(goes_on >> lane & 1));
  r.at = pages8::slot_block(slot, a.n_pages, a.page, a.stride_page, D);
  r.offset = slot < 0 ? 0 : (int)(slot & (pages8::kBlock - 1));
  r.len = lane == 31 ? 1 : __ffs(~(goes_on >> (lane + 1)));                          // (at most 16: a block's positions, or a window's)
  return r;
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
// on the way: not with scales from 2^-90 on, and smaller ones are brought there together with the components.
struct Numbers { float v[16]; };
template <bool ORDINARY = false>
__device__ __forceinline__ uint4 codes_of(Numbers x, float s) {
  if (!ORDINARY && s < 8.0779356694631609e-28f) {      // 2^-90
    const float up = 1.2676506002282294e30f;           // 2^100
    s *= up;
#pragma unroll
    for (int i = 0; i < 16; ++i) x.v[i] *= up;
  }
  const float y = ORDINARY || s > 0.f ? 1.f / s : 0.f;
  uint32_t b[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float q = x.v[i] * y;
    b[i] = __float_as_uint(fmaf(fmaf(-q, s, x.v[i]), y, q) + kMagic);
  }
  auto four = [&](int i) { return __byte_perm(__byte_perm(b[i], b[i + 1], 0x0040), __byte_perm(b[i + 2], b[i + 3], 0x0040), 0x5410); };
  return make_uint4(four(0), four(4), four(8), four(12));
}
// NaN as 0, sizes above 2^127 as 2^127.
__device__ __forceinline__ void tame(Numbers& x) {
#pragma unroll
  for (int i = 0; i < 16; ++i) x.v[i] = x.v[i] != x.v[i] ? 0.f : fminf(fmaxf(x.v[i], -kMost), kMost);
}
// What 16 codes stand for.  A byte below 2^23, its sign turned round, is a float's last bits.
__device__ __forceinline__ Numbers values_of(const uint4& c, float s) {
  const uint32_t w[4] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u, c.z ^ 0x80808080u, c.w ^ 0x80808080u};
  Numbers x;
#pragma unroll
  for (int i = 0; i < 16; ++i) x.v[i] = (__uint_as_float(__byte_perm(w[i >> 2], 0x4b000000u, 0x7440 + (i & 3))) - 8388736.f) * s;
  return x;
}
// Codes for one scale as codes for another.
__device__ __forceinline__ uint4 again(uint4 c, float from, float to) { return from == to ? c : codes_of(values_of(c, from), to); }
// The first n of 16 bytes.
__device__ __forceinline__ uint4 first_bytes(const uint4& c, int n) {
  auto word = [&](uint32_t x, int i) { const int m = n - 4 * i; return m <= 0 ? 0u : m >= 4 ? x : x & ((1u << (8 * m)) - 1); };
  return make_uint4(word(c.x, 0), word(c.y, 1), word(c.z, 2), word(c.w, 3));
}

// N components as they are in memory, and as numbers.
template <class T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Raw { T v[N]; };
template <class T, int N>
__device__ __forceinline__ Raw<T, N> load(const T* p) {
  Raw<T, N> x;
  if constexpr (sizeof(x) >= 16) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(x) / 16; ++i) reinterpret_cast<uint4*>(&x)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  } else if constexpr (sizeof(x) == 8) {
    *reinterpret_cast<uint2*>(&x) = __ldg(reinterpret_cast<const uint2*>(p));
  } else {
    *reinterpret_cast<uint32_t*>(&x) = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
  return x;
}
template <class T, int N>
__device__ __forceinline__ void store(T* p, const float (&x)[N]) {
  Raw<T, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = from_float<T>(x[i]);
  if constexpr (sizeof(r) >= 16) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(r) / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&r)[i];
  } else if constexpr (sizeof(r) == 8) {
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(&r);
  } else {
    *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(&r);
  }
}
// The largest size of two, four, .. numbers, NaN if one is: as bits of a float, so that the larger size is the larger integer.
template <int N>
__device__ __forceinline__ uint32_t most_of(const Raw<float, N>& x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(x.v[i]) & 0x7fffffff);
  return m;
}
template <class T, class T2, int N>
__device__ __forceinline__ uint32_t most_of_pairs(const Raw<T, N>& x) {
  const T2* const p = reinterpret_cast<const T2*>(&x);
  T2 m = __habs2(p[0]);
#pragma unroll
  for (int i = 1; i < N / 2; ++i) m = __hmax2_nan(m, __habs2(p[i]));
  return max(__float_as_uint(to_float(T(m.x))) & 0x7fffffff, __float_as_uint(to_float(T(m.y))) & 0x7fffffff);
}
template <int N> __device__ __forceinline__ uint32_t most_of(const Raw<__nv_bfloat16, N>& x) { return most_of_pairs<__nv_bfloat16, __nv_bfloat162>(x); }
template <int N> __device__ __forceinline__ uint32_t most_of(const Raw<__half, N>& x) { return most_of_pairs<__half, __half2>(x); }

// Of eight positions of two components the lane's own component's 16: `mine` has the first component's codes in x, y and the other's in z, w; the neighbour has the other eight positions.
__device__ __forceinline__ uint4 exchange(const uint4& mine, int h) {
  const uint32_t g0 = __shfl_xor_sync(~0u, h ? mine.x : mine.z, 1), g1 = __shfl_xor_sync(~0u, h ? mine.y : mine.w, 1);
  return h ? make_uint4(g0, g1, mine.z, mine.w) : make_uint4(mine.x, mine.y, g0, g1);
}

// One run of one head, its keys or its values, in turns of 16 codes a lane: of keys components 16 u .. of position r, of values components 2 c, 2 c + 1 of positions 8 h ..
// FULL: the run is a whole block; where its largest component is not an ordinary one nothing is done, and false returned.
template <class T, int D, bool VALUES, bool FULL>
__device__ __forceinline__ bool write_run(unsigned char* block, const T* rows, int64_t stride_t, int offset, int len) {
  constexpr int U = D / 16, kTurns = D / 32, kEach = VALUES ? 8 : 1, kPart = VALUES ? 2 : 16;
  const int lane = threadIdx.x & 31, h = lane & 1, end = offset + len;
  const float old = !FULL && offset ? *reinterpret_cast<const float*>(block + pages8::scales(D) + 4 * VALUES) : 0.f;
  Raw<T, kPart> in[kTurns][kEach];
  uint32_t most = 0;
  // (of keys the lane's positions are 32 / U apart from turn to turn, of values its components 32)
  const T* row = rows + (VALUES ? (8 * h - offset) * stride_t + 2 * (lane >> 1) : (lane / U - offset) * stride_t + 16 * (lane % U));
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int r = VALUES ? 8 * h + j : lane / U + 32 / U * i;
      const T* const from = VALUES ? row + 32 * i : row + 32 / U * i * stride_t;
      if constexpr (FULL) {
        in[i][j] = load<T, kPart>(from);
      } else {
#pragma unroll
        for (int e = 0; e < kPart; ++e) in[i][j].v[e] = from_float<T>(0.f);
        if (r >= offset && r < end) in[i][j] = load<T, kPart>(from);
      }
    }
    if (VALUES) row += stride_t;
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j)
#pragma unroll
    for (int i = 0; i < kTurns; ++i) most = max(most, most_of(in[i][j]));
  most = __reduce_max_sync(~0u, most);
  auto numbers = [&](int i) {
    Numbers x;
#pragma unroll
    for (int e = 0; e < 16; ++e) x.v[e] = VALUES ? to_float(in[i][e & (kEach - 1)].v[(e >> 3) & (kPart - 1)]) : to_float(in[i][0].v[e & (kPart - 1)]);
    return x;
  };
  const bool wild = most > 0x7f000000u;                 // a NaN, or something above 2^127
  if (FULL && (wild || most < 0x17000000u)) return false;       // (below 2^-81)
  if (!FULL && wild) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      Numbers x = numbers(i);
      tame(x);
#pragma unroll
      for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(x.v[e]));
    }
    most = __reduce_max_sync(~0u, __float_as_uint(m));
  }
  const float s = fmaxf(scale_of(__uint_as_float(most)), old);
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int at = lane + 32 * i;
    unsigned char* const to = block + (VALUES ? pages8::value_unit(at, D) : pages8::key_unit(at / U, at % U, D));
    uint4 c = make_uint4(0, 0, 0, 0);
    if (FULL || VALUES || (32 / U * i < end && 32 / U * (i + 1) > offset)) {
      Numbers x = numbers(i);
      if (!FULL && wild) tame(x);
      c = codes_of<FULL>(x, s);
    }
    if constexpr (VALUES) c = exchange(c, h);
    if (!FULL && offset) {
      if constexpr (VALUES) {
        const uint4 kept = first_bytes(again(*reinterpret_cast<const uint4*>(to), old, s), offset);
        c = make_uint4(c.x | kept.x, c.y | kept.y, c.z | kept.z, c.w | kept.w);
      } else if (at / U < offset) {
        c = again(*reinterpret_cast<const uint4*>(to), old, s);
      }
    }
    *reinterpret_cast<uint4*>(to) = c;
  }
  if (lane == 0) *reinterpret_cast<float*>(block + pages8::scales(D) + 4 * VALUES) = s;
  if (lane == 1) *reinterpret_cast<float*>(block + pages8::scales(D) + 8 + 4 * VALUES) = 0.f;
  return true;
}

// One position, as a step writes it: a lane has D / 32 of its components, neighbours of the keys and 32 apart of the values.
template <class T, int D, bool VALUES>
__device__ __forceinline__ void write_position(unsigned char* block, const T* row, int offset) {
  constexpr int U = D / 16, kTurns = D / 32;
  const int lane = threadIdx.x & 31;
  const float old = offset ? *reinterpret_cast<const float*>(block + pages8::scales(D) + 4 * VALUES) : 0.f;
  uint4 was[kTurns];
  float x[kTurns];
  uint32_t most = 0;
  if constexpr (!VALUES) {
    const Raw<T, kTurns> raw = load<T, kTurns>(row + kTurns * lane);
#pragma unroll
    for (int i = 0; i < kTurns; ++i) x[i] = to_float(raw.v[i]);
  }
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    if constexpr (VALUES) {
      x[i] = to_float(__ldg(row + lane + 32 * i));
      was[i] = offset ? *reinterpret_cast<const uint4*>(block + pages8::value_unit(lane + 32 * i, D)) : make_uint4(0, 0, 0, 0);
    }
    x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -kMost), kMost);
    most = max(most, __float_as_uint(fabsf(x[i])));
  }
  const float s = fmaxf(scale_of(__uint_as_float(__reduce_max_sync(~0u, most))), old);
  uint32_t code[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) code[i] = __float_as_uint((s > 0.f ? __fdiv_rn(x[i], s) : 0.f) + kMagic) & 255;
  if constexpr (VALUES) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const uint32_t byte = code[i] << (8 * (offset & 3));
      uint4 c = offset ? first_bytes(again(was[i], old, s), offset) : make_uint4(0, 0, 0, 0);
      const int word = offset >> 2;
      if (word == 0) c.x |= byte;
      else if (word == 1) c.y |= byte;
      else if (word == 2) c.z |= byte;
      else c.w |= byte;
      *reinterpret_cast<uint4*>(block + pages8::value_unit(lane + 32 * i, D)) = c;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int at = lane + 32 * i, r = at / U;
      uint4* const to = reinterpret_cast<uint4*>(block + pages8::key_unit(r, at % U, D));
      if (r > offset) *to = make_uint4(0, 0, 0, 0);
      else if (r < offset && old != s) *to = again(*to, old, s);
    }
    unsigned char* const to = block + pages8::key_unit(offset, kTurns * lane / 16, D) + kTurns * lane % 16;
    if constexpr (kTurns == 4) *reinterpret_cast<uint32_t*>(to) = code[0] | code[1] << 8 | code[kTurns - 2] << 16 | code[kTurns - 1] << 24;
    else *reinterpret_cast<uint16_t*>(to) = (uint16_t)(code[0] | code[1] << 8);
  }
  if (lane == 0) *reinterpret_cast<float*>(block + pages8::scales(D) + 4 * VALUES) = s;
  if (lane == 1) *reinterpret_cast<float*>(block + pages8::scales(D) + 8 + 4 * VALUES) = 0.f;
}

template <class T, int D, bool VALUES, bool FULL>
__device__ __forceinline__ bool read_run(const unsigned char* block, T* rows, int64_t stride_t, int offset, int len) {
  constexpr int U = D / 16, kTurns = D / 32;
  const int lane = threadIdx.x & 31, h = lane & 1;
  uint4 c[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int at = lane + 32 * i;
    c[i] = __ldg(reinterpret_cast<const uint4*>(block + (VALUES ? pages8::value_unit(at, D) : pages8::key_unit(at / U, at % U, D))));
  }
  const float s = __ldg(reinterpret_cast<const float*>(block + pages8::scales(D)) + VALUES);
  T* const row = rows + (VALUES ? (8 * h - offset) * stride_t + 2 * (lane >> 1) : (lane / U - offset) * stride_t + 16 * (lane % U));
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    if constexpr (VALUES) {
      // Eight positions of the first component, then of the other.
      const uint32_t g0 = __shfl_xor_sync(~0u, h ? c[i].x : c[i].z, 1), g1 = __shfl_xor_sync(~0u, h ? c[i].y : c[i].w, 1);
      const Numbers x = values_of(h ? make_uint4(g0, g1, c[i].z, c[i].w) : make_uint4(c[i].x, c[i].y, g0, g1), s);
      T* to = row + 32 * i;
#pragma unroll
      for (int j = 0; j < 8; ++j, to += stride_t) {
        const int r = 8 * h + j;
        const float two[2] = {x.v[j], x.v[8 + j]};
        if (FULL || (r >= offset && r < offset + len)) store<T, 2>(to, two);
      }
    } else {
      const int r = lane / U + 32 / U * i;
      const Numbers x = values_of(c[i], s);
      if (FULL || (r >= offset && r < offset + len)) store<T, 16>(row + 32 / U * i * stride_t, x.v);
    }
  }
  return true;
}

// A few positions' values, byte by byte; and zeros for slots that are none.
template <class T, int D>
__device__ __forceinline__ void read_values(const unsigned char* block, T* rows, int64_t stride_t, int offset, int len) {
  const int lane = threadIdx.x & 31;
  const float s = __ldg(reinterpret_cast<const float*>(block + pages8::scales(D)) + 1);
  for (int r = 0; r < len; ++r, rows += stride_t)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) rows[lane + 32 * i] = from_float<T>((float)(signed char)__ldg(block + pages8::value_unit(lane + 32 * i, D) + offset + r) * s);
}
template <class T, int D>
__device__ __forceinline__ void read_nothing(T* rows, int64_t stride_t, int len) {
  constexpr int kUnits = D * (int)sizeof(T) / 16;
  for (int i = threadIdx.x & 31; i < len * kUnits; i += 32) reinterpret_cast<uint4*>(rows + i / kUnits * stride_t)[i % kUnits] = make_uint4(0, 0, 0, 0);
}

template <bool WRITE, class T, int D>
__global__ void __launch_bounds__(32 * kWarps, 3) rows_kernel(const RowsParams a) {
  const int warp = threadIdx.x / 32, h0 = blockIdx.y * a.heads_each, units = 2 * (min(a.heads, h0 + a.heads_each) - h0);
  const Runs runs = runs_of_window<WRITE, D>(a, blockIdx.x);
  int unit = warp;
  for (uint32_t left = runs.begins; left; left &= left - 1) {
    const int l = __ffs(left) - 1;
    const long long at = __shfl_sync(~0u, runs.at, l);
    const int offset = __shfl_sync(~0u, runs.offset, l), len = __shfl_sync(~0u, runs.len, l);
    const int64_t first = (int64_t)blockIdx.x * a.window + l - 1;
    for (; unit < units; unit += kWarps) {              // (the warps go on with the next run where they end with this one)
      const int head = h0 + unit / 2;
      unsigned char* const block = at < 0 ? nullptr : a.data + at + head * a.stride_head;
      T* const rows = unit & 1 ? static_cast<T*>(a.v) + first * a.v_t + head * a.v_h : static_cast<T*>(a.k) + first * a.k_t + head * a.k_h;
      auto go = [&](auto values, auto full) {
        const int64_t stride_t = values.value ? a.v_t : a.k_t;
        if constexpr (WRITE) return write_run<T, D, values.value, full.value>(block, rows, stride_t, offset, len);
        else return read_run<T, D, values.value, full.value>(block, rows, stride_t, offset, len);
      };
      const bool values = unit & 1;
      if (len == pages8::kBlock && at >= 0 && (values ? go(std::true_type{}, std::true_type{}) : go(std::false_type{}, std::true_type{}))) continue;
      if (WRITE && len == 1) {
        if (values) write_position<T, D, true>(block, rows, offset);
        else write_position<T, D, false>(block, rows, offset);
      } else if (!WRITE && at < 0) {
        read_nothing<T, D>(rows, values ? a.v_t : a.k_t, len);
      } else if (!WRITE && values && len <= 4) {
        read_values<T, D>(block, rows, a.v_t, offset, len);
      } else if (values) go(std::true_type{}, std::false_type{});
      else go(std::false_type{}, std::false_type{});
    }
    unit -= units;
  }
}

template <bool WRITE, class T>
void launch_rows(RowsParams p, int dim, cudaStream_t st) {
  // Few positions: a window for each, as a step's lie in a block each.  More: windows of 16 positions, and all heads by one CTA where that leaves 16 CTAs for each SM all
  // the same, as looking at the slots takes as long as a run; four heads otherwise, a run of each for every warp.  (How many runs a window has, which is what counts, only the device
  // knows: 16 single positions of a window are 16 runs one after the other for a warp.)
  p.window = (int64_t)p.t * p.heads <= 16 * 16 * 148 ? 1 : 16;
  const int64_t windows = ((int64_t)p.t + p.window - 1) / p.window, each = windows * p.heads / (16 * 148);
  p.heads_each = (int)(each < 4 ? (p.heads < 4 ? p.heads : 4) : each > p.heads ? p.heads : each);
  const dim3 grid((unsigned)windows, (unsigned)((p.heads + p.heads_each - 1) / p.heads_each));
  if (dim == 64) rows_kernel<WRITE, T, 64><<<grid, 32 * kWarps, 0, st>>>(p);
  else rows_kernel<WRITE, T, 128><<<grid, 32 * kWarps, 0, st>>>(p);
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
