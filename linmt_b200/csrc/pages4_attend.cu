// pages4_attend.cu -- attention of a few query rows per sentence over a pool of 4-bit pages (linmt_attend_pages4).
//
//   out = sum_t softmax_t(f(scale q . k_t)) v_t,   k_t = sk (codes - 8), v_t = sv (codes - 8) by groups of 32 components
//
// A sentence's beams, and the query heads that share a head of the pool, read the same positions: up to 16 rows are the left
// operand of mma.m16n8k16, so every code is loaded and unpacked once for all of them.  (tcgen05.mma wants both operands of at least 64
// rows, and codes unpacked into shared memory first; with 16 rows the unpacking, not the product, is what takes the time.)
//   Scales stay out of the products: a key's is multiplied onto its group's sum, a value's into the weight on the left, and
//   the codes minus 8 are exact in bf16 and fp16.  So 16-bit queries lose nothing against the 4-bit values as they stand.
//   Weights are rounded to bf16 once for bf16 queries (2^-8 each at most, on average over the positions far less, and the output's own
//   rounding is as large); for fp16 they are taken as two bf16 terms (2^-16), for fp32 weights and queries as three (2^-24).
// Every warp has a ring of tiles of its own (cp.async, no barrier among warps) and its own maximum and sums; the CTA's four are
// joined through shared memory at the end, and where a sentence's positions are split over CTAs a second kernel joins those.
#include <atomic>

#include "device_ops.h"
#include "pages4.h"

namespace linmt {
namespace ops {
namespace {

constexpr int kWarps = 4;
constexpr int kStages = 4;
constexpr int kRows = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;      // the reference maximum follows the true one only when it lags by 2^8: few tiles rescale the sums

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
  int32_t n, g, heads, rep, width, row_tiles, splits;
  float scale, cap;
};

template <class T> struct Terms;
template <> struct Terms<__nv_bfloat16> { static constexpr int q = 1, p = 1; };
template <> struct Terms<__half> { static constexpr int q = 1, p = 2; };
template <> struct Terms<float> { static constexpr int q = 3, p = 3; };

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t lop_and_or(uint32_t x, uint32_t m, uint32_t o) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(m), "r"(o));
  return r;
}
// Codes i (low half) and i + 4 (high half) of a word, minus 8.  An integer below 128 laid into the low bits of 128.0 (bf16) or 1024.0 (fp16) adds
// itself to it.
template <int I>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w) {
  const uint32_t b = lop_and_or(w >> (4 * I), 0x000f000fu, 0x43004300u), off = 0x43084308u;      // 128 + code, 136
  __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&off));
  return *reinterpret_cast<uint32_t*>(&r);
}
template <int I>
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
  const uint32_t b = lop_and_or(w >> (4 * I), 0x000f000fu, 0x64006400u), off = 0x64086408u;      // 1024 + code, 1032
  __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ float bf16_low(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_high(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <class T> __device__ __forceinline__ float tanh_of(float x) {
  // 1 - 2 / (e^2x + 1), good to 2e-7 of 1: what a 16-bit result can see of it.
  const float e = exp2_of(x * (2 * kLog2e));
  return 1.f - __fdividef(2.f, e + 1.f);
}
template <> __device__ __forceinline__ float tanh_of<float>(float x) { return tanhf(x); }

__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <class T, int D>
constexpr int attend_smem() {
  return kWarps * kStages * 18 * D + (Terms<T>::q > 1 ? Terms<T>::q * (D / 16) * 512 : 0);
}

// The pair of query components that a lane's 32 bits of the left operand hold, as term `term` of their bf16 expansion.
template <class T>
__device__ __forceinline__ uint32_t query_pair(const T* row, int d, int term) {
  if (!row) return 0u;
  if constexpr (sizeof(T) == 2) {
    const uint16_t* r = reinterpret_cast<const uint16_t*>(row);
    return (uint32_t)__ldg(r + d) | (uint32_t)__ldg(r + d + 4) << 16;
  } else {
    float lo = __ldg(row + d), hi = __ldg(row + d + 4);
    for (int i = 0; i < term; ++i) {
      lo -= __bfloat162float(__float2bfloat16_rn(lo));
      hi -= __bfloat162float(__float2bfloat16_rn(hi));
    }
    return pack_bf16(lo, hi);
  }
}

template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(const __grid_constant__ AttendParams a) {
  constexpr int NG = D / 32, kTileBytes = pages4::tile_bytes(D), QT = Terms<T>::q, PT = Terms<T>::p;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, c = lane & 3;
  int64_t job = blockIdx.x;
  const int split = (int)(job % a.splits);
  job /= a.splits;
  const int64_t out_tile = job;            // (sentence, head of the pool, row tile)
  const int rt = (int)(job % a.row_tiles);
  job /= a.row_tiles;
  const int kvh = (int)(job % a.pool_heads), sent = (int)(job / a.pool_heads);
  const int n_rows = min(kRows, a.g * a.rep - rt * kRows);

  // The lane's rows gid and gid + 8: query row and head, what they see, their bias.
  const int cap_len = (int)min((int64_t)a.width * a.page, (int64_t)0x7fffffff), len = min(max(__ldg(a.len + sent), 0), cap_len);
  const T* q_row[2];
  int lo[2], hi[2];
  float slope[2], centre[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = gid + 8 * i, at = rt * kRows + r, g = at / a.rep, h = kvh * a.rep + at % a.rep;
    const bool have = r < n_rows;
    q_row[i] = have ? static_cast<const T*>(a.q) + sent * a.q_n + g * a.q_g + h * a.q_h : nullptr;
    lo[i] = have ? (a.first ? max(__ldg(a.first + (int64_t)sent * a.g + g), 0) : 0) : 0x7fffffff;
    hi[i] = have ? (a.last ? min(__ldg(a.last + (int64_t)sent * a.g + g), len) : len) : 0;
    slope[i] = have && a.slope ? __ldg(a.slope + h) * kLog2e : 0.f;
    centre[i] = have && a.slope ? __ldg(a.centre + (int64_t)sent * a.g + g) : 0.f;
  }
  // What any row sees, and what all of them see.
  int any_lo = lo[0] < hi[0] ? lo[0] : 0x7fffffff, any_hi = lo[0] < hi[0] ? hi[0] : 0;
  if (lo[1] < hi[1]) { any_lo = min(any_lo, lo[1]); any_hi = max(any_hi, hi[1]); }
  int all_lo = gid < n_rows ? lo[0] : 0, all_hi = gid < n_rows ? hi[0] : 0x7fffffff;
  if (gid + 8 < n_rows) { all_lo = max(all_lo, lo[1]); all_hi = min(all_hi, hi[1]); }
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    any_lo = min(any_lo, __shfl_xor_sync(~0u, any_lo, o));
    any_hi = max(any_hi, __shfl_xor_sync(~0u, any_hi, o));
    all_lo = max(all_lo, __shfl_xor_sync(~0u, all_lo, o));
    all_hi = min(all_hi, __shfl_xor_sync(~0u, all_hi, o));
  }
  const int tile0 = any_lo < any_hi ? any_lo / pages4::kTile : 0, tile1 = any_lo < any_hi ? (any_hi - 1) / pages4::kTile + 1 : 0;
  const int per_split = (tile1 - tile0 + a.splits - 1) / a.splits;
  const int t0 = min(tile1, tile0 + split * per_split), t1 = min(tile1, t0 + per_split);

  // Queries as left operands: step (group, half) takes components 32 group + 8 c + 2 half + {0, 4 | 1, 5}.
  uint4 qa[QT == 1 ? NG * 2 : 1];
  uint4* const q_smem = reinterpret_cast<uint4*>(smem + kWarps * kStages * kTileBytes);
  if constexpr (QT == 1) {
#pragma unroll
    for (int s = 0; s < NG * 2; ++s) {
      const int d = 32 * (s >> 1) + 8 * c + 2 * (s & 1);
      qa[s] = make_uint4(query_pair(q_row[0], d, 0), query_pair(q_row[1], d, 0), query_pair(q_row[0], d + 1, 0), query_pair(q_row[1], d + 1, 0));
    }
  } else {
    for (int s = warp; s < QT * NG * 2; s += kWarps) {
      const int term = s / (NG * 2), d = 32 * ((s % (NG * 2)) >> 1) + 8 * c + 2 * (s & 1);
      q_smem[s * 32 + lane] = make_uint4(query_pair(q_row[0], d, term), query_pair(q_row[1], d, term), query_pair(q_row[0], d + 1, term), query_pair(q_row[1], d + 1, term));
    }
    __syncthreads();
  }

  float o[NG][4][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const float to_log2 = a.cap > 0.f ? a.scale / a.cap : a.scale * kLog2e, cap_log2 = a.cap * kLog2e;
  unsigned char* const ring = smem + warp * kStages * kTileBytes;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const int32_t* const table = a.table + sent * a.table_stride;
  const unsigned char* const head = a.data + kvh * a.stride_head;
  const int tiles_per_page = a.page / pages4::kTile;
  const int mine = t1 - t0 > warp ? (t1 - t0 - warp + kWarps - 1) / kWarps : 0;        // this warp's tiles: t0 + warp + kWarps i

  // Where this warp's tiles are: looked up 32 at a time, one by each lane, a batch ahead of their use.
  int64_t where = -1;
  uint32_t bad = 0;                // bit of a stage: it holds no tile of the pool
  auto fetch = [&](int i) {
    if ((i & 31) == 0) {
      where = -1;
      if (i + lane < mine) where = pages4::tile_offset(table, t0 + warp + kWarps * (i + lane), tiles_per_page, a.n_pages, a.stride_page, D);
    }
    const int64_t at = __shfl_sync(~0u, where, i & 31);
    const int stage = i % kStages;
    if (i < mine && at >= 0) {
      bad &= ~(1u << stage);
#pragma unroll
      for (int b = 0; b < (kTileBytes + 511) / 512; ++b) {
        const int byte = b * 512 + lane * 16;
        if (byte < kTileBytes) copy16(ring_at + stage * kTileBytes + byte, head + at + byte);
      }
    } else {
      bad |= 1u << stage;
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);

  for (int i = 0; i < mine; ++i) {
    copy_wait<kStages - 2>();
    __syncwarp();                       // every lane's part of tile i is there, and tile i - 1 has been read by all
    fetch(i + kStages - 1);
    if ((bad >> (i % kStages)) & 1) continue;
    const unsigned char* const tile = ring + (i % kStages) * kTileBytes;
    const int pos = (t0 + warp + kWarps * i) * pages4::kTile;

    // scores: x[j][0..3] = rows gid, gid, gid + 8, gid + 8 at positions pos + 8 j + 2 c + {0, 1, 0, 1}
    float x[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t w[NG], sc[NG];
      const unsigned char* const kw = tile + (8 * j + gid) * (D / 2) + c * (4 * NG);
      const unsigned char* const ks = tile + pages4::key_scales(D) + (8 * j + 2 * c) * (2 * NG);
      if constexpr (NG == 4) {
        *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(kw);
        *reinterpret_cast<uint4*>(sc) = *reinterpret_cast<const uint4*>(ks);
      } else {
        *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(kw);
        *reinterpret_cast<uint2*>(sc) = *reinterpret_cast<const uint2*>(ks);
      }
      x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t b[4];
        if constexpr (sizeof(T) == 2 && QT == 1 && PT == 2) {
          b[0] = codes_f16<0>(w[gr]); b[1] = codes_f16<1>(w[gr]); b[2] = codes_f16<2>(w[gr]); b[3] = codes_f16<3>(w[gr]);
          mma_f16(s, qa[2 * gr], b[0], b[1]);
          mma_f16(s, qa[2 * gr + 1], b[2], b[3]);
        } else {
          b[0] = codes_bf16<0>(w[gr]); b[1] = codes_bf16<1>(w[gr]); b[2] = codes_bf16<2>(w[gr]); b[3] = codes_bf16<3>(w[gr]);
#pragma unroll
          for (int term = QT - 1; term >= 0; --term) {      // small terms first
            const uint4 a0 = QT == 1 ? qa[QT == 1 ? 2 * gr : 0] : q_smem[(term * NG * 2 + 2 * gr) * 32 + lane];
            const uint4 a1 = QT == 1 ? qa[QT == 1 ? 2 * gr + 1 : 0] : q_smem[(term * NG * 2 + 2 * gr + 1) * 32 + lane];
            mma_bf16(s, a0, b[0], b[1]);
            mma_bf16(s, a1, b[2], b[3]);
          }
        }
        // scales of position 2 c: halves gr of the first NG, of 2 c + 1: of the second
        const float s0 = gr & 1 ? bf16_high(sc[gr >> 1]) : bf16_low(sc[gr >> 1]);
        const float s1 = gr & 1 ? bf16_high(sc[NG / 2 + (gr >> 1)]) : bf16_low(sc[NG / 2 + (gr >> 1)]);
        x[j][0] = fmaf(s[0], s0, x[j][0]);
        x[j][1] = fmaf(s[1], s1, x[j][1]);
        x[j][2] = fmaf(s[2], s0, x[j][2]);
        x[j][3] = fmaf(s[3], s1, x[j][3]);
      }
    }
    if (a.cap > 0.f) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] = cap_log2 * tanh_of<T>(x[j][e] * to_log2);
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] *= to_log2;
    }
    if (a.slope) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] -= slope[e >> 1] * fabsf((float)(pos + 8 * j + 2 * c + (e & 1)) - centre[e >> 1]);
    }
    const bool edge = pos < all_lo || pos + pages4::kTile > all_hi;
    if (edge) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int p = pos + 8 * j + 2 * c + (e & 1);
          if (p < lo[e >> 1] || p >= hi[e >> 1]) x[j][e] = -INFINITY;
        }
    }
    float top[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[e] = fmaxf(fmaxf(x[0][2 * e], x[0][2 * e + 1]), fmaxf(x[1][2 * e], x[1][2 * e + 1]));
      top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], 1));
      top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], 2));
    }
    const bool up0 = top[0] > m[0] + kSlack || (m[0] == -INFINITY && top[0] > -INFINITY), up1 = top[1] > m[1] + kSlack || (m[1] == -INFINITY && top[1] > -INFINITY);
    if (__any_sync(~0u, up0 || up1)) {
      const float f0 = up0 ? exp2_of(m[0] - top[0]) : 1.f, f1 = up1 ? exp2_of(m[1] - top[1]) : 1.f;
      if (up0) m[0] = top[0];
      if (up1) m[1] = top[1];
      l[0] *= f0;
      l[1] *= f1;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[gr][e][0] *= f0; o[gr][e][1] *= f0;
          o[gr][e][2] *= f1; o[gr][e][3] *= f1;
        }
    }
    const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      x[j][0] = exp2_of(x[j][0] - m0);
      x[j][1] = exp2_of(x[j][1] - m0);
      x[j][2] = exp2_of(x[j][2] - m1);
      x[j][3] = exp2_of(x[j][3] - m1);
      l[0] += x[j][0] + x[j][1];
      l[1] += x[j][2] + x[j][3];
    }

    // out += weights . values, a group of 32 components a time: its scales go into the weights
    uint32_t vs[2][NG];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const unsigned char* const at = tile + pages4::value_scales(D) + (8 * j + 2 * c) * (2 * NG);
      if constexpr (NG == 4) *reinterpret_cast<uint4*>(vs[j]) = *reinterpret_cast<const uint4*>(at);
      else *reinterpret_cast<uint2*>(vs[j]) = *reinterpret_cast<const uint2*>(at);
      if (edge) {            // a position that nobody sees may hold anything: 0 times its scale has to be 0
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (x[j][e] == 0.f && x[j][e + 2] == 0.f) {
#pragma unroll
            for (int i2 = 0; i2 < NG / 2; ++i2) vs[j][e * (NG / 2) + i2] = 0u;
          }
      }
    }
#pragma unroll
    for (int i2 = 0; i2 < NG / 2; ++i2) {
      const uint4 u = *reinterpret_cast<const uint4*>(tile + pages4::value_codes(D) + 16 * (i2 * 32 + lane));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int gr = 2 * i2 + h;
        const uint32_t w0 = h ? u.y : u.x, w1 = h ? u.w : u.z;
        float p[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float s0 = h ? bf16_high(vs[j][i2]) : bf16_low(vs[j][i2]), s1 = h ? bf16_high(vs[j][NG / 2 + i2]) : bf16_low(vs[j][NG / 2 + i2]);
          p[j][0] = x[j][0] * s0;
          p[j][1] = x[j][1] * s1;
          p[j][2] = x[j][2] * s0;
          p[j][3] = x[j][3] * s1;
        }
        uint4 pa[PT];
#pragma unroll
        for (int term = 0; term < PT; ++term) {
          pa[term] = make_uint4(pack_bf16(p[0][0], p[0][1]), pack_bf16(p[0][2], p[0][3]), pack_bf16(p[1][0], p[1][1]), pack_bf16(p[1][2], p[1][3]));
          if (term + 1 < PT) {
            p[0][0] -= bf16_low(pa[term].x); p[0][1] -= bf16_high(pa[term].x);
            p[0][2] -= bf16_low(pa[term].y); p[0][3] -= bf16_high(pa[term].y);
            p[1][0] -= bf16_low(pa[term].z); p[1][1] -= bf16_high(pa[term].z);
            p[1][2] -= bf16_low(pa[term].w); p[1][3] -= bf16_high(pa[term].w);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t b0 = e == 0 ? codes_bf16<0>(w0) : e == 1 ? codes_bf16<1>(w0) : e == 2 ? codes_bf16<2>(w0) : codes_bf16<3>(w0);
          const uint32_t b1 = e == 0 ? codes_bf16<0>(w1) : e == 1 ? codes_bf16<1>(w1) : e == 2 ? codes_bf16<2>(w1) : codes_bf16<3>(w1);
#pragma unroll
          for (int term = PT - 1; term >= 0; --term) mma_bf16(o[gr][e], pa[term], b0, b1);
        }
      }
    }
  }

  // The warps' parts, joined: their rings are free once all have come here.
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(~0u, l[e], 1);
    l[e] += __shfl_xor_sync(~0u, l[e], 2);
  }
  copy_wait<0>();
  __syncthreads();
  float* const part = reinterpret_cast<float*>(smem);              // [warp][row][D]
  __shared__ float part_m[kWarps][kRows], part_l[kWarps][kRows];
  if (c == 0) {
    part_m[warp][gid] = m[0]; part_m[warp][gid + 8] = m[1];
    part_l[warp][gid] = l[0]; part_l[warp][gid + 8] = l[1];
  }
#pragma unroll
  for (int gr = 0; gr < NG; ++gr)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      // columns 2 c and 2 c + 1 of product e are components 8 c + e and 8 c + 4 + e of the group
      float4* const to = reinterpret_cast<float4*>(part + (warp * kRows + gid + 8 * r) * D + 32 * gr + 8 * c);
      to[0] = make_float4(o[gr][0][2 * r], o[gr][1][2 * r], o[gr][2][2 * r], o[gr][3][2 * r]);
      to[1] = make_float4(o[gr][0][2 * r + 1], o[gr][1][2 * r + 1], o[gr][2][2 * r + 1], o[gr][3][2 * r + 1]);
    }
  __syncthreads();
  float* const ws = a.splits > 1 ? a.ws + (out_tile * a.splits + split) * (kRows * (D + 2)) : nullptr;   // [row][D] sums, [row] maximum, [row] weight
  for (int i = tid; i < kRows * (D / 4); i += kWarps * 32) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
    if (r >= n_rows) break;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part_m[w][r]);
    const float base = top == -INFINITY ? 0.f : top;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float weight = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2_of(part_m[w][r] - base);
      const float4 v = *reinterpret_cast<const float4*>(part + (w * kRows + r) * D + d);
      sum.x += f * v.x; sum.y += f * v.y; sum.z += f * v.z; sum.w += f * v.w;
      weight += f * part_l[w][r];
    }
    if (ws) {
      *reinterpret_cast<float4*>(ws + r * D + d) = sum;
      if (d == 0) { ws[kRows * D + r] = top; ws[kRows * D + kRows + r] = weight; }
    } else {
      const int at = rt * kRows + r, g = at / a.rep, h = kvh * a.rep + at % a.rep;
      const float f = weight > 0.f ? 1.f / weight : 0.f;
      T* const to = static_cast<T*>(a.out) + sent * a.o_n + g * a.o_g + h * a.o_h + d;
      to[0] = from_float<T>(sum.x * f); to[1] = from_float<T>(sum.y * f); to[2] = from_float<T>(sum.z * f); to[3] = from_float<T>(sum.w * f);
      if (d == 0 && a.lse) a.lse[((int64_t)sent * a.g + g) * a.heads + h] = weight > 0.f ? (top + log2f(weight)) * 0.69314718055994531f : -INFINITY;
    }
  }
}

// Joins the parts of a row tile: one CTA for each.
template <class T, int D>
__global__ void __launch_bounds__(128) attend_join_kernel(const __grid_constant__ AttendParams a) {
  const int64_t out_tile = blockIdx.x;
  const int rt = (int)(out_tile % a.row_tiles), kvh = (int)(out_tile / a.row_tiles % a.pool_heads), sent = (int)(out_tile / a.row_tiles / a.pool_heads);
  const int n_rows = min(kRows, a.g * a.rep - rt * kRows);
  const float* const ws = a.ws + out_tile * a.splits * (kRows * (D + 2));
  for (int i = threadIdx.x; i < n_rows * (D / 4); i += 128) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
    float top = -INFINITY;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ws[(int64_t)s * (kRows * (D + 2)) + kRows * D + r]);
    const float base = top == -INFINITY ? 0.f : top;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float weight = 0.f;
    for (int s = 0; s < a.splits; ++s) {
      const float* const p = ws + (int64_t)s * (kRows * (D + 2));
      const float f = exp2_of(p[kRows * D + r] - base);
      const float4 v = *reinterpret_cast<const float4*>(p + r * D + d);
      sum.x += f * v.x; sum.y += f * v.y; sum.z += f * v.z; sum.w += f * v.w;
      weight += f * p[kRows * D + kRows + r];
    }
    const int at = rt * kRows + r, g = at / a.rep, h = kvh * a.rep + at % a.rep;
    const float f = weight > 0.f ? 1.f / weight : 0.f;
    T* const to = static_cast<T*>(a.out) + sent * a.o_n + g * a.o_g + h * a.o_h + d;
    to[0] = from_float<T>(sum.x * f); to[1] = from_float<T>(sum.y * f); to[2] = from_float<T>(sum.z * f); to[3] = from_float<T>(sum.w * f);
    if (d == 0 && a.lse) a.lse[((int64_t)sent * a.g + g) * a.heads + h] = weight > 0.f ? (top + log2f(weight)) * 0.69314718055994531f : -INFINITY;
  }
}

template <class T, int D>
cudaError_t launch_attend(const AttendParams& p, int device, cudaStream_t st) {
  constexpr int smem = attend_smem<T, D>();
  static std::atomic<bool> opted_in[kOpMaxDevices] = {};
  if (smem + 1024 > 48 << 10 && !opted_in[device].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(attend_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    opted_in[device].store(true, std::memory_order_release);
  }
  const int64_t tiles = (int64_t)p.n * p.pool_heads * p.row_tiles;
  attend_kernel<T, D><<<(unsigned)(tiles * p.splits), kWarps * 32, smem, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.splits == 1) return e;
  attend_join_kernel<T, D><<<(unsigned)tiles, 128, 0, st>>>(p);
  return cudaGetLastError();
}

int row_tiles_of(const linmt_attend_pages4_args* g) { return (int)(((int64_t)g->g * (g->heads / g->pages.heads) + kRows - 1) / kRows); }

// CTAs that share a row tile's positions: as many as give the GPU three rounds of the four CTAs that an SM holds, but 16 tiles (256
// positions) at least for each.
int splits_of(const linmt_attend_pages4_args* g) {
  const int64_t tiles = (int64_t)g->n * g->pages.heads * row_tiles_of(g), most = ((int64_t)g->width * (g->pages.page / pages4::kTile) + 15) / 16;
  if (tiles == 0 || most <= 1) return 1;
  const int64_t want = (3 * 4 * 148 + tiles - 1) / tiles;
  return (int)(want < most ? want : most);
}

int check(const linmt_attend_pages4_args* g) {
  if (!g || g->size != sizeof(*g)) return op_fail(LINMT_EINVAL, "attend_pages4: not this library's argument struct");
  if (int rc = check_pages4(g->pages, "attend_pages4")) return rc;
  if (g->n < 0 || g->g < 0 || g->heads < 1 || g->heads % g->pages.heads || g->width < 0 || !dtype_ok(g->dtype))
    return op_fail(LINMT_EINVAL, "attend_pages4: n = %d, g = %d, heads = %d (a multiple of the pool's %d), width = %d, dtype = %d", g->n, g->g, g->heads, g->pages.heads, g->width, g->dtype);
  if (!(g->scale - g->scale == 0.f) || !(g->cap >= 0.f) || !(g->cap - g->cap == 0.f)) return op_fail(LINMT_EINVAL, "attend_pages4: scale and cap have to be finite, cap not negative");
  if (g->n == 0 || g->g == 0) return LINMT_OK;
  if (!g->q || !g->out || !g->len || (g->width && !g->table)) return op_fail(LINMT_EINVAL, "attend_pages4: an array is missing");
  if (!g->slope != !g->centre || !g->first != !g->last) return op_fail(LINMT_EINVAL, "attend_pages4: slope goes with centre, first with last");
  const int size = dtype_bytes(g->dtype);
  if (!aligned(g->q, size) || !aligned(g->out, size) || !aligned(g->lse, 4) || !aligned(g->table, 4) || !aligned(g->len, 4) || !aligned(g->slope, 4) || !aligned(g->centre, 4) || !aligned(g->first, 4) || !aligned(g->last, 4))
    return op_fail(LINMT_EINVAL, "attend_pages4: an array is not aligned to its type");
  if ((int64_t)g->g * g->heads > INT32_MAX / 2 || (int64_t)g->n * g->pages.heads * row_tiles_of(g) > (1 << 24))
    return op_fail(LINMT_ELIMIT, "attend_pages4: %d sentences of %d rows and %d heads are too many for one call", g->n, g->g, g->heads);
  return LINMT_OK;
}

int64_t workspace_of(const linmt_attend_pages4_args* g) {
  const int splits = splits_of(g);
  return splits == 1 ? 0 : (int64_t)g->n * g->pages.heads * row_tiles_of(g) * splits * (kRows * (g->pages.dim + 2)) * 4;
}

}  // namespace
}  // namespace ops
}  // namespace linmt

extern "C" {

int64_t linmt_attend_pages4_workspace(const linmt_attend_pages4_args* g) {
  using namespace linmt::ops;
  if (check(g)) return -1;
  return g->n == 0 || g->g == 0 ? 0 : workspace_of(g);
}

int linmt_attend_pages4(const linmt_attend_pages4_args* g) {
  using namespace linmt::ops;
  if (int rc = check(g)) return rc;
  if (g->n == 0 || g->g == 0) return LINMT_OK;
  const int64_t need = workspace_of(g);
  if (need && (!g->workspace || g->workspace_bytes < need || !aligned(g->workspace, 16)))
    return op_fail(LINMT_EINVAL, "attend_pages4: a workspace of %lld bytes is needed, 16-byte aligned", (long long)need);
  if (g->device < 0 || g->device >= kOpMaxDevices) return op_fail(LINMT_EINVAL, "attend_pages4: device = %d", g->device);
  OnDevice on(g->device);
  if (on.err != cudaSuccess) return op_cuda(on.err, "attend_pages4");
  AttendParams p{static_cast<const unsigned char*>(g->pages.data), g->pages.stride_page, g->pages.stride_head, g->pages.n_pages, g->pages.heads, g->pages.page,
                 g->q, g->q_stride_n, g->q_stride_g, g->q_stride_h, g->out, g->out_stride_n, g->out_stride_g, g->out_stride_h, g->lse, g->table, g->table_stride, g->len,
                 g->slope, g->centre, g->first, g->last, static_cast<float*>(g->workspace), g->n, g->g, g->heads, g->heads / g->pages.heads, g->width, row_tiles_of(g), splits_of(g),
                 g->scale, g->cap};
  const cudaStream_t st = static_cast<cudaStream_t>(g->stream);
  cudaError_t e;
  if (g->pages.dim == 64)
    e = g->dtype == LINMT_F32 ? launch_attend<float, 64>(p, g->device, st) : g->dtype == LINMT_BF16 ? launch_attend<__nv_bfloat16, 64>(p, g->device, st) : launch_attend<__half, 64>(p, g->device, st);
  else
    e = g->dtype == LINMT_F32 ? launch_attend<float, 128>(p, g->device, st) : g->dtype == LINMT_BF16 ? launch_attend<__nv_bfloat16, 128>(p, g->device, st) : launch_attend<__half, 128>(p, g->device, st);
  return e == cudaSuccess ? LINMT_OK : op_cuda(e, "attend_pages4");
}

}  // extern "C"
