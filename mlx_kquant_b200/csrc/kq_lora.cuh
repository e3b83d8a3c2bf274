// Low-rank adapters beside a shared projection: the kernel of both products, in . w1^T -> u and base + f u . w2^T -> out.
//
// A cluster of CTAs takes a tile of rows that share an adapter. Each CTA multiplies a part of the contraction, the parts of u
// meet over distributed shared memory in the order of the CTAs, and each CTA makes a part of the output's columns: one launch,
// rows read once, outputs written once, the adapter's matrices read once per tile. The products are mma.sync m16n8k16: a tile's
// work is bound by its bytes, and the fragments come straight from global memory, 16 bytes a lane, under a permutation of the
// contraction (both operands alike) or of the output's columns that makes a lane's share contiguous.
//
// float32 parameters are split into bf16 terms of 8 bits: three where the result is kept in float32 (u), two where it is rounded to
// 16 bits; fp16 rows are then two bf16 terms, exactly. u enters the second product as two terms of the row's type, fp16 ones
// under a power of two per row.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "kq_lora.h"

namespace kq {
namespace lora {

namespace cg = cooperative_groups;
typedef __nv_bfloat16 bf16;

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------------------------------- groups
__device__ __forceinline__ int group_of(const LoraGroups& g, long long e) {
  int id = 0;
  if (g.ids != nullptr) {
    id = g.ids[e / g.slots];
    if ((unsigned)id >= (unsigned)g.G) return -1;
  }
  if (g.experts == nullptr) return id;
  const uint32_t ex = g.experts[e];
  return ex < (uint32_t)g.E ? id * g.E + (int)ex : -1;
}
__device__ __forceinline__ float factor_of(const LoraGroups& g, int group) {
  return g.scaling != nullptr ? g.scale * g.scaling[group / g.E] : g.scale;
}

// ---------------------------------------------------------------------------------------------------- fragments
__device__ __forceinline__ uint32_t pack(bf16 lo, bf16 hi) {
  return (uint32_t)__bfloat16_as_ushort(lo) | (uint32_t)__bfloat16_as_ushort(hi) << 16;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bf16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The leading bits of two floats as a bf16 pair, cut off (never rounded up to infinity), and what is left of them.
__device__ __forceinline__ uint32_t take_bf16(float& f0, float& f1) {
  const uint32_t b0 = __float_as_uint(f0) & 0xffff0000u, b1 = __float_as_uint(f1) & 0xffff0000u;
  // nothing is left of an infinity; a NaN whose bits all lie below stays one in the rest
  f0 = fabsf(f0) == INFINITY ? 0.f : f0 - __uint_as_float(b0);
  f1 = fabsf(f1) == INFINITY ? 0.f : f1 - __uint_as_float(b1);
  return __byte_perm(b0, b1, 0x7632);
}
__device__ __forceinline__ uint32_t round_bf16(float f0, float f1) {
  return pack(__float2bfloat16_rn(f0), __float2bfloat16_rn(f1));
}

// N terms of the pair (f0, f1).
template <int N>
__device__ __forceinline__ void split(float f0, float f1, uint32_t (&t)[N]) {
#pragma unroll
  for (int i = 0; i < N - 1; i++) t[i] = take_bf16(f0, f1);
  t[N - 1] = round_bf16(f0, f1);
}

// Pairs of 16-bit elements as terms of the type that the products are made in (CT): themselves, or an fp16 pair as two bf16.
template <typename XT, typename CT>
struct RowTerms {
  static constexpr int N = std::is_same<XT, CT>::value ? 1 : 2;
  __device__ static __forceinline__ void get(uint32_t v, uint32_t (&t)[N]) {
    if constexpr (N == 1) {
      t[0] = v;
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
      split<2>(f.x, f.y, t);
    }
  }
};

// `N` contiguous elements as pairs of words, guarded: elements from `valid` on are zero.
template <typename T, int N, bool VEC>
struct Load {
  static constexpr int WORDS = N * (int)sizeof(T) / 4;
  uint32_t w[WORDS];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; i++) w[i] = 0;
  }
  __device__ __forceinline__ void get(const T* p, int valid) {
    if constexpr (VEC) {   // all or nothing
      if (valid <= 0) { zero(); return; }
      if constexpr (WORDS >= 4) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
          w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
      } else if constexpr (WORDS == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = v.x; w[1] = v.y;
      } else {
        w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; i++) w[i] = i < valid ? __float_as_uint((float)p[i]) : 0u;
    } else {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < N / 2; i++)
        w[i] = (2 * i < valid ? (uint32_t)h[2 * i] : 0u) | (2 * i + 1 < valid ? (uint32_t)h[2 * i + 1] << 16 : 0u);
    }
  }
};

// the pair (x[i], x[i + 1]) of a load, i even, as terms
template <typename PT, int TERMS, int N, bool VEC>
__device__ __forceinline__ void pair_along(const Load<PT, N, VEC>& l, int i, uint32_t (&t)[TERMS]) {
  if constexpr (sizeof(PT) == 2) t[0] = l.w[i / 2];
  else split<TERMS>(__uint_as_float(l.w[i]), __uint_as_float(l.w[i + 1]), t);
}
// the pair (p[i], q[i]) of two loads
template <typename PT, int TERMS, int N, bool VEC>
__device__ __forceinline__ void pair_across(const Load<PT, N, VEC>& p, const Load<PT, N, VEC>& q, int i, uint32_t (&t)[TERMS]) {
  if constexpr (sizeof(PT) == 2) t[0] = __byte_perm(p.w[i / 2], q.w[i / 2], (i & 1) ? 0x7632 : 0x5410);
  else split<TERMS>(__uint_as_float(p.w[i]), __uint_as_float(q.w[i]), t);
}

template <int XN, int PN, int MOST, typename CT>
__device__ __forceinline__ void mma_terms(float (&c)[4], const uint32_t (&a)[XN][4], const uint32_t (&b0)[PN], const uint32_t (&b1)[PN]) {
  // smallest products first; those below the last term's bits are left out
#pragma unroll
  for (int s = MOST - 1; s >= 0; s--)
#pragma unroll
    for (int i = 0; i < XN; i++)
#pragma unroll
      for (int j = 0; j < PN; j++)
        if (i + j == s) mma(c, a[i], b0[j], b1[j], CT());
}

// ---------------------------------------------------------------------------------------------------- tile
struct TileAt {
  int group, rows;
};

// The tile that this cluster takes, its entries in s_row; rows 0: none.
template <int MT>
__device__ __forceinline__ TileAt find_tile(const LoraArgs& a, int tile, int* s_row, int* s_info) {
  const int tid = threadIdx.x;
  TileAt t;
  if (a.direct) {
    if (tid < 32) {
      const int mine = group_of(a.g, tile);
      int before = 0;
      for (int b = tid; b < tile; b += 32) before += group_of(a.g, b) == mine;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
      int rows = 0;
      if (before % MT == 0) {
        for (int b0 = tile; b0 < (int)a.g.n && rows < MT; b0 += 32) {
          const int b = b0 + tid;
          const bool same = b < (int)a.g.n && group_of(a.g, b) == mine;
          const uint32_t m = __ballot_sync(0xffffffffu, same);
          const int at = rows + __popc(m & ((1u << tid) - 1u));
          if (same && at < MT) s_row[at] = b;
          rows = min(MT, rows + __popc(m));
        }
      }
      for (int i = rows + tid; i < MT; i += 32) s_row[i] = -1;
      if (tid == 0) {
        s_info[0] = mine;
        s_info[1] = rows;
      }
    }
    __syncthreads();
    t.group = s_info[0];
    t.rows = s_info[1];
  } else if (a.plan.tiles != nullptr) {
    const LoraTile d = a.plan.tiles[tile];
    t.group = d.group;
    t.rows = d.rows;
    if (tid < MT) s_row[tid] = tid < d.rows ? a.plan.order[d.start + tid] : -1;
    __syncthreads();
  } else {
    t.group = 0;
    const long long left = a.g.n - (long long)tile * MT;
    t.rows = left < MT ? (int)left : MT;
    if (tid < MT) s_row[tid] = tid < t.rows ? tile * MT + tid : -1;
    __syncthreads();
  }
  return t;
}

template <typename XT>
__device__ __forceinline__ float to_float(XT v) { return static_cast<float>(v); }

// eight neighbouring columns of an output row
template <typename XT>
__device__ __forceinline__ void store8(const LoraArgs& a, int row, int col, int c_end, const float (&v)[8], float f) {
  if (a.out_f32) {
    float* o = static_cast<float*>(a.out) + (long long)row * a.out_stride + (col - a.c0);
    if (a.vec_out && col + 8 <= c_end) {
      reinterpret_cast<float4*>(o)[0] = make_float4(f * v[0], f * v[1], f * v[2], f * v[3]);
      reinterpret_cast<float4*>(o)[1] = make_float4(f * v[4], f * v[5], f * v[6], f * v[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (col + i < c_end) o[i] = f * v[i];
    }
    return;
  }
  XT* o = static_cast<XT*>(a.out) + (long long)row * a.out_stride + (col - a.c0);
  const XT* b = static_cast<const XT*>(a.base) + (long long)row * a.base_stride + (col - a.c0);
  if (a.vec_out && col + 8 <= c_end) {
    uint4 raw = a.base != nullptr ? *reinterpret_cast<const uint4*>(b) : make_uint4(0, 0, 0, 0);
    XT* h = reinterpret_cast<XT*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = XT(fmaf(f, v[i], a.base != nullptr ? to_float(h[i]) : 0.f));
    *reinterpret_cast<uint4*>(o) = raw;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (col + i < c_end) o[i] = XT(fmaf(f, v[i], a.base != nullptr ? to_float(b[i]) : 0.f));
  }
}

// rows without an adapter: the base as it is
template <typename XT>
__device__ __forceinline__ void copy_rows(const LoraArgs& a, const int* s_row, int rows, int lo, int hi) {
  if (a.out == nullptr || (a.out == a.base && !a.out_f32)) return;
  for (int m = 0; m < rows; m++) {
    const int row = s_row[m];
    if (a.out_f32) {
      float* o = static_cast<float*>(a.out) + (long long)row * a.out_stride - a.c0;
      for (int c = lo + threadIdx.x; c < hi; c += kThreads) o[c] = 0.f;
      continue;
    }
    XT* o = static_cast<XT*>(a.out) + (long long)row * a.out_stride - a.c0;
    const XT* b = static_cast<const XT*>(a.base) + (long long)row * a.base_stride - a.c0;
    if (a.vec_out && lo % 8 == 0 && hi % 8 == 0) {
      for (int c = lo + 8 * threadIdx.x; c < hi; c += 8 * kThreads)
        *reinterpret_cast<uint4*>(o + c) = a.base != nullptr ? *reinterpret_cast<const uint4*>(b + c) : make_uint4(0, 0, 0, 0);
    } else {
      for (int c = lo + threadIdx.x; c < hi; c += kThreads) o[c] = a.base != nullptr ? b[c] : XT(0.f);
    }
  }
}

// ---- first product: a warp's part of u, [16 WT rows] x [16 RT ranks], over the 32-blocks k0, k0 + step, ... below k1
template <typename XT, typename PT, typename CT, bool BWD, int RT, int WT, bool VI, bool VW>
__device__ __forceinline__ void shrink_part(const LoraArgs& a, const PT* w1, const int* s_row, int m0, int k0, int k1, int step,
                                            float (&acc)[WT][2 * RT][4]) {
  constexpr int XN = RowTerms<XT, CT>::N, PN = sizeof(PT) == 4 ? 3 : 1;
  constexpr int MOST = PN > XN ? PN : XN;
  constexpr int JV = 2 * RT;
  const int lane = threadIdx.x & 31, i = lane >> 2, q = lane & 3;
  const XT* xp[WT][2];
#pragma unroll
  for (int m = 0; m < WT; m++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int e = s_row[m0 + 16 * m + 8 * h + i];
      xp[m][h] = e < 0 ? nullptr : static_cast<const XT*>(a.in) + (long long)(a.in_div == 1 ? e : e / a.in_div) * a.in_stride;
    }
  for (int k = k0; k < k1; k += step) {
    const int kk = k + 8 * q;
    Load<XT, 8, VI> x[WT][2];
#pragma unroll
    for (int m = 0; m < WT; m++)
#pragma unroll
      for (int h = 0; h < 2; h++) x[m][h].get(xp[m][h] + kk, xp[m][h] == nullptr ? 0 : a.D1 - kk);
    if constexpr (!BWD) {
#pragma unroll
      for (int jt = 0; jt < 2 * RT; jt++) {
        const int j = 8 * jt + i;
        Load<PT, 8, VW> w;
        w.get(w1 + (long long)j * a.D1 + kk, j < a.r ? a.D1 - kk : 0);
#pragma unroll
        for (int s = 0; s < 2; s++) {
          uint32_t b0[PN], b1[PN];
          pair_along<PT, PN>(w, 4 * s, b0);
          pair_along<PT, PN>(w, 4 * s + 2, b1);
#pragma unroll
          for (int m = 0; m < WT; m++) {
            uint32_t xa[XN][4], t0[XN], t1[XN], t2[XN], t3[XN];
            RowTerms<XT, CT>::get(x[m][0].w[2 * s], t0);
            RowTerms<XT, CT>::get(x[m][1].w[2 * s], t1);
            RowTerms<XT, CT>::get(x[m][0].w[2 * s + 1], t2);
            RowTerms<XT, CT>::get(x[m][1].w[2 * s + 1], t3);
#pragma unroll
            for (int n = 0; n < XN; n++) { xa[n][0] = t0[n]; xa[n][1] = t1[n]; xa[n][2] = t2[n]; xa[n][3] = t3[n]; }
            mma_terms<XN, PN, MOST, CT>(acc[m][jt], xa, b0, b1);
          }
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < 2; s++) {
        uint32_t xa[WT][XN][4];
#pragma unroll
        for (int m = 0; m < WT; m++) {
          uint32_t t0[XN], t1[XN], t2[XN], t3[XN];
          RowTerms<XT, CT>::get(x[m][0].w[2 * s], t0);
          RowTerms<XT, CT>::get(x[m][1].w[2 * s], t1);
          RowTerms<XT, CT>::get(x[m][0].w[2 * s + 1], t2);
          RowTerms<XT, CT>::get(x[m][1].w[2 * s + 1], t3);
#pragma unroll
          for (int n = 0; n < XN; n++) { xa[m][n][0] = t0[n]; xa[m][n][1] = t1[n]; xa[m][n][2] = t2[n]; xa[m][n][3] = t3[n]; }
        }
        // rows kk + 4 s .. + 3 of w1, a lane's JV neighbouring ranks of each
        Load<PT, JV, VW> w[4];
#pragma unroll
        for (int n = 0; n < 4; n++) w[n].get(w1 + (long long)(kk + 4 * s + n) * a.r + i * JV, kk + 4 * s + n < a.D1 ? a.r - i * JV : 0);
#pragma unroll
        for (int jt = 0; jt < 2 * RT; jt++) {
          uint32_t b0[PN], b1[PN];
          pair_across<PT, PN>(w[0], w[1], jt, b0);
          pair_across<PT, PN>(w[2], w[3], jt, b1);
#pragma unroll
          for (int m = 0; m < WT; m++) mma_terms<XN, PN, MOST, CT>(acc[m][jt], xa[m], b0, b1);
        }
      }
    }
  }
}

// ---- second product: the CTA's columns [lo, hi), a warp a chunk of 32 (forward) or 64 (backward) after another
template <typename XT, typename PT, typename CT, bool BWD, int RT, int MT, bool VW>
__device__ __forceinline__ void expand_part(const LoraArgs& a, const PT* w2, const int* s_row, const float* s_factor, const uint16_t* s_u,
                                            int rows, int lo, int hi) {
  constexpr int PN = sizeof(PT) == 4 ? 2 : 1, UP = 16 * RT + 8, CH = BWD ? 64 : 32, NT = CH / 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = lane >> 2, q = lane & 3;
  for (int c0 = lo + CH * warp; c0 < hi; c0 += CH * (kThreads / 32)) {
    for (int m = 0; m < MT / 16; m++) {
      if (16 * m >= rows) break;
      float acc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) acc[n][k] = 0.f;
#pragma unroll
      for (int ks = 0; ks < RT; ks++) {
        uint32_t ua[2][4];
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const uint2 p = *reinterpret_cast<const uint2*>(s_u + (t * MT + 16 * m + i) * UP + 16 * ks + 4 * q);
          const uint2 v = *reinterpret_cast<const uint2*>(s_u + (t * MT + 16 * m + 8 + i) * UP + 16 * ks + 4 * q);
          ua[t][0] = p.x; ua[t][1] = v.x; ua[t][2] = p.y; ua[t][3] = v.y;
        }
        const int j = 16 * ks + 4 * q;
        if constexpr (!BWD) {
#pragma unroll
          for (int n = 0; n < NT; n++) {
            const int col = c0 + 8 * (i >> 1) + 2 * n + (i & 1);
            Load<PT, 4, VW> w;
            w.get(w2 + (long long)col * a.r + j, col < hi ? a.r - j : 0);
            uint32_t b0[PN], b1[PN];
            pair_along<PT, PN>(w, 0, b0);
            pair_along<PT, PN>(w, 2, b1);
            mma_terms<2, PN, 2, CT>(acc[n], ua, b0, b1);
          }
        } else {
          Load<PT, 8, VW> w[4];
#pragma unroll
          for (int k = 0; k < 4; k++) w[k].get(w2 + (long long)(j + k) * a.D2 + c0 + 8 * i, j + k < a.r ? hi - (c0 + 8 * i) : 0);
#pragma unroll
          for (int n = 0; n < NT; n++) {
            uint32_t b0[PN], b1[PN];
            pair_across<PT, PN>(w[0], w[1], n, b0);
            pair_across<PT, PN>(w[2], w[3], n, b1);
            mma_terms<2, PN, 2, CT>(acc[n], ua, b0, b1);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int row = s_row[16 * m + 8 * h + i];
        if (row < 0) continue;
        const float f = s_factor[16 * m + 8 * h + i];
        float v[8];
        if constexpr (!BWD) {
#pragma unroll
          for (int n = 0; n < 4; n++) { v[2 * n] = acc[n][2 * h]; v[2 * n + 1] = acc[n][2 * h + 1]; }
          if (c0 + 8 * q < hi) store8<XT>(a, row, c0 + 8 * q, hi, v, f);
        } else {
#pragma unroll
          for (int p = 0; p < 2; p++) {
#pragma unroll
            for (int n = 0; n < 8; n++) v[n] = acc[n][2 * h + p];
            if (c0 + 16 * q + 8 * p < hi) store8<XT>(a, row, c0 + 16 * q + 8 * p, hi, v, f);
          }
        }
      }
    }
  }
}

template <int RT, int MT>
constexpr int tile_smem() {
  constexpr int RP = 16 * RT;
  const int red = kThreads / 32 / 2 * (MT >= 32 ? 32 : 16) * RP * 4;   // the partial sums of half of the warps
  return red + MT * RP * 4 + 2 * MT * (RP + 8) * 2 + MT * 4 * 2 + 16;
}

template <typename XT, typename PT, bool BWD, int RT, int MT>
__global__ void __launch_bounds__(kThreads) tile_kernel(const LoraArgs a) {
  typedef typename std::conditional<sizeof(PT) == 4, bf16, XT>::type CT;
  constexpr int RP = 16 * RT, UP = RP + 8, WT = MT >= 32 ? 2 : 1, TG = MT / (16 * WT), KS = kThreads / 32 / TG;
  constexpr int JV = 2 * RT;
  extern __shared__ __align__(16) uint8_t smem[];
  float* s_red = reinterpret_cast<float*>(smem);                                     // [warps / 2][16 WT][RP]
  float* s_part = s_red + kThreads / 32 / 2 * 16 * WT * RP;                          // [MT][RP]: this CTA's part of u
  uint16_t* s_u = reinterpret_cast<uint16_t*>(s_part + MT * RP);                     // [2][MT][UP]: u as two terms
  float* s_factor = reinterpret_cast<float*>(s_u + 2 * MT * UP);                     // [MT]
  int* s_row = reinterpret_cast<int*>(s_factor + MT);                                // [MT]
  int* s_info = s_row + MT;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, i = lane >> 2, q = lane & 3;
  const TileAt t = find_tile<MT>(a, blockIdx.x / C, s_row, s_info);
  if (t.rows == 0) return;   // (the whole cluster)
  const int chunk = BWD ? 64 : 32, n_chunks = (a.c1 - a.c0 + chunk - 1) / chunk;
  const int lo = a.c0 + (int)((long long)n_chunks * rank / C) * chunk;
  const int hi = min(a.c1, a.c0 + (int)((long long)n_chunks * (rank + 1) / C) * chunk);
  if (t.group < 0) {
    copy_rows<XT>(a, s_row, t.rows, lo, hi);
    if (a.shrink && a.u != nullptr && rank == 0)
      for (int v = tid; v < t.rows * a.r; v += kThreads) a.u[(long long)s_row[v / a.r] * a.r + v % a.r] = 0.f;
    return;
  }
  const float factor = factor_of(a.g, t.group);
  if (a.shrink) {
    const PT* w1 = static_cast<const PT*>(a.w1) + (long long)t.group * a.r * a.D1;
    const int blocks = (a.D1 + 31) / 32;
    const int b0 = (int)((long long)blocks * rank / C), b1 = (int)((long long)blocks * (rank + 1) / C);
    const int tg = warp / KS, ks = warp % KS;
    float acc[WT][2 * RT][4];
#pragma unroll
    for (int m = 0; m < WT; m++)
#pragma unroll
      for (int n = 0; n < 2 * RT; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) acc[m][n][k] = 0.f;
    if (a.vec_in && a.vec_w1)
      shrink_part<XT, PT, CT, BWD, RT, WT, true, true>(a, w1, s_row, 16 * WT * tg, 32 * (b0 + ks), 32 * b1, 32 * KS, acc);
    else
      shrink_part<XT, PT, CT, BWD, RT, WT, false, false>(a, w1, s_row, 16 * WT * tg, 32 * (b0 + ks), 32 * b1, 32 * KS, acc);
    // the warps' parts, halves onto halves
    for (int h = KS / 2; h > 0; h >>= 1) {
      float* mine = s_red + (size_t)(tg * (KS / 2) + (ks % h)) * 16 * WT * RP;
      if (ks >= h && ks < 2 * h) {
#pragma unroll
        for (int m = 0; m < WT; m++)
#pragma unroll
          for (int n = 0; n < 2 * RT; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) mine[((m * 2 * RT + n) * 4 + k) * 32 + lane] = acc[m][n][k];
      }
      __syncthreads();
      if (ks < h) {
#pragma unroll
        for (int m = 0; m < WT; m++)
#pragma unroll
          for (int n = 0; n < 2 * RT; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) acc[m][n][k] += mine[((m * 2 * RT + n) * 4 + k) * 32 + lane];
      }
      __syncthreads();
    }
    if (ks == 0) {
#pragma unroll
      for (int m = 0; m < WT; m++)
#pragma unroll
        for (int n = 0; n < 2 * RT; n++)
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const int row = 16 * (WT * tg + m) + i + 8 * (k >> 1), c = 2 * q + (k & 1);
            s_part[row * RP + (BWD ? c * JV + n : 8 * n + c)] = acc[m][n][k];
          }
    }
    cluster.sync();
  }
  // u of the whole contraction: float32 out, two terms for the second product. A warp a row at a time.
  for (int m = warp; m < MT; m += kThreads / 32) {
    float v[(RP + 31) / 32], most = 0.f;
    const int row = s_row[m];
#pragma unroll
    for (int b = 0; b < (RP + 31) / 32; b++) {
      const int j = 32 * b + lane;
      v[b] = 0.f;
      if (j < a.r && row >= 0) {
        if (a.shrink) {
          for (int c = 0; c < C; c++) v[b] += *cluster.map_shared_rank(s_part + m * RP + j, c);
          if (a.scale_u) v[b] *= factor;
          if (a.u != nullptr && rank == m % C) a.u[(long long)row * a.r + j] = v[b];
        } else {
          v[b] = a.u[(long long)row * a.r + j];
        }
      }
      most = fmaxf(most, fabsf(v[b]));
    }
    float f = 1.f;
    if constexpr (std::is_same<CT, __half>::value) {
      // fp16 terms: the largest of the row comes to lie in [1, 2)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (most > 0.f && most < INFINITY) f = __uint_as_float(max(1u, min(253u, __float_as_uint(most) >> 23)) << 23);
    }
#pragma unroll
    for (int b = 0; b < (RP + 31) / 32; b++) {
      const int j = 32 * b + lane;
      if (j >= RP) continue;
      if constexpr (std::is_same<CT, __half>::value) {
        const float n = v[b] / f;
        const __half h = __float2half_rn(n);
        const float rest = fabsf(n) == INFINITY ? 0.f : n - __half2float(h);
        s_u[m * UP + j] = __half_as_ushort(h);
        s_u[(MT + m) * UP + j] = __half_as_ushort(__float2half_rn(rest));
      } else {
        const uint32_t h = __float_as_uint(v[b]) & 0xffff0000u;
        const float rest = fabsf(v[b]) == INFINITY ? 0.f : v[b] - __uint_as_float(h);
        s_u[m * UP + j] = (uint16_t)(h >> 16);
        s_u[(MT + m) * UP + j] = __bfloat16_as_ushort(__float2bfloat16_rn(rest));
      }
    }
    if (lane == 0) s_factor[m] = a.scale_u ? f : f * factor;
  }
  __syncthreads();
  if (a.shrink) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  if (a.out != nullptr) {
    const PT* w2 = static_cast<const PT*>(a.w2) + (long long)t.group * a.r * a.D2;
    if (a.vec_w2) expand_part<XT, PT, CT, BWD, RT, MT, true>(a, w2, s_row, s_factor, s_u, t.rows, lo, hi);
    else expand_part<XT, PT, CT, BWD, RT, MT, false>(a, w2, s_row, s_factor, s_u, t.rows, lo, hi);
  }
  // nobody leaves while its part of u may still be read
  if (a.shrink) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

template <typename XT, typename PT, bool BWD, int RT, int MT>
cudaError_t launch_tile(const LoraArgs& a, int cluster, cudaStream_t st) {
  constexpr int smem = tile_smem<RT, MT>();
  auto kern = tile_kernel<XT, PT, BWD, RT, MT>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n_clusters * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}
template <typename XT, typename PT, bool BWD, int RT>
cudaError_t launch_mt(const LoraArgs& a, int mt, int cluster, cudaStream_t st) {
  return mt == 16 ? launch_tile<XT, PT, BWD, RT, 16>(a, cluster, st) : launch_tile<XT, PT, BWD, RT, 64>(a, cluster, st);
}
template <typename XT, typename PT, bool BWD>
cudaError_t launch_rt(const LoraArgs& a, int mt, int cluster, cudaStream_t st) {
  if (a.r <= 16) return launch_mt<XT, PT, BWD, 1>(a, mt, cluster, st);
  if (a.r <= 32) return launch_mt<XT, PT, BWD, 2>(a, mt, cluster, st);
  if (a.r <= 64) return launch_mt<XT, PT, BWD, 4>(a, mt, cluster, st);
  return launch_mt<XT, PT, BWD, 8>(a, mt, cluster, st);
}
template <typename XT, typename PT>
cudaError_t launch_types(const LoraArgs& a, bool backward, int mt, int cluster, cudaStream_t st) {
  return backward ? launch_rt<XT, PT, true>(a, mt, cluster, st) : launch_rt<XT, PT, false>(a, mt, cluster, st);
}

}  // namespace lora
}  // namespace kq
