// Low-rank adapters beside a shared projection: the kernel of both products, in . w1^T -> u and base + f u . w2^T -> out.
//
// A cluster of CTAs takes a tile of 16 or 64 rows that share an adapter. Each CTA multiplies a part of the contraction, the parts of
// u meet over distributed shared memory in the order of the CTAs, and each CTA makes a part of the output's columns: one launch,
// rows read once, outputs written once, the adapter's matrices read once per tile. Rows and weights of both products pass through
// one ring of stages in shared memory, filled by 16-byte asynchronous copies (the rows of a tile lie anywhere), so that the second
// product's weights and the base's rows are on their way while the first ends. The products are mma.sync m16n8k16 on ldmatrix
// fragments, sums in float32.
//
// float32 parameters are split into bf16 terms of 8 bits as they are read from shared memory: three where the result is kept in
// float32 (u), two where it is rounded to 16 bits; fp16 rows are then two bf16 terms, exactly. u enters the second product as two
// terms of the row's type, fp16 ones under a power of two per row: 16 bits. It is saved for the gradients as three bf16 terms beside float32
// parameters, as two beside 16-bit ones, whose gradients are rounded to 16 bits.
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

// First in every kernel here: they are launched beside the end of the launch before them and wait for it, and let the next one start
// likewise only then (so that what lies further back has ended for it too).
__device__ __forceinline__ void wait_for_launch() {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;\n" ::: "memory");
}
// cluster: CTAs of a cluster, or 0
template <typename... Params, typename... Args>
cudaError_t launch(void (*kern)(Params...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, Params(args)...);
}

// ---------------------------------------------------------------------------------------------------- groups
__device__ __forceinline__ int group_of(const LoraGroups& g, long long e) {
  int id = 0;
  if (g.ids != nullptr) {
    id = g.ids[g.slots == 1 ? (unsigned)e : (unsigned)e / (unsigned)g.slots];
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
__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
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
// the same from zero
__device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t round_bf16(float f0, float f1) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(f0, f1);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t round_pair(float f0, float f1, bf16) { return round_bf16(f0, f1); }
__device__ __forceinline__ uint32_t round_pair(float f0, float f1, __half) {
  const __half2 v = __floats2half2_rn(f0, f1);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Two floats as the nearest bf16 pair, and what is left of them: 2^-8 of them at most, so that of two such splits' products the one of
// both rests, which the products with two terms leave away, is below 2^-16. (Cut off, the rests were up to 2^-7 and never turned
// down, the product left away up to 2^-14.) FINITE: of an infinity NaN is left, else nothing. (The last 2^-8 below the largest float
// round to infinity.)
template <bool FINITE>
__device__ __forceinline__ uint32_t take_bf16(float& f0, float& f1) {
  const uint32_t t = round_bf16(f0, f1);
  const float t0 = __uint_as_float(t << 16), t1 = __uint_as_float(t & 0xffff0000u);
  f0 = !FINITE && fabsf(t0) == INFINITY ? 0.f : f0 - t0;
  f1 = !FINITE && fabsf(t1) == INFINITY ? 0.f : f1 - t1;
  return t;
}
// N bf16 terms of the pair (f0, f1)
template <int N, bool FINITE = false>
__device__ __forceinline__ void split(float f0, float f1, uint32_t (&t)[N]) {
#pragma unroll
  for (int i = 0; i < N - 1; i++) t[i] = take_bf16<FINITE>(f0, f1);
  t[N - 1] = round_bf16(f0, f1);
}

// Pairs of 16-bit elements as terms of the type that the products are made in (CT): themselves, or an fp16 pair as two bf16.
template <typename XT, typename CT>
struct RowTerms {
  static constexpr int N = std::is_same<XT, CT>::value ? 1 : 2;
  __device__ static __forceinline__ void get(const uint32_t (&v)[4], uint32_t (&t)[N][4]) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if constexpr (N == 1) {
        t[0][k] = v[k];
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[k]));
        uint32_t p[2];
        split<2>(f.x, f.y, p);
        t[0][k] = p[0];
        t[1][k] = p[1];
      }
    }
  }
};

// all products of the terms but those below the last one's bits, smallest first
template <int XN, int PN, typename CT>
__device__ __forceinline__ void mma_terms(float (&c)[4], const uint32_t (&a)[XN][4], const uint32_t (&b0)[PN], const uint32_t (&b1)[PN]) {
  constexpr int MOST = PN > XN ? PN : XN;
#pragma unroll
  for (int s = MOST - 1; s >= 0; s--)
#pragma unroll
    for (int i = 0; i < XN; i++)
#pragma unroll
      for (int j = 0; j < PN; j++)
        if (i + j == s) mma(c, a[i], b0[j], b1[j], CT());
}

// the bf16 products by themselves, c = ...
template <int XN, int PN>
__device__ __forceinline__ void mma_terms_first(float (&c)[4], const uint32_t (&a)[XN][4], const uint32_t (&b0)[PN], const uint32_t (&b1)[PN]) {
  constexpr int MOST = PN > XN ? PN : XN;
  bool first = true;
#pragma unroll
  for (int s = MOST - 1; s >= 0; s--)
#pragma unroll
    for (int i = 0; i < XN; i++)
#pragma unroll
      for (int j = 0; j < PN; j++)
        if (i + j == s) {
          if (first) mma_first(c, a[i], b0[j], b1[j]);
          else mma(c, a[i], b0[j], b1[j], bf16());
          first = false;
        }
}

// ---------------------------------------------------------------------------------------------------- shared-memory tiles
// ROWS x COLS elements in chunks of 16 bytes; a row's chunks are permuted so that the eight rows of a matrix fragment, and eight
// neighbouring chunks of a row, lie in different banks.
template <int COLS, int ES>
struct Tile {
  static constexpr int CHUNKS = COLS * ES / 16, PER = 16 / ES;   // chunks of a row, elements of a chunk
  __device__ static __forceinline__ int chunk(int row, int c) {
    if constexpr (CHUNKS >= 8) return row * CHUNKS + (c ^ (row & 7));
    else return row * CHUNKS + (c ^ ((row / (8 / CHUNKS)) & (CHUNKS - 1)));
  }
  __device__ static __forceinline__ uint32_t at(uint32_t base, int row, int c) { return base + 16 * chunk(row, c); }
};

template <int ES>
__device__ __forceinline__ constexpr int PerChunk() { return 16 / ES; }

// how a matrix's rows can be read: 16 bytes at a time, 8, or element by element
enum { kBy16 = 0, kBy8 = 1, kByElement = 2 };

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// `bytes` of 16, the others zero
__device__ __forceinline__ void cp16_sized(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 8 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

// One chunk: elements [e, e + PER) of a row of which `valid` exist; the others become zero.
template <int ES>
__device__ __forceinline__ void load_chunk(uint32_t dst, const void* row, int e, int valid, int by) {
  constexpr int PER = 16 / ES;
  const uint8_t* p = static_cast<const uint8_t*>(row) + (long long)e * ES;
  if (by == kBy16) {
    cp16(dst, e < valid ? p : row, e < valid);
  } else if (by == kBy8) {
    cp8(dst, e < valid ? p : row, e < valid);
    cp8(dst + 8, e + PER / 2 < valid ? p + 8 : row, e + PER / 2 < valid);
  } else {
    uint32_t w[4];
    if constexpr (ES == 2) {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < 4; i++)
        w[i] = (e + 2 * i < valid ? (uint32_t)h[2 * i] : 0u) | (e + 2 * i + 1 < valid ? (uint32_t)h[2 * i + 1] << 16 : 0u);
    } else {
      const uint32_t* h = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = e + i < valid ? h[i] : 0u;
    }
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
  }
}

// Fragments of the second operand for sixteen columns (two n8 tiles) and a k16 step: b[tile][half][term]. ALONG: the tile's rows are
// the product's columns, the contraction runs along them; otherwise its rows are the contraction.
template <typename PT, int TERMS, int COLS, bool ALONG>
__device__ __forceinline__ void load_b(uint32_t base, int col0, int k0, uint32_t (&b)[2][2][TERMS]) {
  typedef Tile<COLS, sizeof(PT)> W;
  const int l = threadIdx.x & 31;
  if constexpr (sizeof(PT) == 2) {
    uint32_t r[4];
    if constexpr (ALONG) ldsm(r, W::at(base, col0 + (l & 7) + ((l >> 4) & 1) * 8, k0 / 8 + ((l >> 3) & 1)));
    else ldsm_trans(r, W::at(base, k0 + (l & 15), col0 / 8 + (l >> 4)));
    b[0][0][0] = r[0]; b[0][1][0] = r[1]; b[1][0][0] = r[2]; b[1][1][0] = r[3];
  } else {
    const int i = l >> 2, q = l & 3;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float f0, f1;
        if constexpr (ALONG) {
          const uint32_t p = W::at(base, col0 + 8 * t + i, (k0 + 8 * h) / 4 + (q >> 1)) + 8 * (q & 1);
          asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];\n" : "=f"(f0), "=f"(f1) : "r"(p) : "memory");
        } else {
          const int k = k0 + 8 * h + 2 * q, c = (col0 + 8 * t) / 4 + (i >> 2);
          asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(f0) : "r"(W::at(base, k, c) + 4 * (i & 3)) : "memory");
          asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(f1) : "r"(W::at(base, k + 1, c) + 4 * (i & 3)) : "memory");
        }
        split<TERMS, true>(f0, f1, b[t][h]);   // (an infinite float32 parameter makes NaN)
      }
  }
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
      // the groups of up to 128 entries at once; longer calls in turns
      const int n = (int)a.g.n;
      const int mine = group_of(a.g, tile);
      int before = 0, rows = 0;
      for (int b0 = 0; b0 < n; b0 += 128) {
        int key[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int b = b0 + 32 * k + tid;
          key[k] = b < n ? group_of(a.g, b) : -2;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int b = b0 + 32 * k + tid, left = tile - (b0 + 32 * k);   // entries of these 32 that lie ahead of the cluster's own
          const uint32_t m = __ballot_sync(0xffffffffu, key[k] == mine), ahead = left <= 0 ? 0u : left >= 32 ? ~0u : (1u << left) - 1u;
          before += __popc(m & ahead);
          const uint32_t from = m & ~ahead;
          const int at = rows + __popc(from & ((1u << tid) - 1u));
          if ((from >> tid & 1) && at < MT) s_row[at] = b;
          rows = min(MT, rows + __popc(from));
        }
        if (b0 + 128 > tile && (before % MT != 0 || rows == MT)) break;
      }
      if (before % MT != 0) rows = 0;   // another cluster's
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

// Rows without an adapter: columns [lo, hi) of the base as they are, zeros without one. A warp a row, eight accesses of a lane on their
// way at once, of 16 bytes wherever the row starts (as long as base and out start alike).
static __device__ __noinline__ void copy_rows(const uint16_t* base, long long base_stride, uint16_t* out, long long out_stride, const int* s_row, int rows, int lo,
                                       int hi) {
  const int lane = threadIdx.x & 31;
  for (int m = threadIdx.x >> 5; m < rows; m += kThreads / 32) {
    const uint16_t* p = base == nullptr ? nullptr : base + (long long)s_row[m] * base_stride + lo;
    uint16_t* o = out + (long long)s_row[m] * out_stride + lo;
    const int n = hi - lo;
    const bool alike = p == nullptr || ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(o)) & 15) == 0;
    const int head = alike ? min(n, (int)((16 - (reinterpret_cast<uintptr_t>(o) & 15)) & 15) / 2) : n, body = (n - head) / 8;
    auto some = [&](auto* to, const auto* from, int count) {
      for (int v0 = lane; v0 < count; v0 += 256) {
        typename std::remove_reference<decltype(*to)>::type u[8] = {};
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (v0 + 32 * k < count && base != nullptr) u[k] = from[v0 + 32 * k];
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (v0 + 32 * k < count) to[v0 + 32 * k] = u[k];
      }
    };
    some(o, p, head);
    some(reinterpret_cast<uint4*>(o + head), reinterpret_cast<const uint4*>(p + head), body);
    some(o + head + 8 * body, p + head + 8 * body, n - head - 8 * body);
  }
}

// ---------------------------------------------------------------------------------------------------- both products
template <typename PT, bool BWD, int RT, int MT>
struct Shape {
  static constexpr int RP = 16 * RT, PS = sizeof(PT);
  // A warp has MW sixteens of rows, so that a weight fragment (and the split of a float32 one) serves all of them; KS warps share
  // their contraction. float32, 4096 rows, K 4096, N 14336, rank 16: MW 1, 2, 4 forward 86, 75, 80 us, backward 84, 67, 62.
  static constexpr int MW = MT == 16 ? 1 : PS == 4 ? (RT == 8 ? 1 : RT == 4 || !BWD ? 2 : 4) : RT >= 4 ? 1 : 2, WM = MT / 16 / MW, KS = kThreads / 32 / WM;
  static constexpr int KB = MT == 16 ? (RT <= 2 && PS == 2 ? 256 : 128) : RT <= 2 ? 128 : 64;   // contraction of a stage of the first product
  static constexpr int CW = MT == 16 ? (RT <= 2 && PS == 2 ? 32 : 16) : KS == 8 || RT == 4 && PS == 4 ? 16 : 32;   // columns of a warp in a stage of the second
  static constexpr int NB = CW * KS;
  static constexpr int X = MT * KB * 2, W1 = RP * KB * PS, Y = MT * NB * 2, W2 = NB * RP * PS;
  static constexpr int STAGE = X + W1 > Y + W2 ? X + W1 : Y + W2;
  static constexpr int UP = RP + 8;
  // room for the sums of some of the warps, and then for the CTA's part of u, in one place
  static constexpr int SLOTS = MT == 16 ? 4 : KS == 8 ? 2 : 1, SLOT = 16 * MW * RP;
  static constexpr int RED = SLOTS * WM * SLOT * 4, PART = MT * RP * 4, SUM = RED > PART ? RED : PART, U = 2 * MT * UP * 2;
  static constexpr int REST = SUM + U + MT * 8 + 16;
  // two CTAs of an SM where at least three stages of each fit, else one
  static constexpr int TWO = (112 * 1024 - REST) / STAGE, ONE = (224 * 1024 - REST) / STAGE;
  static constexpr int STAGES = TWO >= 3 ? (TWO > 8 ? 8 : TWO) : ONE > 6 ? 6 : ONE;
  static constexpr int SMEM = STAGES * STAGE + REST, CTAS = TWO >= 3 ? 2 : 1;
  static_assert(STAGES >= 2 && SMEM <= 227 * 1024, "does not fit");
};

// One matrix of a stage: ROWS x COLS elements, chunks dealt out to the threads; with a thread's chunks a fixed number of rows apart.
template <int ROWS, int COLS, int ES>
struct Deal {
  typedef Tile<COLS, ES> T;
  static constexpr int CHUNKS = ROWS * T::CHUNKS, EACH = (CHUNKS + kThreads - 1) / kThreads, STEP = kThreads / T::CHUNKS;
  static constexpr bool ALL = CHUNKS % kThreads == 0;   // every thread has EACH chunks
  static_assert(STEP % 8 == 0, "the permutation of a row's chunks would change");
  __device__ static __forceinline__ int row() { return threadIdx.x / T::CHUNKS; }
  __device__ static __forceinline__ int chunk() { return threadIdx.x % T::CHUNKS; }
  __device__ static __forceinline__ bool has(int t) { return ALL || (int)threadIdx.x + t * kThreads < CHUNKS; }
};

// Forward, the second product's columns: a warp's tile of CW columns lies in shared memory so that a lane comes to hold CW / 4
// neighbouring columns of a row of the output. Column n of the stage goes to this row.
template <int CW>
__device__ __forceinline__ int place_of(int n) {
  if constexpr (CW == 32) return (n & ~31) | (n >> 1 & 3) << 3 | (n >> 3 & 3) << 1 | (n & 1);
  else return (n & ~15) | (n >> 1 & 1) << 3 | (n >> 2 & 3) << 1 | (n & 1);
}

// FAST: all rows that are read, and the forward pass' outputs, are whole aligned groups of 16 bytes.
template <typename XT, typename PT, bool BWD, int RT, int MT, bool FAST>
__global__ void __launch_bounds__(kThreads, Shape<PT, BWD, RT, MT>::CTAS) tile_kernel(const LoraArgs a) {
  typedef Shape<PT, BWD, RT, MT> S;
  typedef typename std::conditional<sizeof(PT) == 4, bf16, XT>::type CT;
  constexpr int RP = S::RP, UP = S::UP, KS = S::KS, WM = S::WM, MW = S::MW, KB = S::KB, NB = S::NB, CW = S::CW, PS = S::PS;
  constexpr int XN = RowTerms<XT, CT>::N, P1 = PS == 4 ? 3 : 1, P2 = PS == 4 ? 2 : 1, UT = PS == 4 ? 3 : 2;
  constexpr int W1C = BWD ? RP : KB, W2C = BWD ? NB : RP;   // columns of the stages' weight tiles
  typedef Deal<MT, KB, 2> XD;
  typedef Deal<BWD ? KB : RP, W1C, PS> W1D;
  typedef Deal<BWD ? RP : NB, W2C, PS> W2D;
  typedef Deal<MT, NB, 2> YD;
  typedef typename XD::T XTile;
  typedef typename YD::T YTile;
  extern __shared__ __align__(16) uint8_t smem[];
  float* s_red = reinterpret_cast<float*>(smem + S::STAGES * S::STAGE);   // sums of half of the warps
  float* s_part = s_red;                                                  // then [MT][RP]: this CTA's part of u
  uint16_t* s_u = reinterpret_cast<uint16_t*>(s_red + S::SUM / 4);        // [2][MT][UP]: u as two terms
  float* s_factor = reinterpret_cast<float*>(s_u + S::U / 2);             // [MT]
  int* s_row = reinterpret_cast<int*>(s_factor + MT);                     // [MT]
  int* s_info = s_row + MT;
  wait_for_launch();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, i = lane >> 2, q = lane & 3;
  const int m0 = warp % WM * 16 * MW, ks = warp / WM;   // the warp's first row, its share of the others' work
  const TileAt t = find_tile<MT>(a, blockIdx.x / C, s_row, s_info);
  if (t.rows == 0) return;   // (the whole cluster)
  const int n_chunks = (a.c1 - a.c0 + NB - 1) / NB;
  const int lo = a.c0 + n_chunks * rank / C * NB;
  const int hi = min(a.c1, a.c0 + n_chunks * (rank + 1) / C * NB);
  if (t.group < 0) {
    if (a.out_f32) {
      for (int m = warp; m < t.rows; m += kThreads / 32)
        for (int c = lo + lane; c < hi; c += 32) static_cast<float*>(a.out)[(long long)s_row[m] * a.out_stride + c - a.c0] = 0.f;
    } else if (a.out != nullptr && a.out != a.base) {
      copy_rows(static_cast<const uint16_t*>(a.base), a.base_stride, static_cast<uint16_t*>(a.out), a.out_stride, s_row, t.rows, lo, hi);
    }
    if (a.shrink && a.u != nullptr && rank == 0)
      for (int v = tid; v < t.rows * UT * a.ru; v += kThreads)
        a.u[((long long)(v / a.ru % UT) * a.g.n + s_row[v / (a.ru * UT)]) * a.ru + v % a.ru] = 0;
    return;
  }
  const float factor = factor_of(a.g, t.group);
  const PT* w1 = static_cast<const PT*>(a.w1) + (long long)t.group * a.r * a.D1;
  const PT* w2 = static_cast<const PT*>(a.w2) + (long long)t.group * a.r * a.D2;
  const int blocks = a.shrink ? (a.D1 + KB - 1) / KB : 0;
  const int b0 = blocks * rank / C, n1 = blocks * (rank + 1) / C - b0;
  const int n2 = a.out != nullptr ? (hi - lo + NB - 1) / NB : 0;
  const bool staged = !BWD && (FAST || a.by_out != kByElement);   // the base's rows come with the weights
  const uint32_t ring = smem_at(smem);

  // This thread's chunks: where they come from in the first stage of each product, and where they go. A row or rank that does not
  // exist is read as zero bytes of one that does.
  const XT* xp[XD::EACH];
  bool x_there[XD::EACH];
#pragma unroll
  for (int k = 0; k < XD::EACH; k++) {
    const int e = s_row[XD::row() + k * XD::STEP];
    x_there[k] = e >= 0;
    xp[k] = static_cast<const XT*>(a.in) + (long long)(e < 0 ? 0 : a.in_div == 1 ? e : (int)((unsigned)e / (unsigned)a.in_div)) * a.in_stride + b0 * KB;
  }
  const uint32_t x_to = XTile::at(0, XD::row(), XD::chunk()), w1_to = S::X + W1D::T::at(0, W1D::row(), W1D::chunk());
  const uint32_t y_to = YTile::at(0, YD::row(), YD::chunk());
  // rows of the first weight matrix: the ranks (forward), or the contraction
  const long long l1 = BWD ? a.r : a.D1, l2 = BWD ? a.D2 : a.r;
  const PT* p1 = w1 + (BWD ? (long long)b0 * KB * l1 : (long long)b0 * KB);
  const PT* p2 = w2 + (BWD ? (long long)lo : (long long)lo * l2);
  // Stages that have all of their contraction, or columns, by a shorter way. (Not small 16-bit ranks, whose loop is longer with both:
  // 32768 entries of rank 16 98 us, with it 102; rank 64 or float32 the other way round, 75 to 77 and 170 to 183.)
  constexpr bool QUICK = FAST && (PS == 4 || RT >= 4);
  const int full1 = QUICK ? min(n1, a.D1 / KB - b0) : 0, full2 = QUICK ? (hi - lo) / NB : 0;
  // what the whole stages' weights are read by: of the ranks, those that exist
  const PT* q1 = p1 + (!BWD && W1D::row() >= a.r ? 0 : W1D::row()) * l1 + (BWD && PerChunk<PS>() * W1D::chunk() >= a.r ? 0 : PerChunk<PS>() * W1D::chunk());
  const PT* q2 = p2 + (BWD && W2D::row() >= a.r ? 0 : W2D::row()) * l2 + (!BWD && PerChunk<PS>() * W2D::chunk() >= a.r ? 0 : PerChunk<PS>() * W2D::chunk());

  int next = 0, into = 0;   // the stage to be fetched, its place in the ring
  auto fetch = [&]() {
    const uint32_t at = ring + into * S::STAGE;
    into = into + 1 == S::STAGES ? 0 : into + 1;
    if (QUICK && next < full1) {
#pragma unroll
      for (int k = 0; k < XD::EACH; k++)
        cp16_sized(at + x_to + k * XD::STEP * XTile::CHUNKS * 16, xp[k] + (next * KB + PerChunk<2>() * XD::chunk()), x_there[k] ? 16 : 0);
      const PT* q = q1 + (BWD ? (long long)next * KB * l1 : (long long)next * KB);
#pragma unroll
      for (int k = 0; k < W1D::EACH; k++) {
        const bool there = BWD ? PerChunk<PS>() * W1D::chunk() < a.r : W1D::row() + k * W1D::STEP < a.r;
        if (W1D::has(k)) cp16_sized(at + w1_to + k * W1D::STEP * W1D::T::CHUNKS * 16, BWD || there ? q + k * (W1D::STEP * l1) : q1, there ? 16 : 0);
      }
    } else if (next < n1) {
      const int k0 = next * KB, left = a.D1 - b0 * KB - k0;   // of the contraction
#pragma unroll
      for (int k = 0; k < XD::EACH; k++) {
        const int c = PerChunk<2>() * XD::chunk();
        load_chunk<2>(at + x_to + k * XD::STEP * XTile::CHUNKS * 16, x_there[k] ? xp[k] + k0 : a.in, c, x_there[k] ? left : 0, FAST ? kBy16 : a.by_in);
      }
#pragma unroll
      for (int k = 0; k < W1D::EACH; k++) {
        if (!W1D::has(k)) continue;
        const int m = W1D::row() + k * W1D::STEP, c = PerChunk<PS>() * W1D::chunk();
        const PT* row = p1 + m * l1 + (BWD ? (long long)k0 * l1 : (long long)k0);
        const bool there = BWD ? m < left : m < a.r;
        load_chunk<PS>(at + w1_to + k * W1D::STEP * W1D::T::CHUNKS * 16, there ? row : w1, c, there ? (BWD ? a.r : left) : 0, FAST ? kBy16 : a.by_w1);
      }
    } else if (next < n1 + n2) {
      const int c0 = (next - n1) * NB, left = hi - lo - c0;   // of the columns
      if (QUICK && next - n1 < full2) {
        const PT* q = q2 + (BWD ? (long long)c0 : (long long)c0 * l2);
#pragma unroll
        for (int k = 0; k < W2D::EACH; k++) {
          const int m = W2D::row() + k * W2D::STEP;
          const bool there = BWD ? m < a.r : PerChunk<PS>() * W2D::chunk() < a.r;
          const uint32_t to = W2D::STEP % CW == 0 ? W2D::T::at(0, BWD ? W2D::row() : place_of<CW>(W2D::row()), W2D::chunk()) + k * W2D::STEP * W2D::T::CHUNKS * 16
                                                  : W2D::T::at(0, BWD ? m : place_of<CW>(m), W2D::chunk());
          if (W2D::has(k)) cp16_sized(at + S::Y + to, !BWD || there ? q + k * (W2D::STEP * l2) : q2, there ? 16 : 0);
        }
      } else {
#pragma unroll
        for (int k = 0; k < W2D::EACH; k++) {
          if (!W2D::has(k)) continue;
          const int m = W2D::row() + k * W2D::STEP, c = PerChunk<PS>() * W2D::chunk();
          const PT* row = p2 + m * l2 + (BWD ? (long long)c0 : (long long)c0 * l2);
          const bool there = BWD ? m < a.r : m < left;
          load_chunk<PS>(at + S::Y + W2D::T::at(0, BWD ? m : place_of<CW>(m), W2D::chunk()), there ? row : w2, c, there ? (BWD ? left : a.r) : 0,
                         FAST ? kBy16 : a.by_w2);
        }
      }
      if (staged) {
        const int c = c0 + PerChunk<2>() * YD::chunk();
#pragma unroll
        for (int k = 0; k < YD::EACH; k++) {
          if (!YD::has(k)) continue;
          const int e = s_row[YD::row() + k * YD::STEP];
          const bool there = e >= 0 && c < hi - lo;
          const uint32_t to = at + y_to + k * YD::STEP * YTile::CHUNKS * 16;
          const XT* row = static_cast<const XT*>(a.base) + (there ? (long long)e * a.base_stride + lo : 0);
          if (FAST || a.by_out == kBy16) cp16_sized(to, row + (there ? c : 0), there ? 16 : 0);
          else load_chunk<2>(to, row, c, there ? hi - lo : 0, kBy8);
        }
      } else if (!BWD && !FAST && tid < MT && s_row[tid] >= 0 && c0 < hi - lo) {
        // rows that start anywhere are read by column when the stage is multiplied: from L2 then
        const XT* p = static_cast<const XT*>(a.base) + (long long)s_row[tid] * a.base_stride + lo + c0;
        const uintptr_t from = reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)15, to = (reinterpret_cast<uintptr_t>(p + min(NB, hi - lo - c0)) + 15) & ~(uintptr_t)15;
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"(__cvta_generic_to_global(reinterpret_cast<const void*>(from))), "r"((uint32_t)(to - from)) : "memory");
      }
    }
    next++;
    cp_commit();
  };
#pragma unroll 1
  for (int s = 0; s < S::STAGES - 1; s++) fetch();
  uint32_t at = ring;   // the stage that is next to be multiplied
  auto advance = [&]() { at = at + S::STAGE == ring + S::STAGES * S::STAGE ? ring : at + S::STAGE; };

  if (a.shrink) {
    float acc[MW][2 * RT][4];
#pragma unroll
    for (int m = 0; m < MW; m++)
#pragma unroll
      for (int n = 0; n < 2 * RT; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) acc[m][n][k] = 0.f;
#pragma unroll 1
    for (int s = 0; s < n1; s++) {
      cp_wait<S::STAGES - 2>();
      __syncthreads();
      fetch();
#pragma unroll
      for (int k = 0; k < KB / 16 / KS; k++) {
        const int step = ks + k * KS;
        uint32_t xa[MW][XN][4];
#pragma unroll
        for (int m = 0; m < MW; m++) {
          if (m > 0 && m0 + 16 * m >= t.rows) break;
          uint32_t raw[4];
          ldsm(raw, XTile::at(at, m0 + 16 * m + (lane & 15), 2 * step + (lane >> 4)));
          RowTerms<XT, CT>::get(raw, xa[m]);
        }
#pragma unroll
        for (int n = 0; n < RT; n++) {
          uint32_t b[2][2][P1];
          load_b<PT, P1, W1C, !BWD>(at + S::X, 16 * n, 16 * step, b);
#pragma unroll
          for (int m = 0; m < MW; m++) {
            if (m > 0 && m0 + 16 * m >= t.rows) break;
#pragma unroll
            for (int h = 0; h < 2; h++) {
              if constexpr (PS == 4) {
                // The tensor cores cut off what a sum has below its last bit. Where float32 results are wanted, a step's products
                // are added up by themselves and then, rounded, to the whole.
                float part[4];
                mma_terms_first<XN, P1>(part, xa[m], b[h][0], b[h][1]);
#pragma unroll
                for (int c = 0; c < 4; c++) acc[m][2 * n + h][c] += part[c];
              } else {
                mma_terms<XN, P1, CT>(acc[m][2 * n + h], xa[m], b[h][0], b[h][1]);
              }
            }
          }
        }
      }
      advance();
    }
    // the warps' parts, halves onto halves, as many at a time as there is room for
#pragma unroll
    for (int h = KS / 2; h > 0; h >>= 1)
#pragma unroll
      for (int b = 0; b < h; b += S::SLOTS) {
        float* mine = s_red + (warp % WM * S::SLOTS + (ks >= h ? ks - h - b : ks - b)) * S::SLOT;
        if (ks >= h + b && ks < h + b + S::SLOTS && ks < 2 * h) {
#pragma unroll
          for (int m = 0; m < MW; m++)
#pragma unroll
            for (int n = 0; n < 2 * RT; n++)
              *reinterpret_cast<float4*>(mine + ((m * 2 * RT + n) * 32 + lane) * 4) = make_float4(acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]);
        }
        __syncthreads();
        if (ks >= b && ks < b + S::SLOTS && ks < h) {
#pragma unroll
          for (int m = 0; m < MW; m++)
#pragma unroll
            for (int n = 0; n < 2 * RT; n++) {
              const float4 v = *reinterpret_cast<const float4*>(mine + ((m * 2 * RT + n) * 32 + lane) * 4);
              acc[m][n][0] += v.x;
              acc[m][n][1] += v.y;
              acc[m][n][2] += v.z;
              acc[m][n][3] += v.w;
            }
        }
        __syncthreads();
      }
    if (ks == 0) {
#pragma unroll
      for (int m = 0; m < MW; m++)
#pragma unroll
        for (int n = 0; n < 2 * RT; n++)
#pragma unroll
          for (int h = 0; h < 2; h++)
            *reinterpret_cast<float2*>(s_part + (m0 + 16 * m + i + 8 * h) * RP + 8 * n + 2 * q) = make_float2(acc[m][n][2 * h], acc[m][n][2 * h + 1]);
    }
    if (C > 1) cluster.sync();
    else __syncthreads();
  }
  // u of the whole contraction, saved as bf16 terms and as two terms for the second product. A warp a row at a time.
#pragma unroll 1
  for (int m = warp; m < MT; m += kThreads / 32) {
    float v[(RP + 31) / 32], most = 0.f;
    const int row = s_row[m];
#pragma unroll
    for (int b = 0; b < (RP + 31) / 32; b++) {
      const int j = 32 * b + lane;
      v[b] = 0.f;
      if (j < a.r && row >= 0) {
        if (a.shrink) {
          if (C == 1) {
            v[b] = s_part[m * RP + j];
          } else {
            float p[8];   // all on their way at once, added in the order of the CTAs
#pragma unroll
            for (int c = 0; c < 8; c++) p[c] = c < C ? *cluster.map_shared_rank(s_part + m * RP + j, c) : 0.f;
#pragma unroll
            for (int c = 0; c < 8; c++) v[b] += p[c];
          }
          if (a.scale_u) v[b] *= factor;
        } else {
#pragma unroll
          for (int n = UT - 1; n >= 0; n--) v[b] += __uint_as_float((uint32_t)a.u[((long long)n * a.g.n + row) * a.ru + j] << 16);
        }
      }
      if (j < a.ru && row >= 0 && a.shrink && a.u != nullptr && rank == m % C) {
        uint32_t p[UT];
        split<UT>(v[b], 0.f, p);
#pragma unroll
        for (int n = 0; n < UT; n++) a.u[((long long)n * a.g.n + row) * a.ru + j] = (uint16_t)p[n];
      }
      most = fmaxf(most, fabsf(v[b]));
    }
    float f = 1.f;
    if constexpr (std::is_same<CT, __half>::value) {
      // fp16 terms: the row's largest comes to lie in [2^14, 2^15), so that parts down to 2^-23 of it still have 16 bits in their two
      // terms (fp16's steps end at 2^-24; the largest in [1, 2) left parts of 2^-20 with five)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (most > 0.f && most < INFINITY) f = __uint_as_float((unsigned)max(1, (int)(__float_as_uint(most) >> 23) - 14) << 23);
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
        uint32_t p[2];
        split<2>(v[b], 0.f, p);
        s_u[m * UP + j] = (uint16_t)p[0];
        s_u[(MT + m) * UP + j] = (uint16_t)p[1];
      }
    }
    if (lane == 0) s_factor[m] = a.scale_u ? f : f * factor;
  }
  __syncthreads();
  if (a.shrink && C > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");

  const uint32_t u_at = smem_at(s_u) + ((m0 + (lane & 15)) * UP + 8 * (lane >> 4)) * 2;
  const int cw = CW * ks;
#pragma unroll 1
  for (int s = 0; s < n2; s++) {
    cp_wait<S::STAGES - 2>();
    __syncthreads();
    fetch();
    const int c0 = lo + s * NB;
    if (m0 < t.rows && c0 + cw < hi) {
      // forward, rows that start anywhere: eight rows at a time, a column a lane, so that an access is a run of a row; all at once, and
      // what lies outside is read from the tile's first row or the last column instead
      constexpr int TURN = 32 / CW;   // rows at once
      const bool anywhere = !BWD && !FAST && a.by_out == kByElement;
      const int own = c0 + cw + (lane & (CW - 1));
      uint16_t y[MW][2][8 / TURN];
      if (anywhere) {
        const uint16_t* p = static_cast<const uint16_t*>(a.base) + min(own, hi - 1);
#pragma unroll
        for (int m = 0; m < MW; m++)
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < 8 / TURN; r++) {
              const int e = s_row[m0 + 16 * m + 8 * h + r * TURN + lane / CW];
              y[m][h][r] = p[(long long)(e < 0 ? s_row[0] : e) * a.base_stride];
            }
      }
      float acc[MW][CW / 8][4];
#pragma unroll
      for (int m = 0; m < MW; m++)
#pragma unroll
        for (int n = 0; n < CW / 8; n++)
#pragma unroll
          for (int k = 0; k < 4; k++) acc[m][n][k] = 0.f;
#pragma unroll
      for (int k = 0; k < RT; k++) {
        uint32_t b[CW / 16][2][2][P2];
#pragma unroll
        for (int n = 0; n < CW / 16; n++) load_b<PT, P2, W2C, !BWD>(at + S::Y, cw + 16 * n, 16 * k, b[n]);
#pragma unroll
        for (int m = 0; m < MW; m++) {
          if (m > 0 && m0 + 16 * m >= t.rows) break;
          uint32_t ua[2][4];
#pragma unroll
          for (int n = 0; n < 2; n++) ldsm(ua[n], u_at + ((n * MT + 16 * m) * UP + 16 * k) * 2);
#pragma unroll
          for (int n = 0; n < CW / 8; n++) mma_terms<2, P2, CT>(acc[m][n], ua, b[n / 2][n % 2][0], b[n / 2][n % 2][1]);
        }
      }
#pragma unroll
      for (int m = 0; m < MW; m++) {
        if (m > 0 && m0 + 16 * m >= t.rows) break;
        const int m1 = m0 + 16 * m + i;
        const int row[2] = {s_row[m1], s_row[m1 + 8]};
        const float f[2] = {s_factor[m1], s_factor[m1 + 8]};
        if constexpr (!BWD) {
          // columns c0 + cw + (CW / 4) q .. of two rows
          constexpr int HOLD = CW / 4;
          const int col = c0 + cw + HOLD * q;
          const float (&c)[CW / 8][4] = acc[m];
          if (FAST || a.by_out != kByElement) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
              if (row[h] < 0 || col >= hi) continue;
              XT* o = static_cast<XT*>(a.out) + (long long)row[h] * a.out_stride + col;
              uint32_t v[HOLD / 2];
              const uint32_t p = YTile::at(at, m1 + 8 * h, (cw + HOLD * q) / 8) + (HOLD == 4 ? 8 * (q & 1) : 0);
              if constexpr (HOLD == 8) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(p) : "memory");
              else asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];\n" : "=r"(v[0]), "=r"(v[1]) : "r"(p) : "memory");
#pragma unroll
              for (int n = 0; n < HOLD / 2; n++) {
                const XT* y = reinterpret_cast<const XT*>(&v[n]);
                v[n] = round_pair(fmaf(f[h], c[n][2 * h], to_float(y[0])), fmaf(f[h], c[n][2 * h + 1], to_float(y[1])), XT());
              }
              if constexpr (HOLD == 8) {
                if (FAST || a.by_out == kBy16) {
                  *reinterpret_cast<uint4*>(o) = make_uint4(v[0], v[1], v[2], v[3]);
                } else {
                  *reinterpret_cast<uint2*>(o) = make_uint2(v[0], v[1]);
                  if (col + 4 < hi) *reinterpret_cast<uint2*>(o + 4) = make_uint2(v[2], v[3]);
                }
              } else {
                *reinterpret_cast<uint2*>(o) = make_uint2(v[0], v[1]);
              }
            }
          } else {
            // through shared memory in float32
            float* tile = reinterpret_cast<float*>(smem + (at - ring)) + warp * 8 * CW;
            static_assert(kThreads / 32 * 8 * CW * 4 <= S::Y, "the stage's room for rows");
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
              for (int n = 0; n < CW / 8; n++) *reinterpret_cast<float2*>(tile + i * CW + HOLD * q + 2 * n) = make_float2(f[h] * c[n][2 * h], f[h] * c[n][2 * h + 1]);
              __syncwarp();
#pragma unroll
              for (int r = 0; r < 8 / TURN; r++) {
                const int e = s_row[m0 + 16 * m + 8 * h + r * TURN + lane / CW];
                if (e >= 0 && own < hi) static_cast<XT*>(a.out)[(long long)e * a.out_stride + own] = XT(to_float(*reinterpret_cast<const XT*>(&y[m][h][r])) + tile[(r * TURN + lane / CW) * CW + (lane & (CW - 1))]);
              }
              __syncwarp();
            }
          }
        } else if (a.out_f32) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            if (row[h] < 0) continue;
            float* o = static_cast<float*>(a.out) + (long long)row[h] * a.out_stride - a.c0;
#pragma unroll
            for (int n = 0; n < CW / 8; n++) {
              const int col = c0 + cw + 8 * n + 2 * q;
              if (a.out_stride % 2 == 0 && col + 1 < hi) *reinterpret_cast<float2*>(o + col) = make_float2(f[h] * acc[m][n][2 * h], f[h] * acc[m][n][2 * h + 1]);
              else
#pragma unroll
                for (int k = 0; k < 2; k++)
                  if (col + k < hi) o[col + k] = f[h] * acc[m][n][2 * h + k];
            }
          }
        } else if (a.by_out == kBy16) {
          // through the stage's room for rows, from where whole chunks leave
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int n = 0; n < CW / 8; n++)
              asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(YTile::at(at, m1 + 8 * h, cw / 8 + n) + 4 * q), "r"(round_pair(f[h] * acc[m][n][2 * h], f[h] * acc[m][n][2 * h + 1], XT())) : "memory");
          __syncwarp();
          constexpr int EACH = CW / 8;   // chunks of a row
#pragma unroll
          for (int c = lane; c < 16 * EACH; c += 32) {
            const int mr = m0 + 16 * m + c / EACH, ch = cw / 8 + c % EACH, e = s_row[mr], col = c0 + 8 * ch;
            if (e < 0 || col >= hi) continue;
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(YTile::at(at, mr, ch)) : "memory");
            *reinterpret_cast<uint4*>(static_cast<XT*>(a.out) + (long long)e * a.out_stride + col) = v;
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            if (row[h] < 0) continue;
            XT* o = static_cast<XT*>(a.out) + (long long)row[h] * a.out_stride;
#pragma unroll
            for (int n = 0; n < CW / 8; n++)
#pragma unroll
              for (int k = 0; k < 2; k++)
                if (c0 + cw + 8 * n + 2 * q + k < hi) o[c0 + cw + 8 * n + 2 * q + k] = XT(f[h] * acc[m][n][2 * h + k]);
          }
        }
      }
    }
    advance();
  }
  cp_wait<0>();
  // nobody leaves while its part of u may still be read
  __syncthreads();
  if (a.shrink && C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// A kernel's shared memory, asked for once on each device.
template <typename Kernel>
cudaError_t allow_smem(Kernel kern, int bytes, bool (&done)[16]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev >= 0 && dev < 16 && done[dev])) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 16) done[dev] = true;
  return e;
}

template <typename XT, typename PT, bool BWD, int RT, int MT, bool FAST>
cudaError_t launch_tile(const LoraArgs& a, int cluster, cudaStream_t st) {
  constexpr int smem = Shape<PT, BWD, RT, MT>::SMEM;
  auto kern = tile_kernel<XT, PT, BWD, RT, MT, FAST>;
  if (smem > 48 * 1024) {
    static bool done[16] = {};
    const cudaError_t e = allow_smem(kern, smem, done);
    if (e != cudaSuccess) return e;
  }
  return launch(kern, dim3((unsigned)(a.n_clusters * cluster)), kThreads, smem, cluster, st, a);
}
template <typename XT, typename PT, bool BWD, int RT>
cudaError_t launch_mt(const LoraArgs& a, int mt, int cluster, cudaStream_t st) {
  if (a.by_in == kBy16 && a.by_w1 == kBy16 && a.by_w2 == kBy16 && (BWD || a.by_out == kBy16))
    return mt == 16 ? launch_tile<XT, PT, BWD, RT, 16, true>(a, cluster, st) : launch_tile<XT, PT, BWD, RT, 64, true>(a, cluster, st);
  return mt == 16 ? launch_tile<XT, PT, BWD, RT, 16, false>(a, cluster, st) : launch_tile<XT, PT, BWD, RT, 64, false>(a, cluster, st);
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
