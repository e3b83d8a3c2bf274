// Low-rank adapters: the order of the rows by adapter (plan), the gradients of the adapters' matrices, the sum over a token's
// slots, and which launches a call takes. The products of the rows are in kq_lora.cuh.
#include <algorithm>

#include "kq_lora.cuh"

namespace kq {
namespace lora {
namespace {

// ---------------------------------------------------------------------------------------------------- plan
constexpr int kPlanThreads = 512;

// One CTA per group, the last for the entries without one. It reads every entry's group: how many lie before its own, and its
// own in their order. No counters, nothing to clear, the same order each time. A warp has a run of neighbouring entries and reads
// four a lane at a time; the second pass, which places the group's own, has nothing to do for most of them. Tiles take the list's
// slots from start / height + group on, which no two groups share; slots that are left over hold none. 4072 entries of 128 groups 4.8 us;
// 32768 of 256 groups 27, most of it the 33 MB that the CTAs read from L2: the two launches below take those calls.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const LoraGroups g, int n_groups, int height, int* order, int* offsets, LoraTile* tiles) {
  wait_for_launch();
  constexpr int WARPS = kPlanThreads / 32;
  __shared__ int s_less[WARPS], s_same[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, mine = blockIdx.x;
  const int n = (int)g.n, each = ((n + WARPS - 1) / WARPS + 127) / 128 * 128;   // entries of a warp
  const int w0 = min(n, warp * each), w1 = min(n, w0 + each);
  const bool by4 = ((reinterpret_cast<uintptr_t>(g.experts) | (g.slots == 1 ? reinterpret_cast<uintptr_t>(g.ids) : 0)) & 15) == 0;
  // the keys of entries e .. e + 3, those past the warp's end none's
  auto keys = [&](int e, int (&k)[4]) {
    uint32_t x[4] = {0, 0, 0, 0};
    int id[4] = {0, 0, 0, 0};
    if (g.experts != nullptr) {
      if (by4 && e + 4 <= n) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(g.experts + e));
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (e + i < n) x[i] = g.experts[e + i];
      }
    }
    if (g.ids != nullptr) {
      if (g.slots == 1 && by4 && e + 4 <= n) {
        const int4 v = __ldg(reinterpret_cast<const int4*>(g.ids + e));
        id[0] = v.x; id[1] = v.y; id[2] = v.z; id[3] = v.w;
      } else if (e < n) {
        int token = (int)((unsigned)e / (unsigned)g.slots), slot = e - token * g.slots, a = g.ids[token];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          id[i] = a;
          if (++slot == g.slots && e + i + 1 < n) {
            slot = 0;
            a = g.ids[++token];
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
      k[i] = e + i >= w1 ? 0x7fffffff : (unsigned)id[i] < (unsigned)g.G && x[i] < (uint32_t)g.E ? id[i] * g.E + (int)x[i] : n_groups;
  };
  int less = 0, same = 0;
#pragma unroll 2
  for (int e = w0 + 4 * lane; e < w1; e += 128) {
    int k[4];
    keys(e, k);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      less += k[i] < mine;
      same += k[i] == mine;
    }
  }
  less = __reduce_add_sync(0xffffffffu, less);
  same = __reduce_add_sync(0xffffffffu, same);
  if (lane == 0) {
    s_less[warp] = less;
    s_same[warp] = same;
  }
  __syncthreads();
  int start = 0, count = 0, ahead = 0;
#pragma unroll
  for (int w = 0; w < WARPS; w++) {
    start += s_less[w];
    if (w < warp) ahead += s_same[w];
    count += s_same[w];
  }
  if (tid == 0) {
    offsets[mine] = start;
    if (mine == n_groups) offsets[mine + 1] = start + count;
  }
  // tiles as even as sixteen rows allow
  const int first = start / height + mine, slots = (start + count) / height + mine + 1 - first;
  const int n_tiles = (count + height - 1) / height;
  const int rows = n_tiles > 0 ? ((count + n_tiles - 1) / n_tiles + 15) / 16 * 16 : 0;
  for (int s = tid; s < slots; s += kPlanThreads) {
    const int at = s * rows;
    tiles[first + s] = LoraTile{mine == n_groups ? -1 : mine, start + at, s < n_tiles ? max(0, min(rows, count - at)) : 0, 0};
  }
  if (same == 0) return;
  int at = start + ahead;
  for (int e0 = w0; e0 < w1; e0 += 128) {
    const int e = e0 + 4 * lane;
    int k[4];
    keys(e, k);
    const int c = (k[0] == mine) + (k[1] == mine) + (k[2] == mine) + (k[3] == mine);
    if (!__any_sync(0xffffffffu, c != 0)) continue;
    int upto = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    int to = at + upto - c;
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (k[i] == mine) order[to++] = e + i;
    at += __shfl_sync(0xffffffffu, upto, 31);
  }
}

// The same in two launches, for many entries and fewer than kPlanKeys groups: CTAs count the groups of their chunk of the entries; then
// each adds up the chunks' counts - the chunks ahead of its own say where its entries go - and places them by their rank in the
// warp, the warp's in the chunk. 32768 entries of 256 groups 10 us, of one launch 27.
constexpr int kChunkThreads = 1024, kPlanKeys = 1024, kMostChunks = 128;

__device__ __forceinline__ int key_of(const LoraGroups& g, int e, int n_groups) {
  int id = 0;
  if (g.ids != nullptr) {
    id = g.ids[g.slots == 1 ? e : (int)((unsigned)e / (unsigned)g.slots)];
    if ((unsigned)id >= (unsigned)g.G) return n_groups;
  }
  const uint32_t x = g.experts != nullptr ? g.experts[e] : 0u;
  return x < (uint32_t)g.E ? id * g.E + (int)x : n_groups;
}

__global__ void __launch_bounds__(kChunkThreads) plan_count_kernel(const LoraGroups g, int n_groups, int per, int* counts) {
  wait_for_launch();
  __shared__ int s_count[kPlanKeys];
  const int n = (int)g.n, e0 = blockIdx.x * per, e1 = min(n, e0 + per);
  s_count[threadIdx.x] = 0;
  __syncthreads();
  for (int e = e0 + threadIdx.x; e < e1; e += kChunkThreads) atomicAdd(&s_count[key_of(g, e, n_groups)], 1);
  __syncthreads();
  if ((int)threadIdx.x <= n_groups) counts[blockIdx.x * (n_groups + 1) + threadIdx.x] = s_count[threadIdx.x];
}

__global__ void __launch_bounds__(kChunkThreads) plan_place_kernel(const LoraGroups g, int n_groups, int per, int height, const int* counts, int* order,
                                                                   int* offsets, LoraTile* tiles) {
  wait_for_launch();
  __shared__ int s_base[kPlanKeys], s_warp[32];
  extern __shared__ uint16_t s_rank[];   // [32 warps][n_groups + 1]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = (int)g.n, me = blockIdx.x, chunks = gridDim.x, keys = n_groups + 1;
  int count = 0, before = 0;   // thread = group
  if (tid < keys) {
#pragma unroll 8
    for (int c = 0; c < chunks; c++) {
      const int v = counts[c * keys + tid];
      count += v;
      before += c < me ? v : 0;
    }
  }
  int upto = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) s_warp[warp] = upto;
  __syncthreads();
  int start = upto - count;
  for (int w = 0; w < warp; w++) start += s_warp[w];
  s_base[tid] = start + before;
  if (tid < keys) {
    if (me == 0) {
      offsets[tid] = start;
      if (tid == n_groups) offsets[tid + 1] = start + count;
    }
    const int first = start / height + tid, slots = (start + count) / height + tid + 1 - first;
    const int n_tiles = (count + height - 1) / height;
    const int rows = n_tiles > 0 ? ((count + n_tiles - 1) / n_tiles + 15) / 16 * 16 : 0;
    for (int s = me; s < slots; s += chunks) {
      const int at = s * rows;
      tiles[first + s] = LoraTile{tid == n_groups ? -1 : tid, start + at, s < n_tiles ? max(0, min(rows, count - at)) : 0, 0};
    }
  }
  for (int e0 = me * per; e0 < min(n, me * per + per); e0 += kChunkThreads) {
    for (int v = tid; v < 32 * keys; v += kChunkThreads) s_rank[v] = 0;
    __syncthreads();
    const int e = e0 + tid;
    const bool in = e < n && e < me * per + per;
    const int key = in ? key_of(g, e, n_groups) : kPlanKeys;
    const uint32_t same = __match_any_sync(0xffffffffu, key);
    const int rank = __popc(same & ((1u << lane) - 1u));
    if (in && rank == 0) s_rank[warp * keys + key] = (uint16_t)__popc(same);
    __syncthreads();
    int here = 0;
    if (tid < keys) {
#pragma unroll 8
      for (int w = 0; w < 32; w++) {
        const int v = s_rank[w * keys + tid];
        s_rank[w * keys + tid] = (uint16_t)here;
        here += v;
      }
    }
    __syncthreads();
    if (in) order[s_base[key] + s_rank[warp * keys + key] + rank] = e;
    __syncthreads();
    s_base[tid] += here;   // (a thread's own group; read again behind the barriers of the next turn)
  }
}

// ---------------------------------------------------------------------------------------------------- gradients of the matrices
// A CTA's tile: 128 columns of `in` x 16 RT ranks, over the group's entries in stages of 64. Rows and the terms of u (or v) come by
// asynchronous copies into a ring; both fragments are transposed on the way out of it (the contraction runs over the entries). Four
// warps have 32 columns each, the other four the same columns and the other half of a stage's entries. fp16 rows are two bf16
// terms, exactly. The CTAs of a cluster share a group's stages; all sums meet in a fixed order.
template <typename PT, int RT, bool SHORT>
struct WgradShape {
  static constexpr int RP = 16 * RT, UN = sizeof(PT) == 4 ? 3 : 2, ROWS = 64, COLS = 128;
  static constexpr int IN = ROWS * COLS * 2, UV = ROWS * RP * 2, STAGE = IN + UN * UV;
  // groups of one or two stages: fewer of them, more CTAs of an SM
  static constexpr int STAGES = SHORT ? 2 : 96 * 1024 / STAGE > 5 ? 5 : 96 * 1024 / STAGE < 3 ? 3 : 96 * 1024 / STAGE;
  // the CTA's sums, in the ring's room: [ranks][columns] or [columns][ranks], whichever the gradient is, in rows of these pitches
  static constexpr int PITCH_R = COLS + 4, PITCH_C = RP + 8;
  static constexpr int OUT = (RP * PITCH_R > COLS * PITCH_C ? RP * PITCH_R : COLS * PITCH_C) * 4;
  static constexpr int RING = STAGES * STAGE > OUT ? STAGES * STAGE : OUT;
  static constexpr int SMEM = RING + (STAGES + 1) * ROWS * 4;   // and the entries of the stages
};
template <typename XT, typename PT, int RT, bool FAST, bool SHORT>
__global__ void __launch_bounds__(kThreads, RT == 1 && SHORT ? 4 : RT <= 2 ? 2 : 1) wgrad_kernel(const LoraWgradArgs both) {
  typedef WgradShape<PT, RT, SHORT> S;
  constexpr int XN = RowTerms<XT, bf16>::N, UN = S::UN, RP = S::RP;
  typedef Tile<S::COLS, 2> InTile;
  typedef Tile<RP, 2> UvTile;
  extern __shared__ __align__(16) uint8_t smem[];
  wait_for_launch();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, i = lane >> 2, q = lane & 3, cq = warp & 3, half = warp >> 2;
  // one launch for both gradients: the first's tiles, then the second's
  const int tile = blockIdx.x / C;
  const bool second = tile >= both.tiles;
  const LoraWgrad a = both.of[second];
  const int group = blockIdx.y, j0 = blockIdx.z * 64, c0 = (tile - (second ? both.tiles : 0)) * S::COLS;
  int start = 0, count = (int)both.g.n;
  if (both.offsets != nullptr) {
    start = both.offsets[group];
    count = both.offsets[group + 1] - start;
  }
  const int blocks = (count + S::ROWS - 1) / S::ROWS;
  const int b0 = (int)((long long)blocks * rank / C), nb = (int)((long long)blocks * (rank + 1) / C) - b0;
  const uint32_t ring = smem_at(smem);
  // Entries of the stages, known a stage before their rows are asked for: read two stages ahead into a register, then put here.
  int* s_entry = reinterpret_cast<int*>(smem + S::RING);
  auto entry_of = [&](int s) {
    const int t = (b0 + s) * S::ROWS + tid;
    return tid >= S::ROWS || s >= nb || t >= count ? -1 : both.order != nullptr ? both.order[start + t] : t;
  };
  typedef Deal<S::ROWS, S::COLS, 2> InD;
  const uint32_t in_to = InTile::at(0, InD::row(), InD::chunk());
  const int col = c0 + 8 * InD::chunk();
  int next = 0, into = 0, listed = 0;
  int upcoming = entry_of(S::STAGES);
  auto fetch = [&]() {
    const uint32_t at = ring + into * S::STAGE;
    into = into + 1 == S::STAGES ? 0 : into + 1;
    if (next < nb) {
      const int* entries = s_entry + listed * S::ROWS;
#pragma unroll
      for (int k = 0; k < InD::EACH; k++) {
        const int e = entries[InD::row() + k * InD::STEP];
        const int row = e < 0 || a.in_div == 1 ? e : (int)((unsigned)e / (unsigned)a.in_div);
        const XT* p = static_cast<const XT*>(a.in) + (long long)row * a.in_stride;
        const uint32_t to = at + in_to + k * InD::STEP * InTile::CHUNKS * 16;
        if constexpr (FAST) cp16(to, e >= 0 && col < a.D ? p + col : a.in, e >= 0 && col < a.D);
        else load_chunk<2>(to, e >= 0 ? p : a.in, col, e >= 0 ? a.D : 0, a.by_in);
      }
#pragma unroll
      for (int n = 0; n < UN; n++)
#pragma unroll
        for (int c = tid; c < S::ROWS * UvTile::CHUNKS; c += kThreads) {
          const int m = c / UvTile::CHUNKS, ch = c % UvTile::CHUNKS, e = entries[m];
          const bool there = e >= 0 && j0 + 8 * ch < both.ru;
          cp16(UvTile::at(at + S::IN + n * S::UV, m, ch), there ? a.uv + ((long long)n * both.g.n + e) * both.ru + j0 + 8 * ch : a.uv, there);
        }
    }
    next++;
    listed = listed == S::STAGES ? 0 : listed + 1;
    cp_commit();
  };
  for (int s = 0; s < S::STAGES; s++)
    if (tid < S::ROWS) s_entry[s * S::ROWS + tid] = entry_of(s);
  __syncthreads();
#pragma unroll 1
  for (int s = 0; s < S::STAGES - 1; s++) fetch();
  int put = S::STAGES;   // where the entries of stage s + STAGES go
  float acc[2][2 * RT][4];
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int n = 0; n < 2 * RT; n++)
#pragma unroll
      for (int k = 0; k < 4; k++) acc[m][n][k] = 0.f;
  for (int s = 0; s < nb; s++) {
    cp_wait<S::STAGES - 2>();
    __syncthreads();
    fetch();
    // (the slot's last reader, the fetch of stage s - 1, lies behind the barrier)
    if (tid < S::ROWS) s_entry[put * S::ROWS + tid] = upcoming;
    put = put == S::STAGES ? 0 : put + 1;
    upcoming = entry_of(s + S::STAGES + 1);
    const uint32_t at = ring + s % S::STAGES * S::STAGE;
    const int left = count - (b0 + s) * S::ROWS;
    float part[2][2 * RT][4];   // (a stage's sums by themselves: see the tile kernel)
    if constexpr (sizeof(PT) == 4) {
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
        for (int n = 0; n < 2 * RT; n++)
#pragma unroll
          for (int k = 0; k < 4; k++) part[m][n][k] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int t = 16 * (2 * k + half);
      if (t >= left) continue;
      uint32_t xa[2][XN][4];
#pragma unroll
      for (int m = 0; m < 2; m++) {
        uint32_t raw[4];
        ldsm_trans(raw, InTile::at(at, t + (lane & 7) + ((lane >> 4) & 1) * 8, 4 * cq + 2 * m + ((lane >> 3) & 1)));
        RowTerms<XT, bf16>::get(raw, xa[m]);
      }
#pragma unroll
      for (int n = 0; n < RT; n++) {
        uint32_t b[2][2][UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
          uint32_t r[4];
          ldsm_trans(r, UvTile::at(at + S::IN + u * S::UV, t + (lane & 15), 2 * n + (lane >> 4)));
          b[0][0][u] = r[0]; b[0][1][u] = r[1]; b[1][0][u] = r[2]; b[1][1][u] = r[3];
        }
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            if constexpr (sizeof(PT) == 4) mma_terms<XN, UN, bf16>(part[m][2 * n + h], xa[m], b[h][0], b[h][1]);
            else mma_terms<XN, UN, bf16>(acc[m][2 * n + h], xa[m], b[h][0], b[h][1]);
          }
      }
    }
    if constexpr (sizeof(PT) == 4) {
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
        for (int n = 0; n < 2 * RT; n++)
#pragma unroll
          for (int k = 0; k < 4; k++) acc[m][n][k] += part[m][n][k];
    }
  }
  cp_wait<0>();
  __syncthreads();
  // in shared memory as the gradient lies: one half of the warps, then both; the CTAs of the cluster add and store a part of it each
  float* s_out = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int turn = 1; turn >= 0; turn--) {
    if (half == turn) {
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
        for (int n = 0; n < 2 * RT; n++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int c = 32 * cq + 16 * m + i + 8 * h, j = 8 * n + 2 * q;
            float v0 = acc[m][n][2 * h], v1 = acc[m][n][2 * h + 1];
            if (a.r_first) {
              float *o = s_out + j * S::PITCH_R + c, *p = o + S::PITCH_R;
              *o = turn == 1 ? v0 : *o + v0;
              *p = turn == 1 ? v1 : *p + v1;
            } else {
              float2* o = reinterpret_cast<float2*>(s_out + c * S::PITCH_C + j);
              if (turn == 0) {
                v0 += o->x;
                v1 += o->y;
              }
              *o = make_float2(v0, v1);
            }
          }
    }
    __syncthreads();
  }
  if (C > 1) cluster.sync();
  const float f = a.scaled && count > 0 ? factor_of(both.g, group) : 1.f;   // (zero times a factor may be NaN)
  const int r1 = min(RP, both.r - j0), cols = min(S::COLS, a.D - c0);
  PT* out = static_cast<PT*>(a.out) + (long long)group * both.r * a.D;
  // rows of the gradient's tile: ranks (r_first) or columns; four neighbours a thread
  const int length = a.r_first ? cols : r1, n_rows = a.r_first ? r1 : cols, pitch = a.r_first ? S::PITCH_R : S::PITCH_C;
  const long long stride = a.r_first ? a.D : both.r;
  out += a.r_first ? (long long)j0 * a.D + c0 : (long long)c0 * both.r + j0;
  const int quads = a.r_first ? S::COLS / 4 : RP / 4;   // a power of two
  const bool whole = length % 4 == 0 && stride % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(PT)) == 0;
  const int at = 4 * (tid & (quads - 1));
  for (int row = tid / quads + rank * (kThreads / quads); row < n_rows; row += C * (kThreads / quads)) {
    if (at >= length) break;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int b = 0; b < C; b++) {
      const float4* p = reinterpret_cast<const float4*>(s_out + row * pitch + at);
      const float4 v = C == 1 ? *p : *cluster.map_shared_rank(p, b);
      s[0] += v.x;
      s[1] += v.y;
      s[2] += v.z;
      s[3] += v.w;
    }
    PT* o = out + row * stride + at;
    if (whole) {
      alignas(16) PT v[4] = {PT(s[0] * f), PT(s[1] * f), PT(s[2] * f), PT(s[3] * f)};
      if constexpr (sizeof(PT) == 4) *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(v);
      else *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(v);
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (at + k < length) o[k] = PT(s[k] * f);
    }
  }
  if (C > 1) cluster.sync();
}

template <typename XT, typename PT, int RT, bool FAST, bool SHORT>
cudaError_t wgrad_launch(const LoraWgradArgs& a, int cluster, cudaStream_t st) {
  typedef WgradShape<PT, RT, SHORT> S;
  auto kern = wgrad_kernel<XT, PT, RT, FAST, SHORT>;
  static bool done[16] = {};
  const cudaError_t e = allow_smem(kern, S::SMEM, done);
  if (e != cudaSuccess) return e;
  const int tiles = a.tiles + (a.of[1].out != nullptr ? (a.of[1].D + S::COLS - 1) / S::COLS : 0);
  return launch(kern, dim3((unsigned)(tiles * cluster), (unsigned)a.n_groups, (unsigned)((a.r + 63) / 64)), kThreads, S::SMEM, cluster, st, a);
}
template <typename XT, typename PT, int RT, bool FAST>
cudaError_t wgrad_length(const LoraWgradArgs& a, int cluster, cudaStream_t st) {
  return a.g.n <= 128LL * a.n_groups ? wgrad_launch<XT, PT, RT, FAST, true>(a, cluster, st) : wgrad_launch<XT, PT, RT, FAST, false>(a, cluster, st);
}
template <typename XT, typename PT, bool FAST>
cudaError_t wgrad_rank(const LoraWgradArgs& a, int cluster, cudaStream_t st) {
  if (a.r <= 16) return wgrad_length<XT, PT, 1, FAST>(a, cluster, st);
  if (a.r <= 32) return wgrad_length<XT, PT, 2, FAST>(a, cluster, st);
  return wgrad_length<XT, PT, 4, FAST>(a, cluster, st);
}
template <typename XT, typename PT>
cudaError_t wgrad_read(const LoraWgradArgs& a, int cluster, cudaStream_t st) {
  return a.of[0].by_in == kBy16 && (a.of[1].out == nullptr || a.of[1].by_in == kBy16) ? wgrad_rank<XT, PT, true>(a, cluster, st) : wgrad_rank<XT, PT, false>(a, cluster, st);
}

// ---------------------------------------------------------------------------------------------------- sum over slots
// Rows that start anywhere, again at 16-byte boundaries, zero behind their end: two products read them.
__global__ void __launch_bounds__(kThreads) align_rows_kernel(const uint16_t* in, long long in_stride, int cols, uint16_t* out, int out_stride) {
  wait_for_launch();
  const uint16_t* p = in + (long long)blockIdx.x * in_stride;
  uint16_t* o = out + (long long)blockIdx.x * out_stride;
#pragma unroll 8
  for (int c = threadIdx.x; c < out_stride; c += kThreads) o[c] = c < cols ? p[c] : (uint16_t)0;
}

// four neighbouring columns of a token a thread; part's rows are whole fours where `quads`
template <typename XT>
__global__ void __launch_bounds__(kThreads) sum_slots_kernel(const float* part, int slots, int cols, XT* out, long long out_stride, bool quads) {
  wait_for_launch();
  const long long token = blockIdx.x;
  const int c = 4 * (blockIdx.y * kThreads + threadIdx.x);
  if (c >= cols) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  const float* p = part + token * slots * cols + c;
  XT* o = out + token * out_stride + c;
  if (quads) {
#pragma unroll 8
    for (int j = 0; j < slots; j++) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(p + (long long)j * cols));
      s[0] += v.x;
      s[1] += v.y;
      s[2] += v.z;
      s[3] += v.w;
    }
    const uint2 v = make_uint2(round_pair(s[0], s[1], XT()), round_pair(s[2], s[3], XT()));
    *reinterpret_cast<uint2*>(o) = v;
    return;
  }
  for (int k = 0; k < 4 && c + k < cols; k++) {
    for (int j = 0; j < slots; j++) s[k] += p[(long long)j * cols + k];
    o[k] = XT(s[k]);
  }
}

// Rows whose expert lies outside [0, E) become zero, the others are not touched. A warp a row.
__global__ void __launch_bounds__(kThreads) clear_rows_kernel(uint16_t* y, int rows, int N, const uint32_t* experts, uint32_t E) {
  wait_for_launch();
  const int row = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= rows || experts[row] < E) return;
  uint16_t* p = y + (long long)row * N;
  const int whole = (reinterpret_cast<uintptr_t>(p) & 15) == 0 ? N / 8 : 0;   // groups of 16 bytes
  for (int c = lane; c < whole; c += 32) reinterpret_cast<uint4*>(p)[c] = make_uint4(0, 0, 0, 0);
  for (int c = 8 * whole + lane; c < N; c += 32) p[c] = 0;
}

int sm_count() {
  static int known[16] = {};   // of the devices asked for so far
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev >= 0 && dev < 16 && known[dev] != 0) return known[dev];
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  if (dev >= 0 && dev < 16) known[dev] = sms;
  return sms;
}

// CTAs of a cluster, for that many tiles and as many CTAs as an SM holds: what fills the GPU but still runs at once. Clusters
// stay within a group of SMs, so larger ones leave a few of them empty: a tenth is kept back. Rows in tiles of 64, K 1024, N 2048, rank
// 16, clusters of 2, 3, 4, 6, 8: 30 tiles 15.0, 13.2, 12.5, 12.8, 11.8 us; 40 tiles 15.2, 13.3, 14.3, 13.0, 20.5; 60 tiles 15.5, 17.5,
// 14.4, 23.4, 21.2; 72 tiles 15.7, 17.6, 23.0 (no longer at once); 80 tiles 21.0, 17.7, 23.3; 96 tiles 21.6, 28.0.
// `exact`: no other CTAs are in the grid (those of a plan's empty slots take SMs for a moment, and two CTAs then share one).
int pick_cluster(long long tiles, int per_sm, bool exact) {
  const long long sms = sm_count(), room = per_sm * sms;
  auto fits = [&](int c) { return 10 * tiles * c <= 9 * room; };
  for (int c : {8, 6, 4})
    if (fits(c)) return c;
  if (per_sm > 1 && exact && 2 * tiles <= sms) return 2;   // an SM for each CTA
  return fits(3) ? 3 : 2 * tiles <= room ? 2 : 1;
}

constexpr size_t kSlotBytes = 64u << 20;          // float32 rows of slots that are summed at a time: they stay in L2

cudaError_t tile_launch(int types, const LoraArgs& a, bool backward, int mt, int cluster, cudaStream_t st) {
  switch (types) {
    case kLoraBf16: return launch_lora_tile_bf16(a, backward, mt, cluster, st);
    case kLoraF16: return launch_lora_tile_f16(a, backward, mt, cluster, st);
    case kLoraBf16F32: return launch_lora_tile_bf16_f32(a, backward, mt, cluster, st);
    default: return launch_lora_tile_f16_f32(a, backward, mt, cluster, st);
  }
}

// the rows of a call: planned, found by the kernel, or all of one group
int set_rows(LoraArgs& a, const LoraCall& c, int& cluster) {
  a.g = c.g;
  a.direct = 0;
  a.plan = LoraPlan{};
  const bool grouped = c.g.ids != nullptr || c.g.experts != nullptr;
  int mt;
  if (!grouped) {
    // Low tiles while two CTAs of each run at once, and the matrices that each tile reads are small. K, N 4096, rank 16: 1300 rows 12.9 and
    // 16.0 us in tiles of 16 and 64, 2368 rows 16.0 and 19.8, 2700 rows 23.2 and 20.6; float32 1300 rows 18.4 and 20.5, 1700 24.1 and 20.6.
    const long long matrices = (long long)c.r * ((long long)c.K + c.N) * (c.types == kLoraBf16 || c.types == kLoraF16 ? 2 : 4);
    mt = c.g.n <= (matrices < (512 << 10) ? 16 * sm_count() : 1280) ? 16 : 64;
    a.n_clusters = (int)((c.g.n + mt - 1) / mt);
  } else if (c.plan != nullptr) {
    const LoraPlanLayout l = lora_plan_layout(c.g.n, c.g.G * c.g.E);
    const uint8_t* p = static_cast<const uint8_t*>(c.plan);
    a.plan = LoraPlan{reinterpret_cast<const int*>(p + l.order), reinterpret_cast<const int*>(p + l.offsets),
                      reinterpret_cast<const LoraTile*>(p + l.tiles), l.n_tiles, l.tile_rows};
    mt = l.tile_rows;
    a.n_clusters = l.n_tiles;
  } else {
    a.direct = 1;
    mt = 16;
    a.n_clusters = (int)c.g.n;
  }
  // tiles that have rows, as far as the host knows: those found one by one are no more than the groups; half of the groups' last
  // tiles of a plan are counted (4072 entries of 128 groups: clusters of 1, 2, 4, 8 forward 47, 30, 37, 56 us)
  const long long groups = (long long)c.g.G * c.g.E;
  cluster = pick_cluster(a.direct ? std::min(c.g.n, groups) : grouped ? c.g.n / mt + std::min(c.g.n, groups) / 2 : a.n_clusters,
                         a.r > 64 ? 1 : 2, !grouped);
  return mt;
}

// how rows of `size`-byte elements, `stride` apart from `p` on, of `length` elements, can be read
int by(const void* p, long long stride, int length, int size) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(stride * size) | (uintptr_t)((long long)length * size);
  return (all & 15) == 0 ? kBy16 : (all & 7) == 0 ? kBy8 : kByElement;
}

void set_reads(LoraArgs& a, const LoraCall& c, bool backward) {
  const int ps = c.types == kLoraBf16 || c.types == kLoraF16 ? 2 : 4;
  const int l1 = backward ? a.r : a.D1, l2 = backward ? a.D2 : a.r;
  a.by_in = by(a.in, a.in_stride, a.D1, 2);
  a.by_w1 = by(a.w1, l1, l1, ps);
  a.by_w2 = by(a.w2, l2, l2, ps);
  a.by_out = std::max(by(a.out, a.out_stride, a.D2, 2), a.base != nullptr ? by(a.base, a.base_stride, a.D2, 2) : (int)kBy16);
  a.ru = (a.r + 7) / 8 * 8;
}

}  // namespace
}  // namespace lora

using namespace lora;

LoraPlanLayout lora_plan_layout(long long n, int n_groups) {
  auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
  LoraPlanLayout l;
  // Low tiles while they are few, or groups small: 1000 rows of K, N 4096 and rank 16 with 10 adapters 14.0 us in tiles of 16 rows, 18.1
  // in tiles of 64; with 128 experts 4000 and 8000 rows alike, beyond that the weights are read less often by high ones.
  l.tile_rows = n > 2048 && n >= 24LL * n_groups ? 64 : 16;
  l.n_tiles = (int)(n / l.tile_rows) + n_groups + 1;
  // entries of a CTA where two launches are faster: in one, 4072 entries of 128 groups took 4.8 us, two launches 5.6
  l.chunk = n_groups < kPlanKeys && n * n_groups > (1 << 20) ? (int)((n + kMostChunks - 1) / kMostChunks + kChunkThreads - 1) / kChunkThreads * kChunkThreads : 0;
  l.chunks = l.chunk > 0 ? (int)((n + l.chunk - 1) / l.chunk) : 0;
  l.order = 0;
  l.offsets = up((size_t)n * 4);
  l.tiles = up(l.offsets + ((size_t)n_groups + 2) * 4);
  l.counts = up(l.tiles + (size_t)l.n_tiles * sizeof(LoraTile));
  l.total = up(l.counts + (size_t)l.chunks * (n_groups + 1) * 4);
  return l;
}

cudaError_t launch_lora_plan(const LoraGroups& g, void* plan, cudaStream_t st) {
  const int n_groups = g.G * g.E;
  const LoraPlanLayout l = lora_plan_layout(g.n, n_groups);
  uint8_t* p = static_cast<uint8_t*>(plan);
  int *order = reinterpret_cast<int*>(p + l.order), *offsets = reinterpret_cast<int*>(p + l.offsets), *counts = reinterpret_cast<int*>(p + l.counts);
  LoraTile* tiles = reinterpret_cast<LoraTile*>(p + l.tiles);
  if (l.chunks == 0) {
    return launch(plan_kernel, dim3((unsigned)n_groups + 1), kPlanThreads, 0, 0, st, g, n_groups, l.tile_rows, order, offsets, tiles);
  }
  cudaError_t e = launch(plan_count_kernel, dim3((unsigned)l.chunks), kChunkThreads, 0, 0, st, g, n_groups, l.chunk, counts);
  if (e != cudaSuccess) return e;
  const int smem = 32 * (n_groups + 1) * 2;
  if (smem > 40 * 1024) {
    static bool done[16] = {};
    if ((e = allow_smem(plan_place_kernel, 32 * kPlanKeys * 2, done)) != cudaSuccess) return e;
  }
  return launch(plan_place_kernel, dim3((unsigned)l.chunks), kChunkThreads, smem, 0, st, g, n_groups, l.chunk, l.tile_rows, counts, order, offsets, tiles);
}

cudaError_t launch_lora_wgrad(const LoraWgradArgs& a, int in_dtype, int out_f32, int cluster, cudaStream_t st) {
  if (in_dtype == 1) return out_f32 ? wgrad_read<__half, float>(a, cluster, st) : wgrad_read<__half, __half>(a, cluster, st);
  return out_f32 ? wgrad_read<bf16, float>(a, cluster, st) : wgrad_read<bf16, bf16>(a, cluster, st);
}

cudaError_t launch_lora_sum_slots(const float* part, int slots, long long tokens, int cols, void* out, long long out_stride, int dtype,
                                  cudaStream_t st) {
  const dim3 grid((unsigned)tokens, (unsigned)((cols + 4 * kThreads - 1) / (4 * kThreads)));
  const bool quads = cols % 4 == 0 && out_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(part) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0;
  if (dtype == 1) return launch(sum_slots_kernel<__half>, grid, kThreads, 0, 0, st, part, slots, cols, static_cast<__half*>(out), out_stride, quads);
  return launch(sum_slots_kernel<bf16>, grid, kThreads, 0, 0, st, part, slots, cols, static_cast<bf16*>(out), out_stride, quads);
}

cudaError_t launch_clear_rows(void* y, int rows, int N, const uint32_t* experts, int n_experts, cudaStream_t st) {
  return launch(clear_rows_kernel, dim3((unsigned)((rows + kThreads / 32 - 1) / (kThreads / 32))), kThreads, 0, 0, st, static_cast<uint16_t*>(y), rows, N, experts,
                (uint32_t)n_experts);
}

cudaError_t launch_lora_forward(const LoraCall& c, const void* y, long long y_stride, void* out, long long out_stride, void* u,
                                cudaStream_t st) {
  LoraArgs a{};
  int cluster;
  a.r = c.r;
  const int mt = set_rows(a, c, cluster);
  a.in = c.x;
  a.in_stride = c.x_stride;
  a.in_div = c.shared ? c.g.slots : 1;
  a.D1 = c.K;
  a.D2 = c.N;
  a.w1 = c.a;
  a.w2 = c.b;
  a.base = y;
  a.base_stride = y_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.c1 = c.N;
  a.u = static_cast<uint16_t*>(u);
  a.shrink = 1;
  set_reads(a, c, false);
  return tile_launch(c.types, a, false, mt, cluster, st);
}

// v [n, r], and the slots' rows of as many columns as are summed at a time
static int slot_columns(long long n, int K) {
  const long long fit = (long long)(kSlotBytes / 4) / std::max<long long>(1, n) / 64 * 64;
  return (int)std::min<long long>(K, std::max<long long>(64, fit));
}
size_t lora_saved_bytes(long long n, int r, int param_f32) { return (size_t)n * ((r + 7) / 8 * 8) * (param_f32 ? 6 : 4); }
static size_t v_bytes(long long n, int r, int f32) { return (lora_saved_bytes(n, r, f32) + 255) & ~(size_t)255; }
static size_t aligned_bytes(long long n, int N) { return N % 8 != 0 ? ((size_t)n * ((N + 7) / 8 * 8) * 2 + 255) & ~(size_t)255 : 0; }
size_t lora_backward_workspace_bytes(long long n, int slots, int shared, int K, int N, int r, int param_f32) {
  return v_bytes(n, r, param_f32) + aligned_bytes(n, N) + (shared && slots > 1 ? (size_t)n * slot_columns(n, K) * 4 : 0);
}

cudaError_t launch_lora_backward(const LoraCall& c, const void* dy, long long dy_stride, const void* u, void* dx, long long dx_stride,
                                 void* da, void* db, void* workspace, cudaStream_t st) {
  LoraArgs a{};
  cudaError_t e;
  int cluster;
  const bool summed = c.shared && c.g.slots > 1;
  const int f16 = c.types == kLoraF16 || c.types == kLoraF16F32, f32 = c.types == kLoraBf16F32 || c.types == kLoraF16F32;
  uint16_t* v = static_cast<uint16_t*>(workspace);
  if (c.N % 8 != 0) {
    uint16_t* aligned = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(workspace) + v_bytes(c.g.n, c.r, f32));
    const int stride = (c.N + 7) / 8 * 8;
    if ((e = launch(align_rows_kernel, dim3((unsigned)c.g.n), kThreads, 0, 0, st, static_cast<const uint16_t*>(dy), dy_stride, c.N, aligned, stride)) != cudaSuccess)
      return e;
    dy = aligned;
    dy_stride = stride;
  }
  a.r = c.r;
  const int mt = set_rows(a, c, cluster);
  a.in = dy;
  a.in_stride = dy_stride;
  a.in_div = 1;
  a.D1 = c.N;
  a.D2 = c.K;
  a.w1 = c.b;
  a.w2 = c.a;
  a.c1 = c.K;
  a.u = v;
  a.shrink = 1;
  a.scale_u = 1;
  const long long tokens = c.g.n / c.g.slots;
  float* part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + v_bytes(c.g.n, c.r, f32) + aligned_bytes(c.g.n, c.N));
  const int step = slot_columns(c.g.n, c.K);
  // a token's slots share its row: their parts in float32, as many columns at a time as stay in L2, then the sum
  auto columns = [&](int c0) {
    a.c0 = c0;
    a.c1 = std::min(c.K, c0 + step);
    a.out = part;
    a.out_f32 = 1;
    a.out_stride = a.c1 - c0;
  };
  if (dx != nullptr && summed) {
    columns(0);
  } else if (dx != nullptr) {
    a.out = dx;
    a.out_stride = dx_stride;
  }
  set_reads(a, c, true);
  if (c.N % 8 != 0) a.by_in = kBy16;   // (the rows put at boundaries above)
  if (dx != nullptr || da != nullptr) {
    if ((e = tile_launch(c.types, a, true, mt, cluster, st)) != cudaSuccess) return e;
  }
  if (dx != nullptr && summed) {
    for (int c0 = 0;;) {
      if ((e = launch_lora_sum_slots(part, c.g.slots, tokens, a.c1 - a.c0, static_cast<uint16_t*>(dx) + c0, dx_stride, f16 ? 1 : 2, st)) != cudaSuccess)
        return e;
      if ((c0 = a.c1) >= c.K) break;
      a.shrink = 0;
      columns(c0);
      set_reads(a, c, true);   // (the rows are not read again)
      if ((e = tile_launch(c.types, a, true, mt, cluster, st)) != cudaSuccess) return e;
    }
  }
  if (da == nullptr && db == nullptr) return cudaSuccess;
  auto side = [&](const void* in, long long stride, int div, int D, const void* uv, int scaled, void* out, int r_first) {
    // (dy's rows are zero up to their own stride where they were put at boundaries)
    return LoraWgrad{in, stride, div, D, static_cast<const uint16_t*>(uv), scaled, out, r_first, by(in, stride, in == dy && D % 8 != 0 ? (int)stride : D, 2)};
  };
  LoraWgradArgs w{};
  w.g = c.g;
  w.r = c.r;
  w.ru = a.ru;
  w.n_groups = c.g.G * c.g.E;
  w.order = a.plan.order;
  w.offsets = a.plan.offsets;
  int n = 0;
  if (db != nullptr) w.of[n++] = side(dy, dy_stride, 1, c.N, u, 1, db, 0);
  if (da != nullptr) w.of[n++] = side(c.x, c.x_stride, c.shared ? c.g.slots : 1, c.K, v, 0, da, 1);
  w.tiles = (w.of[0].D + 127) / 128;
  // CTAs of a cluster share a group's stages of 64 entries, where the columns alone leave the GPU empty
  const long long stages = (c.g.n / w.n_groups + 63) / 64, all = w.tiles + (n > 1 ? (w.of[1].D + 127) / 128 : 0);
  cluster = pick_cluster(w.n_groups * all, a.r > 32 ? 1 : 2, true);
  while (cluster > 1 && stages < 2 * cluster) cluster >>= 1;
  return launch_lora_wgrad(w, f16 ? 1 : 2, f32, cluster, st);
}

}  // namespace kq
