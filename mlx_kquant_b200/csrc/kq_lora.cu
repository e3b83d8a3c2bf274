// Low-rank adapters: the order of the rows by adapter (plan), the gradients of the adapters' matrices, the sum over a token's
// slots, and which launches a call takes. The products of the rows are in kq_lora.cuh.
#include <algorithm>

#include "kq_lora.cuh"

namespace kq {
namespace lora {
namespace {

// ---------------------------------------------------------------------------------------------------- plan
constexpr int kPlanThreads = 512, kPlanEach = 8;

// One CTA per group, the last for the entries without one. It reads every entry's group: how many lie before its own, and its
// own in their order. No counters, nothing to clear, the same order each time. Tiles take the list's slots from
// start / height + group on, which no two groups share; slots that are left over hold none.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const LoraGroups g, int n_groups, int height, int* order, int* offsets, LoraTile* tiles) {
  __shared__ int s_warp[2][kPlanThreads / 32];
  __shared__ int s_base;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, mine = blockIdx.x;
  const int n = (int)g.n;
  auto key = [&](int e) {
    const int k = group_of(g, e);
    return k < 0 ? n_groups : k;
  };
  int less = 0, same = 0;
  for (int e = tid; e < n; e += kPlanThreads) {
    const int k = key(e);
    less += k < mine;
    same += k == mine;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    less += __shfl_xor_sync(0xffffffffu, less, o);
    same += __shfl_xor_sync(0xffffffffu, same, o);
  }
  if (lane == 0) {
    s_warp[0][warp] = less;
    s_warp[1][warp] = same;
  }
  __syncthreads();
  int start = 0, count = 0;
  for (int w = 0; w < kPlanThreads / 32; w++) {
    start += s_warp[0][w];
    count += s_warp[1][w];
  }
  if (tid == 0) {
    offsets[mine] = start;
    if (mine == n_groups) offsets[mine + 1] = start + count;
    s_base = start;
  }
  // tiles as even as sixteen rows allow
  const int first = start / height + mine, slots = (start + count) / height + mine + 1 - first;
  const int n_tiles = (count + height - 1) / height;
  const int each = n_tiles > 0 ? ((count + n_tiles - 1) / n_tiles + 15) / 16 * 16 : 0;
  for (int s = tid; s < slots; s += kPlanThreads) {
    const int at = s * each;
    tiles[first + s] = LoraTile{mine == n_groups ? -1 : mine, start + at, s < n_tiles ? max(0, min(each, count - at)) : 0, 0};
  }
  if (count == 0) return;
  for (int e0 = 0; e0 < n; e0 += kPlanThreads * kPlanEach) {
    __syncthreads();
    const int base = s_base;
    uint32_t hits = 0;
#pragma unroll
    for (int v = 0; v < kPlanEach; v++) {
      const int e = e0 + tid * kPlanEach + v;
      if (e < n && key(e) == mine) hits |= 1u << v;
    }
    const int c = __popc(hits);
    int at = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += v;
    }
    if (lane == 31) s_warp[0][warp] = at;
    __syncthreads();
    int ahead = 0, total = 0;
    for (int w = 0; w < kPlanThreads / 32; w++) {
      const int v = s_warp[0][w];
      if (w < warp) ahead += v;
      total += v;
    }
    at += base + ahead - c;
#pragma unroll
    for (int v = 0; v < kPlanEach; v++)
      if (hits >> v & 1) order[at++] = e0 + tid * kPlanEach + v;
    if (tid == 0) s_base = base + total;   // (read again behind the barrier at the top)
  }
}

// ---------------------------------------------------------------------------------------------------- gradients of the matrices
// A warp's tile: 64 columns of `in` x 16 RT ranks, over the group's entries in sixteens. `in`'s fragments come straight from
// memory: a lane holds eight neighbouring columns of four entries. Both operands as bf16 terms: fp16 rows are two, exactly; uv is
// three where the gradient is float32, two where it is rounded to 16 bits. `splits` warps share a tile's entries, and the CTAs of a
// cluster; their sums meet in a fixed order.
template <typename XT, typename PT, int RT, bool VEC>
__global__ void __launch_bounds__(kThreads) wgrad_kernel(const LoraWgradArgs a) {
  constexpr int XN = RowTerms<XT, bf16>::N, UN = sizeof(PT) == 4 ? 3 : 2, MOST = UN, JV = 2 * RT, RP = 16 * RT;
  extern __shared__ float w_smem[];   // [tiles][splits / 2][2 RP][32 lanes] and [tiles][64][RP]
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, i = lane >> 2, q = lane & 3;
  const int S = a.splits, tiles = kThreads / 32 / S, ct = warp / S, sp = warp % S;
  const int group = blockIdx.y, j0 = blockIdx.z * 64;
  const int c0 = (blockIdx.x / C * tiles + ct) * 64;
  long long start = 0, count = a.g.n;
  if (a.offsets != nullptr) {
    start = a.offsets[group];
    count = a.offsets[group + 1] - start;
  }
  float acc[4][2 * RT][4];
#pragma unroll
  for (int m = 0; m < 4; m++)
#pragma unroll
    for (int n = 0; n < 2 * RT; n++)
#pragma unroll
      for (int k = 0; k < 4; k++) acc[m][n][k] = 0.f;
  if (c0 < a.D) {
    const int col = c0 + 8 * i;
    for (long long t0 = 16LL * (rank * S + sp); t0 < count; t0 += 16LL * S * C) {
      Load<XT, 8, VEC> x[4];
      float u[4][JV];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const long long t = t0 + 4 * q + k;
        const long long e = t >= count ? -1 : a.order != nullptr ? a.order[start + t] : t;
        x[k].get(static_cast<const XT*>(a.in) + (e < 0 ? 0 : e / a.in_div) * a.in_stride + col, e < 0 ? 0 : a.D - col);
        const float* up = a.uv + (e < 0 ? 0 : e) * a.r + j0 + i * JV;
#pragma unroll
        for (int j = 0; j < JV; j++) u[k][j] = e >= 0 && j0 + i * JV + j < a.r ? up[j] : 0.f;
      }
      uint32_t xa[4][XN][4];
#pragma unroll
      for (int m = 0; m < 4; m++) {
        const uint32_t p[4] = {__byte_perm(x[0].w[m], x[1].w[m], 0x5410), __byte_perm(x[0].w[m], x[1].w[m], 0x7632),
                               __byte_perm(x[2].w[m], x[3].w[m], 0x5410), __byte_perm(x[2].w[m], x[3].w[m], 0x7632)};
#pragma unroll
        for (int k = 0; k < 4; k++) {
          uint32_t t[XN];
          RowTerms<XT, bf16>::get(p[k], t);
#pragma unroll
          for (int n = 0; n < XN; n++) xa[m][n][k] = t[n];
        }
      }
#pragma unroll
      for (int jt = 0; jt < 2 * RT; jt++) {
        uint32_t b0[UN], b1[UN];
        split<UN>(u[0][jt], u[1][jt], b0);
        split<UN>(u[2][jt], u[3][jt], b1);
#pragma unroll
        for (int m = 0; m < 4; m++) mma_terms<XN, UN, MOST, bf16>(acc[m][jt], xa[m], b0, b1);
      }
    }
  }
  for (int h = S / 2; h > 0; h >>= 1) {
    float* mine = w_smem + (size_t)(ct * (S / 2) + sp % h) * 2 * RP * 16 * 2;
    if (sp >= h && sp < 2 * h) {
#pragma unroll
      for (int m = 0; m < 4; m++)
#pragma unroll
        for (int n = 0; n < 2 * RT; n++)
#pragma unroll
          for (int k = 0; k < 4; k++) mine[((m * 2 * RT + n) * 4 + k) * 32 + lane] = acc[m][n][k];
    }
    __syncthreads();
    if (sp < h) {
#pragma unroll
      for (int m = 0; m < 4; m++)
#pragma unroll
        for (int n = 0; n < 2 * RT; n++)
#pragma unroll
          for (int k = 0; k < 4; k++) acc[m][n][k] += mine[((m * 2 * RT + n) * 4 + k) * 32 + lane];
    }
    __syncthreads();
  }
  // [64 columns][RP ranks] of each tile in shared memory; the CTAs of the cluster add and store a part of it each
  float* s_out = w_smem + (size_t)tiles * (S / 2) * 64 * RP;
  if (sp == 0) {
#pragma unroll
    for (int m = 0; m < 4; m++)
#pragma unroll
      for (int n = 0; n < 2 * RT; n++)
#pragma unroll
        for (int k = 0; k < 4; k++)
          s_out[(ct * 64 + 8 * i + 2 * m + (k >> 1)) * RP + (2 * q + (k & 1)) * JV + n] = acc[m][n][k];
  }
  cluster.sync();
  const float f = a.scaled ? factor_of(a.g, group) : 1.f;
  const int r1 = min(RP, a.r - j0);
  PT* out = static_cast<PT*>(a.out) + (long long)group * a.r * a.D;
  const int per = tiles * 64 * r1;
  for (int v = rank * kThreads + tid; v < per; v += C * kThreads) {
    const int c = a.r_first ? v % (tiles * 64) : v / r1, j = a.r_first ? v / (tiles * 64) : v % r1;
    const long long column = (long long)blockIdx.x / C * tiles * 64 + c;
    if (column >= a.D) continue;
    float s = 0.f;
    for (int b = 0; b < C; b++) s += *cluster.map_shared_rank(s_out + c * RP + j, b);
    out[a.r_first ? (long long)(j0 + j) * a.D + column : column * a.r + j0 + j] = PT(s * f);
  }
  cluster.sync();
}

template <typename XT, typename PT, int RT, bool VEC>
cudaError_t wgrad_launch(const LoraWgradArgs& a, int cluster, cudaStream_t st) {
  constexpr int RP = 16 * RT;
  const int tiles = kThreads / 32 / a.splits;
  const int smem = (tiles * (a.splits / 2) + tiles) * 64 * RP * 4;
  auto kern = wgrad_kernel<XT, PT, RT, VEC>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * 64 * RP * 4);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.D + 64 * tiles - 1) / (64 * tiles) * cluster), (unsigned)a.n_groups, (unsigned)((a.r + 63) / 64));
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
template <typename XT, typename PT>
cudaError_t wgrad_rank(const LoraWgradArgs& a, int cluster, cudaStream_t st) {
  if (a.vec_in) {
    if (a.r <= 16) return wgrad_launch<XT, PT, 1, true>(a, cluster, st);
    if (a.r <= 32) return wgrad_launch<XT, PT, 2, true>(a, cluster, st);
    return wgrad_launch<XT, PT, 4, true>(a, cluster, st);
  }
  if (a.r <= 16) return wgrad_launch<XT, PT, 1, false>(a, cluster, st);
  if (a.r <= 32) return wgrad_launch<XT, PT, 2, false>(a, cluster, st);
  return wgrad_launch<XT, PT, 4, false>(a, cluster, st);
}

// ---------------------------------------------------------------------------------------------------- sum over slots
template <typename XT>
__global__ void __launch_bounds__(kThreads) sum_slots_kernel(const float* part, int slots, int cols, XT* out, long long out_stride) {
  const long long token = blockIdx.x;
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    float s = 0.f;
    for (int j = 0; j < slots; j++) s += part[(token * slots + j) * cols + c];
    out[token * out_stride + c] = XT(s);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return sms;
}

// CTAs of a cluster: as many as fill the GPU twice at most
int pick_cluster(long long tiles) {
  const long long room = 2LL * sm_count();
  for (int c = 8; c > 1; c >>= 1)
    if (tiles * c <= room) return c;
  return 1;
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
    mt = c.g.n <= 512 ? 16 : 64;
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
  cluster = pick_cluster(std::min<long long>(a.n_clusters, c.g.n));
  return mt;
}

void set_vec(LoraArgs& a, const LoraCall& c, bool backward) {
  const int rt = a.r <= 16 ? 1 : a.r <= 32 ? 2 : a.r <= 64 ? 4 : 8;
  a.vec_in = a.D1 % 8 == 0 && a.in_stride % 8 == 0 && aligned16(a.in);
  a.vec_w1 = aligned16(a.w1) && (backward ? a.r % (2 * rt) == 0 : a.D1 % 8 == 0);
  a.vec_w2 = aligned16(a.w2) && (backward ? a.D2 % 8 == 0 : a.r % 4 == 0);
  a.vec_out = a.D2 % 8 == 0 && a.out_stride % 8 == 0 && aligned16(a.out) &&
              (a.base == nullptr || (a.base_stride % 8 == 0 && aligned16(a.base)));
}

}  // namespace
}  // namespace lora

using namespace lora;

LoraPlanLayout lora_plan_layout(long long n, int n_groups) {
  auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
  LoraPlanLayout l;
  l.tile_rows = n >= 24LL * n_groups ? 64 : 16;
  l.n_tiles = (int)(n / l.tile_rows) + n_groups + 1;
  l.order = 0;
  l.offsets = up((size_t)n * 4);
  l.tiles = up(l.offsets + ((size_t)n_groups + 2) * 4);
  l.total = up(l.tiles + (size_t)l.n_tiles * sizeof(LoraTile));
  return l;
}

cudaError_t launch_lora_plan(const LoraGroups& g, void* plan, cudaStream_t st) {
  const int n_groups = g.G * g.E;
  const LoraPlanLayout l = lora_plan_layout(g.n, n_groups);
  uint8_t* p = static_cast<uint8_t*>(plan);
  plan_kernel<<<n_groups + 1, kPlanThreads, 0, st>>>(g, n_groups, l.tile_rows, reinterpret_cast<int*>(p + l.order),
                                                     reinterpret_cast<int*>(p + l.offsets), reinterpret_cast<LoraTile*>(p + l.tiles));
  return cudaGetLastError();
}

cudaError_t launch_lora_wgrad(const LoraWgradArgs& a, int in_dtype, int out_f32, int cluster, cudaStream_t st) {
  if (in_dtype == 1) return out_f32 ? wgrad_rank<__half, float>(a, cluster, st) : wgrad_rank<__half, __half>(a, cluster, st);
  return out_f32 ? wgrad_rank<bf16, float>(a, cluster, st) : wgrad_rank<bf16, bf16>(a, cluster, st);
}

cudaError_t launch_lora_sum_slots(const float* part, int slots, long long tokens, int cols, void* out, long long out_stride, int dtype,
                                  cudaStream_t st) {
  if (dtype == 1) sum_slots_kernel<__half><<<(unsigned)tokens, kThreads, 0, st>>>(part, slots, cols, static_cast<__half*>(out), out_stride);
  else sum_slots_kernel<bf16><<<(unsigned)tokens, kThreads, 0, st>>>(part, slots, cols, static_cast<bf16*>(out), out_stride);
  return cudaGetLastError();
}

cudaError_t launch_lora_forward(const LoraCall& c, const void* y, long long y_stride, void* out, long long out_stride, float* u,
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
  a.u = u;
  a.shrink = 1;
  set_vec(a, c, false);
  return tile_launch(c.types, a, false, mt, cluster, st);
}

// v [n, r], and the slots' rows of as many columns as are summed at a time
static int slot_columns(long long n, int K) {
  const long long fit = (long long)(kSlotBytes / 4) / std::max<long long>(1, n) / 64 * 64;
  return (int)std::min<long long>(K, std::max<long long>(64, fit));
}
static size_t v_bytes(long long n, int r) { return ((size_t)n * r * 4 + 255) & ~(size_t)255; }
size_t lora_backward_workspace_bytes(long long n, int slots, int shared, int K, int r) {
  return v_bytes(n, r) + (shared && slots > 1 ? (size_t)n * slot_columns(n, K) * 4 : 0);
}

cudaError_t launch_lora_backward(const LoraCall& c, const void* dy, long long dy_stride, const float* u, void* dx, long long dx_stride,
                                 void* da, void* db, void* workspace, cudaStream_t st) {
  LoraArgs a{};
  cudaError_t e;
  int cluster;
  const bool summed = c.shared && c.g.slots > 1;
  float* v = static_cast<float*>(workspace);
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
  if (dx != nullptr && !summed) {
    a.out = dx;
    a.out_stride = dx_stride;
  }
  set_vec(a, c, true);
  if (dx != nullptr || da != nullptr) {
    if ((e = tile_launch(c.types, a, true, mt, cluster, st)) != cudaSuccess) return e;
  }
  const int f16 = c.types == kLoraF16 || c.types == kLoraF16F32, f32 = c.types == kLoraBf16F32 || c.types == kLoraF16F32;
  if (dx != nullptr && summed) {
    const long long tokens = c.g.n / c.g.slots;
    float* part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + v_bytes(c.g.n, c.r));
    const int step = slot_columns(c.g.n, c.K);
    a.shrink = 0;
    a.out = part;
    a.out_f32 = 1;
    for (int c0 = 0; c0 < c.K; c0 += step) {
      a.c0 = c0;
      a.c1 = std::min(c.K, c0 + step);
      a.out_stride = a.c1 - a.c0;
      set_vec(a, c, true);
      if ((e = tile_launch(c.types, a, true, mt, cluster, st)) != cudaSuccess) return e;
      if ((e = launch_lora_sum_slots(part, c.g.slots, tokens, a.c1 - a.c0, static_cast<uint16_t*>(dx) + c0, dx_stride, f16 ? 1 : 2, st)) !=
          cudaSuccess)
        return e;
    }
  }
  LoraWgradArgs w{};
  w.g = c.g;
  w.r = c.r;
  w.n_groups = c.g.G * c.g.E;
  w.order = a.plan.order;
  w.offsets = a.plan.offsets;
  // few entries of a group: its warps take columns of their own; many: they share the entries, and the CTAs of a cluster
  const long long rows = c.g.n / w.n_groups;
  w.splits = rows >= 512 ? 8 : rows >= 128 ? 2 : 1;
  auto wgrad = [&](const void* in, long long stride, int div, int D, const float* uv, int scaled, void* out, int r_first) {
    w.in = in;
    w.in_stride = stride;
    w.in_div = div;
    w.D = D;
    w.uv = uv;
    w.scaled = scaled;
    w.out = out;
    w.r_first = r_first;
    w.vec_in = D % 8 == 0 && stride % 8 == 0 && aligned16(in);
    const long long ctas = (long long)w.n_groups * ((D + 64 * (8 / w.splits) - 1) / (64 * (8 / w.splits)));
    return launch_lora_wgrad(w, f16 ? 1 : 2, f32, rows >= 512 ? pick_cluster(ctas) : 1, st);
  };
  if (db != nullptr && (e = wgrad(dy, dy_stride, 1, c.N, u, 1, db, 0)) != cudaSuccess) return e;
  if (da != nullptr && (e = wgrad(c.x, c.x_stride, c.shared ? c.g.slots : 1, c.K, v, 0, da, 1)) != cudaSuccess) return e;
  return cudaSuccess;
}

}  // namespace kq
