// Routing to experts in groups, and its gradient (kq_moe_router_grouped, kq_moe_router_grouped_backward).
//
// Row of logits l[E]: scores s = sigmoid(l) or softmax(l), ranked by q = s + bias (without a bias by l itself: the scores rise
// with it). A group of E / G neighbours counts by the sum of its group_top largest q; the top_groups best groups stay, of
// these the top_k largest q are picked, lowest index first among equals, groups and experts alike. Weights
// w_j = scale * s_ij / (sum s_i + 1e-20), or scale * s_ij.
//
// A warp per token, a lane NI neighbouring experts, all in registers. The order is that of 64 bits, but sums in 64 bits of
// exponentials in 64 bits took 66 us for 16384 tokens of 256 experts. So the kernel ranks floats first, whose error is bounded
// (kRouteSlack): where the neighbours in the order of the picks, the last of them and the best that is left, and the groups around the
// border lie further apart than that, 64 bits would give the same order; where they don't, unless they are bit for bit the same
// logit and bias, the token is ranked again in 64 bits. Logits alone need neither: they are compared as they are.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kq_common.cuh"
#include "kq_route.h"

namespace kq {
namespace {

constexpr int kRouteWarps = 4;
constexpr uint32_t kAll = 0xffffffffu;

__device__ __forceinline__ float rt_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ double rt_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ float rt_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
__device__ __forceinline__ float rt_sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// a float's order as an unsigned number's; NaN does not occur in keys
__device__ __forceinline__ uint32_t rt_order(float f) {
  const uint32_t b = __float_as_uint(f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float rt_unorder(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }

// The largest of the lanes' values and the lowest index that has it: a reduction of the whole warp in one instruction each.
__device__ __forceinline__ float rt_best(float v, int e, int& best) {
  const uint32_t mine = rt_order(v + 0.f), most = __reduce_max_sync(kAll, mine);   // (a negative zero is equal to zero)
  best = (int)__reduce_min_sync(kAll, mine == most ? (uint32_t)e : 0x7fffffffu);
  return rt_unorder(most);
}
__device__ __forceinline__ double rt_best(double v, int e, int& best) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double ov = __shfl_xor_sync(kAll, v, o);
    const int oe = __shfl_xor_sync(kAll, e, o);
    if (ov > v || (ov == v && oe < e)) {
      v = ov;
      e = oe;
    }
  }
  best = e;
  return v;
}

// Error of a float score + bias, relative to 1 + |bias| (scores are at most 1): expf, the sum of up to 1024 exponentials (32 a lane
// and five steps of a tree, each step half a last bit of what is there), the quotient and the sum with the bias are off by less
// than 48 halves of a step.
constexpr float kRouteSlack = 48.f * 0x1p-24f;

// the lane's NI logits, -infinity where there are none
template <typename T, int NI>
__device__ __forceinline__ void load_row(const T* row, int E, bool whole, float (&l)[NI]) {
  const int e0 = NI * (threadIdx.x & 31);
  constexpr int BYTES = NI * (int)sizeof(T);
  if constexpr (BYTES >= 8) {
    if (whole) {
      alignas(16) T v[NI];
      if (e0 < E) {
        if constexpr (BYTES == 8) {
          *reinterpret_cast<uint2*>(v) = __ldg(reinterpret_cast<const uint2*>(row + e0));
        } else {
#pragma unroll
          for (int k = 0; k < BYTES / 16; k++) reinterpret_cast<uint4*>(v)[k] = __ldg(reinterpret_cast<const uint4*>(row + e0) + k);
        }
      }
#pragma unroll
      for (int i = 0; i < NI; i++) l[i] = e0 < E ? static_cast<float>(v[i]) : -INFINITY;
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < NI; i++) l[i] = e0 + i < E ? static_cast<float>(row[e0 + i]) : -INFINITY;
}

template <typename K>
__device__ __forceinline__ void top_two(K v, K& b0, K& b1) {
  if (v > b0) {
    b1 = b0;
    b0 = v;
  } else if (v > b1) {
    b1 = v;
  }
}

// grp[g]: what group g counts, the sum of its group_top largest keys. Groups that are whole lanes are summed up by the lanes
// that hold them, others by a lane each, from shared memory behind the sums.
template <typename K, int NI>
__device__ __forceinline__ void count_groups(const RouteArgs& a, const K (&key)[NI], K* grp) {
  const int lane = threadIdx.x & 31, size = a.size, lanes = size / NI;
  if (size % NI == 0 && 32 % lanes == 0) {
    K b0 = -INFINITY, b1 = -INFINITY;
#pragma unroll
    for (int i = 0; i < NI; i++) top_two(key[i], b0, b1);
    for (int o = 1; o < lanes; o <<= 1) {
      const K c0 = __shfl_xor_sync(kAll, b0, o), c1 = __shfl_xor_sync(kAll, b1, o);
      top_two(c0, b0, b1);
      top_two(c1, b0, b1);
    }
    if (lane % lanes == 0 && lane / lanes < a.G) grp[lane / lanes] = a.group_top > 1 && b1 > -INFINITY ? b0 + b1 : b0;
  } else {
    K* all = grp + a.G;
#pragma unroll
    for (int i = 0; i < NI; i++)
      if (NI * lane + i < a.E) all[NI * lane + i] = key[i];
    __syncwarp();
    for (int g = lane; g < a.G; g += 32) {
      K b0 = -INFINITY, b1 = -INFINITY;
      for (int j = 0; j < size; j++) top_two(all[g * size + j], b0, b1);
      grp[g] = a.group_top > 1 && b1 > -INFINITY ? b0 + b1 : b0;
    }
  }
  __syncwarp();
}

// The groups that stay, a bit each. With a slack, returns whether sums that lie within it decide about one.
template <typename K>
__device__ __forceinline__ bool keep_groups(const RouteArgs& a, const K* grp, K slack, uint32_t* bits) {
  const int lane = threadIdx.x & 31;
  bool close = false;
  for (int g0 = 0; g0 < a.G; g0 += 32) {
    const int g = g0 + lane;
    bool in = false, near = false;
    if (g < a.G) {
      const K mine = grp[g];
      int ahead = 0, surely = 0, behind = 0;
      for (int h = 0; h < a.G; h++) {
        const K o = grp[h];
        ahead += o > mine || (o == mine && h < g);
        surely += o > mine + slack;
        behind += o < mine - slack;
      }
      in = ahead < a.top_groups;
      // neither out nor in whatever the doubtful ones are
      near = slack > 0 && surely < a.top_groups && a.G - 1 - behind >= a.top_groups;
    }
    const uint32_t m = __ballot_sync(kAll, in);
    if (lane == 0) bits[g0 / 32] = m;
    close = close || __any_sync(kAll, near);
  }
  __syncwarp();
  return close;
}

// keys of experts whose groups do not stay become -infinity
template <typename K, int NI>
__device__ __forceinline__ void drop_groups(const RouteArgs& a, const uint32_t* bits, K (&key)[NI]) {
  const int e0 = NI * (threadIdx.x & 31);
  int g = min(e0 / a.size, a.G - 1), left = (g + 1) * a.size - e0;
  uint32_t in = bits[g / 32] >> (g & 31) & 1;
#pragma unroll
  for (int i = 0; i < NI; i++) {
    if (left == 0 && g + 1 < a.G) {
      g++;
      left = a.size;
      in = bits[g / 32] >> (g & 31) & 1;
    }
    left--;
    if (!in) key[i] = -INFINITY;
  }
}

// The top_k largest keys, lowest index first among equals; lane r returns the r-th, -1 where none is left. With a slack: `close` is set,
// and the picks are void, where neighbours in the order lie within it and are not the same logit and bias in every bit.
template <typename T, typename K, int NI>
__device__ __forceinline__ int pick(const RouteArgs& a, const T* row, K (&key)[NI], const float (&l)[NI], const float (&bias)[NI], K slack, bool& close) {
  const int lane = threadIdx.x & 31, e0 = NI * lane;
  int win = -1, before = 0;
  K last = 0;
  for (int r = 0; r < a.top_k; r++) {
    K bv = -INFINITY;
    int be = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < NI; i++)
      if (key[i] > bv) {
        bv = key[i];
        be = e0 + i;
      }
    int best;
    const K top = rt_best(bv, be, best);
    if (best >= a.E) return win;   // no expert is left
    if (slack > 0 && r > 0 && !(last - top > slack) &&
        !(static_cast<float>(row[best]) == static_cast<float>(row[before]) && a.bias[best] == a.bias[before])) {
      close = true;
      return win;
    }
#pragma unroll
    for (int i = 0; i < NI; i++)
      if (e0 + i == best) key[i] = -INFINITY;
    last = top;
    before = best;
    if (lane == r) win = best;
  }
  if (slack > 0) {
    // the best of what is left and not the last pick's equal
    const float ll = static_cast<float>(row[before]), lb = a.bias[before];
    K bv = -INFINITY;
#pragma unroll
    for (int i = 0; i < NI; i++)
      if (!(l[i] == ll && bias[i] == lb) && key[i] > bv) bv = key[i];
    close = __any_sync(kAll, bv > -INFINITY && !(last - bv > slack));
  }
  return win;
}

template <typename T, int NI>
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(const RouteArgs a) {
  extern __shared__ double route_smem[];   // per warp, with groups: what they count, E keys, bits
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int token = blockIdx.x * kRouteWarps + warp;
  if (token >= a.T) return;
  double* grp = route_smem + (size_t)warp * (a.G + a.E + 16);
  uint32_t* bits = reinterpret_cast<uint32_t*>(grp + a.G + a.E);
  const T* row = static_cast<const T*>(a.logits) + (long long)token * a.E;
  const int e0 = NI * lane;
  float l[NI], key[NI], bias[NI];
  load_row<T, NI>(row, a.E, a.whole, l);
#pragma unroll
  for (int i = 0; i < NI; i++) bias[i] = a.bias != nullptr && e0 + i < a.E ? a.bias[e0 + i] : 0.f;
  float fm = 0.f, fz = 1.f;   // softmax: the largest logit, the sum of exponentials
  if (a.scoring == 0) {
    float m = -INFINITY, s = 0.f;
#pragma unroll
    for (int i = 0; i < NI; i++) m = fmaxf(m, l[i]);
    fm = rt_max(m);
#pragma unroll
    for (int i = 0; i < NI; i++) s += l[i] == -INFINITY ? 0.f : expf(l[i] - fm);
    fz = rt_sum(s);
  }
  // what experts are ranked by, and groups
  const bool by_score = a.bias != nullptr, groups_by_score = by_score || a.group_top > 1;
  auto by_logit = [&](float x) { return x == x ? x : INFINITY; };   // NaN comes first, so that it is seen
  float slack = kRouteSlack;
  if (by_score || (a.G > 1 && groups_by_score)) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const float q = (a.scoring == 0 ? expf(l[i] - fm) / fz : rt_sigmoid(l[i])) + bias[i];
      key[i] = l[i] == -INFINITY ? -INFINITY : by_logit(q);
      if (fabsf(bias[i]) < INFINITY) most = fmaxf(most, fabsf(bias[i]));
    }
    if (by_score) slack *= 1.f + rt_max(most);
  } else {
#pragma unroll
    for (int i = 0; i < NI; i++) key[i] = by_logit(l[i]);
  }
  bool close = false;
  int win = -1;
  if (a.G > 1) {
    float* g32 = reinterpret_cast<float*>(grp);
    count_groups<float, NI>(a, key, g32);
    close = keep_groups<float>(a, g32, groups_by_score ? 4.f * slack : 0.f, bits);   // (each of two sums of two)
    if (!by_score) {
#pragma unroll
      for (int i = 0; i < NI; i++) key[i] = by_logit(l[i]);
    }
    drop_groups<float, NI>(a, bits, key);
  }
  if (!close) win = pick<T, float, NI>(a, row, key, l, bias, by_score ? 2.f * slack : 0.f, close);
  if (close) {
    double z = 1., q[NI];
    if (a.scoring == 0) {
      double s = 0.;
#pragma unroll
      for (int i = 0; i < NI; i++) s += l[i] == -INFINITY ? 0. : exp((double)l[i] - (double)fm);
      z = rt_sum(s);
    }
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const double v = (a.scoring == 0 ? exp((double)l[i] - (double)fm) / z : 1. / (1. + exp(-(double)l[i]))) + (double)bias[i];
      q[i] = l[i] == -INFINITY ? -INFINITY : v == v ? v : INFINITY;
    }
    if (a.G > 1) {
      __syncwarp();   // (the floats' sums have been read)
      count_groups<double, NI>(a, q, grp);
      keep_groups<double>(a, grp, 0., bits);
      if (!by_score) {
#pragma unroll
        for (int i = 0; i < NI; i++) q[i] = by_logit(l[i]);
      }
      drop_groups<double, NI>(a, bits, q);
    }
    win = pick<T, double, NI>(a, row, q, l, bias, 0., close);
  }
  float score = 0.f;
  if (win >= 0) {
    const float x = static_cast<float>(row[win]);
    score = a.scoring == 0 ? expf(x - fm) / fz : rt_sigmoid(x);
  }
  if (a.norm) score /= rt_sum(score) + 1e-20f;
  if (lane < a.top_k) {
    const long long at = (long long)token * a.top_k + lane;
    a.indices[at] = win;
    a.weights[at] = a.scale * score;
  }
}

// dl from dw. A warp per token; everything but the picks is zero, except with softmax scores that are not renormalised.
template <typename T, int NI>
__global__ void __launch_bounds__(32 * kRouteWarps) route_backward_kernel(const RouteArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int token = blockIdx.x * kRouteWarps + warp;
  if (token >= a.T) return;
  const T* row = static_cast<const T*>(a.logits) + (long long)token * a.E;
  T* out = static_cast<T*>(a.dlogits) + (long long)token * a.E;
  const int e0 = NI * lane;
  int idx = -1;
  float x = 0.f, s = 0.f, dw = 0.f;
  if (lane < a.top_k) {
    idx = a.indices[(long long)token * a.top_k + lane];
    if (idx >= a.E) idx = -1;
    if (idx >= 0) {
      dw = a.scale * a.dw[(long long)token * a.top_k + lane];
      x = static_cast<float>(row[idx]);
    }
  }
  float l[NI], fm = 0.f, fz = 1.f;
  if (a.scoring == 0) {
    load_row<T, NI>(row, a.E, a.whole, l);
    float m = -INFINITY, z = 0.f;
#pragma unroll
    for (int i = 0; i < NI; i++) m = fmaxf(m, l[i]);
    fm = rt_max(m);
#pragma unroll
    for (int i = 0; i < NI; i++) z += l[i] == -INFINITY ? 0.f : expf(l[i] - fm);
    fz = rt_sum(z);
  }
  if (idx >= 0) s = a.scoring == 0 ? expf(x - fm) / fz : rt_sigmoid(x);
  float ds = dw;
  if (a.norm) {
    const float S = rt_sum(s) + 1e-20f;
    ds = (dw - rt_sum(dw * (s / S))) / S;
  }
  const float dl = a.scoring == 1 ? ds * s * rt_sigmoid(-x) : ds * s;
  float d[NI];
  const float all = a.scoring == 0 && !a.norm ? rt_sum(dl) : 0.f;
#pragma unroll
  for (int i = 0; i < NI; i++) d[i] = a.scoring == 0 && !a.norm && l[i] != -INFINITY ? -(expf(l[i] - fm) / fz) * all : 0.f;
  for (int r = 0; r < a.top_k; r++) {
    const int e = __shfl_sync(kAll, idx, r);
    const float v = __shfl_sync(kAll, dl, r);
#pragma unroll
    for (int i = 0; i < NI; i++)
      if (e0 + i == e) d[i] += v;
  }
  constexpr int BYTES = NI * (int)sizeof(T);
  if constexpr (BYTES >= 8) {
    if (a.whole) {
      if (e0 >= a.E) return;
      alignas(16) T v[NI];
#pragma unroll
      for (int i = 0; i < NI; i++) v[i] = static_cast<T>(d[i]);
      if constexpr (BYTES == 8) {
        *reinterpret_cast<uint2*>(out + e0) = *reinterpret_cast<const uint2*>(v);
      } else {
#pragma unroll
        for (int k = 0; k < BYTES / 16; k++) reinterpret_cast<uint4*>(out + e0)[k] = reinterpret_cast<const uint4*>(v)[k];
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < NI; i++)
    if (e0 + i < a.E) out[e0 + i] = static_cast<T>(d[i]);
}

template <typename T, int NI>
cudaError_t route_launch(RouteArgs& a, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.T + kRouteWarps - 1) / kRouteWarps);
  // a lane's experts lie whole on a boundary of 16 bytes, or of their size
  constexpr int BYTES = NI * (int)sizeof(T), STEP = BYTES < 16 ? BYTES : 16;
  const uintptr_t all = reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.dlogits) | (uintptr_t)(a.E * sizeof(T));
  a.whole = a.E % NI == 0 && all % STEP == 0;
  if (a.dlogits != nullptr) {
    route_backward_kernel<T, NI><<<grid, 32 * kRouteWarps, 0, st>>>(a);
    return cudaGetLastError();
  }
  a.size = a.E / a.G;
  const size_t smem = a.G > 1 ? (size_t)kRouteWarps * (a.E + a.G + 16) * sizeof(double) : 0;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(route_kernel<T, NI>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  route_kernel<T, NI><<<grid, 32 * kRouteWarps, smem, st>>>(a);
  return cudaGetLastError();
}
template <typename T>
cudaError_t route_width(RouteArgs& a, cudaStream_t st) {
  if (a.E <= 64) return route_launch<T, 2>(a, st);
  if (a.E <= 128) return route_launch<T, 4>(a, st);
  if (a.E <= 256) return route_launch<T, 8>(a, st);
  if (a.E <= 512) return route_launch<T, 16>(a, st);
  return route_launch<T, 32>(a, st);
}

}  // namespace

cudaError_t launch_route(RouteArgs a, cudaStream_t st) {
  if (a.dtype == F32) return route_width<float>(a, st);
  if (a.dtype == F16) return route_width<__half>(a, st);
  return route_width<__nv_bfloat16>(a, st);
}

}  // namespace kq
