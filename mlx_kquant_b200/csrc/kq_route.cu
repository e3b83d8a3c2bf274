// Routing to experts in groups, and its gradient (kq_moe_router_grouped, kq_moe_router_grouped_backward).
//
// Row of logits l[E]: scores s = sigmoid(l) or softmax(l), ranked by q = s + bias (without a bias by l itself: the scores rise
// with it). A group of E / G neighbours counts by the sum of its group_top largest q; the top_groups best groups stay, of
// these the top_k largest q are picked, lowest index first among equals, groups and experts alike. Weights
// w_j = scale * s_ij / (sum s_i + 1e-20), or scale * s_ij.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kq_common.cuh"
#include "kq_route.h"

namespace kq {
namespace {

constexpr int kRouteWarps = 4;

template <typename T>
__device__ __forceinline__ float rt_float(T v) { return static_cast<float>(v); }

__device__ __forceinline__ double rt_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float rt_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float rt_sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// One warp per token; lane l holds experts l, l + 32, ...
template <typename T, int NI>
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(const RouteArgs a) {
  extern __shared__ double route_smem[];   // per warp: E keys, G group scores
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int token = blockIdx.x * kRouteWarps + warp;
  if (token >= a.T) return;
  double* key_s = route_smem + (size_t)warp * (a.E + a.G);
  double* grp_s = key_s + a.E;
  const T* row = static_cast<const T*>(a.logits) + (long long)token * a.E;
  float l[NI];
  double key[NI];
#pragma unroll
  for (int i = 0; i < NI; i++) {
    const int e = lane + 32 * i;
    l[i] = e < a.E ? rt_float(row[e]) : -INFINITY;
  }
  float fm = 0.f, fz = 1.f;   // softmax: largest logit, sum of exponentials
  if (a.scoring == 0) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NI; i++) m = fmaxf(m, l[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NI; i++) s += l[i] == -INFINITY ? 0.f : expf(l[i] - m);
    fz = rt_sum(s);
    fm = m;
  }
  const bool scored = a.bias != nullptr || (a.G > 1 && a.group_top > 1);   // else the logits say all
  double z = 1.;
  if (scored && a.scoring == 0) {
    double s = 0.;
#pragma unroll
    for (int i = 0; i < NI; i++) s += l[i] == -INFINITY ? 0. : exp((double)l[i] - (double)fm);
    z = rt_sum(s);
  }
#pragma unroll
  for (int i = 0; i < NI; i++) {
    const int e = lane + 32 * i;
    double q = l[i];
    if (scored) {
      q = a.scoring == 0 ? exp((double)l[i] - (double)fm) / z : 1. / (1. + exp(-(double)l[i]));
      if (a.bias != nullptr && e < a.E) q += a.bias[e];
    }
    if (q != q) q = INFINITY;               // NaN comes first, so that it is seen
    key[i] = l[i] == -INFINITY ? -INFINITY : q;
  }
  if (a.G > 1) {
#pragma unroll
    for (int i = 0; i < NI; i++)
      if (lane + 32 * i < a.E) key_s[lane + 32 * i] = key[i];
    __syncwarp();
    const int size = a.E / a.G;
    for (int g = lane; g < a.G; g += 32) {
      double b0 = -INFINITY, b1 = -INFINITY;
      for (int j = 0; j < size; j++) {
        const double v = key_s[g * size + j];
        if (v > b0) { b1 = b0; b0 = v; }
        else if (v > b1) b1 = v;
      }
      grp_s[g] = a.group_top > 1 && b1 > -INFINITY ? b0 + b1 : b0;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const int e = lane + 32 * i;
      if (e >= a.E) continue;
      const int g = e / size;
      const double mine = grp_s[g];
      int ahead = 0;
      for (int h = 0; h < a.G; h++) ahead += grp_s[h] > mine || (grp_s[h] == mine && h < g);
      if (ahead >= a.top_groups) key[i] = -INFINITY;
      else if (a.bias == nullptr) key[i] = l[i] == l[i] ? (double)l[i] : INFINITY;
    }
  }
  int win_i = -1;          // lane r keeps the r-th pick
  float win_s = 0.f, total = 0.f;
  for (int r = 0; r < a.top_k; r++) {
    double bv = -INFINITY;
    int bi = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < NI; i++)
      if (key[i] > bv) {
        bv = key[i];
        bi = lane + 32 * i;
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
      if (ov > bv || (ov == bv && oi < bi)) {
        bv = ov;
        bi = oi;
      }
    }
    if (bi == 0x7fffffff) break;            // no expert is left
    float pick = 0.f;
#pragma unroll
    for (int i = 0; i < NI; i++)
      if (lane + 32 * i == bi) {
        pick = l[i];
        key[i] = -INFINITY;
      }
    pick = __shfl_sync(0xffffffffu, pick, bi & 31);
    const float s = a.scoring == 0 ? expf(pick - fm) / fz : rt_sigmoid(pick);
    total += s;
    if (lane == r) {
      win_i = bi;
      win_s = s;
    }
  }
  if (lane < a.top_k) {
    const long long at = (long long)token * a.top_k + lane;
    a.indices[at] = win_i;
    a.weights[at] = win_i < 0 ? 0.f : a.scale * (a.norm ? win_s / (total + 1e-20f) : win_s);
  }
}

// dl from dw. A warp per token; everything but the picks is zero, except with softmax scores that are not renormalised.
template <typename T>
__global__ void __launch_bounds__(32 * kRouteWarps) route_backward_kernel(const RouteArgs a) {
  extern __shared__ double route_smem[];   // per warp: E floats
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int token = blockIdx.x * kRouteWarps + warp;
  if (token >= a.T) return;
  float* d = reinterpret_cast<float*>(route_smem) + (size_t)warp * a.E;
  const T* row = static_cast<const T*>(a.logits) + (long long)token * a.E;
  T* out = static_cast<T*>(a.dlogits) + (long long)token * a.E;
  float fm = 0.f, fz = 1.f;
  if (a.scoring == 0) {
    float m = -INFINITY;
    for (int e = lane; e < a.E; e += 32) m = fmaxf(m, rt_float(row[e]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float s = 0.f;
    for (int e = lane; e < a.E; e += 32) {
      const float v = rt_float(row[e]);
      s += v == -INFINITY ? 0.f : expf(v - m);
    }
    fz = rt_sum(s);
    fm = m;
  }
  int idx = -1;
  float x = 0.f, s = 0.f, dw = 0.f;
  if (lane < a.top_k) {
    idx = a.indices[(long long)token * a.top_k + lane];
    if (idx >= a.E) idx = -1;
    if (idx >= 0) {
      dw = a.scale * a.dw[(long long)token * a.top_k + lane];
      x = rt_float(row[idx]);
      s = a.scoring == 0 ? expf(x - fm) / fz : rt_sigmoid(x);
    }
  }
  float ds = dw;
  if (a.norm) {
    const float S = rt_sum(s) + 1e-20f;
    ds = (dw - rt_sum(dw * (s / S))) / S;
  }
  float dl;
  float all = 0.f;
  if (a.scoring == 1) dl = ds * s * rt_sigmoid(-x);
  else if (a.norm) dl = ds * s;
  else {
    dl = ds * s;
    all = rt_sum(dl);
  }
  for (int e = lane; e < a.E; e += 32) {
    float v = 0.f;
    if (a.scoring == 0 && !a.norm) {
      const float xe = rt_float(row[e]);
      v = xe == -INFINITY ? 0.f : -(expf(xe - fm) / fz) * all;
    }
    d[e] = v;
  }
  __syncwarp();
  if (idx >= 0) d[idx] += dl;
  __syncwarp();
  for (int e = lane; e < a.E; e += 32) out[e] = static_cast<T>(d[e]);
}

template <typename T>
cudaError_t route_launch(const RouteArgs& a, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.T + kRouteWarps - 1) / kRouteWarps);
  if (a.dlogits != nullptr) {
    route_backward_kernel<T><<<grid, 32 * kRouteWarps, kRouteWarps * a.E * sizeof(float), st>>>(a);
    return cudaGetLastError();
  }
  const size_t smem = a.G > 1 ? (size_t)kRouteWarps * (a.E + a.G) * sizeof(double) : 0;
  auto kern = a.E <= 128 ? route_kernel<T, 4> : a.E <= 256 ? route_kernel<T, 8> : a.E <= 512 ? route_kernel<T, 16> : route_kernel<T, 32>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  kern<<<grid, 32 * kRouteWarps, smem, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_route(const RouteArgs& a, cudaStream_t st) {
  if (a.dtype == F32) return route_launch<float>(a, st);
  if (a.dtype == F16) return route_launch<__half>(a, st);
  return route_launch<__nv_bfloat16>(a, st);
}

}  // namespace kq
