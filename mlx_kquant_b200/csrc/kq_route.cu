// Routing to experts in groups, and its gradient (kq_moe_router_grouped, kq_moe_router_grouped_backward).
//
// Row of logits l[E]: scores s = sigmoid(l) or softmax(l), ranked by q = s + bias (without a bias by l itself: the scores rise
// with it). A group of E / G neighbours counts by the sum of its group_top largest q; the top_groups best groups stay, of
// these the top_k largest q are picked, lowest index first among equals, groups and experts alike. Weights
// w_j = scale * s_ij / (sum s_i + 1e-20), or scale * s_ij.
//
// A warp per token, a lane NI neighbouring experts, all in registers. The order is that of 64 bits; exponentials and sums in 64 bits
// for all experts took 66 us for 16384 tokens of 256 experts in 8 groups, this kernel takes 22. It ranks 32-bit codes: what an expert
// is ranked by in the upper bits (score + bias as fixed point over the range of the biases, or a logit's leading bits), its index,
// counted down, in the lower ones. A lane sorts its codes, and each pick is one warp-wide maximum of the lanes' first. The codes'
// error is bounded (kRouteSlack): where neighbours in the order of the picks, the last of them and the best that is left, or the
// sums around the border of the groups lie no further apart than that, and are not the same logit and bias bit for bit (one token
// in 250 of normally distributed logits), the token is ranked again with 64 bits for its 32 best codes and for the experts that
// count for the groups, and if that leaves a doubt with 64 bits for all (which one token alone takes 12 us for). A code holds all
// of a 16-bit logit: without a bias and sums nothing is ever ranked again. Half of the time is instruction issue,
// some 800 a token, a tenth the tokens that are ranked again; the rest is the latency of dependent maxima.
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

// the largest of the lanes' values, and the lowest index that has it
__device__ __forceinline__ void rt_best(double v, int e, int& best) {
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
}

// Error of a float score + bias, relative to 1 + |bias| (scores are at most 1): the exponential and the quotient in their fast forms
// (2 + 1.16 |x| and 2 steps, the former weighted with s (1 - s)), the sum of up to 1024 exponentials (32 a lane and five steps of
// a tree, half a last bit each) and the sum with the bias are off by less than 48 halves of a step.
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

// The top_k largest keys, lowest index first among equals; lane r returns the r-th, -1 where none is left.
template <int NI>
__device__ __forceinline__ int pick(const RouteArgs& a, double (&key)[NI]) {
  const int lane = threadIdx.x & 31, e0 = NI * lane;
  int win = -1;
  for (int r = 0; r < a.top_k; r++) {
    double bv = -INFINITY;
    int be = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < NI; i++)
      if (key[i] > bv) {
        bv = key[i];
        be = e0 + i;
      }
    int best;
    rt_best(bv, be, best);
    if (best >= a.E) return win;   // no expert is left
#pragma unroll
    for (int i = 0; i < NI; i++)
      if (e0 + i == best) key[i] = -INFINITY;
    if (lane == r) win = best;
  }
  return win;
}

__device__ __forceinline__ float rt_first(float x) { return x == x ? x : INFINITY; }   // NaN comes first, so that it is seen

// softmax: the largest logit, and the sum of the exponentials, which replace the logits' in s
template <int NI>
__device__ __forceinline__ void softmax(const float (&l)[NI], float (&s)[NI], float& fm, float& fz) {
  float m = -INFINITY, z = 0.f;
#pragma unroll
  for (int i = 0; i < NI; i++) m = fmaxf(m, l[i]);
  fm = rt_max(m);
#pragma unroll
  for (int i = 0; i < NI; i++) {
    s[i] = l[i] == -INFINITY ? 0.f : expf(l[i] - fm);
    z += s[i];
  }
  fz = rt_sum(z);
}

// lane r has the r-th pick, or -1
template <typename T>
__device__ __forceinline__ void store_picks(const RouteArgs& a, int token, const T* row, int win, float fm, float fz) {
  const int lane = threadIdx.x & 31;
  float score = 0.f;
  if (win >= 0) {
    const float x = static_cast<float>(row[win]);
    // (quotients within two steps)
    score = a.scoring == 0 ? __fdividef(expf(x - fm), fz) : __fdividef(1.f, 1.f + expf(-x));
    if (a.scoring != 0 && x < -80.f) score = expf(x);   // (1 + e^-x beyond the range of that quotient)
  }
  if (a.norm) score = __fdividef(score, rt_sum(score) + 1e-20f);
  if (lane < a.top_k) {
    const long long at = (long long)token * a.top_k + lane;
    a.indices[at] = win;
    a.weights[at] = a.scale * score;
  }
}

// A token as 64 bits have it.
template <typename T, int NI>
__device__ __forceinline__ void route_exactly(const RouteArgs& a, int token, const T* row, double* grp, uint32_t* bits) {
  const int e0 = NI * (threadIdx.x & 31);
  float fm = 0.f, fz = 1.f;
  float l[NI];
  double z = 1., q[NI];
  load_row<T, NI>(row, a.E, a.whole, l);
  if (a.scoring == 0) {
    float e[NI];
    softmax<NI>(l, e, fm, fz);
    double s = 0.;
#pragma unroll
    for (int i = 0; i < NI; i++) s += l[i] == -INFINITY ? 0. : exp((double)l[i] - (double)fm);
    z = rt_sum(s);
  }
#pragma unroll
  for (int i = 0; i < NI; i++) {
    double v = a.scoring == 0 ? exp((double)l[i] - (double)fm) / z : 1. / (1. + exp(-(double)l[i]));
    if (a.bias != nullptr && e0 + i < a.E) v += (double)a.bias[e0 + i];
    q[i] = l[i] == -INFINITY ? -INFINITY : v == v ? v : INFINITY;
  }
  if (a.G > 1) {
    if (a.bias == nullptr && a.group_top == 1) {
#pragma unroll
      for (int i = 0; i < NI; i++) q[i] = rt_first(l[i]);
    }
    __syncwarp();
    count_groups<double, NI>(a, q, grp);
    keep_groups<double>(a, grp, 0., bits);
  }
  if (a.bias == nullptr) {
#pragma unroll
    for (int i = 0; i < NI; i++) q[i] = rt_first(l[i]);
  }
  if (a.G > 1) drop_groups<double, NI>(a, bits, q);
  store_picks<T>(a, token, row, pick<NI>(a, q), fm, fz);
  __syncwarp();
}

__device__ __forceinline__ void sort_pair(uint32_t& a, uint32_t& b) {
  const uint32_t m = max(a, b);
  b = min(a, b);
  a = m;
}
// descending, by a network of odd and even merges
template <int N>
__device__ __forceinline__ void sort_codes(uint32_t (&c)[N]) {
#pragma unroll
  for (int p = 1; p < N; p <<= 1)
#pragma unroll
    for (int k = p; k >= 1; k >>= 1)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; i++)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) sort_pair(c[i + j], c[i + j + k]);
}

__device__ __forceinline__ float fast_sigmoid(float x) {
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(e) : "f"(x * -1.44269504f));
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(s) : "f"(1.f + e));
  return s;
}
// the two largest of (b0, b1) and (c0, c1), both in order
__device__ __forceinline__ void merge_two(uint32_t c0, uint32_t c1, uint32_t& b0, uint32_t& b1) {
  b1 = max(min(b0, c0), max(b1, c1));
  b0 = max(b0, c0);
}

template <int NI>
constexpr int route_ctas() { return NI <= 4 ? 6 : NI == 8 ? 5 : NI == 16 ? 4 : 2; }   // of an SM: more of them spill

template <typename T, int NI>
__global__ void __launch_bounds__(32 * kRouteWarps, route_ctas<NI>()) route_kernel(const RouteArgs a) {
  constexpr int IB = NI == 2 ? 6 : NI == 4 ? 7 : NI == 8 ? 8 : NI == 16 ? 9 : 10;   // bits of an expert's index
  constexpr uint32_t IM = (1u << IB) - 1;
  constexpr float UNITS = (float)(1ull << (32 - IB)) - 1024.f;
  extern __shared__ double route_smem[];   // per warp, with groups: what they count, E keys, bits
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;\n" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = NI * lane;
  double* grp = route_smem + (size_t)warp * (a.G + a.E + 16);
  uint32_t* bits = reinterpret_cast<uint32_t*>(grp + a.G + a.E);
  // what experts are ranked by, and groups; a logit of 16 bits is all in its code
  const bool by_score = a.bias != nullptr, groups_by_score = by_score || a.group_top > 1;
  const bool sure = !by_score && sizeof(T) == 2;
  float bias[NI], lo = 0.f, hi = 1.f, slack = kRouteSlack;
  bool odd = false;        // biases that a code cannot hold
  if (by_score) {
    load_row<float, NI>(a.bias, a.E, a.whole_bias, bias);
    float least = INFINITY, most = -INFINITY;
#pragma unroll
    for (int i = 0; i < NI; i++)
      if (e0 + i < a.E) {
        odd |= !(fabsf(bias[i]) < 1e30f);
        least = fminf(least, bias[i]);
        most = fmaxf(most, bias[i]);
      }
    lo = -rt_max(-least);
    hi = rt_max(most) + 1.f;
    if (a.G > 1 && a.group_top > 1) {   // the range holds zero too, which is what the second of a single available expert counts
      lo = fminf(lo, 0.f);
      hi = fmaxf(hi, 0.f);
    }
    slack *= 1.f + fmaxf(fabsf(lo), fabsf(hi));
    odd = __any_sync(kAll, odd);
  }
  // score + bias as fixed point: unit * s + shift, from 0 at the least bias (or at zero); a code's upper bits are one more
  const float unit = UNITS / (hi - lo);
  const uint32_t nothing = by_score ? (uint32_t)(-lo * unit) + 1u : 0u;   // a sum of two holds the range's offset twice, of one likewise then
  float shift[NI];
#pragma unroll
  for (int i = 0; i < NI; i++) shift[i] = by_score ? (bias[i] - lo) * unit : 0.f;
  const uint32_t unsure = (uint32_t)fminf(2.f * slack * unit + 4.f, 1e9f);   // of two codes
  const uint32_t close_by = by_score ? unsure : 0u, groups_close_by = groups_by_score ? 2 * unsure : 0u;
  const int lanes = a.G > 1 ? a.size / NI : 1;   // of a group
  const bool whole_groups = a.G > 1 && a.G <= 32 && a.size % NI == 0 && 32 % lanes == 0;

  // Up to 32 tokens at a time, then those of them that the codes could not rank: once more with 64 bits for the best 32 codes, and for
  // the experts that count for the groups; and if that too leaves a doubt, with 64 bits for all.
  const int stride = gridDim.x * kRouteWarps;
  int ahead = blockIdx.x * kRouteWarps + warp, first = ahead, it = 0;   // the next token; the first of these 32, how many of them
  uint32_t again = 0;
  bool exactly = false;
  for (;;) {
    int token = ahead;
    if (!exactly && (ahead >= a.T || it == 32)) exactly = true;
    if (exactly) {
      if (again == 0) {
        if (ahead >= a.T) break;
        exactly = false;
        first = ahead;
        it = 0;
        continue;
      }
      token = first + (__ffs(again) - 1) * stride;
      again &= again - 1;
    } else {
      ahead = ahead < a.T - stride ? ahead + stride : a.T;
    }
    const T* row = static_cast<const T*>(a.logits) + (long long)token * a.E;
    if (exactly && a.scoring == 0 && groups_by_score && (by_score || a.G > 1)) {   // (the sum of the exponentials in 64 bits too)
      route_exactly<T, NI>(a, token, row, grp, bits);
      continue;
    }
    float l[NI];
    load_row<T, NI>(row, a.E, a.whole, l);
    float s[NI];
    bool close = odd;
    float fm = 0.f, fz = 1.f;
    if (a.scoring == 0) {
      softmax<NI>(l, s, fm, fz);
      const float over = 1.f / fz;
#pragma unroll
      for (int i = 0; i < NI; i++) s[i] *= over;
    } else if (by_score || (a.G > 1 && groups_by_score)) {
#pragma unroll
      for (int i = 0; i < NI; i++) s[i] = fast_sigmoid(l[i]);
    }
    // a NaN's code would not come first; scores that are not numbers the full form has to deal with
    bool nan = false;
#pragma unroll
    for (int i = 0; i < NI; i++) nan |= l[i] != l[i];
    nan |= fz != fz;
    close |= __any_sync(kAll, nan);
    auto score_of = [&](uint32_t code) {   // of an expert, in 64 bits (sigmoid)
      const int e = (int)(IM - (code & IM));
      const double v = 1. / (1. + exp(-(double)static_cast<float>(row[e])));
      return by_score ? v + (double)a.bias[e] : v;
    };
    uint32_t code[NI], by[NI];   // of the scores, and what experts are ranked by
    if (by_score || (a.G > 1 && groups_by_score)) {
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const uint32_t v = (uint32_t)fmaf(s[i], unit, shift[i]);
        code[i] = l[i] == -INFINITY ? 0u : (v << IB) + ((1u << IB) + IM - (uint32_t)(e0 + i));
      }
    }
    if (!by_score) {
#pragma unroll
      for (int i = 0; i < NI; i++) by[i] = l[i] == -INFINITY ? 0u : (rt_order(l[i] + 0.f) & ~IM) | (IM - (uint32_t)(e0 + i));
    }
    if (a.G > 1) {
      if (whole_groups) {
        uint32_t b0 = 0, b1 = 0;
#pragma unroll
        for (int i = 0; i < NI; i++) merge_two(groups_by_score ? code[i] : by[i], 0, b0, b1);
        for (int o = 1; o < lanes; o <<= 1) merge_two(__shfl_xor_sync(kAll, b0, o), __shfl_xor_sync(kAll, b1, o), b0, b1);
        // lane g comes to have group g: what it counts, and its index counted down; none without an expert
        const uint32_t second = b1 != 0 ? b1 >> IB : b0 != 0 ? nothing : 0u;
        const uint32_t count = __shfl_sync(kAll, a.group_top > 1 ? (b0 >> IB) + second : b0 >> IB, lane * lanes & 31);
        const uint32_t whole = lane < a.G && count != 0 ? count << 5 | (31 - lane) : 0u;
        uint32_t mine = whole, last = 0;
        bool stays = false;
        for (int r = 0; r < a.top_groups; r++) {
          last = __reduce_max_sync(kAll, mine);
          if (mine == last) {
            mine = 0;
            stays = true;
          }
        }
        const uint32_t next = __reduce_max_sync(kAll, mine);
        if (next != 0 && (sizeof(T) == 4 || groups_by_score) && (last >> 5) - (next >> 5) <= groups_close_by) {
          if (!exactly || !groups_by_score) {
            close = true;
          } else {
            // the experts that count, if no other comes near them: their scores' sum
            uint32_t third = 0;
#pragma unroll
            for (int i = 0; i < NI; i++)
              if (code[i] < (a.group_top > 1 ? b1 : b0)) third = max(third, code[i]);
            for (int o = 1; o < lanes; o <<= 1) third = max(third, __shfl_xor_sync(kAll, third, o));
            close |= __any_sync(kAll, third != 0 && ((a.group_top > 1 ? b1 : b0) >> IB) - (third >> IB) <= unsure);
            const uint32_t c0 = __shfl_sync(kAll, b0, lane * lanes & 31), c1 = __shfl_sync(kAll, b1, lane * lanes & 31);
            double v = -INFINITY;
            if (whole != 0) {
              v = score_of(c0);
              if (a.group_top > 1 && c1 != 0) v += score_of(c1);
            }
            int ahead = 0;
            for (int h = 0; h < a.G; h++) {
              const double o = __shfl_sync(kAll, v, h);
              ahead += o > v || (o == v && h < lane);
            }
            stays = whole != 0 && ahead < a.top_groups;
          }
        }
        const uint32_t kept = __ballot_sync(kAll, stays);
        if (!(kept >> (lane / lanes) & 1)) {
#pragma unroll
          for (int i = 0; i < NI; i++) code[i] = by[i] = 0;
        }
      } else {
        float* g32 = reinterpret_cast<float*>(grp);
        float key[NI];
#pragma unroll
        for (int i = 0; i < NI; i++) key[i] = l[i] == -INFINITY ? -INFINITY : !groups_by_score ? l[i] : by_score ? s[i] + bias[i] : s[i];
        __syncwarp();
        count_groups<float, NI>(a, key, g32);
        close |= keep_groups<float>(a, g32, groups_by_score ? 4.f * slack : 0.f, bits);
#pragma unroll
        for (int i = 0; i < NI; i++) key[i] = 0.f;
        drop_groups<float, NI>(a, bits, key);
#pragma unroll
        for (int i = 0; i < NI; i++)
          if (key[i] < 0.f) code[i] = by[i] = 0;
      }
    }
    if (by_score) {
#pragma unroll
      for (int i = 0; i < NI; i++) by[i] = code[i];
    }
    sort_codes<NI>(by);
    uint32_t mine = 0;       // lane r: the r-th pick's code; one more, where it has to be told how near that comes
    const int rounds = exactly ? 32 : sure ? a.top_k : min(32, a.top_k + 1);
    for (int r = 0; r < rounds; r++) {
      const uint32_t top = __reduce_max_sync(kAll, by[0]);
      const bool took = by[0] == top;
      mine = lane == r ? top : mine;
#pragma unroll
      for (int i = 0; i < NI - 1; i++) by[i] = took ? by[i + 1] : by[i];   // (selected, not branched over)
      by[NI - 1] = took ? 0u : by[NI - 1];
    }
    int e = mine != 0 ? (int)(IM - (mine & IM)) : -1;
    if (exactly) {
      const uint32_t end = __shfl_sync(kAll, mine, 31), least = __shfl_sync(kAll, mine, a.top_k - 1);
      close |= a.top_k == 32 || (end != 0 && (least >> IB) - (end >> IB) <= close_by);   // more than 32 come near
      const double v = mine == 0 ? -INFINITY : by_score ? score_of(mine) : (double)static_cast<float>(row[e]);
      int place = 0;
      for (int h = 0; h < 32; h++) {
        const double o = __shfl_sync(kAll, v, h);
        const int f = __shfl_sync(kAll, e, h);
        place += o > v || (o == v && f < e && f >= 0);
      }
      if (e < 0) place = 32;
      int win = -1;
      for (int h = 0; h < 32; h++) {
        const int p = __shfl_sync(kAll, place, h), f = __shfl_sync(kAll, e, h);
        if (p == lane) win = f;
      }
      e = win;
    } else if (!sure) {
      const uint32_t before = __shfl_up_sync(kAll, mine, 1);
      const bool near = lane > 0 && mine != 0 && (before >> IB) - (mine >> IB) <= close_by;
      if (__any_sync(kAll, near)) {
        // equals in every bit keep the order of their indices; what follows the last one is not known
        bool same = false;
        if (near && lane < a.top_k) {
          const int f = (int)(IM - (before & IM));
          same = static_cast<float>(row[e]) == static_cast<float>(row[f]) && (!by_score || a.bias[e] == a.bias[f]);
        }
        close |= __any_sync(kAll, near && !same);
      }
      close |= a.top_k == 32;
    }
    if (!close) store_picks<T>(a, token, row, lane < a.top_k ? e : -1, fm, fz);
    else if (exactly) route_exactly<T, NI>(a, token, row, grp, bits);
    else again |= 1u << it;
    if (!exactly) it++;
  }
}

// dl from dw. A warp per token; everything but the picks is zero, except with softmax scores that are not renormalised (or whose picks'
// sum is next to nothing).
template <typename T, int NI>
__global__ void __launch_bounds__(32 * kRouteWarps) route_backward_kernel(const RouteArgs a) {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;\n" ::: "memory");
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
  // softmax: every expert has -s times the picks' sum of ds s. Renormalised, that is dw's mean over the picks times 1e-20 / S: beside the
  // row's other entries less than half a float's last bit, and left away, as long as S is above 1e-12.
  float ds = dw, all = 0.f;
  bool whole_row = a.scoring == 0;
  if (a.norm) {
    const float S = rt_sum(s) + 1e-20f, mean = rt_sum(dw * (s / S));
    ds = (dw - mean) / S;
    all = mean * (1e-20f / S);
    whole_row = whole_row && S < 1e-12f;
  }
  const float dl = a.scoring == 1 ? ds * s * rt_sigmoid(-x) : ds * s;
  if (!a.norm && whole_row) all = rt_sum(dl);
  float d[NI];
#pragma unroll
  for (int i = 0; i < NI; i++) d[i] = whole_row && l[i] != -INFINITY ? -(expf(l[i] - fm) / fz) * all : 0.f;
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

// beside the end of the launch before it, for which the kernels wait
cudaError_t route_go(void (*kern)(const RouteArgs), unsigned grid, size_t smem, const RouteArgs& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(32 * kRouteWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

template <typename T, int NI>
cudaError_t route_launch(RouteArgs& a, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.T + kRouteWarps - 1) / kRouteWarps);
  // a lane's experts lie whole on a boundary of 16 bytes, or of their size
  constexpr int BYTES = NI * (int)sizeof(T), STEP = BYTES < 16 ? BYTES : 16;
  const uintptr_t all = reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.dlogits) | (uintptr_t)(a.E * sizeof(T));
  a.whole = a.E % NI == 0 && all % STEP == 0;
  if (a.dlogits != nullptr) {
    return route_go(route_backward_kernel<T, NI>, grid, 0, a, st);
  }
  a.whole_bias = a.E % NI == 0 && (reinterpret_cast<uintptr_t>(a.bias) | (uintptr_t)(a.E * 4)) % (NI == 2 ? 8 : 16) == 0;
  a.size = a.E / a.G;
  // as many CTAs as the GPU holds at once: more would wait for the first to be through with all their tokens
  int dev = 0, sms = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (err != cudaSuccess) return err;
  const unsigned room = (unsigned)(route_ctas<NI>() * sms);
  const size_t smem = a.G > 1 ? (size_t)kRouteWarps * (a.E + a.G + 16) * sizeof(double) : 0;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(route_kernel<T, NI>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  return route_go(route_kernel<T, NI>, grid < room ? grid : room, smem, a, st);
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
