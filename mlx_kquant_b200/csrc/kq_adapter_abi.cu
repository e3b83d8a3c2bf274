// The C entry points of the grouped router and of the low-rank adapters: argument checks, then the launches.
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <initializer_list>

#include "../../include/kquant_b200.h"
#include "kq_lora.h"
#include "kq_route.h"

namespace kq {
int set_error(int code, const char* msg);
}

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return kq::set_error(code, buf);
}

int done(const char* what, cudaError_t e) {
  return e == cudaSuccess ? KQ_OK : fail(KQ_ERR_CUDA, "[mlx_kquant] %s: CUDA error: %s", what, cudaGetErrorString(e));
}

// rows, and values of a row: the kernels count them in 32 bits, some steps ahead of the last
constexpr int kMost = 1 << 30;
// rows without an order of their entries: every cluster looks through all indices, rows x rows reads in all
constexpr int kMostDirect = 1 << 16;

struct Operand {
  const char* name;
  const void* p;
  int align;
};
int aligned_check(const char* op, std::initializer_list<Operand> all) {
  for (const Operand& o : all)
    if (reinterpret_cast<uintptr_t>(o.p) % o.align != 0)
      return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] %s must be %d-byte aligned.", op, o.name, o.align);
  return KQ_OK;
}
int size_of(int dtype) { return dtype == KQ_F32 ? 4 : 2; }

int route_check(const char* op, int dtype, long long T, int E, int top_k, const char* scoring, int* code) {
  if (scoring != nullptr && std::strcmp(scoring, "softmax") == 0) *code = 0;
  else if (scoring == nullptr || std::strcmp(scoring, "sigmoid") == 0) *code = 1;
  else return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] unknown scoring '%s'.", op, scoring);
  if (dtype != KQ_F32 && dtype != KQ_F16 && dtype != KQ_BF16)
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] logits must be floating.", op);
  if (E < 1 || E > 1024 || top_k < 1 || top_k > 32 || top_k > E)
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] needs 1 <= top_k <= min(E, 32) and E <= 1024.", op);
  if (T < 0 || T > kMost) return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] bad token count.", op);
  return KQ_OK;
}

// what kq_lora_update and kq_lora_backward have in common
int lora_check(const char* op, int dtype, int param_dtype, long long rows, int K, int N, int rank, int slots, int n_adapters,
               int n_experts, const void* adapter_ids, const void* experts, const void* plan, size_t plan_bytes) {
  if ((dtype != KQ_F16 && dtype != KQ_BF16) || (param_dtype != dtype && param_dtype != KQ_F32))
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] rows must be float16 or bfloat16, parameters of the same type or float32.", op);
  if (K < 1 || N < 1 || K > kMost || N > kMost) return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] bad row length.", op);
  if (rank < 1 || rank > kq::kLoraMaxRank)
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] rank must be 1 to %d but is %d.", op, kq::kLoraMaxRank, rank);
  if (rows < 0 || rows > kMost || slots < 1 || rows % slots != 0)
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] bad row count.", op);
  if (n_adapters < 1 || n_experts < 1 || (long long)n_adapters * n_experts > 65535)
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] needs 1 <= adapters * experts <= 65535.", op);
  if (adapter_ids == nullptr && experts == nullptr) {
    if (n_adapters != 1 || n_experts != 1)
      return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] several adapters or experts and no indices.", op);
  } else if (plan != nullptr && plan_bytes < kq_lora_plan_bytes(rows, n_adapters * n_experts)) {
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] the plan is smaller than kq_lora_plan_bytes.", op);
  }
  return KQ_OK;
}

int types_of(int dtype, int param_dtype) {
  if (param_dtype == KQ_F32) return dtype == KQ_BF16 ? kq::kLoraBf16F32 : kq::kLoraF16F32;
  return dtype == KQ_BF16 ? kq::kLoraBf16 : kq::kLoraF16;
}

}  // namespace

extern "C" {

int kq_moe_router_grouped(const void* logits, int dtype, long long T, int E, int top_k, int n_groups, int top_groups, int group_top,
                          const char* scoring, const float* bias, int norm_topk_prob, float scale, int32_t* indices, float* weights,
                          void* stream) {
  const char* op = "moe_router_grouped";
  kq::RouteArgs a{};
  const int rc = route_check(op, dtype, T, E, top_k, scoring, &a.scoring);
  if (rc != KQ_OK) return rc;
  if (n_groups < 1 || E % n_groups != 0 || top_groups < 1 || top_groups > n_groups)
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] needs E a multiple of n_groups and 1 <= top_groups <= n_groups.", op);
  if (group_top < 1 || group_top > 2) return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] group_top must be 1 or 2.", op);
  if ((long long)top_groups * (E / n_groups) < top_k)
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] the kept groups have fewer than top_k experts.", op);
  if (T == 0) return KQ_OK;
  if (!logits || !indices || !weights) return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] null pointer.", op);
  if (int off = aligned_check(op, {{"logits", logits, size_of(dtype)}, {"bias", bias, 4}, {"indices", indices, 4}, {"weights", weights, 4}})) return off;
  a.logits = logits;
  a.dtype = dtype;
  a.T = (int)T;
  a.E = E;
  a.G = top_groups == n_groups ? 1 : n_groups;   // all groups stay: they choose nothing
  a.top_groups = top_groups;
  a.group_top = group_top;
  a.top_k = top_k;
  a.norm = norm_topk_prob != 0;
  a.bias = bias;
  a.scale = scale;
  a.indices = indices;
  a.weights = weights;
  return done(op, kq::launch_route(a, static_cast<cudaStream_t>(stream)));
}

int kq_moe_router_grouped_backward(const void* logits, int dtype, long long T, int E, int top_k, const char* scoring, int norm_topk_prob,
                                   float scale, const int32_t* indices, const float* dweights, void* dlogits, void* stream) {
  const char* op = "moe_router_grouped_backward";
  kq::RouteArgs a{};
  const int rc = route_check(op, dtype, T, E, top_k, scoring, &a.scoring);
  if (rc != KQ_OK || T == 0) return rc;
  if (!logits || !indices || !dweights || !dlogits) return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] null pointer.", op);
  if (int off = aligned_check(op, {{"logits", logits, size_of(dtype)}, {"indices", indices, 4}, {"dweights", dweights, 4}, {"dlogits", dlogits, size_of(dtype)}}))
    return off;
  a.logits = logits;
  a.dtype = dtype;
  a.T = (int)T;
  a.E = E;
  a.top_k = top_k;
  a.norm = norm_topk_prob != 0;
  a.scale = scale;
  a.indices = const_cast<int32_t*>(indices);
  a.dw = dweights;
  a.dlogits = dlogits;
  return done(op, kq::launch_route(a, static_cast<cudaStream_t>(stream)));
}

size_t kq_lora_plan_bytes(long long rows, int n_groups) {
  return rows < 0 || rows > kMost || n_groups < 1 || n_groups > 65535 ? 0 : kq::lora_plan_layout(rows, n_groups).total;
}

int kq_lora_plan(const int32_t* adapter_ids, const uint32_t* experts, long long rows, int slots, int n_adapters, int n_experts,
                 void* plan, size_t plan_bytes, void* stream) {
  const char* op = "lora_plan";
  const int rc = lora_check(op, KQ_F16, KQ_F16, rows, 1, 1, 1, slots, n_adapters, n_experts, adapter_ids, experts, nullptr, 0);
  if (rc != KQ_OK) return rc;
  if (plan == nullptr || plan_bytes < kq_lora_plan_bytes(rows, n_adapters * n_experts))
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] the plan is smaller than kq_lora_plan_bytes.", op);
  if (adapter_ids == nullptr && experts == nullptr) return KQ_OK;
  if (int off = aligned_check(op, {{"the plan", plan, 256}, {"adapter_ids", adapter_ids, 4}, {"experts", experts, 4}})) return off;
  return done(op, kq::launch_lora_plan(kq::LoraGroups{adapter_ids, experts, slots, n_adapters, n_experts, rows, nullptr, 1.f}, plan,
                                       static_cast<cudaStream_t>(stream)));
}

int kq_lora_update(const void* x, int dtype, long long rows, int K, long long x_row_stride, int slots, int x_shared, const void* a,
                   const void* b, int param_dtype, int rank, int N, int n_adapters, int n_experts, const int32_t* adapter_ids,
                   const uint32_t* experts, const float* scaling, float scale, const void* y, long long y_row_stride, void* out,
                   long long out_row_stride, void* u, const void* plan, size_t plan_bytes, void* stream) {
  const char* op = "lora_update";
  const int rc = lora_check(op, dtype, param_dtype, rows, K, N, rank, slots, n_adapters, n_experts, adapter_ids, experts, plan, plan_bytes);
  if (rc != KQ_OK || rows == 0) return rc;
  if (!x || !a || !b || !y || !out) return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] null pointer.", op);
  if ((adapter_ids != nullptr || experts != nullptr) && plan == nullptr && rows > kMostDirect)
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] needs the plan of its indices beyond %d rows.", op, kMostDirect);
  if (int off = aligned_check(op, {{"x", x, 2}, {"a", a, size_of(param_dtype)}, {"b", b, size_of(param_dtype)}, {"y", y, 2}, {"out", out, 2}, {"saved", u, 16},
                                   {"adapter_ids", adapter_ids, 4}, {"experts", experts, 4}, {"scaling", scaling, 4}, {"the plan", plan, 256}}))
    return off;
  const kq::LoraCall c{types_of(dtype, param_dtype), kq::LoraGroups{adapter_ids, experts, slots, n_adapters, n_experts, rows, scaling, scale},
                       x, x_row_stride, x_shared, K, N, rank, a, b, plan};
  return done(op, kq::launch_lora_forward(c, y, y_row_stride, out, out_row_stride, u, static_cast<cudaStream_t>(stream)));
}

size_t kq_lora_saved_bytes(long long rows, int rank, int param_dtype) {
  return rows < 0 || rank < 1 || rank > kq::kLoraMaxRank ? 0 : kq::lora_saved_bytes(rows, rank, param_dtype == KQ_F32);
}

size_t kq_lora_backward_workspace_bytes(long long rows, int slots, int x_shared, int K, int N, int rank, int param_dtype) {
  return rows < 0 || slots < 1 || K < 1 || N < 1 || rank < 1 || rank > kq::kLoraMaxRank
             ? 0 : kq::lora_backward_workspace_bytes(rows, slots, x_shared, K, N, rank, param_dtype == KQ_F32);
}

int kq_lora_backward(const void* dy, int dtype, long long rows, int N, long long dy_row_stride, const void* x, int K, long long x_row_stride,
                     int slots, int x_shared, const void* a, const void* b, int param_dtype, int rank, int n_adapters, int n_experts,
                     const int32_t* adapter_ids, const uint32_t* experts, const float* scaling, float scale, const void* u, void* dx,
                     void* da, void* db, const void* plan, size_t plan_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "lora_backward";
  const int rc = lora_check(op, dtype, param_dtype, rows, K, N, rank, slots, n_adapters, n_experts, adapter_ids, experts, plan, plan_bytes);
  if (rc != KQ_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {   // the matrices' gradients are whole all the same
    const size_t bytes = (size_t)n_adapters * n_experts * rank * (param_dtype == KQ_F32 ? 4 : 2);
    if (da != nullptr) {
      const cudaError_t e = cudaMemsetAsync(da, 0, bytes * K, st);
      if (e != cudaSuccess) return done(op, e);
    }
    return db != nullptr ? done(op, cudaMemsetAsync(db, 0, bytes * N, st)) : KQ_OK;
  }
  if (!dy || !a || !b || (da && !x) || (db && !u)) return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] null pointer.", op);
  if ((adapter_ids != nullptr || experts != nullptr) && plan == nullptr)
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] needs the plan of its indices.", op);
  if (workspace == nullptr || workspace_bytes < kq_lora_backward_workspace_bytes(rows, slots, x_shared, K, N, rank, param_dtype))
    return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] workspace is smaller than kq_lora_backward_workspace_bytes.", op);
  if (int off = aligned_check(op, {{"dy", dy, 2}, {"x", x, 2}, {"a", a, size_of(param_dtype)}, {"b", b, size_of(param_dtype)}, {"saved", u, 16}, {"dx", dx, 2},
                                   {"da", da, size_of(param_dtype)}, {"db", db, size_of(param_dtype)}, {"adapter_ids", adapter_ids, 4}, {"experts", experts, 4},
                                   {"scaling", scaling, 4}, {"the plan", plan, 256}, {"the workspace", workspace, 256}}))
    return off;
  const kq::LoraCall c{types_of(dtype, param_dtype), kq::LoraGroups{adapter_ids, experts, slots, n_adapters, n_experts, rows, scaling, scale},
                       x, x_row_stride, x_shared, K, N, rank, a, b, plan};
  return done(op, kq::launch_lora_backward(c, dy, dy_row_stride, u, dx, K, da, db, workspace, st));
}

int kq_clear_rows(void* y, long long rows, int N, const uint32_t* experts, int n_experts, void* stream) {
  const char* op = "clear_rows";
  if (rows < 0 || rows > kMost || N < 1 || N > kMost || n_experts < 1) return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] bad row, column or expert count.", op);
  if (rows == 0) return KQ_OK;
  if (!y || !experts) return fail(KQ_ERR_INVALID_ARGUMENT, "[mlx_kquant.%s] null pointer.", op);
  if (int off = aligned_check(op, {{"y", y, 2}, {"experts", experts, 4}})) return off;
  return done(op, kq::launch_clear_rows(y, (int)rows, N, experts, n_experts, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
