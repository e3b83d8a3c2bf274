// Internal interface of the low-rank adapter kernels (kq_lora*.cu) to their C entry points.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace kq {

constexpr int kLoraMaxRank = 128;

// Rows of one group (adapter, or adapter and expert), up to the tile's height: entries order[start .. start + rows). group -1:
// rows without an adapter. rows 0: a slot of the list that holds no tile.
struct LoraTile {
  int group, start, rows, pad;
};

// Which group an entry belongs to. Entry e = token * slots + slot; group = adapter of the token * E + expert of the entry.
struct LoraGroups {
  const int* ids;           // adapter of each token, or nullptr: 0; others than [0, G): none
  const uint32_t* experts;  // expert of each entry, or nullptr: 0; others than [0, E): none
  int slots, G, E;
  long long n;              // entries
  const float* scaling;     // factor of each adapter, or nullptr: 1
  float scale;              // factor of all of them
};

// A plan (launch_lora_plan): entries in the order of their groups, stable; each group's first place; tiles.
struct LoraPlan {
  const int* order;
  const int* offsets;  // [groups + 2]: group g's entries are order[offsets[g] .. offsets[g + 1]), those without one come last
  const LoraTile* tiles;
  int n_tiles;         // slots of the list
  int tile_rows;
};
struct LoraPlanLayout {
  size_t order, offsets, tiles, counts, total;
  int n_tiles, tile_rows;
  int chunk, chunks;   // entries of a CTA, and CTAs, where they are counted and placed in two launches; 0: in one
};
LoraPlanLayout lora_plan_layout(long long n, int n_groups);
cudaError_t launch_lora_plan(const LoraGroups& g, void* plan, cudaStream_t st);

// in . w1^T -> u, base + factor * u . w2^T -> out, in one launch (or one of the two halves).
struct LoraArgs {
  LoraGroups g;
  const void* in;             // shrink: rows of D1 values; entry e reads row e / in_div
  long long in_stride;
  int in_div, D1, D2, r;
  const void *w1, *w2;        // forward: a [groups, r, D1], b [groups, D2, r]; backward: b [groups, D1, r], a [groups, r, D2]
  const void* base;           // rows to add to, or nullptr
  long long base_stride;
  void* out;                  // or nullptr: shrink only
  long long out_stride;
  int out_f32;                // out is float32 and base nullptr
  int c0, c1;                 // columns [c0, c1) of out; column c is stored at c - c0
  uint16_t* u;                // [terms][n][ru] bf16 terms: written by the shrink (if not nullptr), read where shrink == 0
  int ru;                     // r up to a multiple of 8
  int shrink;
  int scale_u;                // the factor goes into u (backward), not into the output
  LoraPlan plan;              // tiles == nullptr: one group, rows in order; or `direct`
  int direct;                 // tiles are found by the kernel itself: cluster c looks for the tile that entry c leads
  int n_clusters;             // tiles
  int by_in, by_w1, by_w2;    // how rows are read: by 16 bytes, 8, or elements
  int by_out;                 // rows of base and out likewise
};
enum LoraTypes { kLoraBf16 = 0, kLoraF16 = 1, kLoraBf16F32 = 2, kLoraF16F32 = 3 };  // rows, and parameters where they are float32
cudaError_t launch_lora_tile_bf16(const LoraArgs& a, bool backward, int mt, int cluster, cudaStream_t st);
cudaError_t launch_lora_tile_f16(const LoraArgs& a, bool backward, int mt, int cluster, cudaStream_t st);
cudaError_t launch_lora_tile_bf16_f32(const LoraArgs& a, bool backward, int mt, int cluster, cudaStream_t st);
cudaError_t launch_lora_tile_f16_f32(const LoraArgs& a, bool backward, int mt, int cluster, cudaStream_t st);

// dw[g] = sum over the group's entries of in^T uv: [D, r] (r_first 0) or [r, D] (1).
struct LoraWgrad {
  const void* in;
  long long in_stride;
  int in_div, D;
  const uint16_t* uv;    // [terms][n][ru]
  int scaled;            // times the adapter's factor
  void* out;             // [groups, r, D] (r_first), else [groups, D, r]; nullptr: none
  int r_first;
  int by_in;
};
struct LoraWgradArgs {
  LoraGroups g;
  LoraWgrad of[2];             // one of them or both, in one launch
  int tiles;                   // of 128 columns of the first
  int r, ru;
  const int *order, *offsets;  // or nullptr: one group, rows in order
  int n_groups;
};
cudaError_t launch_lora_wgrad(const LoraWgradArgs& a, int in_dtype, int out_f32, int cluster, cudaStream_t st);

// out[t] = sum of the slots' float32 rows
cudaError_t launch_lora_sum_slots(const float* part, int slots, long long tokens, int cols, void* out, long long out_stride, int dtype,
                                  cudaStream_t st);

// rows of 16-bit values whose expert lies outside [0, n_experts) become zero
cudaError_t launch_clear_rows(void* y, int rows, int N, const uint32_t* experts, int n_experts, cudaStream_t st);

struct LoraCall {
  int types;                 // LoraTypes
  LoraGroups g;
  const void* x;
  long long x_stride;
  int shared;                // x has one row per token
  int K, N, r;
  const void *a, *b;
  const void* plan;          // or nullptr
};
cudaError_t launch_lora_forward(const LoraCall& c, const void* y, long long y_stride, void* out, long long out_stride, void* u,
                                cudaStream_t st);
size_t lora_saved_bytes(long long n, int r, int param_f32);
size_t lora_backward_workspace_bytes(long long n, int slots, int shared, int K, int N, int r, int param_f32);
cudaError_t launch_lora_backward(const LoraCall& c, const void* dy, long long dy_stride, const void* u, void* dx, long long dx_stride,
                                 void* da, void* db, void* workspace, cudaStream_t st);

}  // namespace kq
