// Shared by the kernels that sum attention weights by key (key_weights*.cu).
#pragma once

#include "internal.h"

namespace aoh {

// One call: the queries of one layer against the layer's retrieval units.
// A unit's query rows are its (token, head of the group) pairs, token major:
// row = token * grp + head.
struct KeyWeightsArgs {
  CacheGeom g;
  const RetrievalRow* rows;  // the layer's retrieval rows
  int unit0;                // first unit of the layer
  int units;                // retrieval rows of the layer: B * n_ret
  int past_len;             // keys cached before these queries
  const int* past_len_dev;  // read instead of past_len when not null
  int max_len;              // keys that `out` and the plan have room for
  int q_len;
  const void* q;            // (B, q_len, Hq, 128) contiguous
  float* out;               // retrieval row r, key j: out[r * out_stride + j]
  long long out_stride;
  int accumulate;
};

// How a call is run and where its workspace's parts begin (bytes).
//   any:     for some query rows after others: their scores and (m, l) by key range, then the sums
//   few:     scores of every (key, query row) and (m, l) by key range, then the sums; or both by a cluster
//   tensor:  (m, l) by key range, the rows' -lse, the sums by row range
enum class KeyWeightsKind { any, few, tensor };
struct KeyWeightsPlan {
  KeyWeightsKind kind = KeyWeightsKind::any;
  int rows = 0;            // query rows of a unit; any: that a pair of launches takes
  int row_tiles = 0, tile_rows = 0;
  int tile_tokens = 0;     // tensor: tokens of a row tile
  int splits = 1;          // key ranges
  int row_splits = 1;      // tensor: row ranges of the sums
  bool one = false;        // few: one launch, no workspace
  bool stream = false;     // tensor: the query rows stay resident in the second pass too
  size_t part = 0, score = 0, lse = 0, sums = 0, bytes = 0;
};

// Launchers of the bf16 kernels (key_weights_sm100.cu).
// false: too many rows and keys
bool plan_key_weights_few(const aoh_kv_cache* c, int units, int max_len, KeyWeightsPlan& p);
void plan_key_weights_tensor(const aoh_kv_cache* c, int units, int max_len, int q_len, KeyWeightsPlan& p);
int launch_key_weights_few(const aoh_kv_cache* c, const KeyWeightsArgs& a, const KeyWeightsPlan& p, char* ws,
                           cudaStream_t st);
int launch_key_weights_tensor(const aoh_kv_cache* c, const KeyWeightsArgs& a, const KeyWeightsPlan& p, char* ws,
                              cudaStream_t st);

// Query rows of a unit that the few-rows kernels take: up to 32 where one launch
// does, else 16 (16 rows x 32768 keys, 2 units: 16 us, on the tensor cores 21).
constexpr int kFewRows = 16, kOneRows = 32;

inline size_t align256(size_t n) { return (n + 255) / 256 * 256; }

#ifdef __CUDACC__
// Keys cached before the queries.  A device length beyond what the caller
// planned for is cut to it, so that no weight lands behind a row of `out`.
__device__ __forceinline__ int key_weights_past(const KeyWeightsArgs& a) {
  return a.past_len_dev ? max(0, min(*a.past_len_dev, a.max_len - a.q_len)) : a.past_len;
}
#endif

// 1 / sqrt(128) * log2(e): scores in the log2 domain
constexpr float kScoreScale = 0.08838834764831845f * 1.4426950408889634f;

}  // namespace aoh
