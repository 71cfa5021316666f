// Shared by the kernels that sum attention weights by key (key_weights*.cu).
#pragma once

#include "internal.h"

namespace aoh {

// One call: the queries of one layer against the layer's retrieval units.
// A unit's query rows are its (token, head of the group) pairs, token major:
// row = token * grp + head.
struct KeyWeightsArgs {
  CacheGeom g;
  const int32_t* unit_row;  // per unit: index among the retrieval units, -1: streaming
  int unit0, row0;          // first unit of the layer, first retrieval row of the layer
  int units;                // B * G units of the layer
  int past_len;             // keys cached before these queries
  const int* past_len_dev;  // read instead of past_len when not null
  int max_len;              // keys that `out` and the plan have room for
  int q_len;
  const void* q;            // (B, q_len, Hq, 128) contiguous
  float* out;               // retrieval row r, key j: out[r * out_stride + j]
  long long out_stride;
  int accumulate;
  float2* part;             // (m, l) of a query row over one key range: part[(split * n_rows_total + row)]
  int splits;
  long long rows_total;     // query rows of all retrieval units
};

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
