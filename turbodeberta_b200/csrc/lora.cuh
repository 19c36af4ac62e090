// What the kernels for adapters share: whose row it is.
#pragma once
#include "tdb_internal.h"

namespace tdb {

struct LoraRows {
  const void* ids;                                   // int32 or int64, one for every rows_per_id rows; null: all rows are adapter 0's
  int id_bytes;
  int64_t rows_per_id, rows;
  int n;                                             // adapters
  const float* scaling;                              // one for each adapter; null: scaling_value
  float scaling_value;
  // Rows sorted by adapter (lora.cu; null: as they come): position -> row, and each adapter's first position.  Ids are then those of positions.
  const int32_t *order, *starts;
};
__device__ __forceinline__ int64_t row_at(const LoraRows& r, int64_t position) { return r.order ? r.order[position] : position; }
__device__ __forceinline__ float scaling_of(const LoraRows& r, int adapter) { return r.scaling ? r.scaling[adapter] : r.scaling_value; }

// -1 for a row without one: its id is not an adapter's.
__device__ __forceinline__ int adapter_of(const LoraRows& r, int64_t row) {
  if (!r.ids) return 0;
  const int64_t i = r.rows_per_id == 1 ? row : row / r.rows_per_id;
  const int64_t id = r.id_bytes == 8 ? static_cast<const int64_t*>(r.ids)[i] : static_cast<const int32_t*>(r.ids)[i];
  return id >= 0 && id < r.n ? (int)id : -1;
}

// Of a call, in the order of its plan where it has one.
inline LoraRows lora_rows(const Lora& l) {
  if (!l.plan) return LoraRows{l.ids, l.id_bytes, l.rows_per_id, l.rows, l.n, l.scaling, l.scaling_value, nullptr, nullptr};
  const int32_t* order = l.plan + l.n + 2;
  return LoraRows{order + l.rows, 4, 1, l.rows, l.n, l.scaling, l.scaling_value, order, l.plan};
}
inline LoraRows lora_rows_as_they_come(const Lora& l) {
  Lora plain = l;
  plain.plan = nullptr;
  return lora_rows(plain);
}

}  // namespace tdb
