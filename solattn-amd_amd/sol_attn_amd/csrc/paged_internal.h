// Parameter blocks and launchers of the paged cache (cache.hip) and of the
// attention over it and under a window (paged.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sol {

// How a cache stores a K or V row (SOL_CACHE_* of the C header).
enum CacheFormat { kBf16 = 0, kInt8 = 1, kFp8 = 2 };

template <int F>
constexpr int kElemBytes = F == kBf16 ? 2 : 1;

// One sequence batch over a cache: rows query_offsets[s] .. [s + 1] - 1 of the
// new tokens belong to sequence s, whose keys (the new ones included) are
// positions 0 .. context_lengths[s] - 1; position p is row p % page_size of
// page page_table[s][p / page_size].  The arrays are the caller's device
// memory and may hold anything: rows outside [0, rows) do not exist (attention
// clamps the offsets, the write looks rows up), a page outside [0, pages) is no
// page (not written, read as zeros, not attended), and neither is there anything
// past the table's last position.  (A length past the table must not move the
// new tokens to the places of stored ones.)
struct PagedBatch {
  const int32_t* table;    // [S, width]
  const int32_t* lengths;  // [S]
  const int32_t* offsets;  // [S + 1]
  int S, width, pages;
  int page_shift;          // page_size = 1 << page_shift, 16 at least
  int rows;                // new rows there are

  __device__ __forceinline__ int offset(int s) const { return min(max(offsets[s], 0), rows); }
  // The position after sequence s's last new token, and how many keys it has in the table.
  __device__ __forceinline__ int end(int s) const { return max(lengths[s], 0); }
  __device__ __forceinline__ int positions() const { return width << page_shift; }
  __device__ __forceinline__ int length(int s) const { return min(end(s), positions()); }
};

struct CacheParams {
  PagedBatch batch;
  const uint16_t* rows[2];  // K, V rows to write: [rows, H, D] by the strides
  int64_t st[2], sh[2];     // element strides {token, head}
  uint8_t* store[2];        // [pages, H, page_size, D] codes
  float* scale[2];          // [pages, H, page_size], or null (BF16)
  uint16_t* out[2];         // cache_read: [S, tokens, H, D]
  int H, start, tokens;
};

struct PagedParams {
  PagedBatch batch;           // table null: plain K / V, S entries of Tq queries and Tk keys
  const uint16_t* q;          // NHD rows (sb ignored) or BTHD
  int64_t q_sb, q_st, q_sh;   // element strides
  const uint8_t* store[2];    // K, V
  const float* scale[2];      // or null
  int64_t sb[2], st[2], sh[2];  // plain: byte strides {entry, row, head}
  uint16_t* out;              // contiguous [rows, Hq, D] (plain: [S, Tq, Hq, D])
  int Tq, Tk;
  int H, G;                   // K / V heads, query heads of each
  float scale_log2;
  int causal;
  int window, sinks;          // window 2^31 - 1: none
  const int32_t* parents;     // a tree of new tokens: each row's parent among its sequence's; or null
  // Keys split over workgroups (take_item in paged.hip); target 0: not split.
  int target, min_tiles;      // workgroups per head; key tiles of a part at least
  int rounds;                 // 2: `target` is two rounds of them, of which take_item may make one
  int64_t headers, records;   // PagedSize's
  int64_t header_bytes, new_rows;
  void* workspace;            // PagedSize::bytes: headers, then records
};

// The launch of a call, from what the host knows of it.
struct PagedSize {
  int64_t rows;               // of a row tile: 16 (step_kernel) or 128 (wide_kernel)
  int64_t tiles;              // row tiles at most
  int64_t target, min_tiles, rounds;
  bool many_parts;            // a row tile has many parts and few rows (merge_kernel)
  int64_t grid;               // workgroups
  int64_t headers;            // split row tiles per head at most, 0 without target
  int64_t records;            // their parts over all heads at most
  int64_t merge_rows;         // rows of a tile that the merge's workgroups take side by side
  int64_t header_bytes;
  int64_t bytes;              // workspace, 0 without target
};

// rows: new tokens in all; keys: what a sequence's see at most; tile_keys: what 16
// neighbouring ones do (of trees, what their row tile streams); step_keys: the same
// as it counts for the choice of kernel; group: query heads per head; ragged:
// sequences may differ in length; tree: the new tokens are trees.
PagedSize paged_size(int64_t rows, int64_t sequences, int64_t keys, int64_t tile_keys, int64_t step_keys, int64_t heads,
                     int64_t group, int64_t head_dim, int format, bool causal, bool ragged, bool tree = false);

hipError_t launch_cache_write(const CacheParams& p, int D, int format, hipStream_t stream);
hipError_t launch_cache_read(const CacheParams& p, int D, int format, hipStream_t stream);
hipError_t launch_paged(const PagedParams& p, const PagedSize& size, int D, int format, hipStream_t stream);

}  // namespace sol
