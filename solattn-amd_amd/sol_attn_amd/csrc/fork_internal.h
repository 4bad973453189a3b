// Parameter blocks and launchers of what happens to a paged cache's sequences
// between calls (fork.hip): kept drafts, forks, pages taken and freed.
#pragma once

#include "paged_internal.h"

namespace sol {

// Kept drafts: row base + kept[s][j] of sequence s goes to row base + j.
struct KeepParams {
  PagedBatch batch;      // rows unused
  const int32_t* kept;   // [S, most]
  int most;
  uint8_t* store[2];     // K, V: [pages, H, page_size, D]
  float* scale[2];       // [pages, H, page_size], or null
  int H;
  int32_t* lengths_out;  // [S]
};

// The next plan of a batch (cache_fork).
struct ForkParams {
  const int32_t* table;      // [S, width]
  const int32_t* lengths;    // [S]: tokens that have pages
  const int32_t* continued;  // [S]: tokens to continue from
  int S, width;
  const int32_t* parents;    // [N]
  const int32_t* new_tokens; // [N]
  int N, new_width;
  const int32_t* refs;       // [pages]: tables that name a page
  int pages, page_shift;
  uint8_t* store[2];
  float* scale[2];
  int H;
  int row_bytes;             // of a K (V) row
  int32_t* new_table;        // [N, new_width]
  int32_t* new_lengths;      // [N]
  int32_t* new_offsets;      // [N + 1]
  int32_t* new_refs;         // [pages]
  int32_t* missing;          // [1]
  uint64_t* absent;          // [1] pages of the new sequences' tokens that their tables do not name; or null
  // Workspace.
  int slices, slice_pages;   // of the pool: up to kForkSlices, of whole kForkStep pages
  int32_t* first;            // [S] first child, N: none
  int32_t* children;         // [S]
  int64_t* start;            // [N + 1] pages taken before sequence i's
  int32_t* lost;             // [1] begun pages that are not to be had
  int32_t* free_count;       // [slices]
  int32_t* free_list;        // [slices, slice_pages]: a slice's free pages in ascending order
};

constexpr int kForkSlices = 1024;
constexpr int kForkStep = 4096;

// Byte offsets of the workspace's parts, 16-byte aligned, and its size.
struct ForkSize {
  int64_t slices, slice_pages;
  int64_t first, children, start, lost, free_count, free_list, bytes;
};
ForkSize fork_size(int64_t sequences, int64_t new_sequences, int64_t pages);

// Lists of at most this many entries are moved by workgroups of 64 threads, longer
// ones by workgroups of 1,024, one or two (rows of 256 bytes) per head of K and of V.
constexpr int keep_small_rows(int row_bytes) { return 4 * 1024 / (row_bytes < 128 ? row_bytes : 128); }

hipError_t launch_keep(const KeepParams& p, int D, int format, hipStream_t stream);
hipError_t launch_fork(const ForkParams& p, hipStream_t stream);

}  // namespace sol
