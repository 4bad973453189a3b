// What happens to the sequences of a paged cache between calls.
//
// cache_keep: of a sequence's n new tokens (positions base .. base + n - 1) the
// kept ones, whose numbers k_0 < k_1 < ... ascend, move together: row base + k_j
// goes to row base + j, K and V and their scales, of every head.
//
// cache_fork: the next plan.  New sequence i continues old sequence p_i from its
// first L tokens (or is empty, L = 0) with a new ones, so it needs ceil((L + a) /
// page_size) pages: the floor(L / page_size) whole pages of its parent, which all
// children share; then, for the parent's first child, the parent's further pages
// that no other table names; and pages of its own for the rest, taken in order
// of sequences and their places, lowest free page first.  The page that position L
// lies in, where the parent has rows before it, is copied.  A page is free if
// no table named it before the call: pages that a call frees are taken from the
// next call on, so that no page is read and written by one call, and everything
// follows from the state before it.  A begun page that the parent does not have
// (none was free, then) its children do not have either.  `missing` counts the
// pages that this call was to take or go on in and could not; `absent` those that
// the new sequences' tokens need and their tables do not name, for whatever reason:
// those, whole pages that a parent lacks, and what new_width has no room for.
// Reference counts change by whole numbers, in any order.
#include <algorithm>

#include "fork_internal.h"
#include "sol_device.h"

namespace sol {

namespace {

// ---- kept rows --------------------------------------------------------------

// Entry j of a sequence's list stands if the entries ascend up to it, inside
// [0, n).
__device__ __forceinline__ bool kept_ascends(const int32_t* kept, int j, int64_t n) {
  const int x = kept[j];
  return x > (j ? kept[j - 1] : -1) && x < n;
}

// How many entries of the list stand, for all threads: those before the first that
// does not ascend.
template <int NT>
__device__ __forceinline__ int kept_count(const int32_t* kept, int most, int64_t n) {
  constexpr int kEach = 4;  // entries that a thread reads at once
  __shared__ int s_least[NT / kWave];
  for (int j0 = 0; j0 < most; j0 += kEach * NT) {
    bool bad[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int j = j0 + k * NT + int(threadIdx.x);
      bad[k] = j >= most || !kept_ascends(kept, j, n);
    }
    int least = 0x7FFFFFFF;
#pragma unroll
    for (int k = kEach - 1; k >= 0; --k) {
      const uint64_t lanes = __builtin_amdgcn_ballot_w64(bad[k]);
      if (lanes) least = j0 + k * NT + int(threadIdx.x & ~63u) + __builtin_ctzll(lanes);
    }
    if constexpr (NT > kWave) {
      s_least[threadIdx.x >> 6] = least;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NT / kWave; ++w) least = min(least, s_least[w]);
      __syncthreads();
    }
    if (least != 0x7FFFFFFF) return min(least, most);
  }
  return most;
}

// A workgroup moves the rows of one (sequence, head, K or V), 128 bytes of them at
// most (longer rows take two workgroups).  Rows only move forward, k_j >= j, and in
// ascending order, so that a row is read before another takes its place: a batch
// of rows is read whole before it is written, and the batches follow one another.
// So the time is that of a batch's chain of reads (the list, the table, the rows),
// and the workgroups are large: two frames of 4,032 tokens, thinned to 927 and 23, 24
// heads of 128, BF16, 18 MB: 9.0 us (15.6 with whole rows, 512 to a batch, and a wait
// for each row's entry, page and bytes); 48 sequences' paths of up to 13 INT8 drafts,
// 8 heads: 3.7 us.
template <int ROW, int WAVES, int U>
__global__ __launch_bounds__(WAVES * kWave) void keep_kernel(KeepParams p) {
  constexpr int NT = WAVES * kWave, kPiece = ROW < 128 ? ROW : 128, kPieces = ROW / kPiece;
  constexpr int kLanes = kPiece / 16, kRows = NT / kLanes;
  constexpr uint32_t kStays = 0xFFFFFFFFu;
  const PagedBatch& bt = p.batch;
  const int piece = int(blockIdx.x) % kPieces, unit = int(blockIdx.x) / kPieces;
  const int kv = unit & 1, h = (unit >> 1) % p.H, s = (unit >> 1) / p.H;
  const int64_t n = int64_t(bt.offsets[s + 1]) - bt.offsets[s], base = int64_t(bt.lengths[s]) - max(n, int64_t(0));
  const int32_t* kept = p.kept + int64_t(s) * p.most;
  const int c = threadIdx.x % kLanes;
  uint8_t* store = p.store[kv] + kPiece * piece + 16 * c;
  const bool scales = p.scale[kv] && piece == 0 && c == 0;
  const int32_t* table = bt.table + int64_t(s) * bt.width;
  // Row of the cache at position `at`, whose page number is `page` (a cache of 2^32
  // rows does not fit the card), kStays: none.
  auto page_at = [&](int64_t at) { return table[min(max(at >> bt.page_shift, int64_t(0)), int64_t(bt.width - 1))]; };
  auto row_of = [&](int64_t at, int page) -> uint32_t {
    if (at < 0 || at >= bt.positions() || page < 0 || page >= bt.pages) return kStays;
    return uint32_t((uint64_t(uint32_t(page)) * p.H + h) << bt.page_shift) + uint32_t(at & ((1 << bt.page_shift) - 1));
  };
  const bool speaks = unit == 2 * p.H * s && piece == 0 && threadIdx.x == 0;  // for the sequence
  if (p.most == 0 && speaks) p.lengths_out[s] = int(max(base, int64_t(0)));
  int count = p.most;  // known once the first batch is on its way
  for (int j0 = 0; j0 < count; j0 += U * kRows) {
    // Of all rows the list's entries, then their pages, then the rows, without a
    // branch in between, so that each is one wait.
    const int first = j0 + int(threadIdx.x) / kLanes;
    u32x4 x[U];
    float scale[U];
    uint32_t to[U], from[U];
    int k[U], pages[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = kept[min(first + u * kRows, p.most - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      pages[u][0] = page_at(base + k[u]);
      pages[u][1] = page_at(base + first + u * kRows);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = first + u * kRows;
      const bool moves = j < count && k[u] != j && k[u] >= 0 && k[u] < n;
      from[u] = moves ? row_of(base + k[u], pages[u][0]) : kStays;
      to[u] = moves ? row_of(base + j, pages[u][1]) : kStays;
      const uint64_t at = from[u] == kStays ? 0 : from[u];
      x[u] = *reinterpret_cast<const u32x4*>(store + at * ROW);
      scale[u] = scales ? p.scale[kv][at] : 0.f;
    }
    if (j0 == 0) {
      count = kept_count<NT>(kept, p.most, n);
      if (speaks) p.lengths_out[s] = int(max(base + count, int64_t(0)));
    }
    // Every read of the batch has returned before anything is written.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (WAVES > 1) __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (to[u] != kStays && first + u * kRows < count) {
        const bool none = from[u] == kStays;  // what has no page reads as zeros
        *reinterpret_cast<u32x4*>(store + uint64_t(to[u]) * ROW) = none ? zero_u32x4() : x[u];
        if (scales) p.scale[kv][to[u]] = none ? 0.f : scale[u];
      }
  }
}

template <int ROW>
void keep_variant(const KeepParams& p, hipStream_t stream) {
  constexpr int kPieces = ROW > 128 ? ROW / 128 : 1, kRows = kWave * 16 * kPieces / ROW;  // of a wave's load
  const dim3 grid(unsigned(int64_t(p.batch.S) * p.H * 2 * kPieces));
  static_assert(4 * kRows == keep_small_rows(ROW), "the C entry's check of the grid");
  if (p.most <= 4 * kRows)
    hipLaunchKernelGGL((keep_kernel<ROW, 1, 4>), grid, dim3(64), 0, stream, p);
  else
    hipLaunchKernelGGL((keep_kernel<ROW, 16, 8>), grid, dim3(1024), 0, stream, p);
}

// ---- forks ------------------------------------------------------------------

constexpr int kPlanThreads = 1024;
constexpr int kFewPages = 32;         // that one thread looks up
constexpr int kHeldSequences = 4096;  // old ones whose children a workgroup counts in LDS

// What a new sequence takes over from its parent.
struct Child {
  int parent;           // -1: none
  int kept, after;      // tokens before and with the new ones
  int full, held, used; // whole pages shared; pages of the parent; pages needed (of the new table's width)
  bool first;           // the parent's first child
  bool lost;            // page `full` is begun, and the parent does not have it
};

__device__ __forceinline__ int pages_of(int64_t tokens, int shift) {
  return int((tokens + (1 << shift) - 1) >> shift);
}

// Tokens that old sequence s has, and is continued from.
__device__ __forceinline__ int length_of(const ForkParams& p, int s) { return max(p.lengths[s], 0); }
__device__ __forceinline__ int kept_of(const ForkParams& p, int s) {
  return min(max(p.continued[s], 0), length_of(p, s));
}

__device__ __forceinline__ int page_of(const ForkParams& p, int s, int e) {
  return p.table[int64_t(s) * p.width + e];
}

__device__ __forceinline__ Child child_of(const ForkParams& p, int i, int first) {
  Child x;
  x.parent = p.parents[i];
  if (x.parent < 0 || x.parent >= p.S) x.parent = -1;
  const int length = x.parent >= 0 ? length_of(p, x.parent) : 0;
  x.kept = x.parent >= 0 ? kept_of(p, x.parent) : 0;
  x.after = int(min(int64_t(x.kept) + max(p.new_tokens[i], 0), int64_t(0x7FFFFFFF)));
  x.full = x.kept >> p.page_shift;
  x.held = min(pages_of(length, p.page_shift), p.width);
  x.used = min(pages_of(x.after, p.page_shift), p.new_width);
  x.first = first == i;
  x.lost = false;
  if ((x.kept & ((1 << p.page_shift) - 1)) && x.full < x.used) {
    const int page = x.full < x.held ? page_of(p, x.parent, x.full) : -1;
    x.lost = page < 0 || page >= p.pages;
  }
  return x;
}

// Whether the first child goes on in its parent's page e (>= full, < held): no other table names it.
__device__ __forceinline__ bool goes_on(const ForkParams& p, int s, int e) {
  const int page = page_of(p, s, e);
  return page >= 0 && page < p.pages && p.refs[page] == 1;
}

// Up to which of its parent's pages the child may go on (from `full`).
__device__ __forceinline__ int goes_until(const Child& x) { return x.first ? min(x.used, x.held) : x.full; }

// How many of its pages [full, e) the child takes, of which it goes on in `going`.
__device__ __forceinline__ int taken_before(const Child& x, int e, int going) {
  return max(e - x.full - (x.lost ? 1 : 0), 0) - going;
}

template <typename T>
__device__ __forceinline__ T wave_scan(T x, int lane) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const T y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  return x;
}

// Workgroup 0: first children, and the new sequences' lengths, offsets and numbers
// of pages.  The others: a slice of the pool each, whose counts they copy and
// whose free pages they list.
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(ForkParams p) {
  constexpr int kPlanWaves = kPlanThreads / kWave, kAtOnce = 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (blockIdx.x > 0) {
    __shared__ int s_count[kPlanWaves];
    constexpr int kEach = kForkStep / kPlanThreads;
    const int slice = blockIdx.x - 1;
    const int64_t from = int64_t(slice) * p.slice_pages, to = min(from + p.slice_pages, int64_t(p.pages));
    int32_t* list = p.free_list + from;
    int found = 0;
    for (int64_t a = from; a < to; a += kForkStep) {
      int refs[kEach], mine = 0;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        const int64_t page = a + tid * kEach + k;
        refs[k] = page < to ? p.refs[page] : 1;
        if (page < to) p.new_refs[page] = refs[k];
        mine += refs[k] <= 0;
      }
      const int end = wave_scan(mine, lane);
      if (lane == 63) s_count[wave] = end;
      __syncthreads();
      int at = found + end - mine;
#pragma unroll
      for (int w = 0; w < kPlanWaves; ++w) {
        at += w < wave ? s_count[w] : 0;
        found += s_count[w];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kEach; ++k)
        if (refs[k] <= 0) list[at++] = int(a) + tid * kEach + k;
    }
    if (tid == 0) p.free_count[slice] = found;
    return;
  }
  __shared__ int64_t s_taken[kPlanWaves], s_tokens[kPlanWaves];
  __shared__ int s_first[kHeldSequences], s_children[kHeldSequences], s_lost;
  if (tid == 0) s_lost = 0;
  // First children and numbers of children: in LDS, or, of more sequences, in
  // memory, where each of the two barriers waits for the card's caches.  (48 beams:
  // 10.6 us that way, 3.8 in LDS.)
  const bool held = p.S <= kHeldSequences;
  for (int s = tid; s < p.S; s += kPlanThreads) {
    if (held) {
      s_first[s] = p.N;
      s_children[s] = 0;
    } else {
      __hip_atomic_store(p.first + s, p.N, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(p.children + s, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (!held) __threadfence();
  __syncthreads();
  for (int i = tid; i < p.N; i += kPlanThreads) {
    const int s = p.parents[i];
    if (s < 0 || s >= p.S) continue;
    if (held) {
      atomicMin(s_first + s, i);
      atomicAdd(s_children + s, 1);
    } else {
      atomicMin(p.first + s, i);
      atomicAdd(p.children + s, 1);
    }
  }
  if (!held) __threadfence();
  __syncthreads();
  if (held)
    for (int s = tid; s < p.S; s += kPlanThreads) p.first[s] = s_first[s], p.children[s] = s_children[s];
  auto first_of = [&](int i) {
    const int s = p.parents[i];
    if (s < 0 || s >= p.S) return -1;
    return held ? s_first[s] : __hip_atomic_load(p.first + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  int64_t taken = 0, tokens = 0;
  for (int i0 = 0; i0 < p.N; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int64_t n = 0, a = 0;
    Child x = {};
    int going = 0;
    if (i < p.N) {
      x = child_of(p, i, first_of(i));
      if (goes_until(x) - x.full <= kFewPages)
        for (int e = x.full; e < goes_until(x); e += kAtOnce) {
          int page[kAtOnce], refs[kAtOnce];  // without a branch, so that each is one wait
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k) page[k] = page_of(p, x.parent, min(e + k, goes_until(x) - 1));
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k) refs[k] = p.refs[min(max(page[k], 0), p.pages - 1)];
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k)
            going += e + k < goes_until(x) && page[k] >= 0 && page[k] < p.pages && refs[k] == 1;
        }
    }
    // Sequences that go back far: the wave counts their pages together.
    for (uint64_t far = __builtin_amdgcn_ballot_w64(goes_until(x) - x.full > kFewPages); far; far &= far - 1) {
      const int of = __builtin_ctzll(far), s = __shfl(x.parent, of), end = __shfl(goes_until(x), of);
      int found = 0;
      for (int e0 = __shfl(x.full, of); e0 < end; e0 += kWave)
        found += __builtin_popcountll(__builtin_amdgcn_ballot_w64(e0 + lane < end && goes_on(p, s, e0 + lane)));
      if (lane == of) going = found;
    }
    if (i < p.N) {
      n = taken_before(x, x.used, going);
      a = x.after - x.kept;
      if (x.lost) atomicAdd(&s_lost, 1);
    }
    int64_t n_end = wave_scan(n, lane), a_end = wave_scan(a, lane);
    if (lane == 63) s_taken[wave] = n_end, s_tokens[wave] = a_end;
    __syncthreads();
    int64_t n_at = taken + n_end - n, a_at = tokens + a_end - a;
    for (int w = 0; w < kPlanWaves; ++w) {
      if (w < wave) n_at += s_taken[w], a_at += s_tokens[w];
      taken += s_taken[w];
      tokens += s_tokens[w];
    }
    __syncthreads();
    if (i < p.N) {
      p.start[i] = n_at;
      p.new_offsets[i] = int(min(a_at, int64_t(0x7FFFFFFF)));
      p.new_lengths[i] = x.after;
    }
  }
  if (tid == 0) {
    p.start[p.N] = taken;
    *p.lost = s_lost;
    if (p.absent) *p.absent = 0;
    p.new_offsets[p.N] = int(min(tokens, int64_t(0x7FFFFFFF)));
    if (p.N == 0) *p.missing = 0;  // (otherwise sequence 0's workgroup writes it)
  }
}

constexpr int kForkThreads = 256;
constexpr int kForkWaves = kForkThreads / kWave;
constexpr int kCopyBytes = 32768;  // of a page's rows that a workgroup copies

// The pool's free pages by their rank.
struct FreePages {
  int* ends;  // LDS [kForkSlices]: free pages up to a slice's end
  int total;

  // Every thread of the workgroup calls it.
  __device__ __forceinline__ FreePages(const ForkParams& p, int* lds) : ends(lds) {
    __shared__ int s_sum[kForkWaves];
    constexpr int kEach = kForkSlices / kForkThreads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int n[kEach], mine = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int slice = tid * kEach + k;
      n[k] = slice < p.slices ? p.free_count[slice] : 0;
      mine += n[k];
    }
    const int end = wave_scan(mine, lane);
    if (lane == 63) s_sum[wave] = end;
    __syncthreads();
    int at = end - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < kForkWaves; ++w) {
      at += w < wave ? s_sum[w] : 0;
      total += s_sum[w];
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) ends[tid * kEach + k] = at += n[k];
    __syncthreads();
  }
  // The free page of a rank, -1: there is none.
  __device__ __forceinline__ int page(const ForkParams& p, int64_t rank) const {
    if (rank >= total) return -1;
    int lo = 0, hi = p.slices - 1;  // the first slice whose end is past the rank
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > rank)
        hi = mid;
      else
        lo = mid + 1;
    }
    return p.free_list[int64_t(lo) * p.slice_pages + rank - (lo ? ends[lo - 1] : 0)];
  }
};

// Workgroups [0, N): a new sequence's table; [N, N + S): an old sequence's counts;
// the others: pieces of the pages that are copied.
__global__ __launch_bounds__(kForkThreads) void fork_kernel(ForkParams p, int pieces) {
  __shared__ int s_ends[kForkSlices];
  const int tid = threadIdx.x;
  const int64_t id = blockIdx.x;
  if (id >= p.N && id < int64_t(p.N) + p.S) {
    const int s = int(id - p.N), first = p.first[s], children = p.children[s];
    const int held = min(pages_of(length_of(p, s), p.page_shift), p.width), full = kept_of(p, s) >> p.page_shift;
    const int used = children ? child_of(p, first, first).used : 0;
    for (int e = tid; e < held; e += kForkThreads) {
      const int page = page_of(p, s, e);
      if (page < 0 || page >= p.pages) continue;
      const int more = e < full ? (e < p.new_width ? children : 0) : (e < used && goes_on(p, s, e) ? 1 : 0);
      if (more != 1) atomicAdd(p.new_refs + page, more - 1);
    }
    return;
  }
  if (id < p.N) {
    const int i = int(id), s = p.parents[i];
    const Child x = child_of(p, i, s >= 0 && s < p.S ? p.first[s] : -1);
    const FreePages free(p, s_ends);
    const int64_t start = p.start[i];
    if (i == 0 && tid == 0)
      *p.missing = int(min(max(p.start[p.N] - free.total, int64_t(0)) + *p.lost, int64_t(0x7FFFFFFF)));
    const int end = goes_until(x);
    __shared__ int s_going[kForkWaves];
    int going = 0;  // pages below e0 that the child goes on in
    uint64_t absent = tid == 0 ? uint64_t(pages_of(x.after, p.page_shift) - x.used) : 0;
    for (int e0 = 0; e0 < p.new_width; e0 += kForkThreads) {
      const int e = e0 + tid;
      const bool goes = e >= x.full && e < end && goes_on(p, x.parent, e);
      int before = going;  // pages below e
      if (e0 < end && e0 + kForkThreads > x.full) {
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(goes);
        if ((tid & 63) == 0) s_going[tid >> 6] = __builtin_popcountll(lanes);
        __syncthreads();
        before += __builtin_popcountll(lanes & ((uint64_t(1) << (tid & 63)) - 1));
#pragma unroll
        for (int w = 0; w < kForkWaves; ++w) {
          before += w < tid >> 6 ? s_going[w] : 0;
          going += s_going[w];
        }
        __syncthreads();
      }
      if (e >= p.new_width) continue;
      int page = -1;
      if (e < x.used) {
        if (e < x.full) {
          if (e < p.width) page = page_of(p, x.parent, e);
        } else if (goes) {
          page = page_of(p, x.parent, e);
        } else if (!x.lost || e > x.full) {
          page = free.page(p, start + taken_before(x, e, before));
          if (page >= 0) atomicAdd(p.new_refs + page, 1);
        }
        absent += page < 0 || page >= p.pages;
      }
      p.new_table[int64_t(i) * p.new_width + e] = page;
    }
    if (p.absent && absent)
      atomicAdd(reinterpret_cast<unsigned long long*>(p.absent), static_cast<unsigned long long>(absent));
    return;
  }
  const int64_t unit = id - p.N - p.S;
  const int piece = int(unit % pieces), kv = int(unit / pieces) & 1;
  const int h = int(unit / pieces / 2 % p.H), i = int(unit / pieces / 2 / p.H);
  const int s = p.parents[i];
  if (s < 0 || s >= p.S) return;
  const Child x = child_of(p, i, p.first[s]);
  const int rows = x.kept & ((1 << p.page_shift) - 1);
  if (rows == 0 || x.full >= x.used || x.lost || piece * int64_t(kCopyBytes) >= int64_t(rows) * p.row_bytes) return;
  const int from = page_of(p, s, x.full);
  if (x.first && p.refs[from] == 1) return;
  const FreePages free(p, s_ends);
  const int to = free.page(p, p.start[i]);
  if (to < 0) return;
  const int64_t source = (int64_t(from) * p.H + h) << p.page_shift, target = (int64_t(to) * p.H + h) << p.page_shift;
  const int64_t a = int64_t(piece) * kCopyBytes, b = min(a + kCopyBytes, int64_t(rows) * p.row_bytes);
  const uint8_t* in = p.store[kv] + source * p.row_bytes;
  uint8_t* out = p.store[kv] + target * p.row_bytes;
  constexpr int kAtOnce = 4;
  for (int64_t at = a + 16 * tid; at < b; at += kAtOnce * 16 * kForkThreads) {
    u32x4 x[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      x[k] = *reinterpret_cast<const u32x4*>(in + min(at + k * 16 * kForkThreads, b - 16));
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (at + k * 16 * kForkThreads < b) *reinterpret_cast<u32x4*>(out + at + k * 16 * kForkThreads) = x[k];
  }
  if (p.scale[kv] && piece == 0)
    for (int r = tid; r < rows; r += kForkThreads) p.scale[kv][target + r] = p.scale[kv][source + r];
}

}  // namespace

ForkSize fork_size(int64_t sequences, int64_t new_sequences, int64_t pages) {
  ForkSize s;
  const int64_t steps = (pages + kForkStep - 1) / kForkStep;
  s.slice_pages = (steps + kForkSlices - 1) / kForkSlices * kForkStep;
  s.slices = (pages + s.slice_pages - 1) / s.slice_pages;
  int64_t at = 0;
  auto part = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 15) / 16 * 16;
    return here;
  };
  s.first = part(4 * sequences);
  s.children = part(4 * sequences);
  s.start = part(8 * (new_sequences + 1));
  s.lost = part(4);
  s.free_count = part(4 * s.slices);
  s.free_list = part(4 * s.slices * s.slice_pages);
  s.bytes = at;
  return s;
}

hipError_t launch_keep(const KeepParams& p, int D, int format, hipStream_t stream) {
  const int row = D * (format == kBf16 ? 2 : 1);
  if (row == 256) keep_variant<256>(p, stream);
  else if (row == 128) keep_variant<128>(p, stream);
  else keep_variant<64>(p, stream);
  return hipGetLastError();
}

hipError_t launch_fork(const ForkParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(fork_plan_kernel, dim3(unsigned(1 + p.slices)), dim3(kPlanThreads), 0, stream, p);
  const int64_t page_bytes = int64_t(p.row_bytes) << p.page_shift;
  const int pieces = int((page_bytes + kCopyBytes - 1) / kCopyBytes);
  const int64_t grid = int64_t(p.N) + p.S + (p.S ? int64_t(p.N) * p.H * 2 * pieces : 0);
  if (grid) hipLaunchKernelGGL(fork_kernel, dim3(unsigned(grid)), dim3(kForkThreads), 0, stream, p, pieces);
  return hipGetLastError();
}

}  // namespace sol
