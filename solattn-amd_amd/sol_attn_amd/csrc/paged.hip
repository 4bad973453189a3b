// Attention of new tokens over a paged cache, and over plain K / V under a
// sliding window with first tokens that stay visible.
//
// Query i of an entry with n queries and L keys has position p = L - n + i (L as
// the caller gives it, also past the keys that a page table names); key j < L is
// visible iff (j <= p or not causal) and (|p - j| < window or j <
// sinks).  O = sum_j softmax_j(scale q . k_j) v_j over the visible keys, 0 for
// a query that sees none.  Scores, softmax statistics and sums are FP32; the
// probabilities (times V's scales) are rounded to BF16 for their product with V
// on the matrix cores, as everywhere in this library (half a step each, 2^-8 at
// most, which averages out over the keys; the denominator sums the unrounded
// ones), where few rows leave them time as two BF16 terms.  (Two terms in
// wide_kernel would be half as many products again in a kernel whose matrix
// cores are busy for half of its time and more.)
//
// The rows of a (sequence, K/V head) are its new tokens times the G query
// heads that share the head, token by token: row r is token r / G, query head
// r % G of the group.  They are cut into tiles of R rows; a tile's keys are the
// union of what its rows see, in key tiles, and may be split over several
// workgroups ("parts"), whose softmax states the merge kernel joins.
//   step_kernel  R = 16, for few rows per sequence (single tokens) and small
//                calls: four waves, each with key tiles of its own
//   wide_kernel  R = 128, for chunks: four waves of 32 rows share every key tile
// paged_size() at the end chooses and says what both sides took.
//
// Cached INT8 and FP8 codes are converted to BF16 (exact); a key's scale
// multiplies its score, a value's scale its probability.
#include <algorithm>
#include <type_traits>

#include "attn_common.h"
#include "paged_internal.h"

namespace sol {

namespace {

constexpr int kNT = 256;  // threads per workgroup
constexpr int kWaves = kNT / kWave;

__device__ __forceinline__ int cdiv_i(int a, int b) { return (a + b - 1) / b; }

// ---- what is visible --------------------------------------------------------

// The keys a position sees: [lo, hi] and [0, sink).
struct Visible {
  int lo, hi, sink;
};

// Positions lie from -2^30 on and may be past every key, windows reach 2^31 - 1
// (none).
__device__ __forceinline__ Visible visible(const PagedParams& p, int pos, int length) {
  Visible v;
  v.lo = max(pos, p.window - 1) - (p.window - 1);
  v.hi = p.causal ? min(pos, length - 1) : min(pos, length - p.window) + p.window - 1;
  v.sink = min(p.sinks, p.causal ? v.hi + 1 : length);
  return v;
}

// The key tiles (of TK keys) that positions first .. last see: tiles [0, ns)
// and n - ns tiles from w0.
struct Span {
  int ns, w0, n;
  __device__ __forceinline__ int tile(int i) const { return i < ns ? i : w0 + (i - ns); }
};

template <int TK>
__device__ __forceinline__ Span span_of(const PagedParams& p, int first, int last, int length) {
  const int lo = visible(p, first, length).lo;
  const Visible v = visible(p, last, length);
  Span s;
  s.ns = v.sink > 0 ? (v.sink - 1) / TK + 1 : 0;
  s.w0 = max(s.ns, lo / TK);
  s.n = s.ns + (v.hi >= lo ? max(0, v.hi / TK + 1 - s.w0) : 0);
  return s;
}

// ---- which rows and keys a workgroup takes ----------------------------------

struct Item {
  int s, off, n, length;  // the sequence: first row, new tokens, keys
  int pos0;               // position of its first new token
  int r0, rows;           // the tile's rows r0 .. r0 + rows - 1 of the sequence's n G
  int part, parts;        // its share of the tile's keys
  int record;             // where its partial state goes, if there are several parts
};

// What the merge kernel has to join: a header per (split row tile, head), the
// tiles in order of sequences.
struct Header {
  int parts;         // 0: nothing
  int off, r0, rows; // Item's
  uint32_t first, step;  // record of its first part, and from one part to the next
};

// Partial states of split tiles, after the headers: per part (record) and row D
// sums, the maximum, the denominator and whether a key was seen.
template <int D>
constexpr int kRecordRow = D + 4;

template <int D, int R>
__device__ __forceinline__ float* record(const PagedParams& p, int64_t i) {
  return reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + p.header_bytes) + i * R * kRecordRow<D>;
}

// Header of split row tile `tile` for this workgroup's head.  Every thread writes
// the same: a branch on the thread made the compiler hold the keys' addresses,
// which the DMA takes from scalar registers, in vector ones.
__device__ __forceinline__ void write_header(const PagedParams& p, int64_t tile, const Header& hd) {
  if (tile >= 0 && tile < p.headers) static_cast<Header*>(p.workspace)[tile * p.H + blockIdx.x % p.H] = hd;
}

// Marks the headers past the last split tile as nothing, by the workgroups
// that have no item: the launch's last `idle` ones per head, of which this is
// number i.
__device__ __forceinline__ void clear_headers(const PagedParams& p, int64_t split_tiles, int64_t i, int64_t idle) {
  for (int64_t t = split_tiles + i; t < p.headers; t += idle) write_header(p, t, Header{0, 0, 0, 0, 0, 0});
}

// Record `part` of this workgroup's head.  (Lengths that change while the launch
// reads them could name one that there is not.)
__device__ __forceinline__ int record_of(const PagedParams& p, int64_t part) {
  return int(min(max(part, int64_t(0)) * p.H, p.records - p.H)) + int(blockIdx.x % p.H);
}

// Item `id` of the launch, in order of sequences, parts and row tiles; false
// past the last one.  Every workgroup forms the whole plan from the lengths on
// the device (two scans over the sequences, a few microseconds), so that a
// captured launch follows them and no launch or copy comes before this one.
// With p.target, parts are of at most z key tiles, z such that about p.target
// workgroups per head share all key tiles evenly: sum ceil(n_s / z) tiles_s is
// below target + sum tiles_s, the grid.  Without, one part each.  No tile has
// more than kMaxParts parts: the merge's time grows with them.
// A split tile has more than z >= sum / target key tiles, so there are fewer than
// target of them, and ceil(n / z) < 2 n / z makes their parts fewer than 2
// target: the headers and records of a launch, however many row tiles it has.
constexpr int kMaxParts = 128;

// A tile's key tiles at most in a part, of `sum` key tiles per head.
__device__ __forceinline__ int part_tiles(const PagedParams& p, int64_t sum) {
  return int(min(int64_t(1) << 30, max(int64_t(p.min_tiles), (sum + p.target - 1) / p.target)));
}

// Entries of plain K / V are all alike: the item by divisions alone.
template <int R, int TK>
__device__ __forceinline__ bool take_plain_item(const PagedParams& p, int id, Item& it) {
  const int rt = (p.Tq * p.G - 1) / R + 1, kt = max(1, span_of<TK>(p, p.Tk - p.Tq, p.Tk - 1, p.Tk).n);
  const int z = p.target ? part_tiles(p, int64_t(p.batch.S) * rt * kt) : 1 << 30;
  it.parts = __builtin_amdgcn_readfirstlane((kt - 1) / max(z, cdiv_i(kt, kMaxParts)) + 1);
  const int items = rt * it.parts;  // of an entry; all of them are fewer than 2^24 (the grid)
  it.s = __builtin_amdgcn_readfirstlane(id / items);
  if (it.s >= p.batch.S) {
    const int all = p.batch.S * items;
    if (p.records) clear_headers(p, it.parts > 1 ? p.batch.S * rt : 0, id - all, int(gridDim.x) / p.H - all);
    return false;
  }
  const int k = id - it.s * items;
  it.part = __builtin_amdgcn_readfirstlane(k / rt);
  const int tile = k - it.part * rt, row_tile = p.causal ? rt - 1 - tile : tile;
  it.off = it.s * p.Tq;
  it.n = p.Tq;
  it.length = p.Tk;
  it.pos0 = p.Tk - p.Tq;
  it.r0 = row_tile * R;
  it.rows = min(R, it.n * p.G - it.r0);
  if (it.parts > 1) {
    it.record = record_of(p, id);
    if (it.part == 0)
      write_header(p, int64_t(it.s) * rt + tile,
                   Header{it.parts, it.off, it.r0, it.rows, uint32_t(it.record), uint32_t(rt) * uint32_t(p.H)});
  }
  return true;
}

template <int R, int TK, bool PAGED>
__device__ __forceinline__ bool take_item(const PagedParams& p, int64_t id, Item& it) {
  if constexpr (!PAGED) return take_plain_item<R, TK>(p, int(id), it);
  __shared__ int64_t s_total[kWaves];
  __shared__ uint64_t s_split[kWaves];
  __shared__ int s_found[10];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int S = p.batch.S;
  // A sequence's first row, new tokens and end, and its row tiles and key tiles
  // (which matter with p.target alone).
  struct Sizes {
    int off, n, end, row_tiles, key_tiles;
  };
  auto sizes = [&](int s) {
    Sizes x = {0, 0, 0, 0, 0};
    if (s < S) {
      x.off = p.batch.offset(s);
      x.n = p.batch.offset(s + 1) - x.off;
      x.end = p.batch.end(s);
      x.row_tiles = x.n > 0 ? (x.n * p.G - 1) / R + 1 : 0;
      if (p.target && x.n > 0)
        x.key_tiles = max(1, span_of<TK>(p, x.end - x.n, x.end - 1, min(x.end, p.batch.positions())).n);
    }
    return x;
  };
  const Sizes mine0 = sizes(tid);  // read once where there are no more sequences than threads
  int z = 1 << 30;
  if (p.target) {
    int64_t sum = 0;
#pragma unroll 4
    for (int s = tid; s < S; s += kNT) {
      const Sizes x = s == tid ? mine0 : sizes(s);
      sum += int64_t(x.row_tiles) * x.key_tiles;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if (lane == 0) s_total[wave] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += s_total[w];
    sum = int64_t(uniform64(uint64_t(sum)));
    z = part_tiles(p, sum);
    __syncthreads();
  }
  int64_t base = 0;
  uint64_t split = 0;  // of the sequences before s0: parts of split tiles, times 2^32, and the tiles
  auto parts_of = [&](const Sizes& x) {
    return p.target && x.row_tiles ? (x.key_tiles - 1) / max(z, cdiv_i(x.key_tiles, kMaxParts)) + 1 : 1;
  };
  auto split_of = [&](const Sizes& x, int64_t items) {
    return items > x.row_tiles ? (uint64_t(items) << 32) + uint32_t(x.row_tiles) : 0ull;
  };
  // Larger batches: kEach consecutive sequences per thread, as a step of the scan
  // costs two barriers (4,096 sequences of 256 keys, 8 heads: 1,172 us, 1,297
  // with one each).
  constexpr int kEach = 8;
  const int each = S <= kNT ? 1 : kEach;
  for (int s0 = 0; s0 < S; s0 += kNT * each) {
    int s = s0 + tid * each;
    Sizes mine_of[kEach] = {mine0};
    int64_t mine = 0;
    uint64_t mine_split = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      if (j && each == 1) break;
      if (each > 1) mine_of[j] = sizes(s + j);
      const int64_t items = int64_t(mine_of[j].row_tiles) * parts_of(mine_of[j]);
      mine += items;
      mine_split += split_of(mine_of[j], items);
    }
    int64_t end = mine;  // inclusive sums over the wave
    uint64_t split_end = mine_split;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t a = __shfl_up(end, off);
      if (lane >= off) end += a;
      if (p.target) {
        const uint64_t b = uint64_t(__shfl_up(int64_t(split_end), off));
        if (lane >= off) split_end += b;
      }
    }
    if (lane == 63) s_total[wave] = end, s_split[wave] = split_end;
    __syncthreads();
    int64_t all = 0;
    uint64_t all_split = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) end += all + base, split_end += all_split + split;
      all += s_total[w];
      all_split += s_split[w];
    }
    if (id >= end - mine && id < end) {
      // Row tile by row tile of a part (they read the same keys), the longest first.
      int64_t first = end - mine;
      uint64_t before = split_end - mine_split;
      Sizes x = mine_of[0];
#pragma unroll
      for (int j = 1; j < kEach; ++j) {
        if (each == 1) break;
        const int64_t items = int64_t(x.row_tiles) * parts_of(x);
        if (id < first + items) break;
        first += items;
        before += split_of(x, items);
        x = mine_of[j];
        s += 1;
      }
      const int k = int(id - first), rt = x.row_tiles;
      s_found[0] = s;
      s_found[1] = p.causal ? rt - 1 - k % rt : k % rt;
      s_found[2] = k / rt;
      s_found[3] = parts_of(x);
      s_found[4] = int(uint32_t(before)) + k % rt;
      s_found[5] = rt;
      s_found[6] = x.off;
      s_found[7] = x.n;
      s_found[8] = x.end;
      s_found[9] = int(before >> 32) + k;
    }
    __syncthreads();
    base += int64_t(uniform64(uint64_t(all)));
    split += uniform64(all_split);
    if (id < base) break;
  }
  if (id >= base) {
    if (p.records) clear_headers(p, uint32_t(split), id - base, int(gridDim.x) / p.H - base);
    return false;
  }
  it.s = __builtin_amdgcn_readfirstlane(s_found[0]);
  it.off = __builtin_amdgcn_readfirstlane(s_found[6]);
  it.n = __builtin_amdgcn_readfirstlane(s_found[7]);
  const int end = __builtin_amdgcn_readfirstlane(s_found[8]);
  it.length = min(end, p.batch.positions());
  it.pos0 = end - it.n;
  it.r0 = __builtin_amdgcn_readfirstlane(s_found[1]) * R;
  it.rows = min(R, it.n * p.G - it.r0);
  it.part = __builtin_amdgcn_readfirstlane(s_found[2]);
  it.parts = __builtin_amdgcn_readfirstlane(s_found[3]);
  if (it.parts > 1) {
    it.record = record_of(p, __builtin_amdgcn_readfirstlane(s_found[9]));
    if (it.part == 0)
      write_header(p, __builtin_amdgcn_readfirstlane(s_found[4]),
                   Header{it.parts, it.off, it.r0, it.rows, uint32_t(it.record),
                          uint32_t(__builtin_amdgcn_readfirstlane(s_found[5])) * uint32_t(p.H)});
  }
  return true;
}

// ---- where the keys lie -----------------------------------------------------

// Key tiles are cut into groups of 16 rows, each of which lies in one page (a
// page holds at least 16); a bit for each group that has a page.
template <int TK>
constexpr uint32_t kAllGroups = (1u << (TK / 16)) - 1u;

// K and V rows of one (sequence, head): in a cache, rows of kRowBytes that
// both operands (and their scales) have at the same index; or plain, at strides
// of their own.
template <int D, int F, bool PAGED>
struct Keys {
  static constexpr uint32_t kRowBytes = D * kElemBytes<F>;
  const uint8_t* base[2];
  const float* scale[2];
  const int32_t* table;
  uint32_t st[2];             // plain: bytes between rows
  int shift, pages, H, h, last;  // last: the last key

  __device__ __forceinline__ Keys(const PagedParams& p, const Item& it, int head) {
    shift = p.batch.page_shift;
    pages = p.batch.pages;
    H = p.H;
    h = head;
    last = it.length - 1;
    table = PAGED ? p.batch.table + int64_t(it.s) * p.batch.width : nullptr;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      base[kv] = p.store[kv] + (PAGED ? 0 : int64_t(h) * p.sh[kv] + int64_t(it.s) * p.sb[kv]);
      scale[kv] = p.scale[kv];
      st[kv] = PAGED ? kRowBytes : uint32_t(p.st[kv]);
    }
  }
};

// Where the groups of kTiles key tiles of a list begin, one lane per group:
// byte offsets from the cache's first K (V) row, handed out through the scalar
// registers.  (Page numbers read one by one through the scalar cache made every
// wait for an LDS read wait for all of them, and their address arithmetic came
// before each tile's products.)
template <int D, int F, bool PAGED, int TK>
struct PageWindow {
  static constexpr int kGroups = TK / 16, kTiles = 64 / kGroups;
  static constexpr uint32_t kRowBytes = D * kElemBytes<F>;
  int id, pos;
  uint32_t lo, hi;
  uint64_t ok;

  // Starts the read of a window's page numbers; groups past the last key take
  // its page.  tile_of(i): tile i of the window.
  template <typename TileOf>
  __device__ __forceinline__ void fetch(const Keys<D, F, PAGED>& keys, TileOf tile_of, int lane) {
    if constexpr (PAGED) {
      pos = tile_of(lane / kGroups) * TK + 16 * (lane % kGroups);
      id = keys.table[min(pos, keys.last) >> keys.shift];
    }
  }
  // Makes the window read last the current one.
  __device__ __forceinline__ void turn(const Keys<D, F, PAGED>& keys) {
    if constexpr (PAGED) {
      const bool in = uint32_t(id) < uint32_t(keys.pages);
      ok = __builtin_amdgcn_ballot_w64(in);
      const uint64_t row = ((uint64_t(in ? uint32_t(id) : 0u) * uint32_t(keys.H) + uint32_t(keys.h)) << keys.shift) +
                           uint32_t(pos & ((1 << keys.shift) - 1));
      lo = uint32_t(row * kRowBytes);
      hi = uint32_t(row * kRowBytes >> 32);
    }
  }
  // Group g of tile i.
  __device__ __forceinline__ uint64_t offset(int i, int g) const {
    if constexpr (!PAGED) return 0;
    const uint32_t l = uint32_t(__builtin_amdgcn_readlane(lo, i * kGroups + g));
    const uint32_t h = uint32_t(__builtin_amdgcn_readlane(hi, i * kGroups + g));
    return uint64_t(h) << 32 | l;
  }
  // Row of the cache (of both operands and their scales) of row `row` of tile i, per lane.
  __device__ __forceinline__ uint64_t row(int i, int row) const {
    const int from = i * kGroups + (row >> 4);
    return (uint64_t(uint32_t(__shfl(int(hi), from))) << 32 | uint32_t(__shfl(int(lo), from))) / kRowBytes + (row & 15);
  }
  __device__ __forceinline__ uint32_t valid(int i) const {
    if constexpr (!PAGED) return kAllGroups<TK>;
    return uint32_t(ok >> (i * kGroups)) & kAllGroups<TK>;
  }
};

// ---- codes ------------------------------------------------------------------

typedef const u32x4 __attribute__((address_space(1)))* global_chunk_ptr;

__device__ __forceinline__ u32x4 load_chunk(const uint8_t* p) { return *(global_chunk_ptr)(uintptr_t)p; }

// Eight codes as BF16 (exact: at most 8 significant bits).
template <int F>
__device__ __forceinline__ u32x4 codes_to_bf16(uint32_t lo, uint32_t hi) {
  u32x4 o;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint32_t c = w ? hi : lo;
    if constexpr (F == kInt8) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = float(int32_t(c << (24 - 8 * i)) >> 24);
      o[2 * w] = pack_bf16x2(v[0], v[1]);
      o[2 * w + 1] = pack_bf16x2(v[2], v[3]);
    } else {
      o[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, false));
      o[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, true));
    }
  }
  return o;
}

// LDS image of a key tile of TK rows: K then V, BF16, in TileLayout's order.
template <int D, int TK>
struct TileImage {
  static constexpr int kElems = TK * D;
  static constexpr int CPR = D / 8;
  __device__ static __forceinline__ void put(uint16_t* slot, int kv, int row, int chunk, const u32x4& x) {
    const int at = kv ? kElems + TileLayout<D>::v_offset(row, chunk) : TileLayout<D>::k_offset(row, chunk);
    *reinterpret_cast<u32x4*>(slot + at) = x;
  }
  // This lane's K operand of half t, k-step ks.
  __device__ static __forceinline__ u32x4 k(const uint16_t* slot, int col, int hh, int t, int ks) {
    const int at = (32 * t + col) * D + (TileLayout<D>::k_lane_xor(col, hh) ^ (16 * ks));
    return *reinterpret_cast<const u32x4*>(slot + at);
  }
  // This lane's V^T operand (FragLane's addresses): feature 32 dt + col, keys
  // 32 t + 16 c4 + 4 hh + {0..3, 8..11}.
  __device__ static __forceinline__ u32x4 v(const uint16_t* slot, int col, int hh, int t, int c4, int dt) {
    const int chunk = hh * 4 * CPR + 4 * ((col >> 2) & 3) + 2 * (col >> 4) + ((col & 3) >> 1);
    const uint32_t lane = lds_address(slot) + uint32_t(2 * (kElems + 8 * chunk + 4 * (col & 1)));
    const uint32_t a = lane + uint32_t(64 * CPR * (8 * t + 4 * c4) + 256 * dt);
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SOL_LDS i16x4*)(uintptr_t)a);
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SOL_LDS i16x4*)(uintptr_t)(a + 128u * CPR));
    const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
    const u32x4 r = {x[0], x[1], y[0], y[1]};
    return r;
  }
};

// ---- the softmax and P V of 32 keys -----------------------------------------

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Bit 15 of every 16-bit half that is an infinity or a NaN.
__device__ __forceinline__ uint32_t nonfinite(uint32_t x) { return ((x & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }

// Adds V's elements that are not finite, of half t of a tile, to the sums of the
// queries that see their keys.  (A product with P = 0 must not spread them to
// the others, so the matrix cores take zeros for them.)  Rare: a loop over the
// keys, written for few registers; the sums are added to in place.
template <int D, int TK>
__device__ __forceinline__ void add_nonfinite(State<D>& st, const uint16_t* slot, int t, int hh, uint32_t seen) {
  using Image = TileImage<D, TK>;
  // The adds below are inline assembly, before which the compiler does not keep
  // the distance that a vector instruction needs from the matrix instruction
  // whose result it reads (19 wait states at most).
#pragma unroll
  for (int dt = 0; dt < Shape<D>::DT; ++dt) asm volatile("s_nop 15\n\ts_nop 7" : "+v"(st.acc[dt]));
  // Key r is score element 4 (r / 8) + r % 4 of lane half (r / 4) % 2.
  const auto both = __builtin_amdgcn_permlane32_swap(seen, seen, false, false);
#pragma unroll 1
  for (int r = 0; r < 32; ++r) {
    const bool on = (((r & 4) ? both[1] : both[0]) >> (4 * (r >> 3) + (r & 3))) & 1u;
#pragma unroll
    for (int dt = 0; dt < Shape<D>::DT; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int at = Image::kElems + TileLayout<D>::v_offset(32 * t + r, 4 * dt + q) + 4 * hh;
        const u32x2 x = *reinterpret_cast<const u32x2*>(slot + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t b = (i & 1) ? x[i >> 1] >> 16 : x[i >> 1] & 0xFFFFu;
          const float add = on && (b & 0x7F80u) == 0x7F80u ? bf16_bits_to_f32(b) : 0.f;
          asm volatile("v_add_f32 %0, %0, %1" : "+v"(st.acc[dt][4 * q + i]) : "v"(add));
        }
      }
  }
}

// This lane's query: its position, and whether it saw a key.
struct LaneRow {
  int pos;
  bool any;
};

// Sixteen per-key factors of this lane's score elements of a half (key 8 (e /
// 4) + 4 hh + e % 4), from LDS.
__device__ __forceinline__ f32x16 key_factors(const float* half, int hh) {
  f32x16 f;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(half + 8 * q + 4 * hh);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[4 * q + i] = x[i];
  }
  return f;
}

// Online softmax of raw scores s (half t of the tile in `slot`, keys from j0 on)
// and O^T += V^T P^T, hidden keys taking no part, whatever their score, value
// and scale hold.
// `valid`: bits of the half's two groups of 16 rows that have a page.  scales:
// the half's K scales times c in LDS (V's scales TK floats on), or null.
template <int D, int TK, int F>
__device__ __forceinline__ void attend_masked(const PagedParams& p, int length, State<D>& st, LaneRow& row, f32x16 s,
                                              const uint16_t* slot, int t, int j0, uint32_t valid, int lane_col,
                                              int lane_hh, const float* scales) {
  const int col = fresh(lane_col), hh = fresh(lane_hh);
  const float c = scales ? 1.f : p.scale_log2;
  const Visible v = visible(p, fresh(row.pos), length);  // not held in registers over the stream
  if (scales) {
    const f32x16 sk = key_factors(scales, hh);
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] *= sk[e];
  }
  uint32_t seen = 0;
  const int a = j0 + 4 * hh;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int j = a + 8 * (e >> 2) + (e & 3);
    const bool in = (((j <= v.hi) & (j >= v.lo)) | (j < v.sink)) & (((valid >> (e >> 3)) & 1u) != 0);
    s[e] = in ? s[e] : kNegInf;
    seen |= in ? 1u << e : 0u;
  }
  row.any |= seen != 0;
  float mx = s[0];
#pragma unroll
  for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
  mx = pair_max(mx) * c;
  if (__builtin_amdgcn_ballot_w64(mx > st.m)) {
    const float mnew = fmaxf(st.m, mx);
    const float alpha = mnew == kNegInf ? 1.f : fast_exp2(st.m - mnew);
    st.m = mnew;
    st.den *= alpha;
    rescale_acc<D>(st, alpha);
  }
  const float neg_m = st.m == kNegInf ? 0.f : -st.m;
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    s[e] = fast_exp2(fmaf(s[e], c, neg_m));
    sum += s[e];
  }
  st.den += sum;
  if (scales) {
    const f32x16 sv = key_factors(scales + TK, hh);
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = (seen >> e) & 1u ? s[e] * sv[e] : 0.f;
  }
  const bf16x8 pb[2] = {pack8(s, 0), pack8(s, 8)};
  // Scheduled apart from the scores: V's operands are not held meanwhile.
  chunk_end();
  u32x4 vt[2][Shape<D>::DT];
  u16x2 most = {0, 0};  // magnitudes compare like their bits
#pragma unroll
  for (int c4 = 0; c4 < 2; ++c4)
#pragma unroll
    for (int dt = 0; dt < Shape<D>::DT; ++dt) {
      vt[c4][dt] = TileImage<D, TK>::v(slot, col, hh, t, c4, dt);
      if constexpr (F != kInt8)  // INT8 codes are finite
#pragma unroll
        for (int i = 0; i < 4; ++i)
          most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, vt[c4][dt][i] & 0x7FFF7FFFu));
    }
  const bool some = F != kInt8 && __builtin_amdgcn_ballot_w64(nonfinite(__builtin_bit_cast(uint32_t, most)) != 0) != 0;
  if (some) {
#pragma unroll
    for (int c4 = 0; c4 < 2; ++c4)
#pragma unroll
      for (int dt = 0; dt < Shape<D>::DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) vt[c4][dt][i] &= ~((nonfinite(vt[c4][dt][i]) >> 15) * 0xFFFFu);
  }
#pragma unroll
  for (int c4 = 0; c4 < 2; ++c4)
#pragma unroll
    for (int dt = 0; dt < Shape<D>::DT; ++dt) st.acc[dt] = mfma32x32x16(as_bf16x8(vt[c4][dt]), pb[c4], st.acc[dt]);
  if (some) add_nonfinite<D, TK>(st, slot, t, hh, seen);
}

// ---- results ----------------------------------------------------------------

// Element offset of row r (of a sequence's n G) of the output.
template <int D>
__device__ __forceinline__ int64_t output_row(const PagedParams& p, int off, int r, int h) {
  return ((int64_t(off) + r / p.G) * (p.H * p.G) + h * p.G + r % p.G) * D;
}

// Four features of a finished row.
__device__ __forceinline__ void store4(uint16_t* out, const f32x4& x, float den, bool any) {
  const float inv = __fdiv_rn(1.f, den);
  u32x2 o;
  o[0] = pack_bf16x2(quotient(x[0], den, inv), quotient(x[1], den, inv));
  o[1] = pack_bf16x2(quotient(x[2], den, inv), quotient(x[3], den, inv));
  if (!any) o[0] = o[1] = 0u;
  *reinterpret_cast<u32x2*>(out) = o;
}

// Joins the parts of split tiles: m = max_s m_s, O = sum_s 2^(m_s - m) acc_s /
// sum_s 2^(m_s - m) den_s.  A workgroup per (row tile, head) and some of its
// rows.  D / 4 lanes take 4 features each.  Tiles of 16 rows have many parts
// and few rows: a row at a time, the 1,024 / D such groups of lanes take the
// parts in turn, kMergeAhead each in flight, and their states join in a fixed
// order.  Tiles of 128 rows have few parts: each group takes a row of its own.
// Bound by its launch (5 us with its reads' latency) or by memory: two parts of
// 4,032 rows of 24 heads of 128, 129 MB, 43 us after the attention, 3.0 TB/s (148
// us a row at a time).
constexpr int kMergeAhead = 8;

// A state of the merge: sums of 4 features, and the row's maximum, denominator
// and whether a key was seen.
struct Joined {
  f32x4 o;
  float m, den, any;
  __device__ __forceinline__ void add(const Joined& x) {
    any += x.any;
    const float mn = fmaxf(m, x.m);
    // A side that has scored nothing (or only -inf) has no sums, but may have a
    // NaN, which stays.
    const float a = m == kNegInf ? 1.f : fast_exp2(m - mn), b = x.m == kNegInf ? 1.f : fast_exp2(x.m - mn);
    m = mn;
    den = den * a + x.den * b;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = o[k] * a + x.o[k] * b;
  }
};

// Joins every `stride`-th part of a row from part `first` on; `row`: its record
// in part 0, `step` floats on the next part's.
template <int D>
__device__ __forceinline__ Joined join_parts(const float* row, int64_t step, int parts, int first, int stride, int c) {
  Joined mine = {{0.f, 0.f, 0.f, 0.f}, kNegInf, 0.f, 0.f};
  for (int s0 = first; s0 < parts; s0 += stride * kMergeAhead) {
    f32x4 tail[kMergeAhead], x[kMergeAhead];
#pragma unroll
    for (int u = 0; u < kMergeAhead; ++u) {
      const float* at = row + min(s0 + u * stride, parts - 1) * step;
      tail[u] = *reinterpret_cast<const f32x4*>(at + D);
      x[u] = *reinterpret_cast<const f32x4*>(at + 4 * c);
    }
#pragma unroll
    for (int u = 0; u < kMergeAhead; ++u)
      if (s0 + u * stride < parts) mine.add(Joined{x[u], tail[u][0], tail[u][1], tail[u][2]});
  }
  return mine;
}

// Rows that a workgroup of the merge takes at once.
template <int D, int R>
constexpr int kMergeRows = R == 16 ? 1 : kNT / (D / 4);

template <int D, int R>
__global__ __launch_bounds__(kNT) void merge_kernel(PagedParams p) {
  constexpr int kLanes = D / 4, kSlots = kNT / kLanes;
  __shared__ Joined s_state[kWaves][kLanes];
  Header hd = static_cast<const Header*>(p.workspace)[blockIdx.x];
  // Offsets that do not ascend can leave headers of another call here, and name
  // more parts than the launch has: nothing outside the tensors is touched.
  if (hd.parts <= 1 || int64_t(hd.first) >= p.records || hd.step == 0 || hd.rows <= 0 || hd.rows > R || hd.off < 0 ||
      hd.r0 < 0 || int64_t(hd.off) + (int64_t(hd.r0) + hd.rows - 1) / p.G >= p.new_rows)
    return;
  hd.parts = int(min(int64_t(hd.parts), (p.records - 1 - hd.first) / hd.step + 1));
  const int h = blockIdx.x % p.H, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % kLanes;
  const int slot = threadIdx.x / kLanes;
  const int64_t step = int64_t(hd.step) * R * kRecordRow<D>;
  const float* base = record<D, R>(p, hd.first);
  auto store = [&](int r, const Joined& x) {
    store4(p.out + output_row<D>(p, hd.off, hd.r0 + r, h) + 4 * c, x.o, x.den, x.any != 0.f);
  };
  if constexpr (kMergeRows<D, R> > 1) {
    for (int r = blockIdx.y * kSlots + slot; r < hd.rows; r += gridDim.y * kSlots)
      store(r, join_parts<D>(base + r * kRecordRow<D>, step, hd.parts, 0, 1, c));
  } else {
    for (int r = blockIdx.y; r < hd.rows; r += gridDim.y) {
      Joined mine = join_parts<D>(base + r * kRecordRow<D>, step, hd.parts, slot, kSlots, c);
#pragma unroll
      for (int off = kLanes; off < kWave; off <<= 1) {
        Joined other;
#pragma unroll
        for (int k = 0; k < 4; ++k) other.o[k] = __shfl_xor(mine.o[k], off);
        other.m = __shfl_xor(mine.m, off);
        other.den = __shfl_xor(mine.den, off);
        other.any = __shfl_xor(mine.any, off);
        mine.add(other);
      }
      if (lane < kLanes) s_state[wave][lane] = mine;
      __syncthreads();
      if (wave == 0 && lane < kLanes) {
#pragma unroll
        for (int w = 1; w < kWaves; ++w) mine.add(s_state[w][lane]);
        store(r, mine);
      }
      __syncthreads();
    }
  }
}

// ---- few rows ---------------------------------------------------------------
//
// Matrix products of 16 x 16 x 32: S^T = K Q^T has a query per column and four
// keys per lane, O^T = V^T P^T a query per column and four features per lane, so
// the softmax's vector work per key is half of the 32 x 32 form's.  A operand:
// lane l supplies row l % 16, k-slots 8 (l / 16) .. + 7; B operand: column l %
// 16, the same slots; C: lane l holds column l % 16, rows 4 (l / 16) + e.

__device__ __forceinline__ f32x4 mfma16x16x32(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Keeps a wave's LDS writes and reads of its own slot in program order (the
// hardware runs them in order; nothing is emitted).
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Every LDS read of the wave has returned: its slot may be written.
__device__ __forceinline__ void lds_returned() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Maximum / sum over the four lanes (l % 16 alike) that share a query.
__device__ __forceinline__ float quad_max(float x) {
  x = pair_max(x);
  const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}

__device__ __forceinline__ float quad_sum(float x) {
  x = pair_sum(x);
  const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}

// Key tiles of the step kernel: 16 KB of stored K and V rows each, which a wave
// moves through its LDS slot as they are (8-bit codes are converted as they are
// read).  Chunks are 16 bytes.
//   K, row by row, chunk c of row r at c ^ k_swizzle(r): the 16 rows that a
//      phase of an operand read takes meet different banks.
//   V, BF16: row quads, chunk c of row r at chunk (c >> 2) 16 + (r & 3) 4 + ((c &
//      3) ^ 2 (quad & 1)) of quad r >> 2; a 16-bit transpose read takes 16
//      features of a quad per lane group, neighbouring quads from different
//      banks.
//   V, codes: row by row, chunk c of row r at c ^ v_swizzle(r); an 8-bit
//      transpose read takes 16 features of 8 rows per lane group: lane j reads
//      row j >> 1, bytes 8 (j & 1) .. + 7, and gets feature j of the 8 rows.
// The scores of a pair of key blocks (32 keys from 32 h on) sit so that a lane's
// eight are the keys of its V^T operand: element e of block 2 h + b in lane group
// g is key 32 h + 16 b + 4 g + e with BF16, 32 h + 8 g + 4 b + e with codes.
template <int D, int F>
struct StepSlot {
  static constexpr bool kCodes = F != kBf16;
  static constexpr int kRow = D * kElemBytes<F>;  // bytes
  static constexpr int TK = 8192 / kRow;
  static constexpr int kPlane = 8192;             // bytes of K, then of V
  static constexpr int kQuad = 4 * kRow;
  static constexpr int kReads = kCodes ? D / 64 : D / 32;  // K chunks per lane and key block
  uint32_t k_lane;     // LDS address of this lane's K chunk 0 of key block 0
  uint32_t v_lane[2];  // of its V reads (BF16: for even and odd feature blocks)

  __device__ __forceinline__ static int k_swizzle(int r) {
    if (!kCodes) return TileLayout<D>::k_swizzle(r);
    return D == 128 ? ((r >> 1) & 1) | ((r >> 3) & 3) << 1 : (r >> 3) & 3;
  }
  __device__ __forceinline__ static int v_swizzle(int r) { return D == 128 ? (r >> 1) & 7 : (r >> 2) & 3; }
  // Byte offset of chunk c of row r.
  __device__ __forceinline__ static int offset(int kv, int r, int c) {
    if (!kv) return r * kRow + 16 * (c ^ k_swizzle(r));
    if (kCodes) return kPlane + r * kRow + 16 * (c ^ v_swizzle(r));
    const int quad = r >> 2;
    return kPlane + quad * kQuad + 16 * ((c >> 2) * 16 + (r & 3) * 4 + ((c & 3) ^ (2 * (quad & 1))));
  }
  // Key of score element e of block kb in lane group g.
  __device__ __forceinline__ static int key(int kb, int g, int e) {
    return kCodes ? 32 * (kb >> 1) + 8 * g + 4 * (kb & 1) + e : 16 * kb + 4 * g + e;
  }

  __device__ __forceinline__ StepSlot(const uint8_t* slot, int lane) {
    const int i = lane & 15, g = lane >> 4;
    const uint32_t base = lds_address(slot);
    const int r = kCodes ? 8 * (i >> 2) + (i & 3) : i;  // the K row of A operand row i
    k_lane = base + r * kRow + 16 * (g ^ k_swizzle(r));
    if constexpr (kCodes) {
      const int vr = 8 * g + (i >> 1);
      v_lane[0] = v_lane[1] = base + kPlane + vr * kRow + 16 * v_swizzle(vr) + 8 * (i & 1);
    } else {
      const uint32_t at = base + kPlane + g * kQuad + 64 * (i >> 2) + 16 * ((i >> 1) & 1) + 8 * (i & 1);
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) v_lane[odd] = at + 32u * (odd ^ (g & 1));
    }
  }
  // K chunk n of key block kb: features 32 n + 8 g .. + 7, or the codes 64 n + 16 g .. + 15.
  __device__ __forceinline__ u32x4 k(int kb, int n) const {
    const uint32_t block = kCodes ? (kb >> 1) * 32 * kRow + (kb & 1) * 4 * kRow : kb * 16 * kRow;
    return *(const SOL_LDS u32x4*)(uintptr_t)((k_lane ^ (64u * n)) + block);
  }
  // V^T of feature block fb (16 features) for the 32 keys from 32 h on.
  __device__ __forceinline__ u32x4 v(int h, int fb) const {
    if constexpr (kCodes) {
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          (SOL_LDS i32x2*)(uintptr_t)((v_lane[0] ^ (16u * fb)) + 32 * h * kRow));
      return codes_to_bf16<F>(x[0], x[1]);
    } else {
      const uint32_t a = v_lane[fb & 1] + uint32_t(8 * h * kQuad + 256 * (fb >> 1));
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SOL_LDS i16x4*)(uintptr_t)a);
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SOL_LDS i16x4*)(uintptr_t)(a + 4u * kQuad));
      const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
      const u32x4 r = {x[0], x[1], y[0], y[1]};
      return r;
    }
  }
};

// 4-byte global -> LDS DMA per lane, each from an address of its own; lane l's
// bytes land at LDS address m + 4 l (dma16's notes).
__device__ __forceinline__ void dma4(uint64_t address, uint32_t m) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %1, off"
      :
      : "s"(m), "v"(address)
      : "memory", "m0");
}

// The DMA of a wave's next key tile into its slot, K and V apart: 1 KB pieces
// of kRows rows each, whose rows lie in one page.  A lane's place in a piece
// names the (row, chunk) it reads, the row's swizzle taken from the piece's
// first row and the lane's by exclusive or.
template <int D, int F, bool PAGED>
struct StepDma {
  using Slot = StepSlot<D, F>;
  using Source = Keys<D, F, PAGED>;
  static constexpr int TK = Slot::TK;
  static constexpr int kPieces = 8;
  static constexpr int kRows = TK / kPieces;
  static_assert(kRows <= 16, "the rows of a piece lie in one page");
  static constexpr int kScales = F == kBf16 ? 0 : TK / 64;
  static constexpr int kLoads = kPieces + kScales;  // of K, and of V
  int row[2];         // this lane's row of a piece
  uint32_t chunk[2];  // its chunk, in bytes
  uint32_t slot, scales;
  int tile, lane;
  uint32_t valid;
  uint64_t group[PAGED ? TK / 16 : 1];  // where each group begins
  uint64_t scale_row[kScales ? kScales : 1];

  __device__ __forceinline__ StepDma(uint32_t slot_lds, uint32_t scales_lds, int l)
      : slot(slot_lds), scales(scales_lds), lane(l) {
    constexpr int kRowLanes = Slot::kRow / 16;
    row[0] = l / kRowLanes;
    chunk[0] = 16u * ((l % kRowLanes) ^ Slot::k_swizzle(row[0]));
    if constexpr (Slot::kCodes) {
      row[1] = row[0];
      chunk[1] = 16u * ((l % kRowLanes) ^ Slot::v_swizzle(row[1]));
    } else {
      const int quad = D == 128 ? 0 : l >> 5, m = D == 128 ? l : l & 31;  // of the piece's quads
      row[1] = 4 * quad + ((m >> 2) & 3);
      chunk[1] = 16u * (4 * (m >> 4) + ((m & 3) ^ (2 * (quad & 1))));
    }
  }

  // Tile t, the window's tile i.
  template <typename Window>
  __device__ __forceinline__ void prepare(const Window& window, int i, int t) {
    tile = t;
    valid = window.valid(i);
    if constexpr (PAGED) {
#pragma unroll
      for (int g = 0; g < TK / 16; ++g) group[g] = window.offset(i, g);
#pragma unroll
      for (int n = 0; n < kScales; ++n) scale_row[n] = window.row(i, 64 * n + lane);
    }
  }

  // Starts K's (V's) loads of the prepared tile; the slot's reads have returned.
  __device__ __forceinline__ void issue(const Source& keys, int kv) const {
    const uint64_t base = reinterpret_cast<uint64_t>(keys.base[kv]);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int r = kRows * i;
      const uint32_t flip = kv ? (Slot::kCodes ? 16u * Slot::v_swizzle(r) : (D == 128 ? 32u * (i & 1) : 0u))
                               : 16u * Slot::k_swizzle(r);
      const uint32_t dst = slot + uint32_t(kv * Slot::kPlane + i * 1024);
      if constexpr (PAGED) {
        dma16(base + group[r / 16] + uint32_t(r % 16) * Slot::kRow,
              row[kv] * Slot::kRow + (chunk[kv] ^ flip), dst);
      } else {
        const int first = min(tile * TK + r, keys.last);
        const uint32_t off = uint32_t(min(tile * TK + r + row[kv], keys.last) - first) * keys.st[kv];
        dma16(base + uint64_t(uint32_t(first)) * keys.st[kv] + round_offset(0u), off + (chunk[kv] ^ flip), dst);
      }
    }
#pragma unroll
    for (int n = 0; n < kScales; ++n)
      dma4(reinterpret_cast<uint64_t>(keys.scale[kv] + scale_row[n]),
           scales + uint32_t(kv * TK + 64 * n) * 4u);
  }
};

// A wave's state for its 16 queries.
template <int D>
struct StepState {
  f32x4 acc[D / 16];
  float m, den;
};

// Adds V's elements that are not finite to the sums of the queries that see
// their keys (as add_nonfinite: the products took zeros for them).  Bit 4 kb +
// e of `seen`: this lane's query sees that score element's key.
template <int D, int F>
__device__ __forceinline__ void step_nonfinite(StepState<D>& st, const uint8_t* slot, int lane, uint32_t seen) {
  using Slot = StepSlot<D, F>;
  // Distance of the inline assembly below from the matrix instructions.
#pragma unroll
  for (int fb = 0; fb < D / 16; ++fb) asm volatile("s_nop 15\n\ts_nop 7" : "+v"(st.acc[fb]));
  const int g = lane >> 4;
#pragma unroll 1
  for (int r = 0; r < Slot::TK; ++r) {
    // The lane group and element that hold key r.
    const int rg = Slot::kCodes ? r >> 3 & 3 : r >> 2 & 3;
    const int kb = Slot::kCodes ? 2 * (r >> 5) + (r >> 2 & 1) : r >> 4;
    const uint32_t bits = uint32_t(__shfl(int(seen), (lane & 15) + 16 * rg));
    const bool on = (bits >> (4 * kb + (r & 3))) & 1u;
#pragma unroll
    for (int fb = 0; fb < D / 16; ++fb) {
      // Features 16 fb + 4 g .. + 3.
      uint32_t w[2];
      if constexpr (Slot::kCodes) {
        const uint32_t c = *reinterpret_cast<const uint32_t*>(slot + Slot::offset(1, r, fb) + 4 * g);
        const u32x4 x = codes_to_bf16<F>(c, 0u);
        w[0] = x[0], w[1] = x[1];
      } else {
        const u32x2 x = *reinterpret_cast<const u32x2*>(slot + Slot::offset(1, r, 2 * fb + (g >> 1)) + 8 * (g & 1));
        w[0] = x[0], w[1] = x[1];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t b = (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu;
        const float add = on && (b & 0x7F80u) == 0x7F80u ? bf16_bits_to_f32(b) : 0.f;
        asm volatile("v_add_f32 %0, %0, %1" : "+v"(st.acc[fb][e]) : "v"(add));
      }
    }
  }
}

// One key tile against the wave's queries.  MASKED: hidden keys take no part,
// whatever their score, value and scale hold.
// keys_read() runs once K has been read, values_due() before V is, which starts
// the next tile's K and waits for this one's V.
template <int D, int F, bool MASKED, typename KeysRead, typename ValuesDue>
__device__ __forceinline__ void step_tile(const PagedParams& p, int length, StepState<D>& st, LaneRow& row,
                                          const bf16x8 (&qf)[D / 32], const uint8_t* slot, const StepSlot<D, F>& at,
                                          const float* scales, int tile, uint32_t valid, int lane, KeysRead keys_read,
                                          ValuesDue values_due) {
  using Slot = StepSlot<D, F>;
  constexpr int TK = Slot::TK, KB = TK / 16, FB = D / 16;
  constexpr bool SCALED = F != kBf16;
  const float c = p.scale_log2;
  const int g = lane >> 4;
  f32x4 s[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    s[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < Slot::kReads; ++n) {
      const u32x4 x = at.k(kb, n);
      if constexpr (Slot::kCodes) {
        s[kb] = mfma16x16x32(as_bf16x8(codes_to_bf16<F>(x[0], x[1])), qf[2 * n], s[kb]);
        s[kb] = mfma16x16x32(as_bf16x8(codes_to_bf16<F>(x[2], x[3])), qf[2 * n + 1], s[kb]);
      } else {
        s[kb] = mfma16x16x32(as_bf16x8(x), qf[n], s[kb]);
      }
    }
    if constexpr (Slot::kCodes) chunk_end();  // few operands in flight: their conversions take registers
  }
  if constexpr (SCALED) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const f32x4 sk = *reinterpret_cast<const f32x4*>(scales + Slot::key(kb, g, 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) s[kb][e] *= sk[e];
    }
  }
  keys_read();
  uint32_t seen = 0;
  if constexpr (MASKED) {
    const Visible v = visible(p, fresh(row.pos), length);  // not held in registers over the stream
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = Slot::key(kb, g, e), j = tile * TK + r;
        const bool in = (((j <= v.hi) & (j >= v.lo)) | (j < v.sink)) & (((valid >> (r >> 4)) & 1u) != 0);
        s[kb][e] = in ? s[kb][e] : kNegInf;
        seen |= in ? 1u << (4 * kb + e) : 0u;
      }
    row.any |= seen != 0;
  } else {
    row.any = true;
  }
  float mx = s[0][0];
#pragma unroll
  for (int i = 1; i < 4 * KB; ++i) mx = fmaxf(mx, s[i / 4][i % 4]);
  mx = quad_max(mx) * c;
  if (__builtin_amdgcn_ballot_w64(mx > st.m)) {
    const float mnew = fmaxf(st.m, mx);
    const float alpha = mnew == kNegInf ? 1.f : fast_exp2(st.m - mnew);
    st.m = mnew;
    st.den *= alpha;
#pragma unroll
    for (int fb = 0; fb < FB; ++fb)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.acc[fb][e] *= alpha;
  }
  const float neg_m = st.m == kNegInf ? 0.f : -st.m;
  float sum = 0.f;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[kb][e] = fast_exp2(fmaf(s[kb][e], c, neg_m));
      sum += s[kb][e];
    }
  st.den += sum;
  values_due();
  if constexpr (SCALED) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const f32x4 sv = *reinterpret_cast<const f32x4*>(scales + TK + Slot::key(kb, g, 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) s[kb][e] = MASKED && !((seen >> (4 * kb + e)) & 1u) ? 0.f : s[kb][e] * sv[e];
    }
  }
  // The probabilities as two BF16 terms, the upper half and the rest (16
  // significant bits, 2^-16 at most): the kernel waits for memory, and the
  // products have time.  Neither term is negative.  In a whole BF16 tile neither
  // is 0, so that an infinite value stays one: 2^-126 is added at most, of the
  // largest probability's 1.  In a masked tile hidden keys have 0, and values that
  // are not finite are added apart.
  constexpr bool kCheck = MASKED && F != kInt8;  // INT8 codes are finite
  constexpr float kLeast = !MASKED && F == kBf16 ? 0x1p-126f : 0.f;
  uint32_t bad = 0;
#pragma unroll
  for (int h = 0; h < TK / 32; ++h) {
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4& x = s[2 * h + (i >> 1)];
      uint32_t u[2];
      float rest[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float y = kLeast > 0.f ? fmaxf(x[2 * (i & 1) + j], kLeast) : x[2 * (i & 1) + j];
        u[j] = __float_as_uint(y);
        rest[j] = y - __uint_as_float(u[j] & 0xFFFF0000u);
        if (kLeast > 0.f) rest[j] = fmaxf(rest[j], kLeast);
      }
      hi[i] = __builtin_amdgcn_perm(u[1], u[0], 0x07060302u);
      lo[i] = pack_bf16x2(rest[0], rest[1]);
    }
#pragma unroll
    for (int fb = 0; fb < FB; ++fb) {
      u32x4 v = at.v(h, fb);
      if constexpr (kCheck) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t b = nonfinite(v[i]);
          bad |= b;
          v[i] &= ~((b >> 15) * 0xFFFFu);
        }
      }
      st.acc[fb] = mfma16x16x32(as_bf16x8(v), as_bf16x8(hi), st.acc[fb]);
      st.acc[fb] = mfma16x16x32(as_bf16x8(v), as_bf16x8(lo), st.acc[fb]);
      if (Slot::kCodes && fb % 2) chunk_end();
    }
  }
  if constexpr (kCheck) {
    if (__builtin_amdgcn_ballot_w64(bad != 0)) step_nonfinite<D, F>(st, slot, lane, seen);
  }
}

// Bound by reading the keys, so that bytes in flight count: every wave moves
// tiles of its own into its own slot, without a barrier, the next tile's keys
// under way while this one's values are, and two workgroups per CU keep 128 KB
// asked for.  Heads of 128, four query heads each: 64 sequences of 8,192 keys of
// 8 heads, BF16 2.15 GB in 371 us, 5.8 TB/s; INT8 1.11 GB 211 us, 5.3 TB/s; FP8
// 210 us.  (BF16 tiles through registers, 32 x 32 products: 48 sequences of up to
// 19,003 keys 256 us, 183 now.)  One sequence of 84,672 INT8 keys: 179 MB in 38
// us and the merge's 5.  Small calls are a chain of latencies: three single
// tokens over up to 317 keys 7.5 us.
template <int D, int F, bool PAGED>
__global__ __launch_bounds__(kNT, 2) void step_kernel(PagedParams p) {
  using Slot = StepSlot<D, F>;
  constexpr int R = 16, TK = Slot::TK;
  constexpr bool SCALED = F != kBf16;
  __shared__ __align__(256) uint8_t s_tile[kWaves][2 * Slot::kPlane];
  __shared__ __align__(16) float s_scale[kWaves][SCALED ? 2 * TK : 1];
  __shared__ float s_md[kWaves][3][kWave];

  const int h = blockIdx.x % p.H;
  Item it;
  if (!take_item<R, TK, PAGED>(p, blockIdx.x / p.H, it)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g = lane >> 4;

  // This lane's query, straight into its operand registers (StepSlot::k's features).
  const int pos0 = it.pos0;
  const int r = it.r0 + min(col, it.rows - 1);
  const int token = r / p.G;
  const uint16_t* q = p.q + (PAGED ? (it.off + token) * p.q_st : it.s * p.q_sb + token * p.q_st) +
                      (h * p.G + r % p.G) * p.q_sh;
  bf16x8 qf[D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks)
    qf[ks] = as_bf16x8(load16(q + (SCALED ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g)));
  LaneRow row;
  row.pos = pos0 + token;
  row.any = false;
  const int first = pos0 + it.r0 / p.G, last = pos0 + (it.r0 + it.rows - 1) / p.G;
  const Span span = span_of<TK>(p, first, last, it.length);
  const int t0 = int(int64_t(it.part) * span.n / it.parts), t1 = int(int64_t(it.part + 1) * span.n / it.parts);
  // Tiles inside these bounds are seen whole by every row.
  const Visible va = visible(p, first, it.length), vb = visible(p, last, it.length);

  StepState<D> st;
#pragma unroll
  for (int fb = 0; fb < D / 16; ++fb) st.acc[fb] = f32x4{0.f, 0.f, 0.f, 0.f};
  st.m = kNegInf;
  st.den = 0.f;
  const Keys<D, F, PAGED> keys(p, it, h);
  uint8_t* slot = s_tile[wave];
  float* scales = s_scale[wave];
  const Slot at(slot, lane);

  // The wave's tiles are every kWaves-th of the part's: tile k of its list.
  const int count = t1 - t0 > wave ? (t1 - t0 - wave - 1) / kWaves + 1 : 0;
  auto tile_of = [&](int k) { return span.tile(t0 + wave + kWaves * min(k, count - 1)); };
  if (count > 0) {
    using Window = PageWindow<D, F, PAGED, TK>;
    using Dma = StepDma<D, F, PAGED>;
    Window window;
    Dma dma(lds_address(slot), lds_address(scales), lane);
    auto prepare = [&](int k) {
      if (k % Window::kTiles == 0) {
        window.fetch(keys, [&](int i) { return tile_of(k + i); }, lane);
        window.turn(keys);
      }
      dma.prepare(window, k % Window::kTiles, tile_of(k));
    };
    // Tile k: its K is awaited, then its V, with the next tile's K on its way
    // meanwhile and its V from the end on (each wave on its own, no barrier).
    auto step = [&](int k, auto masked) {
      const bool more = k + 1 < count;
      const uint32_t valid = dma.valid;
      wait_vmcnt<Dma::kLoads>();
      step_tile<D, F, decltype(masked)::value>(
          p, it.length, st, row, qf, slot, at, scales, tile_of(k), valid, lane,
          [&] {
            if (more) {
              prepare(k + 1);
              lds_returned();
              dma.issue(keys, 0);
            }
          },
          [&] {
            if (more)
              wait_vmcnt<Dma::kLoads>();
            else
              wait_vmcnt<0>();
          });
      if (more) {
        lds_returned();
        dma.issue(keys, 1);
      }
    };
    auto whole = [&](int k) {
      const int a = tile_of(k) * TK, b = a + TK - 1;
      return k < count && dma.valid == kAllGroups<TK> && b <= va.hi && (a >= vb.lo || b < va.sink);
    };
    prepare(0);
    dma.issue(keys, 0);
    dma.issue(keys, 1);
    int k = 0;
    while (k < count) {
      // Whole tiles, the common kind, run in a loop of their own.
      while (whole(k)) step(k++, std::false_type{});
      if (k < count) step(k++, std::true_type{});
    }
  }

  // Join the four waves' states: each writes its sums over its own tiles.
  wave_order();
  f32x4* mine = reinterpret_cast<f32x4*>(slot);
  constexpr int FB = D / 16;
#pragma unroll
  for (int fb = 0; fb < FB; ++fb) mine[fb * kWave + lane] = st.acc[fb];
  s_md[wave][0][lane] = st.m;
  s_md[wave][1][lane] = st.den;
  s_md[wave][2][lane] = row.any ? 1.f : 0.f;
  __syncthreads();
  float m = kNegInf, den = 0.f, w[kWaves], seen = 0.f;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) m = fmaxf(m, s_md[i][0][lane]);
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const float mi = s_md[i][0][lane];
    w[i] = mi == kNegInf ? 1.f : fast_exp2(mi - m);
    den += w[i] * s_md[i][1][lane];
    seen += s_md[i][2][lane];
  }
  // The four lanes of a query saw different keys of each tile.
  den = quad_sum(den);
  seen = quad_sum(seen);
  if (col >= it.rows) return;
  float* row_out = it.parts > 1 ? record<D, R>(p, it.record) + col * kRecordRow<D> : nullptr;
  uint16_t* out = p.out + output_row<D>(p, it.off, it.r0 + col, h);
#pragma unroll
  for (int fb = wave; fb < FB; fb += kWaves) {
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const f32x4 x = reinterpret_cast<const f32x4*>(s_tile[i])[fb * kWave + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += w[i] * x[e];
    }
    if (it.parts > 1)
      *reinterpret_cast<f32x4*>(row_out + 16 * fb + 4 * g) = o;
    else
      store4(out + 16 * fb + 4 * g, o, den, seen > 0.f);
  }
  if (it.parts > 1 && wave == 0 && g == 0) {
    const f32x4 tail = {m, den, seen, 0.f};
    *reinterpret_cast<f32x4*>(row_out + D) = tail;
  }
}

// ---- many rows --------------------------------------------------------------

// The DMA of a BF16 key tile into an LDS slot, in kRounds rounds per wave of 1
// KB each: round r of K (then of V) moves rows R0 = r kRoundRows + wave
// kPieceRows on, all in one group of 16.  In a cache a round's address is its
// group's, and a lane's offset the same in every round (the swizzles repeat; a
// page's rows past the last key exist).  Plain keys take the tile's first row
// and a lane's own, which stops at the last key: no branch for the tail tile
// (one per round took 5% of the kernel's time).
template <int D, bool PAGED>
struct DmaTile {
  using Source = Keys<D, kBf16, PAGED>;
  static constexpr int kHalf = 64 * D * 2 / 16 / kNT;
  static constexpr int kRounds = 2 * kHalf;
  static constexpr int kRoundRows = kNT * 16 / (2 * D);
  static constexpr int kPieceRows = kRoundRows / kWaves;
  // What a lane keeps over the stream, per operand: paged, its offset; plain,
  // its row and its chunk of the row.
  struct Lane {
    uint32_t off[2];
    uint32_t row[2];
    __device__ __forceinline__ Lane(int w, int l) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int m = D == 128 ? l : l % 32;  // of a quad (V)
        const int r = kv ? (D == 128 ? 0 : 4 * (l / 32)) + ((m >> 2) & 3) : l / (D / 8);
        const int c = kv ? 4 * (m >> 4) + (m & 3) : (l % (D / 8)) ^ TileLayout<D>::k_swizzle(w * kPieceRows + r);
        row[kv] = w * kPieceRows + r;
        off[kv] = PAGED ? (w * kPieceRows % 16 + r) * Source::kRowBytes + 16 * c : c;
      }
    }
  };
  const Lane& lane;
  uint64_t src[2], off[PAGED ? kHalf : 1];
  uint32_t lds, st[2];
  int last;  // plain: the last key's row of the tile

  // Tile `tile`, the window's tile i.
  template <typename Window>
  __device__ __forceinline__ DmaTile(const Source& keys, const Window& window, int i, int tile, uint32_t dst, int w,
                                     const Lane& lanes)
      : lane(lanes) {
    last = keys.last - tile * 64;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      src[kv] = reinterpret_cast<uint64_t>(keys.base[kv]);
      if constexpr (!PAGED) src[kv] += uint64_t(uint32_t(tile * 64)) * keys.st[kv];
      st[kv] = keys.st[kv] / 16;  // below 2^21: token strides are below 2^24 elements
    }
    if constexpr (PAGED) {
      // The wave's piece begins w kPieceRows % 16 rows into its group (Lane).
#pragma unroll
      for (int r = 0; r < kHalf; ++r) off[r] = window.offset(i, D == 128 ? r : 2 * r + (w >> 1));
    }
    lds = dst + uint32_t(w) * 1024u;
  }
  __device__ __forceinline__ void round(int i) const {
    const int kv = i / kHalf, r = i % kHalf;
    const uint32_t dst = lds + uint32_t(kv * 64 * D * 2 + r * kNT * 16);
    if constexpr (PAGED) {
      dma16(src[kv] + off[r], lane.off[kv], dst);
    } else {
      const uint32_t row = min(int(lane.row[kv]) + r * kRoundRows, last);
      dma16(src[kv] + round_offset(0u), (__umul24(row, st[kv]) + lane.off[kv]) * 16u, dst);
    }
  }
  __device__ __forceinline__ void all() const {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) round(r);
  }
  template <int N>
  __device__ __forceinline__ void after_step(int k) const {
#pragma unroll
    for (int r = k * kRounds / N; r < (k + 1) * kRounds / N; ++r) round(r);
  }
  __device__ __forceinline__ void late() const {}
  template <int N>
  __device__ __forceinline__ void late_step(int) const {}
};

// An 8-bit key tile on its way, in the workgroup's registers: loaded while
// the tile before it is attended, converted into its slot afterwards.
template <int D, int F>
struct CodeTile {
  static constexpr int kRowLanes = D / 16;
  static constexpr int kLoads = 64 * kRowLanes / kNT;
  u32x4 x[2][kLoads];
  float scale;

  // The window's tile i.
  template <typename Window>
  __device__ __forceinline__ void load(const Keys<D, F, true>& keys, const Window& window, int i, int wave, int lane) {
    const int l = fresh(lane);
    // A wave's 64 chunks are 8 (D = 128) or 16 rows of one group.
    const uint32_t row = uint32_t(wave * kWave / kRowLanes % 16 + l / kRowLanes);
    const uint32_t off = row * keys.kRowBytes + 16u * (l % kRowLanes);
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const uint64_t at = window.offset(i, D == 128 ? 2 * n + (wave >> 1) : wave);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) x[kv][n] = load_chunk(keys.base[kv] + at + off);
    }
    // Wave 0 the keys' scales, wave 1 the values'.
    if (wave < 2) scale = (wave ? keys.scale[1] : keys.scale[0])[window.row(i, l)];
  }
  // Converts piece n of kPieces (16 codes of a row) into its place.
  static constexpr int kPieces = 2 * kLoads;
  __device__ __forceinline__ void put(uint16_t* slot, int n, int thread) const {
    using Image = TileImage<D, 64>;
    const int tid = fresh(thread), kv = n / kLoads, i = n % kLoads;
    const int row = (i * kNT + tid) / kRowLanes, c = tid % kRowLanes;
    Image::put(slot, kv, row, 2 * c, codes_to_bf16<F>(x[kv][i][0], x[kv][i][1]));
    Image::put(slot, kv, row, 2 * c + 1, codes_to_bf16<F>(x[kv][i][2], x[kv][i][3]));
  }
};

// The next tile's codes beside a tile's products: they are converted beside
// half 1's P V, which has no other vector work, or at the end.  K's scales are
// kept times c.
template <int D, int F>
struct CodeRefill {
  const CodeTile<D, F>& code;
  uint16_t* slot;
  float* scales;
  int tid;
  float c;
  __device__ __forceinline__ void all() const {}
  template <int N>
  __device__ __forceinline__ void after_step(int) const {}
  // Step k of N.
  template <int N>
  __device__ __forceinline__ void late_step(int k) const {
    constexpr int P = CodeTile<D, F>::kPieces;
    static_assert(N % P == 0, "a piece every N / P steps");
    if (k % (N / P) == 0) code.put(slot, k / (N / P), tid);
    if (k == N - 1 && tid < 128) scales[tid] = tid < 64 ? code.scale * c : code.scale;
  }
  __device__ __forceinline__ void late() const {
#pragma unroll
    for (int n = 0; n < CodeTile<D, F>::kPieces; ++n) late_step<CodeTile<D, F>::kPieces>(n);
  }
};

// FastHalf with per-key factors (SCALED): the scores take K's scales (times c)
// in the place of c, four at a time, and the probabilities V's before they are
// packed.
template <int D, bool SCALED>
struct WideHalf : FastHalf<D> {
  f32x4 factor;  // of the next four scores

  // half: the half's K factors in LDS, V's 64 floats on.
  __device__ __forceinline__ void ask(const float* half, int q, int hh) {
    if constexpr (SCALED) factor = *reinterpret_cast<const f32x4*>(half + 8 * q + 4 * hh);
  }
  template <int N>
  __device__ __forceinline__ void step(int k, State<D>& st, float c, const float* half, int hh) {
#pragma unroll
    for (int i = k * 8 / N; i < (k + 1) * 8 / N; ++i) {
      if (SCALED && i < 4) {
        const f32x4 f = factor;
        if (i < 3) ask(half, i + 1, hh);
#pragma unroll
        for (int e = 0; e < 4; ++e) this->s[4 * i + e] *= f[e];
      }
      if (SCALED && i == 5) scale(this->s, half + 64, hh);
      this->stage(i, st, SCALED ? 1.f : c);
    }
  }
  __device__ static __forceinline__ void scale(f32x16& x, const float* factors, int hh) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 f = *reinterpret_cast<const f32x4*>(factors + 8 * q + 4 * hh);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * q + i] *= f[i];
    }
  }
  template <typename Raw>
  __device__ __forceinline__ void finish(State<D>& st, float c, const float* half, int hh, Raw raw) {
    if (this->redo) {
      HalfSoftmax<D> full;
      full.s = raw();
      const int fh = fresh(hh);
      if (SCALED) scale(full.s, half, fh);
      const float cs = SCALED ? 1.f : c;
      chunk_end();
#pragma unroll
      for (int i = 0; i < 6; ++i) full.stage(i, st, cs);
      chunk_end();
      if (SCALED) scale(full.s, half + 64, fh);
      full.stage(6, st, cs);
      full.stage(7, st, cs);
      if (full.rescale) rescale_acc<D>(st, full.alpha);
      this->pw[0] = full.pw[0];
      this->pw[1] = full.pw[1];
    }
  }
};

// A key tile that every row of the wave sees whole, pipelined over its two
// halves inside the wave so that the softmax's vector work runs beside the
// matrix products:
//   KT products    half 0's scores
//   KT products    half 1's scores; half 0's softmax
//   2 DT products  half 0's P V; half 1's softmax
//   2 DT products  half 1's P V
// Operands are read kAhead products before their use, and the next tile's DMA
// rounds are spread over the score products.  (More ahead spills with heads of
// 128, where codes under way leave registers for two; heads of 64 have some for
// eight.)
template <int D, bool SCALED, typename Refill>
__device__ __forceinline__ void wide_tile(State<D>& st, const uint16_t* buf, const float* scales,
                                          const bf16x8 (&qf)[Shape<D>::KT], int col, int hh, float c,
                                          const Refill& refill) {
  constexpr int KT = Shape<D>::KT, DT = Shape<D>::DT;
  constexpr int kAhead = SCALED ? 2 : (D == 64 ? 8 : 4);
  const FragLane<D> fl(fresh(col), fresh(hh));
  const uint32_t vbase = fl.v_base(buf);
  // Operand n of the tile's 2 KT K and 4 DT V operands.
  auto operand = [&](int n) {
    const int f = n - 2 * KT;
    return n < 2 * KT ? fl.k(buf, n / KT, n % KT) : fl.v(vbase, f / (2 * DT), f / DT % 2, f % DT);
  };
  auto raw = [&](int t) {
    const FragLane<D> fr(fresh(col), fresh(hh));
    f32x16 s = zero16();
#pragma unroll
    for (int ks = 0; ks < KT; ++ks) {
      s = mfma32x32x16(as_bf16x8(fr.k(buf, t, ks)), qf[ks], s);
      chunk_end();
    }
    return s;
  };
  u32x4 o[kAhead];
#pragma unroll
  for (int n = 0; n < kAhead; ++n) o[n] = operand(n);
  WideHalf<D, SCALED> h0, h1;
  h0.s = zero16();
  h1.s = zero16();
  chunk_end();
  // Operand n is taken, then the one kAhead on asked for in its place.
  auto next = [&](int n) { return as_bf16x8(o[n % kAhead]); };
  auto ask = [&](int n) {
    if (n + kAhead < 2 * KT + 4 * DT) o[n % kAhead] = operand(n + kAhead);
  };
#pragma unroll
  for (int n = 0; n < KT; ++n) {
    h0.s = mfma32x32x16(next(n), qf[n], h0.s);
    ask(n);
    refill.template after_step<2 * KT>(n);
    chunk_end();
  }
  h0.ask(scales, 0, hh);
#pragma unroll
  for (int n = 0; n < KT; ++n) {
    h1.s = mfma32x32x16(next(KT + n), qf[n], h1.s);
    ask(KT + n);
    h0.template step<KT>(n, st, c, scales, hh);
    refill.template after_step<2 * KT>(KT + n);
    chunk_end();
  }
  h0.finish(st, c, scales, hh, [&] { return raw(0); });
  h1.ask(scales + 32, 0, hh);
#pragma unroll
  for (int f = 0; f < 2 * DT; ++f) {
    st.acc[f % DT] = mfma32x32x16(next(2 * KT + f), h0.pb(f / DT), st.acc[f % DT]);
    ask(2 * KT + f);
    h1.template step<2 * DT>(f, st, c, scales + 32, hh);
    chunk_end();
  }
  h1.finish(st, c, scales + 32, hh, [&] { return raw(1); });
#pragma unroll
  for (int f = 0; f < 2 * DT; ++f) {
    st.acc[f % DT] = mfma32x32x16(next(2 * KT + 2 * DT + f), h1.pb(f / DT), st.acc[f % DT]);
    ask(2 * KT + 2 * DT + f);
    refill.template late_step<2 * DT>(f);
    chunk_end();
  }
}

// Bound by the softmax's vector work beside the products: a half's 16 products
// are 512 cycles of the matrix core, its exponentials, sums and packing about
// 420 of the vector unit, of each of two waves.  4,096 queries of 16 heads of 128
// over 16,384 keys, 550 GFLOP: BF16 494 us, 1.11 PFLOP/s (dense_attention_kernel
// 485); heads of 64 317 us, 0.87 PFLOP/s.  8-bit codes add a conversion of 64
// codes and 64 multiplications by scales per lane and tile: FP8 645 us, INT8
// 688.  Two workgroups per CU hold 256 registers a wave and a ring of two tiles
// each; with heads of 128 that leaves 6 (BF16) to 17 (codes) registers spilled.
template <int D, int F, bool PAGED>
__global__ __launch_bounds__(kNT, 2) void wide_kernel(PagedParams p) {
  using S = Shape<D>;
  constexpr int R = 128, TK = 64;
  constexpr bool SCALED = F != kBf16;
  __shared__ __align__(256) uint16_t ring[2][S::TILE];
  __shared__ __align__(16) float s_scale[2][SCALED ? 2 * TK : 1];

  const int h = blockIdx.x % p.H;
  Item it;
  if (!take_item<R, TK, PAGED>(p, blockIdx.x / p.H, it)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, hh = lane >> 5;
  const int wrows = min(32, it.rows - 32 * wave);  // this wave's rows (none: it only moves tiles)

  const int pos0 = it.pos0;
  const int r = it.r0 + min(32 * wave + col, it.rows - 1);
  const int token = r / p.G;
  const uint16_t* q = p.q + (PAGED ? (it.off + token) * p.q_st : it.s * p.q_sb + token * p.q_st) +
                      (h * p.G + r % p.G) * p.q_sh;
  bf16x8 qf[S::KT];
#pragma unroll
  for (int ks = 0; ks < S::KT; ++ks) qf[ks] = as_bf16x8(load16(q + 16 * ks + 8 * hh));
  LaneRow row;
  row.pos = pos0 + token;
  row.any = false;

  const Span span = span_of<TK>(p, pos0 + it.r0 / p.G, pos0 + (it.r0 + it.rows - 1) / p.G, it.length);
  const int t0 = int(int64_t(it.part) * span.n / it.parts), t1 = int(int64_t(it.part + 1) * span.n / it.parts);
  const Visible va = visible(p, pos0 + (it.r0 + 32 * wave) / p.G, it.length);
  const Visible vb = visible(p, pos0 + (it.r0 + 32 * wave + max(wrows, 1) - 1) / p.G, it.length);

  State<D> st;
  state_init(st);
  const Keys<D, F, PAGED> keys(p, it, h);
  auto at = [&](int i) { return span.tile(min(i, t1 - 1)); };
  const uint32_t ring_lds = lds_address(ring[0]);

  // How the wave's rows see a tile: not at all, in part, or whole.
  enum Kind { kHidden, kPart, kWhole };
  auto kind_of = [&](int tile, uint32_t valid) {
    const int a = tile * TK, b = a + TK - 1;
    if (wrows <= 0 || ((a > vb.hi || b < va.lo) && a >= vb.sink)) return kHidden;
    return valid == kAllGroups<TK> && b <= va.hi && (a >= vb.lo || b < va.sink) ? kWhole : kPart;
  };
  auto hidden = [&](int, uint32_t, const uint16_t*, const float*, const auto& refill) {
    refill.all();
    refill.late();
  };
  auto whole = [&](int, uint32_t, const uint16_t* buf, const float* scales, const auto& refill) {
    wide_tile<D, SCALED>(st, buf, scales, qf, col, hh, p.scale_log2, refill);
  };
  auto part = [&](int tile, uint32_t valid, const uint16_t* buf, const float* scales, const auto& refill) {
    refill.all();
#pragma unroll 1
    for (int t = 0; t < 2; ++t) {
      const int fcol = fresh(col), fhh = fresh(hh);
      f32x16 s = zero16();
#pragma unroll
      for (int ks = 0; ks < S::KT; ++ks)
        s = mfma32x32x16(as_bf16x8(TileImage<D, TK>::k(buf, fcol, fhh, t, ks)), qf[ks], s);
      chunk_end();
      attend_masked<D, TK, F>(p, it.length, st, row, s, buf, t, tile * TK + 32 * t, valid >> (2 * t), col, hh,
                           SCALED ? scales + 32 * t : nullptr);
    }
    refill.late();
  };
  // One tile after another; consecutive tiles of a kind run in a loop of their
  // own, so that the sums are not split across a branch per tile.  The waves of
  // a workgroup may be in different loops: each meets one barrier per tile.
  auto stream = [&](auto&& step, const uint32_t& valid) {
    int i = t0;
    while (i < t1) {
      const Kind kind = kind_of(at(i), valid);
      if (kind == kWhole) {
        row.any = true;
        do step(i, whole);
        while (++i < t1 && kind_of(at(i), valid) == kWhole);
      } else if (kind == kPart) {
        do step(i, part);
        while (++i < t1 && kind_of(at(i), valid) == kPart);
      } else {
        do step(i, hidden);
        while (++i < t1 && kind_of(at(i), valid) == kHidden);
      }
    }
  };

  if (t0 < t1) {
    using Window = PageWindow<D, F, PAGED, TK>;
    Window window;
    auto fetch = [&](int i) { window.fetch(keys, [&](int k) { return at(i + k); }, lane); };
    // Makes tile i's pages current, in order of i; returns its place in the
    // window.  The next window is read half a window ahead.
    auto turn_to = [&](int i) {
      const int k = (i - t0) % Window::kTiles;
      if (k == 0) window.turn(keys);
      if (k == Window::kTiles / 2) fetch(i + Window::kTiles / 2);
      return k;
    };
    fetch(t0);
    int k = turn_to(t0);
    uint32_t valid = window.valid(k);  // of the tile at hand
    if constexpr (!SCALED) {
      const typename DmaTile<D, PAGED>::Lane lanes(wave, lane);
      DmaTile<D, PAGED>(keys, window, k, at(t0), ring_lds, wave, lanes).all();
      stream([&](int i, auto&& attend) {
        wait_vmcnt<0>();
        lds_barrier();
        const int slot = (i - t0) & 1;
        const uint32_t now = valid;
        k = turn_to(i + 1);
        valid = window.valid(k);
        // Past the last tile that tile again, into the slot nobody reads.
        const DmaTile<D, PAGED> refill(keys, window, k, at(i + 1), ring_lds + uint32_t((slot ^ 1) * S::TILE * 2), wave,
                                       lanes);
        attend(at(i), now, ring[slot], static_cast<const float*>(nullptr), refill);
      }, valid);
      wait_vmcnt<0>();
    } else {
      CodeTile<D, F> code;
      code.load(keys, window, k, wave, lane);
      CodeRefill<D, F>{code, ring[0], s_scale[0], tid, p.scale_log2}.late();
      stream([&](int i, auto&& attend) {
        lds_barrier();
        const int slot = (i - t0) & 1;
        const uint32_t now = valid;
        k = turn_to(i + 1);
        valid = window.valid(k);
        code.load(keys, window, k, wave, lane);
        attend(at(i), now, ring[slot], s_scale[slot],
               CodeRefill<D, F>{code, ring[slot ^ 1], s_scale[slot ^ 1], tid, p.scale_log2});
      }, valid);
    }
  }

  const float den = pair_sum(st.den), seen = pair_sum(row.any ? 1.f : 0.f);
  if (col >= wrows) return;
  float* row_out = it.parts > 1 ? record<D, R>(p, it.record) + (32 * wave + col) * kRecordRow<D> : nullptr;
  uint16_t* out = p.out + output_row<D>(p, it.off, r, h);
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    const f32x4 o = {st.acc[c / 4][4 * (c % 4)], st.acc[c / 4][4 * (c % 4) + 1], st.acc[c / 4][4 * (c % 4) + 2],
                     st.acc[c / 4][4 * (c % 4) + 3]};
    const int feature = 32 * (c / 4) + 8 * (c % 4) + 4 * hh;
    if (it.parts > 1)
      *reinterpret_cast<f32x4*>(row_out + feature) = o;
    else
      store4(out + feature, o, den, seen > 0.f);
  }
  if (it.parts > 1 && hh == 0) {
    const f32x4 tail = {st.m, den, seen, 0.f};
    *reinterpret_cast<f32x4*>(row_out + D) = tail;
  }
}

// ---- launches ---------------------------------------------------------------

template <int D, int R>
void launch_merge(const PagedParams& p, const PagedSize& size, hipStream_t stream) {
  const unsigned rows = unsigned((size.merge_rows - 1) / kMergeRows<D, R> + 1);
  hipLaunchKernelGGL((merge_kernel<D, R>), dim3(unsigned(p.headers * p.H), rows), dim3(kNT), 0, stream, p);
}

template <int D, int F, bool PAGED>
void launch_variant(const PagedParams& p, const PagedSize& size, hipStream_t stream) {
  const dim3 grid(unsigned(size.grid)), block(kNT);
  if (size.rows == 16) {
    hipLaunchKernelGGL((step_kernel<D, F, PAGED>), grid, block, 0, stream, p);
    if (p.records) launch_merge<D, 16>(p, size, stream);
  } else {
    hipLaunchKernelGGL((wide_kernel<D, F, PAGED>), grid, block, 0, stream, p);
    if (p.records) launch_merge<D, 128>(p, size, stream);
  }
}

template <int D>
void launch_format(const PagedParams& p, const PagedSize& size, int format, hipStream_t stream) {
  if (!p.batch.table) launch_variant<D, kBf16, false>(p, size, stream);
  else if (format == kBf16) launch_variant<D, kBf16, true>(p, size, stream);
  else if (format == kInt8) launch_variant<D, kInt8, true>(p, size, stream);
  else launch_variant<D, kFp8, true>(p, size, stream);
}

}  // namespace

namespace {

constexpr int64_t kResident = 512;  // workgroups of either kernel that the card holds at once (two per CU)

// Workgroups per head that the wide kernel's keys are split for, or 0, where all
// row tiles have as many key tiles.  `tiles` row tiles per head of `key_tiles` key
// tiles each run in rounds of kResident workgroups; in q parts each they take
// ceil(q tiles heads / kResident) rounds of key_tiles / q key tiles, and kPartCost
// more for every part (its set-up, its partial state written and joined).  (128
// queries of 8 heads over 32,768 keys: 46 us in 32 parts, 54 in 64, 561 in one.
// 2,048 queries over themselves, 32 heads: 54 us in one part, 59 in two.)
int64_t wide_target(int64_t tiles, int64_t heads, int64_t key_tiles, int64_t min_tiles) {
  constexpr double kPartCost = 6.0;
  auto cost = [&](int64_t q) {
    const int64_t rounds = (q * tiles * heads + kResident - 1) / kResident;
    return double(rounds) * (double(key_tiles) / double(q) + (q > 1 ? 2.0 : 1.0) * kPartCost);
  };
  int64_t best = 1;
  for (int64_t q = 2; q <= 32 && key_tiles / q >= min_tiles; ++q)
    if (cost(q) < cost(best)) best = q;
  return best > 1 && cost(best) < 0.95 * cost(1) ? best * tiles : 0;
}

}  // namespace

PagedSize paged_size(int64_t rows, int64_t sequences, int64_t keys, int64_t tile_keys, int64_t heads, int64_t group,
                     int64_t head_dim, int format, bool causal, bool ragged) {
  PagedSize s;
  auto likely_tiles = [&](int64_t R) { return (rows * group + R - 1) / R + (sequences - 1) / 2; };
  // The step kernel, whose tiles are 16 rows, for few rows per sequence; and for
  // small calls, which its tiles spread over more of the card: up to two rounds of
  // workgroups that read 128 MB of BF16 keys and values, some of them again and
  // again.  (Heads of 128: 193 queries of 2 heads, 317 keys 11.8 us, 17.8 with tiles
  // of 128; 256 of 16 heads, 1,024 keys, 128 MB: 16 and 21; 1,000 of 16 heads
  // under a window of 100, 1,008 workgroups: 18 and 27, 2,000: 46 and 36; 4 x 12
  // x 4 of 8 heads, 9,000 keys, 440 MB: 48 and 40.)
  const int64_t small = likely_tiles(16) * heads;
  const bool step = rows * group <= 32 * sequences ||
                    (small <= 2 * kResident && small * tile_keys <= (int64_t(128) << 20) / (4 * head_dim));
  s.rows = step ? 16 : 128;
  const int64_t TK = step ? 8192 / (head_dim * (format == kBf16 ? 2 : 1)) : 64;  // StepSlot::TK
  s.tiles = rows * group / s.rows + sequences;  // row tiles: sum ceil(n_s G / R) at most
  const int64_t likely = likely_tiles(s.rows);
  const int64_t key_tiles = (std::min(keys, tile_keys + (step ? 0 : 128)) + TK - 1) / TK;  // of a row tile, at most
  // Row tiles that differ in their keys: other sequences, or the rows of a triangle.
  const bool uneven = (ragged && sequences > 1) || (causal && 2 * rows > keys * sequences);
  s.target = 0;
  if (step) {
    // A second launch costs 5 us, as much as 16 queries over 48 BF16 key tiles or
    // 20 of codes take alone (16 sequences, 4 heads: 1,024 BF16 keys 13.6 us whole,
    // 18.3 split; 4,096 33.5 and 30.7; INT8 1,024 18.0 and 19.8, 2,048 29 and 20).
    // One round of workgroups (one sequence of 84,672 INT8 keys, 8 heads: 44 us,
    // 51 in two rounds), but two where the sequences alone fill half the card
    // and may differ (48 of 300 .. 19,003 keys: 318 us, 330 in one round; 64 of
    // 8,192: 373 and 361).
    s.min_tiles = 8;
    const int64_t rounds = ragged && 2 * sequences * heads >= kResident ? 2 : 1;
    if (key_tiles > (format == kBf16 ? 48 : 20)) s.target = (rounds * kResident + heads - 1) / heads;
  } else if (uneven && 2 * likely * heads * key_tiles >= 3 * kResident * 24) {
    // Enough keys for one and a half rounds of parts of 24 tiles: those even the
    // lengths out (8 sequences of 600 .. 12,000 keys, 512 new tokens of 8 x 4
    // heads: 505 us, 687 with the rule below; 8,192 queries over themselves, 4
    // heads: 116 and 135).
    // A triangle of more row tiles than that holds no part (19,003 queries
    // under a window, 16 heads: the second launch took 10 of 700 us).
    s.min_tiles = 24;
    const int64_t target = (3 * kResident / 2 + heads - 1) / heads;
    if (key_tiles > s.min_tiles && ((ragged && sequences > 1) || likely < 2 * target)) s.target = target;
  } else {
    s.min_tiles = 4;
    if (key_tiles > s.min_tiles) s.target = wide_target(likely, heads, key_tiles, s.min_tiles);
  }
  s.grid = (s.target + s.tiles) * heads;
  s.headers = std::min(s.target, s.tiles);  // (take_item's bounds)
  s.records = std::min(2 * s.target, s.target ? s.target + s.tiles : 0) * heads;
  s.header_bytes = (s.headers * heads * int64_t(sizeof(Header)) + 15) / 16 * 16;
  s.merge_rows = std::min(s.rows, (rows * group + sequences - 1) / sequences);
  s.bytes = s.header_bytes + s.records * s.rows * (head_dim + 4) * 4;
  return s;
}

hipError_t launch_paged(const PagedParams& params, const PagedSize& size, int D, int format, hipStream_t stream) {
  PagedParams p = params;
  p.target = int(size.target);
  p.min_tiles = int(size.min_tiles);
  p.headers = size.headers;
  p.records = size.records;
  p.header_bytes = size.header_bytes;
  p.new_rows = p.batch.table ? p.batch.rows : int64_t(p.batch.S) * p.Tq;
  if (D == 128) launch_format<128>(p, size, format, stream);
  else launch_format<64>(p, size, format, stream);
  return hipGetLastError();
}

}  // namespace sol
