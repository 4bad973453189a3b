// A paged K/V cache: quantising rows as they are written, reading them back.
//
// Write, per (token, head) row x of K and of V:
//   BF16   the row as it is
//   INT8   a = max |x|, scale = a / 127, code = x 127 / a rounded half to even
//   FP8    a = max |x|, scale = a / 448, code = the e4m3 value nearest x 448 / a
// A row of zeros has scale 0 and codes 0; a row with an infinity or a NaN has
// scale NaN, so that it reads back as NaN and not as something finite.
// Read: code * scale in FP32, rounded once to BF16; zeros past a sequence's
// keys.
//
// Both are bound by memory.  D / 8 lanes hold a row, 16 bytes of BF16 each, so
// a wave holds 512 / D rows, which are consecutive tokens of one head: stored
// rows of neighbouring tokens of a page are contiguous (page-major, then head,
// then row), and the BF16 side is read or written in whole rows.  A copy of 4
// GiB reaches 4.9 TB/s on this card.  Writing 4,032 tokens of 24 heads of 128 in
// BF16, 99 MB: 17 us where the caches hold them, 23 where not, 4.3 TB/s; nine
// prompts of up to 4,801 tokens, 12 heads of 64, FP8, 111 MB: 28 us, 4.0 TB/s (more
// rows per wave: 29 to 30).  Reading 40,320 tokens of 24 heads of 128 from INT8, 751
// MB: 145 us, 5.2 TB/s; 19,003 of 16 heads, 236 MB: 39 us where the caches hold a
// part.  Small calls are 5 us, less than the 12 that the host takes to make one.
#include "paged_internal.h"
#include "sol_device.h"

namespace sol {

namespace {

constexpr int kCacheThreads = 256;
constexpr int kOffsetsMax = 1024;  // sequence offsets a workgroup keeps in LDS

template <int D>
constexpr int kRowLanes = D / 8;
template <int D>
constexpr int kWaveRows = 64 / kRowLanes<D>;

// Largest s in [0, S) with offset(s) <= i (0 if none): offsets ascend.
template <typename Offset>
__device__ __forceinline__ int sequence_of(Offset offset, int S, int i) {
  int lo = 0, hi = S;  // offset(lo) <= i or lo = 0; offset(hi) > i or hi = S
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offset(mid) <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Maximum over the LANES (8 or 16) lanes that hold a row.
template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
#pragma unroll
  for (int off = 1; off < LANES; off <<= 1) x = max(x, uint32_t(__shfl_xor(int(x), off)));
  return x;
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pk_max_u16(uint32_t a, uint32_t b) {
  const u16x2 x = __builtin_bit_cast(u16x2, a), y = __builtin_bit_cast(u16x2, b);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, y));
}

// x / a, correctly rounded in all but rare cases and exact wherever the
// quotient is representable, from inv = fl(1 / a): the product and its
// remainder (exact in one fused step).  x = 127 v or 448 v and a hold at most
// 15 and 8 significant bits, so x / a is either exactly half-way between two
// codes, and then representable, or at least 1 / 2 a from it in units of v's
// last place: the code is that of the exact quotient.
__device__ __forceinline__ float exact_quotient(float x, float a, float inv) {
  const float q = x * inv;
  return fmaf(fmaf(-q, a, x), inv, q);
}

template <int D, int F>
__device__ __forceinline__ void write_row(const CacheParams& p, int kv, const u32x4& x, int64_t row, int lane) {
  const int c = lane % kRowLanes<D>;
  if constexpr (F == kBf16) {
    if (row >= 0) *reinterpret_cast<u32x4*>(p.store[kv] + row * D * 2 + 16 * c) = x;
  } else {
    constexpr float kLevels = F == kInt8 ? 127.f : 448.f;
    // Magnitudes compare like their bits, infinities and NaN above all others.
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = pk_max_u16(m, x[i] & 0x7FFF7FFFu);
    m = row_max<kRowLanes<D>>(max(m & 0xFFFFu, m >> 16));
    const float a = bf16_bits_to_f32(m);
    const bool finite = m < 0x7F80u;
    // Products with 448 and 1 / a stay normal: very large and very small rows
    // are moved by a power of two first.
    const float f = a > 0x1p64f ? 0x1p-64f : (a < 0x1p-64f ? 0x1p64f : 1.f);
    const float af = a * f;
    const float inv = a > 0.f && finite ? __fdiv_rn(1.f, af) : 0.f;
    const float up = f * kLevels;  // a power of two times a level: x up is exact
    uint32_t codes[2] = {0u, 0u};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b = x[2 * w + (i >> 1)];
        v[i] = exact_quotient(bf16_bits_to_f32((i & 1) ? (b >> 16) : (b & 0xFFFFu)) * up, af, inv);
        if (!finite) v[i] = 0.f;
      }
      if constexpr (F == kInt8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) codes[w] |= (uint32_t(int(rintf(v[i]))) & 0xFFu) << (8 * i);
      } else {
        codes[w] = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        codes[w] = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], codes[w], true);
      }
    }
    if (row >= 0) {
      const u32x2 out = {codes[0], codes[1]};
      *reinterpret_cast<u32x2*>(p.store[kv] + row * D + 8 * c) = out;
      if (c == 0) p.scale[kv][row] = finite ? __fdiv_rn(a, kLevels) : __builtin_nanf("");
    }
  }
}

// A wave writes U kWaveRows consecutive new rows of one head, K and V.
template <int D, int F, int U>
__global__ __launch_bounds__(kCacheThreads) void cache_write_kernel(CacheParams p) {
  __shared__ int32_t s_off[kOffsetsMax];
  const PagedBatch& bt = p.batch;
  const bool in_lds = bt.S < kOffsetsMax;
  if (in_lds) {
    for (int s = threadIdx.x; s <= bt.S; s += kCacheThreads) s_off[s] = bt.offsets[s];
    __syncthreads();
  }
  const int lane = threadIdx.x & 63;
  const int64_t unit = int64_t(blockIdx.x) * (kCacheThreads / 64) + (threadIdx.x >> 6);
  const int h = int(unit % p.H);
  const int64_t start = unit / p.H * (U * kWaveRows<D>);
  if (start >= bt.rows) return;
  // Rows past the last read that one and are not written.
  auto place = [&](int u) { return start + u * kWaveRows<D> + lane / kRowLanes<D>; };
  u32x4 x[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = int(min(place(u), int64_t(bt.rows - 1)));
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
      x[u][kv] = load16(p.rows[kv] + i * p.st[kv] + h * p.sh[kv] + 8 * (lane % kRowLanes<D>));
  }
  auto offset = [&](int s) { return in_lds ? s_off[s] : bt.offsets[s]; };
  int64_t row[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = int(min(place(u), int64_t(bt.rows - 1)));
    const int s = sequence_of(offset, bt.S, i);
    const int first = offset(s), end = offset(s + 1);
    // From the length as it is: clamped to the table it would move the row to the place of a stored one.
    const int64_t pos = int64_t(bt.lengths[s]) - (int64_t(end) - i);
    row[u] = -1;
    if (place(u) < bt.rows && i >= first && i < end && pos >= 0 && pos < bt.positions()) {
      const int page = bt.table[int64_t(s) * bt.width + (pos >> bt.page_shift)];
      if (page >= 0 && page < bt.pages)
        row[u] = ((int64_t(page) * p.H + h) << bt.page_shift) + (pos & ((1 << bt.page_shift) - 1));
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) write_row<D, F>(p, kv, x[u][kv], row[u], lane);
}

template <int F>
__device__ __forceinline__ u32x4 dequantised(u32x2 codes, float scale) {
  u32x4 o;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float v[4];
    if constexpr (F == kInt8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = float(int32_t(codes[w] << (24 - 8 * i)) >> 24);
    } else {
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes[w], false);
      const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes[w], true);
      v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
    }
    o[2 * w] = pack_bf16x2(v[0] * scale, v[1] * scale);
    o[2 * w + 1] = pack_bf16x2(v[2] * scale, v[3] * scale);
  }
  return o;
}

// Groups of kWaveRows positions that a wave reads.  Rows of codes are half as
// long: two groups, all of whose codes and scales are on their way together
// (40,320 tokens of 24 heads of 128 from FP8 173 us with one whose K is stored
// before V is asked for, 149 with one, 141 with two, 143 with four; BF16 169, 170,
// 182, 186).
template <int F>
constexpr int kReadGroups = F == kBf16 ? 1 : 2;

// A wave reads consecutive positions of one sequence and head, K and V.
template <int D, int F>
__global__ __launch_bounds__(kCacheThreads) void cache_read_kernel(CacheParams p) {
  constexpr int U = kReadGroups<F>, kRows = U * kWaveRows<D>;
  const PagedBatch& bt = p.batch;
  const int lane = threadIdx.x & 63, c = lane % kRowLanes<D>;
  const int64_t unit = int64_t(blockIdx.x) * (kCacheThreads / 64) + (threadIdx.x >> 6);
  const int groups = (p.tokens + kRows - 1) / kRows;
  const int h = int(unit % p.H);
  const int64_t sg = unit / p.H;
  const int s = int(sg / groups);
  if (s >= bt.S) return;
  const int t0 = int(sg % groups) * kRows + lane / kRowLanes<D>;
  const int length = bt.length(s);
  int64_t row[U];  // -1: not there
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t pos = int64_t(p.start) + t0 + u * kWaveRows<D>;
    int page = -1;
    if (pos < length) page = bt.table[int64_t(s) * bt.width + (pos >> bt.page_shift)];
    row[u] = page >= 0 && page < bt.pages
                 ? ((int64_t(page) * p.H + h) << bt.page_shift) + (pos & ((1 << bt.page_shift) - 1))
                 : -1;
  }
  auto out = [&](int u, int kv) {
    const int64_t token = int64_t(s) * p.tokens + t0 + u * kWaveRows<D>;
    return reinterpret_cast<u32x4*>(p.out[kv] + (token * p.H + h) * D + 8 * c);
  };
  if constexpr (F == kBf16) {
    if (t0 >= p.tokens) return;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      u32x4 o = zero_u32x4();
      if (row[0] >= 0) o = *reinterpret_cast<const u32x4*>(p.store[kv] + row[0] * D * 2 + 16 * c);
      *out(0, kv) = o;
    }
  } else {
    u32x2 x[U][2];
    float scale[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int64_t at = max(row[u], int64_t(0));  // row 0 for what is not there
        x[u][kv] = *reinterpret_cast<const u32x2*>(p.store[kv] + at * D + 8 * c);
        scale[u][kv] = p.scale[kv][at];
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t0 + u * kWaveRows<D> >= p.tokens) return;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) *out(u, kv) = row[u] >= 0 ? dequantised<F>(x[u][kv], scale[u][kv]) : zero_u32x4();
    }
  }
}

template <int D, int F, int U>
void write_rows(const CacheParams& p, hipStream_t stream) {
  const int64_t units = (int64_t(p.batch.rows) + U * kWaveRows<D> - 1) / (U * kWaveRows<D>) * p.H;
  hipLaunchKernelGGL((cache_write_kernel<D, F, U>), dim3(unsigned((units + 3) / 4)), dim3(kCacheThreads), 0, stream, p);
}

template <int D, int F>
void write_variant(const CacheParams& p, hipStream_t stream) {
  // BF16 rows, which need no arithmetic, four groups to a wave where that makes
  // one round of waves of one and a half to four.  Kernel time with one group and
  // with four, rows and pages out of the caches (in them), 24 heads of 128; 8
  // heads, and heads of 64, are within 3% of these:
  //    8,300 waves  11.4 and 11.8 us (7.2 and 7.7)     24,000  24.0 and 23.2 (17.9 and 17.1)
  //   10,000        12.7 and 12.7 (8.0 and 8.8)        28,000  26.2 and 27.4 (19.7 and 19.0)
  //   12,000        14.5 and 13.8 (10.1 and 10.1)      32,000  29.7 and 26.2 (22.1 and 21.2)
  //   16,000        17.2 and 15.8 (12.9 and 12.6)      40,000  35.7 and 39.5 (26.8 and 26.0)
  constexpr int64_t kCardWaves = 8192;  // 256 CUs of 32
  const int64_t waves = (int64_t(p.batch.rows) + kWaveRows<D> - 1) / kWaveRows<D> * p.H;
  if constexpr (F == kBf16) {
    if (waves > kCardWaves * 3 / 2 && waves <= 4 * kCardWaves) return write_rows<D, F, 4>(p, stream);
  }
  write_rows<D, F, 1>(p, stream);
}

template <int D, int F>
void read_variant(const CacheParams& p, hipStream_t stream) {
  constexpr int kRows = kReadGroups<F> * kWaveRows<D>;
  const int64_t units = int64_t(p.batch.S) * ((p.tokens + kRows - 1) / kRows) * p.H;
  hipLaunchKernelGGL((cache_read_kernel<D, F>), dim3(unsigned((units + 3) / 4)), dim3(kCacheThreads), 0, stream, p);
}

}  // namespace

hipError_t launch_cache_write(const CacheParams& p, int D, int format, hipStream_t stream) {
  if (D == 128) {
    if (format == kBf16) write_variant<128, kBf16>(p, stream);
    else if (format == kInt8) write_variant<128, kInt8>(p, stream);
    else write_variant<128, kFp8>(p, stream);
  } else {
    if (format == kBf16) write_variant<64, kBf16>(p, stream);
    else if (format == kInt8) write_variant<64, kInt8>(p, stream);
    else write_variant<64, kFp8>(p, stream);
  }
  return hipGetLastError();
}

hipError_t launch_cache_read(const CacheParams& p, int D, int format, hipStream_t stream) {
  if (D == 128) {
    if (format == kBf16) read_variant<128, kBf16>(p, stream);
    else if (format == kInt8) read_variant<128, kInt8>(p, stream);
    else read_variant<128, kFp8>(p, stream);
  } else {
    if (format == kBf16) read_variant<64, kBf16>(p, stream);
    else if (format == kInt8) read_variant<64, kInt8>(p, stream);
    else read_variant<64, kFp8>(p, stream);
  }
  return hipGetLastError();
}

}  // namespace sol
