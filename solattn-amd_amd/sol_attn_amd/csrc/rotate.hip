// Norms of the heads' rows of Q and K, and their rotation by the tokens'
// positions, in one pass.
//
// A row x of D elements, w its norm's weight (no norm: y = x):
//   y = x w / sqrt(mean x^2 + eps)
// Pair j is elements j and j + D / 2 (halves) or 2 j and 2 j + 1 (pairs); its
// angle is a = position[axis_j] f_j, and
//   (y0, y1) -> (y0 cos a - y1 sin a, y0 sin a + y1 cos a)
// rounded once to BF16; everything before is FP32.  An angle is formed and
// reduced to a part of a turn in FP64: position 2^31 times f = 1 still leaves an
// error of 2^-22, where FP32 would leave hundreds of turns.
//
// Bound by memory: every row is read and written once.  84,672 tokens of 24 + 24
// heads of 128, norms and three axes, 2.08 GB: 389 us, 5.35 TB/s (a copy of 4 GiB
// 4.83).  19,003 tokens of 12 + 3 heads of 64, 73 MB: 14.8 us, 4.9 TB/s.  A decoding
// step of 48 tokens of 24 + 8 heads is a chain of latencies, 5.9 us, less than the
// 12 that the host takes to make the call.  (The angles' arithmetic is not what
// bounds it: sines of four multiply-adds each instead of the library's took 0 to 3%
// off.)
#include "rotate_internal.h"
#include "sol_device.h"

namespace sol {

namespace {

constexpr int kRotateThreads = 256;

// D / 16 lanes hold a row, two 16-byte chunks each: chunk c and chunk c + D / 16,
// so that both elements of a pair of halves lie in one lane, and eight pairs in
// either layout.  A wave holds one head's rows of 1024 / D consecutive tokens and
// goes from head to head, so the angles are formed once per token and wave.
template <int D>
constexpr int kRotateLanes = D / 16;
template <int D>
constexpr int kRotateTokens = 64 / kRotateLanes<D>;

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, false));
}

// Sum over the lanes that hold a row.
template <int D>
__device__ __forceinline__ float row_sum(float x) {
  x = dpp_add<0xB1>(x);  // lane ^ 1
  x = dpp_add<0x4E>(x);  // lane ^ 2
  if constexpr (kRotateLanes<D> == 8) x = dpp_add<0x141>(x);  // the row's other four
  return x;
}

// Pair i (of a lane's eight) of the row.
template <int D, bool PAIRS>
__device__ __forceinline__ int pair_of(int c, int i) {
  return PAIRS ? (i < 4 ? 4 * c + i : D / 4 + 4 * c + i - 4) : 8 * c + i;
}

// A lane's elements of one row: pair i is a[i], b[i].  (Arrays in their place went
// through LDS in the layout of pairs: 1,448 tokens of 64 + 8 heads of 64 21 us, 8.9.)
typedef float f32x8 __attribute__((ext_vector_type(8)));
struct LanePairs {
  f32x8 a, b;
};

template <bool PAIRS>
__device__ __forceinline__ LanePairs unpack(const u32x4 (&x)[2]) {
  LanePairs y;
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float lo = bf16_bits_to_f32(x[n][i] & 0xFFFFu), hi = __uint_as_float(x[n][i] & 0xFFFF0000u);
      if constexpr (PAIRS) {
        y.a[4 * n + i] = lo, y.b[4 * n + i] = hi;
      } else {
        if (n) y.b[2 * i] = lo, y.b[2 * i + 1] = hi; else y.a[2 * i] = lo, y.a[2 * i + 1] = hi;
      }
    }
  return y;
}

template <bool PAIRS>
__device__ __forceinline__ void pack(const LanePairs& y, u32x4 (&x)[2]) {
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (PAIRS)
        x[n][i] = pack_bf16x2(y.a[4 * n + i], y.b[4 * n + i]);
      else
        x[n][i] = n ? pack_bf16x2(y.b[2 * i], y.b[2 * i + 1]) : pack_bf16x2(y.a[2 * i], y.a[2 * i + 1]);
    }
}

// Divides a row by sqrt(mean x^2 + eps).  Squares of very large or very small
// rows leave FP32's range: those rows are moved by a power of two first.
template <int D>
__device__ __forceinline__ void normalise(LanePairs& y, float eps) {
  auto squares = [&](float f) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = y.a[i] * f, b = y.b[i] * f;
      s = fmaf(a, a, fmaf(b, b, s));
    }
    return row_sum<D>(s);
  };
  float s = squares(1.f), f = 1.f;
  const bool out = !(s < 0x1p100f) || (s < 0x1p-90f && eps < 0x1p-90f);
  if (__builtin_amdgcn_ballot_w64(out)) {
    const float f2 = s < 1.f ? 0x1p100f : 0x1p-70f;
    const float s2 = squares(f2);
    if (out) s = s2, f = f2, eps = eps * f2 * f2;
  }
  const float r = __fdiv_rn(1.f, __fsqrt_rn(fmaf(s, 1.f / D, eps)));
#pragma unroll
  for (int i = 0; i < 8; ++i) y.a[i] = y.a[i] * f * r, y.b[i] = y.b[i] * f * r;
}

template <int D, bool PAIRS>
__global__ __launch_bounds__(kRotateThreads) void rotate_kernel(RotateParams p, int heads_each) {
  constexpr int U = 4;  // heads on their way together
  const int lane = threadIdx.x & 63, c = lane % kRotateLanes<D>;
  const int heads = p.x[0].heads + p.x[1].heads;
  const int groups = (heads + heads_each - 1) / heads_each;
  const int64_t unit = int64_t(blockIdx.x) * (kRotateThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t first = unit / groups * kRotateTokens<D>;
  if (first >= p.rows) return;
  const int h0 = int(unit % groups) * heads_each, h1 = min(h0 + heads_each, heads);
  // Tokens past the last one read that one and store nothing.
  const bool mine = first + lane / kRotateLanes<D> < p.rows;
  const int64_t row = min(first + lane / kRotateLanes<D>, p.rows - 1);
  const int64_t b = row / p.tokens, t = row % p.tokens;

  // The wave's heads h .. to - 1 of Q (n = 0), then of K.
  int n = h0 < p.x[0].heads ? 0 : 1;
  auto from = [&] { return max(h0 - (n ? p.x[0].heads : 0), 0); };
  auto until = [&] { return min(h1 - (n ? p.x[0].heads : 0), p.x[n].heads); };
  int h = from(), to = until();
  u32x4 v[U][2];
  auto load = [&] {
    const RotateOperand& x = p.x[n];
    const uint16_t* in = x.rows + b * x.sb + t * x.st + 8 * c;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < 2; ++k) v[u][k] = load16(in + min(h + u, to - 1) * x.sh + k * (D / 2));
  };
  load();
  asm volatile("" ::: "memory");  // on their way while the angles are formed

  // The axes of all eight pairs, then all their positions: without a branch, so that
  // each is one wait (a pair of no axis reads one).
  float cs[8], sn[8];
  bool still[8];  // the pair has no axis and stays as it is: a product with a sine of 0 is NaN next to an infinity
  const int32_t* at = p.positions + b * p.pb + t * p.pt;
  int axis[8], position[8];
  double frequency[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    axis[i] = p.axis[pair_of<D, PAIRS>(c, i)];
    frequency[i] = p.frequencies[pair_of<D, PAIRS>(c, i)];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) position[i] = at[min(max(axis[i], 0), p.axes - 1)];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    still[i] = axis[i] < 0 || axis[i] >= p.axes;
    const double turns = still[i] ? 0. : double(position[i]) * frequency[i] * 0.15915494309189533577;
    float s, c1;
    sincospif(2.f * float(turns - rint(turns)), &s, &c1);
    sn[i] = s, cs[i] = c1;
  }

  for (;;) {
    const RotateOperand& x = p.x[n];
    f32x8 wa, wb;
    auto weights = [&](auto at) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = pair_of<D, PAIRS>(c, i);
        wa[i] = at(PAIRS ? 2 * j : j);
        wb[i] = at(PAIRS ? 2 * j + 1 : j + D / 2);
      }
    };
    if (!x.weight)
      weights([](int) { return 1.f; });
    else if (p.weights_bf16)
      weights([&](int e) { return bf16_bits_to_f32(static_cast<const uint16_t*>(x.weight)[e]); });
    else
      weights([&](int e) { return static_cast<const float*>(x.weight)[e]; });
    uint16_t* out = x.out + b * x.ob + t * x.ot + 8 * c;
    for (;;) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        LanePairs y = unpack<PAIRS>(v[u]);
        if (x.weight) {
          normalise<D>(y, p.eps);
#pragma unroll
          for (int i = 0; i < 8; ++i) y.a[i] *= wa[i], y.b[i] *= wb[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a = y.a[i], bb = y.b[i];
          y.a[i] = still[i] ? a : a * cs[i] - bb * sn[i];
          y.b[i] = still[i] ? bb : a * sn[i] + bb * cs[i];
        }
        pack<PAIRS>(y, v[u]);
        if (mine && h + u < to) {
#pragma unroll
          for (int k = 0; k < 2; ++k) *reinterpret_cast<u32x4*>(out + (h + u) * x.oh + k * (D / 2)) = v[u][k];
        }
      }
      h += U;
      if (h >= to) break;
      load();
    }
    if (n == 1) return;
    n = 1;
    h = from(), to = until();
    if (h >= to) return;
    load();
  }
}

template <int D, bool PAIRS>
void rotate_variant(const RotateParams& p, hipStream_t stream) {
  const int64_t groups = (p.rows + kRotateTokens<D> - 1) / kRotateTokens<D>;
  const int heads = p.x[0].heads + p.x[1].heads;
  // Four heads to a wave, eight where that makes 2,000 waves and more: a wave has the
  // angles to form first, and neighbouring waves of few heads read neighbouring rows.
  // Four and eight: 4,032 tokens of 24 + 24 heads of 128 22.1 and 20.1 us, 40,000 of 8
  // + 1 40.1 and 37.9, 2,000 of 32 + 8 (2,500 waves of four) 12.5 and 13.3; eight
  // and sixteen: 84,672 of 24 + 24 389 and 403.
  const int each = groups * ((heads + 3) / 4) > 4096 ? 8 : 4;
  const int64_t units = groups * ((heads + each - 1) / each);
  hipLaunchKernelGGL((rotate_kernel<D, PAIRS>), dim3(unsigned((units + 3) / 4)), dim3(kRotateThreads), 0, stream, p,
                     each);
}

}  // namespace

hipError_t launch_rotate(const RotateParams& p, int D, bool pairs, hipStream_t stream) {
  if (D == 128)
    pairs ? rotate_variant<128, true>(p, stream) : rotate_variant<128, false>(p, stream);
  else
    pairs ? rotate_variant<64, true>(p, stream) : rotate_variant<64, false>(p, stream);
  return hipGetLastError();
}

}  // namespace sol
