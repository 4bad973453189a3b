// Attention of new tokens over a paged cache, and over plain K / V under a
// sliding window with first tokens that stay visible.
//
// Query i of an entry with n queries and L keys has position p = L - n + i; key
// j < L is visible iff (j <= p or not causal) and (|p - j| < window or j <
// sinks).  O = sum_j softmax_j(scale q . k_j) v_j over the visible keys, 0 for
// a query that sees none.  Scores, softmax statistics and sums are FP32.
#include "paged_internal.h"
#include "sol_device.h"

namespace sol {

namespace {

// The keys a position sees: [lo, hi] and [0, sink).
struct Visible {
  int lo, hi, sink;
};

__device__ __forceinline__ Visible visible(const PagedParams& p, int pos, int length) {
  Visible v;
  v.lo = max(0, pos - p.window + 1);
  v.hi = p.causal ? pos : min(length - 1, pos + p.window - 1);
  v.sink = min(p.sinks, p.causal ? pos + 1 : length);
  return v;
}

template <int F>
__device__ __forceinline__ float element(const uint8_t* row, int i) {
  if constexpr (F == kBf16) return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(row)[i]);
  else if constexpr (F == kInt8) return float(int8_t(row[i]));
  else return __builtin_amdgcn_cvt_pk_f32_fp8(int(row[i]), false)[0];
}

// One wave per (query row, query head): a key per lane for the scores, a
// feature (two at D = 128) per lane for the values.
template <int D, int F>
__global__ __launch_bounds__(64) void attend_rows_kernel(PagedParams p) {
  const PagedBatch& bt = p.batch;
  const int lane = threadIdx.x;
  const int heads = p.H * p.G;
  const int64_t row = blockIdx.x / heads;
  const int hq = int(blockIdx.x % heads), h = hq / p.G;
  int s, i, n, length;
  if (bt.table) {
    s = 0;
    while (s + 1 < bt.S && bt.offset(s + 1) <= row) ++s;
    if (row < bt.offset(s) || row >= bt.offset(s + 1)) return;
    n = bt.offset(s + 1) - bt.offset(s);
    i = int(row) - bt.offset(s);
    length = bt.length(s);
  } else {
    s = int(row / p.Tq);
    i = int(row % p.Tq);
    n = p.Tq;
    length = p.Tk;
  }
  const Visible v = visible(p, length - n + i, length);
  const uint16_t* q = p.q + (bt.table ? row * p.q_st : s * p.q_sb + i * p.q_st) + hq * p.q_sh;
  auto address = [&](int kv, int j) -> const uint8_t* {
    int64_t unit = s;
    if (bt.table) {
      unit = bt.table[int64_t(s) * bt.width + (j >> bt.page_shift)];
      if (unit < 0 || unit >= bt.pages) return nullptr;
      return p.store[kv] + unit * p.sb[kv] + h * p.sh[kv] + (j & ((1 << bt.page_shift) - 1)) * p.st[kv];
    }
    return p.store[kv] + unit * p.sb[kv] + h * p.sh[kv] + j * p.st[kv];
  };
  auto scale_of = [&](int kv, int j) {
    if (F == kBf16) return 1.f;
    const int64_t page = bt.table[int64_t(s) * bt.width + (j >> bt.page_shift)];
    return p.scale[kv][((page * p.H + h) << bt.page_shift) + (j & ((1 << bt.page_shift) - 1))];
  };
  float m = -__builtin_huge_valf(), den = 0.f, acc[2] = {0.f, 0.f};
  bool any = false;
  for (int j0 = 0; j0 <= max(v.hi, v.sink - 1); j0 += 64) {
    if (j0 + 63 < v.lo && j0 >= v.sink) continue;
    const int j = j0 + lane;
    const bool in = (j <= v.hi && j >= v.lo) || j < v.sink;
    const uint8_t* k = in ? address(0, j) : nullptr;
    float x = -__builtin_huge_valf();
    if (k) {
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot = fmaf(bf16_bits_to_f32(q[d]), element<F>(k, d), dot);
      x = dot * scale_of(0, j) * p.scale_log2;
    }
    const uint64_t seen = __builtin_amdgcn_ballot_w64(k != nullptr);
    if (!seen) continue;
    any = true;
    float top = x;
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    const float mn = fmaxf(m, top), ms = mn == -__builtin_huge_valf() ? 0.f : mn;
    const float alpha = fast_exp2(m - ms);
    const float e = k ? fast_exp2(x - ms) : 0.f;
    float sum = e;
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    den = den * alpha + sum;
    m = mn;
    acc[0] *= alpha;
    acc[1] *= alpha;
    for (int r = 0; r < 64; ++r) {
      if (!((seen >> r) & 1)) continue;
      const float w = __shfl(e, r) * scale_of(1, j0 + r);
      const uint8_t* vr = address(1, j0 + r);
#pragma unroll
      for (int t = 0; t < D / 64; ++t) acc[t] = fmaf(w, element<F>(vr, lane + 64 * t), acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < D / 64; ++t)
    p.out[(row * heads + hq) * D + lane + 64 * t] = f32_to_bf16_bits(any ? acc[t] / den : 0.f);
}

template <int D, int F>
void launch_rows(const PagedParams& p, hipStream_t stream) {
  const int64_t rows = p.batch.table ? p.batch.rows : int64_t(p.batch.S) * p.Tq;
  hipLaunchKernelGGL((attend_rows_kernel<D, F>), dim3(unsigned(rows * p.H * p.G)), dim3(64), 0, stream, p);
}

}  // namespace

hipError_t launch_paged(const PagedParams& p, int D, int format, hipStream_t stream) {
  if (D == 128) {
    if (format == kBf16) launch_rows<128, kBf16>(p, stream);
    else if (format == kInt8) launch_rows<128, kInt8>(p, stream);
    else launch_rows<128, kFp8>(p, stream);
  } else {
    if (format == kBf16) launch_rows<64, kBf16>(p, stream);
    else if (format == kInt8) launch_rows<64, kInt8>(p, stream);
    else launch_rows<64, kFp8>(p, stream);
  }
  return hipGetLastError();
}

}  // namespace sol
