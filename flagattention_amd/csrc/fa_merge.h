// Merge of the splits' partial rows of packed prompts and of 4-bit decode:
// lse = logsumexp_s lse_s, out = sum_s exp(lse_s - lse) o_s.
//
// A split without a visible key holds lse -inf and no values; one with a NaN holds lse +inf, whose
// weight is NaN.  The weights, 1 at most, are taken at 2^-16 of their size (there are fewer than 2^16
// splits), so that the sum stays within fp32 wherever the result does: two splits of bf16's largest
// value would be past it.
//
// Bound by the latency of its loads up to kAheadRows rows: the values of a lane's first splits are
// requested beside the lse that their weights wait for, up to kWaveSplits splits by a wave per row,
// more by four (one token over 8,192 keys, 32 heads: 13.3 us a call, 14.8 with a wave per row that
// waits for the lse first; 32,000 cached keys 12.4 and 12.8).  With more rows bound by bytes: only the
// values of splits with a visible key are read, after the lse (a causal batch leaves many without: 4
// prompts of up to 1,866 tokens, head dim 256, 53.8 us, 56.5 with all of them).
#pragma once

#include "fa_common.h"
#include "fa_wave.h"

namespace fa {

struct MergeArgs {
  const float* o_part;    // [rows][splits][D]
  const float* lse_part;  // [rows][splits]
  void* out;              // row r at (r / inner) * stride_outer + (r % inner) * stride_inner
  float* lse;             // [rows], or NULL
  int64_t stride_outer, stride_inner;
  int rows, inner, splits;
};

constexpr int kWaveSplits = 16;
constexpr int kAheadRows = 8192;

// Rows that a grid holds, whose lanes number less than 2^32.
inline int64_t max_merge_rows(int splits) {
  return splits <= kWaveSplits ? (int64_t{1} << 26) - 4 : (int64_t{1} << 24) - 1;
}

template <typename T, int D, int kRowWaves, bool kAhead>
__global__ __launch_bounds__(256) void merge_kernel(const MergeArgs a) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  constexpr int kLanes = D / 4, kPar = 64 / kLanes;  // lanes per split, splits side by side
  constexpr int kBatch = kRowWaves == 1 ? 4 : 8, kStep = kPar * kRowWaves;
  __shared__ floatx4 sacc[kRowWaves > 1 ? kRowWaves * kLanes : 1];
  __shared__ float sl[kRowWaves];
  const int part = wave_id() % kRowWaves;
  const int row = blockIdx.x * (4 / kRowWaves) + wave_id() / kRowWaves;
  if (row >= a.rows) return;  // whole waves; never where there is a barrier
  const int lane = threadIdx.x & 63, sub = lane / kLanes, d4 = lane % kLanes;
  const int S = a.splits;
  const float ninf = -__builtin_inff();
  const float* const lp = a.lse_part + static_cast<long long>(row) * S;
  const float* const op = a.o_part + static_cast<long long>(row) * S * D + 4 * d4;
  float lv[kBatch];
  floatx4 ov[kBatch];
  auto request = [&](int s0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int s = s0 + kStep * i;
      lv[i] = s < S ? lp[min(s, S - 1)] : ninf;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int s = min(s0 + kStep * i, S - 1);
      if (kAhead || lv[i] != ninf)
        ov[i] = *reinterpret_cast<const floatx4*>(op + static_cast<long long>(s) * D);
    }
  };
  int s0 = part * kPar + sub;
  request(s0);
  float m = ninf;
  for (int s = lane; s < S; s += 64) m = fmaxf(m, lp[s]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
  float l = 0.f;
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  for (;;) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (lv[i] == ninf) continue;  // no values
      const float w = expf(lv[i] - m) * 0x1p-16f;
      l += w;
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[x] += w * ov[i][x];
    }
    s0 += kStep * kBatch;
    if (s0 - sub >= S) break;  // uniform over the wave
    request(s0);
  }
#pragma unroll
  for (int off = 32; off >= kLanes; off >>= 1) {
    l += __shfl_xor(l, off);
#pragma unroll
    for (int x = 0; x < 4; ++x) acc[x] += __shfl_xor(acc[x], off);
  }
  if constexpr (kRowWaves > 1) {
    if (sub == 0) sacc[part * kLanes + d4] = acc;
    if (lane == 0) sl[part] = l;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int i = 1; i < kRowWaves; ++i) {
      l += sl[i];
      const floatx4 o = sacc[i * kLanes + d4];
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[x] += o[x];
    }
  }
  const bool seen = !(l == 0.f);  // else no visible key: out 0, lse -inf (NaN stays NaN)
  const float inv = seen ? 1.f / l : 0.f;
  const int outer = row / a.inner, inner = row - outer * a.inner;
  if (sub == 0) {
    T4 w;
#pragma unroll
    for (int x = 0; x < 4; ++x) w[x] = static_cast<T>(acc[x] * inv);
    *reinterpret_cast<T4*>(static_cast<T*>(a.out) + outer * a.stride_outer +
                           inner * a.stride_inner + 4 * d4) = w;
  }
  if (part == 0 && lane == 0 && a.lse) a.lse[row] = seen ? m + logf(l * 0x1p16f) : ninf;
}

template <typename T, int D>
void launch_merge_d(const MergeArgs& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.splits <= kWaveSplits ? (a.rows + 3ll) / 4 : a.rows));
  if (a.splits > kWaveSplits)
    hipLaunchKernelGGL((merge_kernel<T, D, 4, true>), grid, dim3(256), 0, stream, a);
  else if (a.rows <= kAheadRows)
    hipLaunchKernelGGL((merge_kernel<T, D, 1, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((merge_kernel<T, D, 1, false>), grid, dim3(256), 0, stream, a);
}

template <typename T>
void launch_merge(const MergeArgs& a, int d, hipStream_t stream) {
  if (d == 64)
    launch_merge_d<T, 64>(a, stream);
  else if (d == 128)
    launch_merge_d<T, 128>(a, stream);
  else
    launch_merge_d<T, 256>(a, stream);
}

}  // namespace fa
