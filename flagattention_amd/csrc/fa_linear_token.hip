// One step of linear attention per sequence for gfx950: S' = e^a S + k v^T, o = scale q S' for every
// query head of the KV head's group.
//
// Bound by the state, read and written once.  A work-group takes kCols columns of one (sequence, KV
// head): columns of the state are independent of each other, so no work-group waits for another.  A
// thread keeps its part -- four columns of every (kThreads / (kCols / 4))th row -- in registers from
// the load to the store, and every load is on its way before the first is used.  The sums over
// rows go through the lanes of a wave, then through LDS.  256 sequences of 16 KV heads, D = 256: 441 us,
// 4.9 TB/s read and written (a large copy: 5.1); 61 of 32, D = 128: 55 us, 4.7; one of 8, D = 64: 3.4 us.
#include "fa_common.h"
#include "fa_divide.h"
#include "fa_linear.h"
#include "fa_wave.h"
#include "flagattention_amd_linear.h"

namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 8;  // query heads whose sums are taken at once

// The value of the lane kBy places on, around a row of 16.
template <int kBy>
__device__ inline float ror16(float x) {
  return __uint_as_float(static_cast<unsigned int>(__builtin_amdgcn_update_dpp(
      0, static_cast<int>(__float_as_uint(x)), 0x120 + kBy, 0xF, 0xF, false)));
}

template <typename T, int D, int kCols>
__global__ __launch_bounds__(kThreads) void linear_token_kernel(const fa_linear_args a,
                                                                const Divisor h_kv) {
  constexpr int kLanes = kCols / 4;           // lanes of a row
  constexpr int kRows = kThreads / kLanes;    // rows at once
  constexpr int kSteps = D / kRows;
  static_assert(kSteps >= 1 && kSteps * kRows == D, "whole steps");
  __shared__ float ks[D], qs[kGroup][D];
  __shared__ __attribute__((aligned(16))) float sums[4][kGroup][kCols];

  const int tid = threadIdx.x;
  const int b = divide(blockIdx.x, h_kv);
  const int hk = blockIdx.x - b * a.h_kv;
  const int col0 = blockIdx.y * kCols;
  const int group = a.h_q / a.h_kv;
  const int slot = a.state_indices ? a.state_indices[b] : b;
  T* const out = static_cast<T*>(a.out) +
                 (static_cast<long long>(b) * a.h_q + hk * group) * D + col0;
  if (slot < 0 || slot >= a.num_slots) {  // uniform
    for (int i = tid; i < group * kCols; i += kThreads)
      out[static_cast<long long>(i / kCols) * D + i % kCols] = static_cast<T>(0.f);
    return;
  }
  const int row0 = tid / kLanes, col = 4 * (tid % kLanes);
  float* const state = a.state + slot * a.state_stride_s + hk * a.state_stride_h + col0 + col;
  floatx4 s[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    s[i] = *reinterpret_cast<const floatx4*>(state + (row0 + i * kRows) * D);
  const T* const k = static_cast<const T*>(a.k) + b * a.k_stride_t + hk * a.k_stride_h;
  const T* const v = static_cast<const T*>(a.v) + b * a.v_stride_t + hk * a.v_stride_h + col0 + col;
  const T* const q = static_cast<const T*>(a.q) + b * a.q_stride_t +
                     static_cast<long long>(hk) * group * a.q_stride_h;
  for (int i = tid; i < D; i += kThreads) ks[i] = static_cast<float>(k[i]);
  floatx4 vs;
#pragma unroll
  for (int x = 0; x < 4; ++x) vs[x] = static_cast<float>(v[x]);
  const Fall fall = fall_of(a.log_decay[hk], 1);  // uniform

  for (int g0 = 0; g0 < group; g0 += kGroup) {
    const int heads = min(kGroup, group - g0);
    for (int i = tid; i < heads * D; i += kThreads)
      qs[i / D][i % D] = static_cast<float>(q[(g0 + i / D) * a.q_stride_h + i % D]);
    __syncthreads();
    if (g0 == 0) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const float kr = ks[row0 + i * kRows];
#pragma unroll
        for (int x = 0; x < 4; ++x)
          s[i][x] = add_fallen(s[i][x], fall, kr * vs[x]);  // (an exact product)
        *reinterpret_cast<floatx4*>(state + (row0 + i * kRows) * D) = s[i];
      }
    }
    for (int g = 0; g < heads; ++g) {
      floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const float qr = qs[g][row0 + i * kRows];
#pragma unroll
        for (int x = 0; x < 4; ++x) o[x] = __builtin_fmaf(qr, s[i][x], o[x]);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (kLanes <= 8) o[x] += ror16<8>(o[x]);
        if (kLanes <= 16) o[x] = sum_xor16(o[x]);
        o[x] = sum_xor32(o[x]);
      }
      if ((tid & 63) < kLanes) *reinterpret_cast<floatx4*>(&sums[tid >> 6][g][col]) = o;
    }
    __syncthreads();
    for (int i = tid; i < heads * kCols; i += kThreads) {
      const int g = i / kCols, c = i % kCols;
      const float o = (sums[0][g][c] + sums[1][g][c]) + (sums[2][g][c] + sums[3][g][c]);
      out[static_cast<long long>(g0 + g) * D + c] = static_cast<T>(a.scale * o);
    }
    __syncthreads();
  }
}

template <typename T, int D, int kCols>
void launch(const fa_linear_args& a, hipStream_t stream) {
  hipLaunchKernelGGL((linear_token_kernel<T, D, kCols>),
                     dim3(static_cast<unsigned>(a.num_seqs * a.h_kv), D / kCols), dim3(kThreads), 0,
                     stream, a, divisor(a.h_kv));
}

// Columns of a work-group.  With few of them the state's rows are cut finer, so that more of the card
// loads them (89 sequences of 2 KV heads, D = 128: 8.1 us with 32, 8.3 with 64; one of 16, D = 256: 4.3
// / 4.9; 16 of 32, D = 128: 12.1 / 12.4); with many, wider pieces of rows come faster (64 of 32, D =
// 128: 59.4 / 57.7; 64 of 64, D = 64: 23.8 / 22.0).  16 columns are 16 and 25% slower in these.
constexpr int kManyWgs = 2048;

template <typename T, int D>
void launch_dim(const fa_linear_args& a, hipStream_t stream) {
  if (static_cast<int64_t>(a.num_seqs) * a.h_kv * (D / 64) < kManyWgs)
    launch<T, D, 32>(a, stream);
  else
    launch<T, D, 64>(a, stream);
}

template <typename T>
void launch_type(const fa_linear_args& a, hipStream_t stream) {
  if (a.d == 64)
    launch_dim<T, 64>(a, stream);
  else if (a.d == 128)
    launch_dim<T, 128>(a, stream);
  else
    launch_dim<T, 256>(a, stream);
}

}  // namespace
}  // namespace fa

extern "C" int fa_linear_token(const fa_linear_args* args, void* stream) {
  FA_CHECK_ARG(args != nullptr, "args is NULL");
  const fa_linear_args& a = *args;
  const int rc = fa::check_linear(a);
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(a.total == a.num_seqs, "%d tokens of %d sequences", a.total, a.num_seqs);
  FA_CHECK_ARG(static_cast<int64_t>(a.num_seqs) * a.h_kv < 1 << 22, "too many sequences or heads");
  if (a.num_seqs == 0) return FA_OK;
  FA_CHECK_ARG(a.state != nullptr, "state is NULL");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  a.dtype == 1 ? fa::launch_type<fa::bf16>(a, s) : fa::launch_type<_Float16>(a, s);
  FA_CHECK_HIP(hipGetLastError());
  return FA_OK;
}
