// Linear attention with a decay per head over packed sequences for gfx950: fp16 or bf16, head dim 64,
// 128, 256.  Per KV head with log decay a, S_t = e^a S_{t-1} + k_t v_t^T, o_t = scale q_t S_t.
//
// A work-group takes one (sequence, KV head) through its tokens, 32 at a time.  For such a chunk of c
// tokens, counted from 0, with S the state before it:
//   O^T = (S^T Q^T) diag(scale e^{a (i+1)}) + V^T P^T,  P^T[j, i] = scale e^{a (i-j)} (K Q^T)[j, i], j <= i
//   S'  = e^{a c} S + K^T diag(e^{a (c-1-j)}) V
// No factor is above 1 for a decay (a <= 0), however long the chunk or fast the decay.
//
// Wave w owns columns 32w .. 32w + 31 of S, in fp32 in its accumulators for the whole sequence, and the
// same dims of the output; D / 32 waves.  All products are MFMA 32x32x16.  Nothing but the inputs goes
// through LDS: S and P^T leave the accumulators as the operands of the next products (the rows of a
// state tile are dealt to dims so that a lane's 8 registers are the 8 dims of its part of a step), and
// every wave works the scores of a chunk out for itself, a fifth of its products.
//
// Bound by q, k, v and out.  Inputs come three chunks deep into LDS.
//
// Rounding: scores, sums and states are fp32.  P and the state's copy are rounded to the input type to
// meet V and Q, as the output is.  The weighted values that a state takes in are split in two such
// numbers, whose rest is 2^-16: the state is an output in fp32.  fp16 operands are taken relative to a
// power of two of the largest, since states, scores and products of tiny inputs leave its range.
#include "fa_common.h"
#include "fa_divide.h"
#include "fa_linear.h"
#include "fa_rows_tile.h"
#include "fa_wave.h"
#include "flagattention_amd_linear.h"

namespace fa {

int check_linear(const fa_linear_args& a) {
  FA_CHECK_ARG(a.d == 64 || a.d == 128 || a.d == 256, "head dim %d is not 64, 128 or 256", a.d);
  FA_CHECK_ARG(a.dtype == 0 || a.dtype == 1, "dtype %d", a.dtype);
  FA_CHECK_ARG(a.h_kv >= 1 && a.h_q >= 1 && a.h_q % a.h_kv == 0,
               "%d query heads are no multiple of %d", a.h_q, a.h_kv);
  FA_CHECK_ARG(static_cast<int64_t>(a.h_q) * a.d < 1 << 23, "too many heads");
  FA_CHECK_ARG(a.num_seqs >= 0 && a.num_seqs <= 65535 && a.total >= 0,
               "%d sequences, %d tokens out of range", a.num_seqs, a.total);
  if (a.total > 0) {
    FA_CHECK_ARG(a.q && a.k && a.v && a.log_decay && a.out, "NULL pointer");
    for (const void* p : {a.q, a.k, a.v, static_cast<const void*>(a.out)})
      FA_CHECK_ARG((reinterpret_cast<uintptr_t>(p) & 15) == 0, "rows must be 16-byte aligned");
    for (const int64_t st : {a.q_stride_t, a.q_stride_h, a.k_stride_t, a.k_stride_h, a.v_stride_t,
                             a.v_stride_h})
      FA_CHECK_ARG(st >= 0 && st % 8 == 0, "stride %lld", static_cast<long long>(st));
    FA_CHECK_ARG(a.q_stride_t < 1 << 23 && a.k_stride_t < 1 << 23 && a.v_stride_t < 1 << 23,
                 "tokens are too far apart");
  }
  if (a.state)
    FA_CHECK_ARG(a.num_slots >= 0 && (reinterpret_cast<uintptr_t>(a.state) & 15) == 0 &&
                     a.state_stride_s % 4 == 0 && a.state_stride_h % 4 == 0,
                 "states must be 16-byte aligned");
  return FA_OK;
}

namespace {

constexpr int kChunk = 32;
constexpr int kStages = 3;
// fp16: the least power of two that operands are relative to.  What is below it by 2^-25 is below half
// of the smallest step of the output for any q or v in range.
constexpr int kLeastPower = -40;

// Where 16 bytes c of row r of a chunk lie in it: c ^ swizzle(r).  Rows are read 16 bytes a lane, one
// row per lane (16 rows have 16 places), and transposed, 8 bytes of 4 rows in a row by 4 lanes each
// (rows r .. r + 3 lie in different quarters).
template <int C>
__device__ inline int swizzle(int r) {
  return C >= 16 ? ((r & 3) << 2) | ((r >> 1) & 2) | ((r >> 3) & 1)
                 : ((r & 2) << 1) | ((r >> 1) & 2) | ((r >> 3) & 1);
}

// A barrier that no access to memory passes.
__device__ inline void sync() {
  asm volatile("" ::: "memory");
  barrier();
  asm volatile("" ::: "memory");
}

// Power of two above |x|, 0 for 0, infinities and NaN.
__device__ inline int power_of(float x) { return __builtin_amdgcn_frexp_expf(x); }
__device__ inline float times_power(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }

template <typename T, int D>
__global__ __launch_bounds__(2 * D, 2) void linear_kernel(const fa_linear_args a,
                                                          const Divisor h_kv) {
  typedef typename PVec<T>::v8 T8;
  typedef typename PVec<T>::v4 T4;
  constexpr bool kHalf = !__is_same(T, __bf16);
  constexpr int C = D / 8;
  constexpr int kRowB = 2 * D;
  constexpr int kTileB = kChunk * kRowB;
  constexpr int kCopies = 2;  // of 1 KiB a wave and tile
  constexpr int kRowsPerCopy = 512 / D;
  constexpr int kKSteps = D / 16;
  constexpr int kTiles = D / 32;
  static_assert(kCopies * kTiles * 1024 == kTileB, "whole copies per wave");
  // [q, k, v][stage]
  __shared__ __attribute__((aligned(16))) unsigned char bufs[3 * kStages * kTileB];

  const int wave = wave_id();
  const int lane = threadIdx.x & 63;
  const int h = lane >> 5, c32 = lane & 31;
  const int group = a.h_q / a.h_kv;

  // rows of no sequence: everybody takes a share of their 16 bytes
  {
    const int first = min(max(a.cu_seqlens[0], 0), a.total);
    const int behind = max(first, min(max(a.cu_seqlens[a.num_seqs], 0), a.total));
    const long long row16 = static_cast<long long>(a.h_q) * C;
    const long long head = first * row16, all = a.total * row16, tail = behind * row16;
    uintx4* const out16 = static_cast<uintx4*>(a.out);
    const long long step = static_cast<long long>(gridDim.x) * (2 * D);
    const long long me = static_cast<long long>(blockIdx.x) * (2 * D) + threadIdx.x;
    for (long long i = me; i < head; i += step) out16[i] = uintx4{0, 0, 0, 0};
    for (long long i = tail + me; i < all; i += step) out16[i] = uintx4{0, 0, 0, 0};
  }

  const int seq = divide(blockIdx.x, h_kv);
  const int hk = blockIdx.x - seq * a.h_kv;
  if (seq >= a.num_seqs) return;  // uniform
  const int start = min(max(sload(a.cu_seqlens + seq), 0), a.total);
  const int n = min(max(sload(a.cu_seqlens + seq + 1), start), a.total) - start;
  if (n == 0) return;
  const float log_decay = sload(a.log_decay + hk);
  float* state = nullptr;  // where the state stays
  bool kept = false;
  if (a.state) {
    const int slot = a.state_indices ? sload(a.state_indices + seq) : seq;
    if (slot >= 0 && slot < a.num_slots) {
      state = a.state + slot * a.state_stride_s + hk * a.state_stride_h;
      kept = a.has_state == nullptr || a.has_state[seq] != 0;
    }
  }

  const unsigned char* const qp =
      static_cast<const unsigned char*>(a.q) +
      2 * (start * a.q_stride_t + static_cast<long long>(hk) * group * a.q_stride_h);
  const unsigned char* const kp = static_cast<const unsigned char*>(a.k) +
                                  2 * (start * a.k_stride_t + hk * a.k_stride_h);
  const unsigned char* const vp = static_cast<const unsigned char*>(a.v) +
                                  2 * (start * a.v_stride_t + hk * a.v_stride_h);
  const unsigned int q_tb = 2 * a.q_stride_t, k_tb = 2 * a.k_stride_t, v_tb = 2 * a.v_stride_t;

  // Items are (chunk, query head of the group), heads innermost; k and v come with the first head.
  const int chunks = cdiv(n, kChunk);
  const int items = chunks * group;
  const int crow = lane / C, cslot = lane % C;
  auto copy = [&](const unsigned char* src, unsigned int row_b, int first, unsigned char* dst) {
    const unsigned char* const from = src + static_cast<long long>(first) * row_b;
    const int last = n - 1 - first;  // rows past the end repeat the last one
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int r = (kCopies * wave + i) * kRowsPerCopy + crow;
      lds_dma16_off(from, min(r, last) * row_b + 16 * (cslot ^ swizzle<C>(r)),
                    (FA_LDS void*)(dst + (kCopies * wave + i) * 1024));
    }
  };
  auto tile = [&](int which, int stage) { return bufs + (which * kStages + stage) * kTileB; };
  // the item to be fetched next
  int next_item = 0, next_head = 0, next_chunk = 0, next_q = 0, next_kv = 0;
  auto fetch = [&]() {
    if (next_item >= items) return;
    copy(qp + 2 * next_head * a.q_stride_h, q_tb, next_chunk * kChunk, tile(0, next_q));
    if (next_head == 0) {
      copy(kp, k_tb, next_chunk * kChunk, tile(1, next_kv));
      copy(vp, v_tb, next_chunk * kChunk, tile(2, next_kv));
    }
    ++next_item;
    next_q = next_q == kStages - 1 ? 0 : next_q + 1;
    if (++next_head == group) {
      next_head = 0;
      ++next_chunk;
      next_kv = next_kv == kStages - 1 ? 0 : next_kv + 1;
    }
  };
  fetch();
  fetch();

  // Row rho of a 32-row tile of the state (or of O^T) is dim 16 (rho / 16) + 8 ((rho / 4) % 2) +
  // 4 ((rho / 8) % 2) + rho % 4: accumulator register r of half h is then dim 16 (r / 8) + 8h + r % 8.
  const int pi = (c32 & 16) + 8 * ((c32 >> 2) & 1) + 4 * ((c32 >> 3) & 1) + (c32 & 3);
  floatx16 s[kTiles];
  {
    const float* const from = state + 32 * wave + pi;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[t][r] = kept ? from[(32 * t + 16 * (r >> 3) + 8 * h + (r & 7)) * D] : 0.f;
  }

  // Token of register r in P^T's rows, and of element r of the values' operands.
  auto token = [&](int r) { return 8 * (r >> 2) + 4 * h + (r & 3); };
  float wp[16], wv[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int j = token(r);
    wp[r] = j <= c32 ? a.scale * decay(log_decay, c32 - j) : 0.f;
    wv[r] = decay(log_decay, kChunk - 1 - j);
  }
  const float since = a.scale * decay(log_decay, c32 + 1);
  Fall fall = fall_of(log_decay, kChunk);

  const int row_at = c32 * kRowB + 16 * (h ^ swizzle<C>(c32));
  // transposed reads: lanes 4e + x of 16 point at 4 dims of token row e
  const int e = (lane & 15) >> 2, x4 = lane & 3, p16 = (lane >> 4) & 1;
  const int tr_at = (4 * h + e) * kRowB + 16 * ((2 * p16 + (x4 & 1)) ^ swizzle<C>(4 * h + e)) +
                    8 * (x4 >> 1);
  // dims 32t .. 32t + 31 of tokens token(8 ss) .. token(8 ss + 7), transposed
  auto transposed = [&](const unsigned char* from, int t, int ss) -> T8 {
    const T4 lo = lds_tr_read4<T>(from + (tr_at ^ (64 * t)) + 16 * ss * kRowB);
    const T4 hi = lds_tr_read4<T>(from + (tr_at ^ (64 * t) ^ 16) + (16 * ss + 8) * kRowB);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  int item = 0, q_stage = 0, kv_stage = 0;
  for (int chunk = 0; chunk < chunks; ++chunk) {
    const int left = min(n - chunk * kChunk, kChunk);
    unsigned char* const kb = tile(1, kv_stage);
    unsigned char* const vb = tile(2, kv_stage);
    T8 va[2];
    bool odd = false;
    for (int g = 0; g < group; ++g, ++item) {
      // all but what was issued after this item's copies: the next item's, and the last one's stores
      if (item + 1 < items && item > 0) {
        if (g + 1 == group)
          wait_vmem<3 * kCopies + 2>();
        else
          wait_vmem<kCopies + 2>();
      } else {
        wait_vmem<0>();
      }
      sync();
      fetch();
      const unsigned char* const qb = tile(0, q_stage);
      q_stage = q_stage == kStages - 1 ? 0 : q_stage + 1;
      if (g == 0) {
        if (left < kChunk) {  // uniform: rows past the end become zeros
          for (int i = left * kRowB / 16 + threadIdx.x; i < kTileB / 16; i += 2 * D) {
            reinterpret_cast<uintx4*>(kb)[i] = uintx4{0, 0, 0, 0};
            reinterpret_cast<uintx4*>(vb)[i] = uintx4{0, 0, 0, 0};
          }
          sync();
        }
        // An infinity or a NaN in v would reach the tokens before its own through weights of 0.
        bool is_odd = false;
#pragma unroll
        for (int ss = 0; ss < 2; ++ss) {
          va[ss] = transposed(vb, wave, ss);
#pragma unroll
          for (int x = 0; x < 8; ++x)
            is_odd |= !(fabsf(static_cast<float>(va[ss][x])) < __builtin_inff());
        }
        odd = __ballot(is_odd) != 0ull;
      }

      // scores and S^T Q^T: a step of Q meets both
      int s_power = 0, p_power = 0;
      if constexpr (kHalf) {
        float most = 0.f;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(s[t][r]));
        if (__ballot(most == __builtin_inff()) != 0ull) {  // uniform: of those that are finite
          most = 0.f;
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              most = fabsf(s[t][r]) < __builtin_inff() ? fmaxf(most, fabsf(s[t][r])) : most;
        }
#pragma unroll
        for (int m = 1; m < 64; m *= 2) most = fmaxf(most, __shfl_xor(most, m));
        s_power = max(power_of(most), kLeastPower);
      }
      floatx16 p = {}, o = {};
#pragma unroll
      for (int ks = 0; ks < kKSteps; ++ks) {
        const T8 qa = *reinterpret_cast<const T8*>(qb + (row_at ^ (32 * ks)));
        const T8 ka = *reinterpret_cast<const T8*>(kb + (row_at ^ (32 * ks)));
        p = mfma_32x32x16(ka, qa, p);
        T8 sa;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float f = s[ks >> 1][8 * (ks & 1) + x];
          sa[x] = static_cast<T>(kHalf ? times_power(f, -s_power) : f);
        }
        o = mfma_32x32x16(sa, qa, o);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] = token(r) <= c32 ? p[r] * wp[r] : 0.f;
      if constexpr (kHalf) {
        float top = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(p[r]));
        p_power = max(power_of(max_xor32(top)), kLeastPower);
      }
      // O^T, relative to 2^p_power
      const float by = kHalf ? times_power(since, s_power - p_power) : since;
#pragma unroll
      for (int r = 0; r < 16; ++r) o[r] *= by;
#pragma unroll
      for (int ss = 0; ss < 2; ++ss) {
        T8 pb, v8 = va[ss];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float f = p[8 * ss + x];
          pb[x] = static_cast<T>(kHalf ? times_power(f, -p_power) : f);
        }
        if (odd) {  // uniform
#pragma unroll
          for (int x = 0; x < 8; ++x)
            v8[x] = fabsf(static_cast<float>(v8[x])) < __builtin_inff() ? v8[x]
                                                                       : static_cast<T>(0.f);
        }
        o = mfma_32x32x16(v8, pb, o);
      }
      if constexpr (kHalf) {
#pragma unroll
        for (int r = 0; r < 16; ++r) o[r] = times_power(o[r], p_power);
      }
      if (odd) {  // those values, for the tokens that see them
        for (int j = 0; j < left; ++j) {
          float w = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) w = 8 * (r >> 2) + (r & 3) == (j & ~4) ? p[r] : w;
          w = __shfl(w, c32 + 32 * ((j >> 2) & 1));
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const T8 v8 = *reinterpret_cast<const T8*>(
                vb + j * kRowB + 16 * ((4 * wave + 2 * half + h) ^ swizzle<C>(j)));
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const float f = static_cast<float>(v8[x]);
              o[8 * half + x] += j <= c32 && !(fabsf(f) < __builtin_inff()) ? w * f : 0.f;
            }
          }
        }
      }

      T* const out = static_cast<T*>(a.out) +
                     ((static_cast<long long>(start) + chunk * kChunk + c32) * a.h_q +
                      hk * group + g) * D + 32 * wave + 8 * h;
      if (c32 < left) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          T8 y;
#pragma unroll
          for (int x = 0; x < 8; ++x) y[x] = static_cast<T>(o[8 * half + x]);
          *reinterpret_cast<T8*>(out + 16 * half) = y;
        }
      }
    }
    if (chunk + 1 == chunks && state == nullptr) break;

    if (left < kChunk) {
#pragma unroll
      for (int r = 0; r < 16; ++r) wv[r] = decay(log_decay, max(left - 1 - token(r), 0));
      fall = fall_of(log_decay, left);
    }
    T8 hi[2], lo[2];
    int v_power = 0;
    if constexpr (kHalf) {
      float top = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        top = fmaxf(top, fabsf(static_cast<float>(va[r >> 3][r & 7]) * wv[r]));
      v_power = max(power_of(max_xor32(top)), -100);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float f = static_cast<float>(va[r >> 3][r & 7]) * wv[r];
      if (kHalf) f = times_power(f, -v_power);
      hi[r >> 3][r & 7] = static_cast<T>(f);
      lo[r >> 3][r & 7] = static_cast<T>(f - static_cast<float>(hi[r >> 3][r & 7]));
    }
    if (odd) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!(fabsf(static_cast<float>(hi[r >> 3][r & 7])) < __builtin_inff()))
          lo[r >> 3][r & 7] = static_cast<T>(0.f);
    }
    if (fall.slow) {  // uniform
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = __builtin_fmaf(s[t][r], fall.by, s[t][r]);
    } else {
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] *= fall.by;
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      if constexpr (kHalf) {
        floatx16 add = {};
#pragma unroll
        for (int ss = 0; ss < 2; ++ss) {
          const T8 ka = transposed(kb, t, ss);
          add = mfma_32x32x16(ka, hi[ss], add);
          add = mfma_32x32x16(ka, lo[ss], add);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] += times_power(add[r], v_power);
      } else {
#pragma unroll
        for (int ss = 0; ss < 2; ++ss) {
          const T8 ka = transposed(kb, t, ss);
          s[t] = mfma_32x32x16(ka, hi[ss], s[t]);
          s[t] = mfma_32x32x16(ka, lo[ss], s[t]);
        }
      }
    }
    kv_stage = kv_stage == kStages - 1 ? 0 : kv_stage + 1;
  }

  if (state != nullptr) {
    float* const to = state + 32 * wave + pi;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        to[(32 * t + 16 * (r >> 3) + 8 * h + (r & 7)) * D] = s[t][r];
  }
}

template <typename T, int D>
void launch(const fa_linear_args& a, hipStream_t stream) {
  const int seqs = a.num_seqs > 0 ? a.num_seqs : 1;  // rows of no sequence are there too
  hipLaunchKernelGGL((linear_kernel<T, D>), dim3(static_cast<unsigned>(seqs * a.h_kv)), dim3(2 * D),
                     0, stream, a, divisor(a.h_kv));
}

}  // namespace
}  // namespace fa

extern "C" int64_t fa_linear_args_size(void) {
  return static_cast<int64_t>(sizeof(fa_linear_args));
}

extern "C" int fa_linear_prompt(const fa_linear_args* args, void* stream) {
  FA_CHECK_ARG(args != nullptr, "args is NULL");
  const fa_linear_args& a = *args;
  const int rc = fa::check_linear(a);
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(static_cast<int64_t>(a.num_seqs) * a.h_kv < 1 << 22, "too many sequences or heads");
  FA_CHECK_ARG(a.total <= INT32_MAX - 256, "too many tokens");
  if (a.total == 0) return FA_OK;
  FA_CHECK_ARG(a.cu_seqlens != nullptr, "cu_seqlens is NULL");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf = a.dtype == 1;
  if (a.d == 64)
    bf ? fa::launch<fa::bf16, 64>(a, s) : fa::launch<_Float16, 64>(a, s);
  else if (a.d == 128)
    bf ? fa::launch<fa::bf16, 128>(a, s) : fa::launch<_Float16, 128>(a, s);
  else
    bf ? fa::launch<fa::bf16, 256>(a, s) : fa::launch<_Float16, 256>(a, s);
  FA_CHECK_HIP(hipGetLastError());
  return FA_OK;
}
