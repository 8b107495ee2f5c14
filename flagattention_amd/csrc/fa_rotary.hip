// Rotary positions for gfx950: q and k turned by the angles of their tokens' positions (of up to four
// axes), into new rows, in place, or k and v into a paged cache.
//
// A thread takes one unit of a token -- kVec pairs, whose two pieces are kVec dims each -- over a few
// heads: it works the sines out once and uses them for each.  The angle of a pair is a product in
// 64 bits, counted in revolutions, whose whole part is taken away there; what is left goes to the
// hardware's sine and cosine (which count revolutions too) in 32.
#include "fa_common.h"
#include "fa_divide.h"
#include "flagattention_amd_linear.h"

namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 4;  // rows that a thread takes at most

struct RotaryPlan {
  Divisor units, chunks;  // units of a row; threads that share a token's rows
  int rows;               // rows of a token: q's heads, k's, and with caches v's
  long long threads;
};

template <typename T, int kVec>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const fa_rotary_args a,
                                                          const RotaryPlan plan) {
  typedef T Vec __attribute__((ext_vector_type(kVec)));
  const long long id = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= plan.threads) return;
  const int of_block = divide(static_cast<int>(id), plan.units);  // below 2^31 (host)
  const int unit = static_cast<int>(id) - of_block * static_cast<int>(plan.units.by);
  const int t = divide(of_block, plan.chunks);
  const int chunk = of_block - t * static_cast<int>(plan.chunks.by);

  // the unit's two pieces of kVec dims
  const int turning = a.pairs / kVec;
  const bool turns = unit < turning;
  int first, second;
  if (turns) {
    first = a.adjacent ? 2 * kVec * unit : kVec * unit;
    second = first + (a.adjacent ? kVec : a.pairs);
  } else {
    first = 2 * a.pairs + 2 * kVec * (unit - turning);
    second = first + kVec;
  }
  const bool both = second < a.d;

  float c[kVec], s[kVec];
  if (turns) {
#pragma unroll
    for (int x = 0; x < kVec; ++x) {
      const int i = kVec * unit + x;
      int axis = 0;
      if (a.axes > 1) {
        if (a.mixed) {
          const int of = i % a.axes;
          axis = i / a.axes < a.sections[of] ? of : 0;
        } else {
          int end = a.sections[0];
#pragma unroll
          for (int n = 1; n < FA_ROTARY_MAX_AXES; ++n) {
            axis = n < a.axes && i >= end ? n : axis;
            end += a.sections[n];
          }
        }
      }
      const long long at = axis * a.pos_stride_a + t;
      const long long pos = a.pos64 ? static_cast<const long long*>(a.positions)[at]
                                    : static_cast<const int*>(a.positions)[at];
      constexpr double kPerTurn = 0.15915494309189533577;  // 1 / (2 pi)
      const double turn = static_cast<double>(pos) * static_cast<double>(a.inv_freq[i]) * kPerTurn;
      const float part = static_cast<float>(turn - __builtin_rint(turn));
      c[x] = __builtin_amdgcn_cosf(part);
      s[x] = __builtin_amdgcn_sinf(part);
    }
  }

  long long slot = 0, block = 0, row_of = 0;
  bool kept = true;
  if (a.key_cache) {
    slot = a.slots64 ? static_cast<const long long*>(a.slots)[t]
                     : static_cast<const int*>(a.slots)[t];
    kept = slot >= 0 && slot < a.num_blocks * a.block_size;
    block = kept ? slot / a.block_size : 0;
    row_of = kept ? slot - block * a.block_size : 0;
  }
  for (int n = 0; n < kHeads; ++n) {
    const int row = chunk + n * static_cast<int>(plan.chunks.by);
    if (row >= plan.rows) break;
    const T* src;
    T* dst;
    bool turn = turns, write = true;
    if (row < a.h_q) {
      src = static_cast<const T*>(a.q) + t * a.q_stride_t + row * a.q_stride_h;
      dst = static_cast<T*>(a.q_out) + t * a.q_out_stride_t + row * a.q_out_stride_h;
    } else if (row < a.h_q + a.h_kv) {
      const int h = row - a.h_q;
      src = static_cast<const T*>(a.k) + t * a.k_stride_t + h * a.k_stride_h;
      if (a.key_cache) {
        dst = static_cast<T*>(a.key_cache) + block * a.kc_stride_0 + h * a.kc_stride_h +
              row_of * a.kc_stride_t;
        write = kept;
      } else {
        dst = static_cast<T*>(a.k_out) + t * a.k_out_stride_t + h * a.k_out_stride_h;
      }
    } else {
      const int h = row - a.h_q - a.h_kv;
      src = static_cast<const T*>(a.v) + t * a.v_stride_t + h * a.v_stride_h;
      dst = static_cast<T*>(a.value_cache) + block * a.vc_stride_0 + h * a.vc_stride_h +
            row_of * a.vc_stride_t;
      write = kept;
      turn = false;
    }
    if (!write) continue;
    const Vec p = *reinterpret_cast<const Vec*>(src + first);
    Vec q = p;
    if (both) q = *reinterpret_cast<const Vec*>(src + second);
    Vec y = p, z = q;
    if (turn) {
      if (a.adjacent) {
#pragma unroll
        for (int x = 0; x < kVec; ++x) {
          // pair x of the unit is elements 2x, 2x + 1 of its 2 kVec
          const float u = static_cast<float>(2 * x < kVec ? p[(2 * x) % kVec] : q[(2 * x) % kVec]);
          const float w = static_cast<float>(2 * x + 1 < kVec ? p[(2 * x + 1) % kVec]
                                                              : q[(2 * x + 1) % kVec]);
          const T yu = static_cast<T>(u * c[x] - w * s[x]), yw = static_cast<T>(w * c[x] + u * s[x]);
          if (2 * x < kVec) y[(2 * x) % kVec] = yu; else z[(2 * x) % kVec] = yu;
          if (2 * x + 1 < kVec) y[(2 * x + 1) % kVec] = yw; else z[(2 * x + 1) % kVec] = yw;
        }
      } else {
#pragma unroll
        for (int x = 0; x < kVec; ++x) {
          const float u = static_cast<float>(p[x]), w = static_cast<float>(q[x]);
          y[x] = static_cast<T>(u * c[x] - w * s[x]);
          z[x] = static_cast<T>(w * c[x] + u * s[x]);
        }
      }
    }
    *reinterpret_cast<Vec*>(dst + first) = y;
    if (both) *reinterpret_cast<Vec*>(dst + second) = z;
  }
}

bool rows_of_16(const void* p, int64_t s0, int64_t s1) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s0 % 8 == 0 && s1 % 8 == 0;
}

template <typename T, int kVec>
void launch(const fa_rotary_args& a, hipStream_t stream) {
  RotaryPlan plan;
  // in place the dims that do not turn are there already
  const bool rest = a.key_cache || (a.h_q > 0 ? a.q != a.q_out : a.k != a.k_out);
  const int units = a.pairs / kVec + (rest ? (a.d - 2 * a.pairs + 2 * kVec - 1) / (2 * kVec) : 0);
  plan.rows = a.h_q + a.h_kv * (a.key_cache ? 2 : 1);
  const int chunks = (plan.rows + kHeads - 1) / kHeads;
  plan.units = divisor(units);
  plan.chunks = divisor(chunks);
  plan.threads = static_cast<long long>(units) * chunks * a.tokens;
  hipLaunchKernelGGL((rotary_kernel<T, kVec>),
                     dim3(static_cast<unsigned>((plan.threads + kThreads - 1) / kThreads)),
                     dim3(kThreads), 0, stream, a, plan);
}

}  // namespace
}  // namespace fa

extern "C" int64_t fa_rotary_args_size(void) {
  return static_cast<int64_t>(sizeof(fa_rotary_args));
}

extern "C" int fa_rotary(const fa_rotary_args* args, void* stream) {
  FA_CHECK_ARG(args != nullptr, "args is NULL");
  const fa_rotary_args& a = *args;
  FA_CHECK_ARG(a.tokens >= 0 && a.h_q >= 0 && a.h_kv >= 0 && a.h_q + a.h_kv >= 1 &&
                   a.h_q <= 65535 && a.h_kv <= 65535,
               "tokens %d, heads %d / %d out of range", a.tokens, a.h_q, a.h_kv);
  FA_CHECK_ARG(a.d >= 2 && a.d <= 4096 && a.pairs >= 1 && 2 * a.pairs <= a.d,
               "head dim %d, %d pairs out of range", a.d, a.pairs);
  FA_CHECK_ARG(a.axes >= 1 && a.axes <= FA_ROTARY_MAX_AXES, "%d axes", a.axes);
  FA_CHECK_ARG(a.dtype == 0 || a.dtype == 1, "dtype %d", a.dtype);
  if (a.axes > 1) {
    int64_t sum = 0;
    for (int n = 0; n < a.axes; ++n) {
      FA_CHECK_ARG(a.sections[n] >= 0, "section %d is negative", n);
      sum += a.sections[n];
    }
    FA_CHECK_ARG(sum == a.pairs, "sections sum to %lld, not to %d pairs",
                 static_cast<long long>(sum), a.pairs);
  }
  FA_CHECK_ARG(a.tokens == 0 || (a.positions && a.inv_freq), "NULL pointer");
  FA_CHECK_ARG(a.tokens == 0 || a.h_q == 0 || (a.q && a.q_out), "NULL pointer");
  const bool cache = a.key_cache != nullptr;
  if (cache) {
    FA_CHECK_ARG(a.value_cache && a.slots && (a.tokens == 0 || a.h_kv == 0 || (a.k && a.v)),
                 "NULL pointer");
    FA_CHECK_ARG(a.num_blocks >= 1 && a.num_blocks <= INT32_MAX && a.block_size >= 1,
                 "the cache has no blocks or too many");
  } else {
    FA_CHECK_ARG(a.tokens == 0 || a.h_kv == 0 || (a.k && a.k_out), "NULL pointer");
    FA_CHECK_ARG(a.h_q == 0 || a.h_kv == 0 || (a.q == a.q_out) == (a.k == a.k_out),
                 "q and k have to be turned in place both or neither");
  }
  if (a.tokens == 0) return FA_OK;
  // a thread per unit and heads: ids of 31 bits
  FA_CHECK_ARG(static_cast<int64_t>(a.tokens) * (a.h_q + 2 * a.h_kv) * a.d < int64_t{1} << 40 &&
                   static_cast<int64_t>(a.tokens) * ((a.h_q + 2 * a.h_kv + fa::kHeads - 1) / fa::kHeads) *
                           (a.d / 2 + 1) < INT32_MAX - fa::kThreads,
               "too many tokens or heads");
  bool wide = a.pairs % 8 == 0 && a.d % 8 == 0;
  if (a.h_q > 0)
    wide = wide && fa::rows_of_16(a.q, a.q_stride_t, a.q_stride_h) &&
           fa::rows_of_16(a.q_out, a.q_out_stride_t, a.q_out_stride_h);
  if (a.h_kv > 0) wide = wide && fa::rows_of_16(a.k, a.k_stride_t, a.k_stride_h);
  if (a.h_kv > 0 && cache)
    wide = wide && fa::rows_of_16(a.v, a.v_stride_t, a.v_stride_h) &&
           fa::rows_of_16(a.key_cache, a.kc_stride_h, a.kc_stride_t) && a.kc_stride_0 % 8 == 0 &&
           fa::rows_of_16(a.value_cache, a.vc_stride_h, a.vc_stride_t) && a.vc_stride_0 % 8 == 0;
  if (a.h_kv > 0 && !cache)
    wide = wide && fa::rows_of_16(a.k_out, a.k_out_stride_t, a.k_out_stride_h);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.dtype == 1)
    wide ? fa::launch<fa::bf16, 8>(a, s) : fa::launch<fa::bf16, 1>(a, s);
  else
    wide ? fa::launch<_Float16, 8>(a, s) : fa::launch<_Float16, 1>(a, s);
  FA_CHECK_HIP(hipGetLastError());
  return FA_OK;
}
