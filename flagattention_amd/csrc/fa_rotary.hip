// Rotary positions for gfx950: q and k turned by the angles of their tokens' positions (of up to four
// axes), into new rows, in place, or k and v into a paged cache (and k into new rows beside it).
//
// A thread takes one unit of a token -- kVec pairs, whose two pieces are kVec dims each -- over a few
// heads: it works the sines out once and uses them for each.  The angle of a pair is a product in
// 64 bits, counted in revolutions, whose whole part is taken away there; what is left goes to the
// hardware's sine and cosine (which count revolutions too) in 32.
//
// Bound by the rows, read and written once: 16,384 tokens of 64 heads and 8 of k and v, D = 128, into a
// cache 131 us, 20,001 of 16 and 16, D = 256, 125 us, 5.1 and 5.3 TB/s (a large copy: 5.1); 8,192 of 32
// and 8 35 to 39 us, 4.8 to 4.3.  A few tokens take 3 to 4.4 us, the launch and two trips to memory.  The
// turned k beside the cache is k's rows once more (16,384 tokens of 64 heads and 8: 129 us without it, 135
// with it, 244 by two calls).
#include <algorithm>

#include "fa_common.h"
#include "fa_divide.h"
#include "flagattention_amd_linear.h"

namespace fa {
namespace {

constexpr int kThreads = 256;

struct RotaryPlan {
  Divisor units, chunks;  // units of a row; threads that share a token's rows
  Divisor axes, block;    // block: where a slot fits 31 bits
  bool small_slots;
  int rows;               // rows of a token: q's heads, k's, with caches v's, and k's for k_out
  int threads;
};

template <typename T, int kVec, int kHeads, bool kAdjacent>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const fa_rotary_args a,
                                                          const RotaryPlan plan) {
  typedef T Vec __attribute__((ext_vector_type(kVec)));
  const int id = blockIdx.x * kThreads + threadIdx.x;  // below 2^31 (host)
  if (id >= plan.threads) return;
  const int of_block = divide(id, plan.units);
  const int unit = id - of_block * static_cast<int>(plan.units.by);
  const int t = divide(of_block, plan.chunks);
  const int chunk = of_block - t * static_cast<int>(plan.chunks.by);

  // the unit's two pieces of kVec dims
  const int turning = a.pairs / kVec;
  const bool turns = unit < turning;
  int first, second;
  if (turns) {
    first = kAdjacent ? 2 * kVec * unit : kVec * unit;
    second = first + (kAdjacent ? kVec : a.pairs);
  } else {
    first = 2 * a.pairs + 2 * kVec * (unit - turning);
    second = first + kVec;
  }
  const bool both = second < a.d;

  // where the rows come from and go to; every load is on its way before the first is used
  const T* src[kHeads];
  T* dst[kHeads];
  bool turn[kHeads], write[kHeads];
  long long k_at = 0, v_at = 0;
  bool kept = true;
  if (a.key_cache) {
    const long long slot = a.slots64 ? static_cast<const long long*>(a.slots)[t]
                                     : static_cast<const int*>(a.slots)[t];
    kept = slot >= 0 && slot < a.num_blocks * a.block_size;
    const long long block = !kept ? 0 : plan.small_slots ? divide(static_cast<int>(slot), plan.block)
                                                         : slot / a.block_size;
    const long long row = kept ? slot - block * a.block_size : 0;
    k_at = block * a.kc_stride_0 + row * a.kc_stride_t;
    v_at = block * a.vc_stride_0 + row * a.vc_stride_t;
  }
#pragma unroll
  for (int n = 0; n < kHeads; ++n) {
    const int row = chunk + n * static_cast<int>(plan.chunks.by);
    write[n] = row < plan.rows;
    turn[n] = turns;
    if (row < a.h_q) {
      src[n] = static_cast<const T*>(a.q) + t * a.q_stride_t + row * a.q_stride_h;
      dst[n] = static_cast<T*>(a.q_out) + t * a.q_out_stride_t + row * a.q_out_stride_h;
    } else if (row < a.h_q + a.h_kv) {
      const int h = row - a.h_q;
      src[n] = static_cast<const T*>(a.k) + t * a.k_stride_t + h * a.k_stride_h;
      if (a.key_cache) {
        dst[n] = static_cast<T*>(a.key_cache) + k_at + h * a.kc_stride_h;
        write[n] = kept;
      } else {
        dst[n] = static_cast<T*>(a.k_out) + t * a.k_out_stride_t + h * a.k_out_stride_h;
      }
    } else if (row >= a.h_q + 2 * a.h_kv) {
      const int h = row - a.h_q - 2 * a.h_kv;
      src[n] = static_cast<const T*>(a.k) + t * a.k_stride_t + h * a.k_stride_h;
      dst[n] = static_cast<T*>(a.k_out) + t * a.k_out_stride_t + h * a.k_out_stride_h;
    } else {
      const int h = row - a.h_q - a.h_kv;
      src[n] = static_cast<const T*>(a.v) + t * a.v_stride_t + h * a.v_stride_h;
      dst[n] = static_cast<T*>(a.value_cache) + v_at + h * a.vc_stride_h;
      write[n] = write[n] && kept;
      turn[n] = false;
    }
  }
  Vec p[kHeads], q[kHeads];
#pragma unroll
  for (int n = 0; n < kHeads; ++n) {
    if (!write[n]) continue;
    p[n] = *reinterpret_cast<const Vec*>(src[n] + first);
    if (both) q[n] = *reinterpret_cast<const Vec*>(src[n] + second);
  }

  float c[kVec], s[kVec];
  if (turns) {
    // every axis at once (past the last one, the last one again): one trip to memory
    long long whole[FA_ROTARY_MAX_AXES];
    if (a.pos64) {
#pragma unroll
      for (int n = 0; n < FA_ROTARY_MAX_AXES; ++n)
        whole[n] = static_cast<const long long*>(a.positions)[min(n, a.axes - 1) * a.pos_stride_a + t];
    } else {
#pragma unroll
      for (int n = 0; n < FA_ROTARY_MAX_AXES; ++n)
        whole[n] = static_cast<const int*>(a.positions)[min(n, a.axes - 1) * a.pos_stride_a + t];
    }
    double at[FA_ROTARY_MAX_AXES];
#pragma unroll
    for (int n = 0; n < FA_ROTARY_MAX_AXES; ++n) at[n] = static_cast<double>(whole[n]);
    // mixed: pair i is number `round` of axis `of`
    int round = 0, of = 0;
    if (a.mixed) {
      round = divide(kVec * unit, plan.axes);
      of = kVec * unit - round * a.axes;
    }
#pragma unroll
    for (int x = 0; x < kVec; ++x) {
      const int i = kVec * unit + x;
      double pos = at[0];
      if (a.axes > 1) {
        int end = a.sections[0];
#pragma unroll
        for (int n = 1; n < FA_ROTARY_MAX_AXES; ++n) {
          if (n >= a.axes) break;
          const bool takes = a.mixed ? of == n && round < a.sections[n] : i >= end;
          pos = takes ? at[n] : pos;
          end += a.sections[n];
        }
        if (a.mixed && ++of == a.axes) {
          of = 0;
          ++round;
        }
      }
      constexpr double kPerTurn = 0.15915494309189533577;  // 1 / (2 pi)
      const double turned = pos * static_cast<double>(a.inv_freq[i]) * kPerTurn;
      const float part = static_cast<float>(turned - __builtin_rint(turned));
      c[x] = __builtin_amdgcn_cosf(part);
      s[x] = __builtin_amdgcn_sinf(part);
    }
  }

#pragma unroll
  for (int n = 0; n < kHeads; ++n) {
    if (!write[n]) continue;
    Vec y = p[n], z = q[n];
    if (turn[n]) {
#pragma unroll
      for (int x = 0; x < kVec; ++x) {
        // pair x of adjacent ones is elements 2x and 2x + 1 of the unit's 2 kVec
        constexpr auto lower = [](int e) { return e < kVec; };
        const int e = 2 * x;
        const float u = static_cast<float>(!kAdjacent ? p[n][x] : lower(e) ? p[n][e % kVec]
                                                                            : q[n][e % kVec]);
        const float w = static_cast<float>(!kAdjacent      ? q[n][x]
                                           : lower(e + 1) ? p[n][(e + 1) % kVec]
                                                          : q[n][(e + 1) % kVec]);
        const T yu = static_cast<T>(u * c[x] - w * s[x]), yw = static_cast<T>(w * c[x] + u * s[x]);
        if (!kAdjacent) {
          y[x] = yu;
          z[x] = yw;
        } else {
          if (lower(e)) y[e % kVec] = yu; else z[e % kVec] = yu;
          if (lower(e + 1)) y[(e + 1) % kVec] = yw; else z[(e + 1) % kVec] = yw;
        }
      }
    }
    *reinterpret_cast<Vec*>(dst[n] + first) = y;
    if (both) *reinterpret_cast<Vec*>(dst[n] + second) = z;
  }
}

bool rows_of_16(const void* p, int64_t s0, int64_t s1) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s0 % 8 == 0 && s1 % 8 == 0;
}

int rows_of(const fa_rotary_args& a) {
  return a.h_q + a.h_kv * (!a.key_cache ? 1 : a.k_out ? 3 : 2);
}

// Rows of a thread: one while the launch leaves the card idle, four to share the sines then.  A thread's
// rows come one after the other (three of 10 heads, D = 64: 4.8 us with four, 3.0 with one).
constexpr int kFewThreads = 1 << 18;

template <typename T, int kVec, int kHeads, bool kAdjacent>
void launch_kernel(const fa_rotary_args& a, RotaryPlan plan, hipStream_t stream) {
  const int chunks = cdiv(plan.rows, kHeads);
  plan.chunks = divisor(chunks);
  plan.threads = static_cast<int>(plan.units.by) * chunks * a.tokens;
  hipLaunchKernelGGL((rotary_kernel<T, kVec, kHeads, kAdjacent>),
                     dim3(static_cast<unsigned>(cdiv(plan.threads, kThreads))), dim3(kThreads), 0,
                     stream, a, plan);
}

template <typename T, int kVec>
void launch(const fa_rotary_args& a, hipStream_t stream) {
  RotaryPlan plan;
  // in place the dims that do not turn are there already
  const bool rest = a.key_cache || (a.h_q > 0 ? a.q != a.q_out : a.k != a.k_out);
  const int units = a.pairs / kVec + (rest ? cdiv(a.d - 2 * a.pairs, 2 * kVec) : 0);
  plan.rows = rows_of(a);
  plan.units = divisor(units);
  plan.axes = divisor(a.axes);
  plan.small_slots = a.key_cache && a.num_blocks * a.block_size <= INT32_MAX;
  plan.block = divisor(plan.small_slots ? a.block_size : 1);
  const bool few = static_cast<int64_t>(units) * plan.rows * a.tokens <= kFewThreads;
  if (a.adjacent)
    few ? launch_kernel<T, kVec, 1, true>(a, plan, stream)
        : launch_kernel<T, kVec, 4, true>(a, plan, stream);
  else
    few ? launch_kernel<T, kVec, 1, false>(a, plan, stream)
        : launch_kernel<T, kVec, 4, false>(a, plan, stream);
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
    FA_CHECK_ARG(!a.k_out || a.k_out != a.k, "k is read for the cache while it is turned in place");
  } else {
    FA_CHECK_ARG(a.tokens == 0 || a.h_kv == 0 || (a.k && a.k_out), "NULL pointer");
    FA_CHECK_ARG(a.h_q == 0 || a.h_kv == 0 || (a.q == a.q_out) == (a.k == a.k_out),
                 "q and k have to be turned in place both or neither");
  }
  if (a.tokens == 0) return FA_OK;
  // a thread per unit and heads: ids of 31 bits
  const int rows = std::max(fa::rows_of(a), a.h_q + 2 * a.h_kv);
  FA_CHECK_ARG(static_cast<int64_t>(a.tokens) * rows * a.d < int64_t{1} << 40 &&
                   static_cast<int64_t>(a.tokens) * ((rows + 3) / 4) * (a.d / 2 + 1) <
                       INT32_MAX - fa::kThreads,
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
  if (a.h_kv > 0 && a.k_out)
    wide = wide && fa::rows_of_16(a.k_out, a.k_out_stride_t, a.k_out_stride_h);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.dtype == 1)
    wide ? fa::launch<fa::bf16, 8>(a, s) : fa::launch<fa::bf16, 1>(a, s);
  else
    wide ? fa::launch<_Float16, 8>(a, s) : fa::launch<_Float16, 1>(a, s);
  FA_CHECK_HIP(hipGetLastError());
  return FA_OK;
}
