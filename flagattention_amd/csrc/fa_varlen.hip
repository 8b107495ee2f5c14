// Prompt attention over packed sequences for gfx950: fp16 or bf16, head dim 64, 128, 256.
//
// A work-group = 4 waves = 128 query rows of one (sequence, KV head), 32 per wave, which share
// every K/V tile through LDS.  A query row is a (position, query head of the group) pair, positions
// outermost.  Row blocks lie inside one sequence, so the grid is the bound that the host knows --
// every sequence rounds its last block up -- and a work-group finds its sequence from the starts,
// which only the device knows.
//
// Per tile of 64 keys (32 at head dim 256) and wave, all MFMA 32x32x16, fp32 accumulation:
//   S^T[keys, 32 rows] = K Q^T, softmax down the columns (lane % 32 = row), O^T[D, 32 rows] +=
//   V^T P^T with P^T the lane's own scores (the k order only has to agree between the operands).
//
// Two waves per SIMD (three at head dim 64): one's softmax fills the other's matrix instructions.
// Long prompts are bound by power: 6 sequences of up to 8,192 tokens, 32 heads of 8 KV heads, D = 128,
// take 712 .. 778 us at 1.94 GHz, 960 .. 1,050 TF (a product of 8,192^3 reaches 1,253), both pipes busy
// for 52% of the cycles.  16 of up to 2,048 take 170 .. 189 us, 725 .. 805 TF, at 2.1 GHz: 3,400 work-groups of ten tiles on
// average with their starts and ends.  64 rows per wave would halve the reads of LDS, but spill
// (830 TF where these reach 1,045); a step whose QK runs beside the last one's softmax took 5%
// fewer cycles and the same time.
#include <algorithm>

#include "fa_common.h"
#include "fa_divide.h"
#include "fa_merge.h"
#include "fa_rows_tile.h"
#include "fa_wave.h"
#include "flagattention_amd_packed.h"

namespace fa {
namespace {

constexpr int kLWaves = 4;
constexpr int kLThreads = 64 * kLWaves;
constexpr int kLWaveRows = 32;
constexpr int kLRows = kLWaves * kLWaveRows;
// Past this reference (log2 units) the scores are scaled in a pass of their own: a fused
// multiply-add does not round their product with the scale, which the reference is made of.
constexpr float kFusedMax = 1024.f;
// P is relative to a reference per row, which moves where the row's maximum is more than kLag (log2
// units) past its last place; in bf16 it then goes kAbove over the maximum, so that P reaches
// 2^(kLag - kAbove) at most.  The sums of 2^10 keys of such a weight and the largest finite V stay
// within fp32, those of 2^16 of equal weights (a reference at the maximum made an infinity of a single
// such V whose weight was past 1).  P ends at 2^-126, so weights below 2^-110 of the largest are 0.
// fp16 keeps 0: its P would lose bits below 2^-14, and its V is below 2^16.
//
// Between moves the accumulators are left alone, but the largest P is then no power of two, whose
// rounding to 16 bits would cost nothing.  Following every new maximum instead (kLag = 0): bf16 error
// against 64 bits at 300 / 512 / 2,048 / 6,144 keys 2.07 / 2.10 / 2.10 / 2.20e-3 where this has 2.17 /
// 2.20 / 2.29 / 2.33e-3, fp16 2.58 .. 2.75e-4 where this has 2.71 .. 2.91e-4; 6 x 8,192 tokens take 763
// instead of 733 us, 16 x 2,048 179 instead of 170, unmasked ones at head dim 256 120 instead of 110.5.
// kLag = 2: 2.14 .. 2.28e-3, 743, 174 and 116 us.  Blocks of few rows, bound by bytes, follow (kFollow).
constexpr float kLag = 6.f;
template <typename T>
constexpr float kAbove = __is_same(T, __bf16) ? 16.f : 0.f;
constexpr int kCus = 256;  // the order of work-groups counts on these
// Keys past which a row block of one wave's rows has them dealt out to the waves: 32 each.
constexpr int kFewKeys = 128;

// Largest |x| of packed 16-bit values as unsigned bit patterns, folded into best.
__device__ inline void fold_bits(unsigned int& best, uintx4 w) {
  typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    best = __builtin_bit_cast(
        unsigned int, __builtin_elementwise_max(__builtin_bit_cast(ushortx2, best),
                                                __builtin_bit_cast(ushortx2, w[i] & 0x7FFF7FFFu)));
}

// What a launch works out once for its work-groups.
struct Plan {
  Divisor group, h_kv;
  int shift;  // log2 of about a row block's positions
  int round;  // items that start at once, if they are ordered by their cost, else 0
};

struct Item {
  int q0, m;     // first packed position, positions of the sequence
  int k0, n;     // first packed key, keys
  int block;     // row block, -1: none left
};

__device__ inline int clip(int x, int hi) { return min(max(x, 0), hi); }

// One lane's sequence: lanes go through the sequences, the rows behind the last one and those
// before the first (two more, without keys).
struct Seq {
  int q0, m, k0, n;
};
__device__ inline Seq seq_of(const fa_varlen_args& a, int s) {
  // every lane loads, so that all of it is one trip to memory
  const int first = s <= a.num_seqs ? s : 0, next = min(first + 1, a.num_seqs);
  const int q0 = clip(a.cu_seqlens_q[first], a.total_q), q1 = clip(a.cu_seqlens_q[next], a.total_q);
  const int k0 = clip(a.cu_seqlens_k[first], a.total_k), k1 = clip(a.cu_seqlens_k[next], a.total_k);
  if (s < a.num_seqs) return Seq{q0, max(q1 - q0, 0), k0, max(k1 - k0, 0)};
  if (s == a.num_seqs) return Seq{q0, a.total_q - q0, 0, 0};
  return Seq{0, s == a.num_seqs + 1 ? q0 : 0, 0, 0};
}
__device__ inline Item item_of(const Seq& x, int l, int block) {
  Item it;
  it.q0 = __builtin_amdgcn_readlane(x.q0, l);
  it.m = __builtin_amdgcn_readlane(x.m, l);
  it.k0 = __builtin_amdgcn_readlane(x.k0, l);
  it.n = __builtin_amdgcn_readlane(x.n, l);
  it.block = block;
  return it;
}

// Inclusive prefix maximum over the lanes (non-negative values), as wave_incl_scan.
__device__ inline int wave_incl_max(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false));  // row_shr:1
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false));  // row_shr:2
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false));  // row_shr:4
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false));  // row_shr:8
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false));  // row_bcast:15
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false));  // row_bcast:31
  return x;
}

// The sequence and row block of work item `item`: blocks of the sequences one after the other,
// each one's last (the longest under a causal mask) first.
__device__ inline Item find_in_order(const fa_varlen_args& a, int group, int item) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < a.num_seqs + 2; base += 64) {
    const Seq x = seq_of(a, base + lane);
    const int upto = wave_incl_scan(cdiv(x.m * group, kLRows));
    const unsigned long long past = __ballot(upto > item);
    if (past != 0ull) {
      const int l = __builtin_ctzll(past);
      return item_of(x, l, __builtin_amdgcn_readlane(upto, l) - 1 - item);
    }
    item -= __builtin_amdgcn_readlane(upto, 63);
  }
  return Item{0, 0, 0, 0, -1};
}

// The same with the items ordered by the keys that they walk, the longest first, so that a launch
// of several work-groups per CU ends with short ones (up to 62 sequences, a lane each).  In units
// of about a row block's positions, block j of a causal sequence costs low + j, low from its
// prefix, and a block of a full one low.  How many blocks cost c or more is a sum over the
// sequences; 64 values of c are summed at once, a lane each (the sequences come from LDS, `table`:
// 512 bytes of the wave's own), and the item is among the blocks of the largest with more than `item`.
// By bisection, a sum over the lanes per value, it took 1,000 cycles more at 16 sequences; in order
// it takes 1,700 less.
__device__ inline Item find_by_cost(const fa_varlen_args& a, int group, int item, int shift,
                                    int round, int* table) {
  const int lane = threadIdx.x & 63;
  const Seq x = seq_of(a, lane);
  const int blocks = cdiv(x.m * group, kLRows);
  const bool rises = a.causal && lane < a.num_seqs;
  // (a block of one wave's rows walks its keys four times as fast)
  const int fast = x.m * group <= kLWaveRows && x.n > kFewKeys ? shift + 2 : shift;
  const int low = rises ? (max(x.n - x.m, 0) >> fast) + 1
                        : static_cast<int>((static_cast<unsigned int>(x.n) + (1u << fast) - 1) >> fast);
  const int end = low + (rises ? blocks : 1);  // past the highest cost
  auto costing = [&](int c) -> int {           // this lane's blocks that cost c or more
    return rises ? min(max(end - c, 0), blocks) : low >= c ? blocks : 0;
  };
  table[2 * lane] = end;
  table[2 * lane + 1] = lane < a.num_seqs ? blocks : 0;
  const int all = __builtin_amdgcn_readlane(wave_incl_scan(blocks), 63);
  const int top = __builtin_amdgcn_readlane(wave_incl_max(blocks > 0 ? end : 0), 63);
  if (item >= all) return Item{0, 0, 0, 0, -1};
  // the second round from its far end: a CU's first two work-groups then sum to about the same
  // (2,048 tokens behind 4,096 keys, 512 work-groups: 189 -> 182 us)
  if (item >= round && item < 2 * round) item = round + min(2 * round, all) - 1 - item;
  // costs in at most 64 steps: a step's blocks go in any order
  const int stride = cdiv(top, 64);
  const int c = (lane + 1) * stride;
  int sum = 0;
  for (int s = 0; s < a.num_seqs; s += 4) {  // lanes past the last sequence hold no block
    const int4 p = *reinterpret_cast<const int4*>(table + 2 * s);
    const int4 q = *reinterpret_cast<const int4*>(table + 2 * s + 4);
    if (a.causal) {
      sum += min(max(p.x - c, 0), p.y) + min(max(p.z - c, 0), p.w);
      sum += min(max(q.x - c, 0), q.y) + min(max(q.z - c, 0), q.w);
    } else {
      sum += (p.x > c ? p.y : 0) + (p.z > c ? p.w : 0) + (q.x > c ? q.y : 0) + (q.z > c ? q.w : 0);
    }
  }
  const int k = __builtin_popcountll(__ballot(sum > item));  // sums fall with c
  const int lo = k * stride;                                 // the item costs lo .. lo + stride - 1
  const int rank = item - (k < 64 ? __builtin_amdgcn_readlane(sum, k) : 0);
  const int here = costing(lo) - costing(lo + stride);
  const int upto = wave_incl_scan(here);
  const int l = __builtin_ctzll(__ballot(upto > rank));
  const int before = __builtin_amdgcn_readlane(upto - here, l);
  const int from = __builtin_amdgcn_readlane(low, l);
  const bool up = __builtin_amdgcn_readlane(static_cast<int>(rises), l) != 0;
  return item_of(x, l, (up ? max(lo - from, 0) : 0) + rank - before);
}

// One 32-row tile's softmax state and operands (lane % 32 = row, g = lane / 32).
template <typename T, int D>
struct RowState {
  typedef typename PVec<T>::v8 T8;
  T8 qf[D / 16];         // Q^T operand: dims 16kk + 8g..+7
  floatx16 acc[D / 32];  // O^T: dim 32dt + 8(i / 4) + 4g + i % 4
  float mref, lsum;      // reference and sum of the weights, base 2
};

// The lane's parts of the LDS reads.
template <int D>
struct LaneReads {
  static constexpr int C = D / 8;
  static constexpr int kRowB = 2 * D;
  static constexpr int kVBases = D / 32 < 4 ? D / 32 : 4;  // fv < 8: dt + 4 is 256 bytes on
  int k;
  int v[kVBases];
  __device__ inline explicit LaneReads(int lane) {
    const int g = lane >> 5, c32 = lane & 31;
    k = c32 * kRowB + 16 * (g ^ fk<C>(c32));  // chunk 2kk + g: xor 32 kk
    const int h16 = lane >> 4, e = (lane & 15) >> 2, qd = lane & 3;
    const int vtok = 4 * g + e;  // token within 8
#pragma unroll
    for (int dt = 0; dt < kVBases; ++dt)
      v[dt] = vtok * kRowB + 32 * ((2 * dt + (h16 & 1)) ^ fv<C>(vtok)) + 16 * (qd >> 1) +
              8 * (qd & 1);
  }
};

// Weights of 32 kSub keys at kb for the 32 rows: scores, mask, running maximum, exponentials.  A
// masked tile's first `sees` keys (from the lane's own, 4g) are seen by the lane's row.
template <typename T, int D, int kSub, bool kFollow>
__device__ inline void weigh(RowState<T, D>& r, const unsigned char* kb, const LaneReads<D>& at,
                             bool masked, int sees, bool prescale, float prescale_by,
                             float scale_log2, typename PVec<T>::v8 (&pb)[2 * kSub]) {
  typedef typename PVec<T>::v8 T8;
  constexpr int kKSteps = D / 16;
  const float ninf = -__builtin_inff();
  // K operands one k-step ahead of their MFMAs (the fences keep them there)
  floatx16 s[kSub];
  T8 ka[2][kSub];
  auto k_read = [&](int kk, int tt) -> T8 {
    return *reinterpret_cast<const T8*>(kb + 32 * tt * 2 * D + (at.k ^ (32 * kk)));
  };
#pragma unroll
  for (int tt = 0; tt < kSub; ++tt) {
    s[tt] = floatx16{};
    ka[0][tt] = k_read(0, tt);
  }
#pragma unroll
  for (int kk = 0; kk < kKSteps; ++kk) {
    if (kk + 1 < kKSteps) {
#pragma unroll
      for (int tt = 0; tt < kSub; ++tt) ka[(kk + 1) & 1][tt] = k_read(kk + 1, tt);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int tt = 0; tt < kSub; ++tt) s[tt] = mfma_32x32x16(ka[kk & 1][tt], r.qf[kk], s[tt]);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (prescale) {
#pragma unroll
    for (int tt = 0; tt < kSub; ++tt)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[tt][i] *= prescale_by;
  }
  if (masked) {
#pragma unroll
    for (int tt = 0; tt < kSub; ++tt)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = 32 * tt + 8 * (i >> 2) + (i & 3);  // + 4g: the key of s[tt][i]
        s[tt][i] = j < sees ? s[tt][i] : ninf;
      }
  }
  float mx = s[0][0];
#pragma unroll
  for (int tt = 0; tt < kSub; ++tt)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[tt][i]);
  mx = max_xor32(mx) * scale_log2;
  // only the rows that are up move: a row's result does not depend on those beside it
  const bool up = mx > r.mref + ((kFollow ? 0.f : kLag) - kAbove<T>);
  if (__ballot(up) != 0ull) {  // uniform
    const float m_new = up ? mx + kAbove<T> : r.mref;
    const float alpha = up ? __builtin_amdgcn_exp2f(r.mref - m_new) : 1.f;
    r.lsum *= alpha;
    r.mref = m_new;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) r.acc[dt][i] *= alpha;
  }
  const float nm = r.mref == ninf ? 0.f : -r.mref;
  float c = scale_log2;
  const bool far = fabsf(nm) > kFusedMax;
  if (__ballot(far) != 0ull) {  // uniform
    const float by = far ? c : 1.f;
#pragma unroll
    for (int tt = 0; tt < kSub; ++tt)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[tt][i] *= by;
    c = far ? 1.f : c;
  }
  float ps = 0.f;
#pragma unroll
  for (int ss = 0; ss < 2 * kSub; ++ss)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ss >> 1][8 * (ss & 1) + i], c, nm));
      ps += p;
      pb[ss][i] = static_cast<T>(p);
    }
  r.lsum += ps;
}

// acc += V^T P^T of the 32 kSub keys at vb.
template <typename T, int D, int kSub>
__device__ inline void add_values(RowState<T, D>& r, const unsigned char* vb,
                                  const LaneReads<D>& at,
                                  const typename PVec<T>::v8 (&pb)[2 * kSub]) {
  typedef typename PVec<T>::v8 T8;
  typedef typename PVec<T>::v4 T4;
  constexpr int kRowB = 2 * D;
#pragma unroll
  for (int ss = 0; ss < 2 * kSub; ++ss)
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      const unsigned char* const p = vb + 16 * ss * kRowB + 256 * (dt >> 2) + at.v[dt & 3];
      const T4 lo = lds_tr_read4<T>(p);
      const T4 hi = lds_tr_read4<T>(p + 8 * kRowB);
      const T8 va = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      r.acc[dt] = mfma_32x32x16(va, pb[ss], r.acc[dt]);
    }
}

// Infinities and NaNs of the keys at vb go to the rows that see their key as they are.
template <typename T, int D>
__device__ inline void add_odd_values(RowState<T, D>& r, const unsigned char* vb, int g, int keys,
                                      int sees) {
  typedef typename PVec<T>::v4 T4;
  for (int j = 0; j < keys; ++j) {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // dims 32dt + 8i + 4g..+3: chunk 4dt + i
        const T4 v4 = *reinterpret_cast<const T4*>(
            vb + j * 2 * D + 16 * ((4 * dt + i) ^ (fv<D / 8>(j) << 1)) + 8 * g);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float f = static_cast<float>(v4[x]);
          r.acc[dt][4 * i + x] += j < sees && !(fabsf(f) < __builtin_inff()) ? f : 0.f;
        }
      }
  }
}

// Whether a lane's part of a copy (16 bytes) holds an infinity or a NaN: the largest bit pattern.
template <typename T>
__device__ inline bool is_odd(unsigned int best) {
  constexpr unsigned int kInf = __is_same(T, __bf16) ? 0x7F80u : 0x7C00u;
  return (best & 0xFFFFu) >= kInf || (best >> 16) >= kInf;
}
template <typename T>
__device__ inline void clean16(unsigned char* at) {
  typedef typename PVec<T>::v8 T8;
  T8* const p = reinterpret_cast<T8*>(at);
  T8 w = *p;
#pragma unroll
  for (int x = 0; x < 8; ++x)
    w[x] = fabsf(static_cast<float>(w[x])) < __builtin_inff() ? w[x] : static_cast<T>(0.f);
  *p = w;
}

// Copies of 32 rows of K (or V) from position `start` on into dst; rows past t1 repeat the last one.
template <int D, bool kValues>
__device__ inline void copy32(const unsigned char* base, unsigned int row_b, int start, int t1,
                              unsigned char* dst) {
  constexpr int C = D / 8, kRowsPerCopy = 512 / D;
  int lane = threadIdx.x & 63;
  if (D == 256) asm volatile("" : "+v"(lane));  // offsets afresh: kept, they would be spilled
  const int crow = lane / C, cslot = lane % C;
  const unsigned char* const src = base + static_cast<long long>(start) * row_b;
  const int last = t1 - 1 - start;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const int r = i * kRowsPerCopy + crow;
    const int from = last < 31 ? min(r, last) : r;
    const unsigned int off = from * row_b + 16 * (cslot ^ (kValues ? fv<C>(r) << 1 : fk<C>(r)));
    lds_dma16_off(src, off, (FA_LDS void*)(dst + 1024 * i));
  }
}

// Nothing the compiler moves passes here.
__device__ inline void fence() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// A row block of at most 32 rows (a batch's single tokens, the ends of prompts): its rows are every
// wave's, and the keys are dealt out, 32 at a time and round-robin, each wave's through its own
// quarter of the tile buffers without a barrier.  The next tile's K is on its way from the end of
// this one's scores, its V from the end of its values; at head dim 256 the quarter holds one of them
// at a time.  The wave's first copies are on their way already: K, and V where both fit.  Bound by
// the keys' bytes: 32 single tokens over up to 7,218 keys (head dim 64, 8 KV heads, 190 MB) 98 us with
// one wave at work on every tile of 64, 57 so, 43 with four work-groups per CU.
template <typename T, int D>
__device__ inline void walk_few(RowState<T, D>& r, const LaneReads<D>& at, unsigned char* mine,
                                const unsigned char* kp, unsigned int k_tb,
                                const unsigned char* vp, unsigned int v_tb, int first, int t1,
                                int end, int min_lim, int lim, bool prescale, float prescale_by,
                                float scale_log2) {
  constexpr int kCopies = D / 16;
  constexpr bool kBoth = D <= 128;
  const int lane = threadIdx.x & 63;
  unsigned char* const vb = mine + (kBoth ? 64 * D : 0);
  for (int start = first; start < end; start += 32 * kLWaves) {
    const int next = start + 32 * kLWaves;
    wait_vmem<kBoth ? kCopies : 0>();  // K
    fence();
    typename PVec<T>::v8 pb[2];
    weigh<T, D, 1, true>(r, mine, at, start + 32 > min_lim, lim - start - 4 * (lane >> 5), prescale,
                   prescale_by, scale_log2, pb);
    fence();
    wait_lds();  // K is read
    if (!kBoth) copy32<D, true>(vp, v_tb, start, t1, vb);
    if (kBoth && next < end) {
      copy32<D, false>(kp, k_tb, next, t1, mine);
      wait_vmem<kCopies>();  // V
    } else {
      wait_vmem<0>();
    }
    fence();
    if (start + 32 > min_lim) {  // as in the kernel, a wave's own
      unsigned int best = 0u;
#pragma unroll
      for (int i = 0; i < kCopies; ++i)
        fold_bits(best, *reinterpret_cast<const uintx4*>(vb + 1024 * i + 16 * lane));
      if (__ballot(is_odd<T>(best)) != 0ull) {
        add_odd_values<T, D>(r, vb, lane >> 5, 32, lim - start);
        fence();
#pragma unroll
        for (int i = 0; i < kCopies; ++i) clean16<T>(vb + 1024 * i + 16 * lane);
        fence();
        wait_lds();
      }
    }
    add_values<T, D, 1>(r, vb, at, pb);
    fence();
    wait_lds();  // V is read
    if (next < end) {
      if (kBoth)
        copy32<D, true>(vp, v_tb, next, t1, vb);
      else
        copy32<D, false>(kp, k_tb, next, t1, mine);
    }
  }
}

template <typename T, int D>
__global__ __launch_bounds__(kLThreads, 2) void varlen_kernel(const fa_varlen_args a,
                                                             const Plan plan) {
  typedef typename PVec<T>::v8 T8;
  typedef typename PVec<T>::v4 T4;
  constexpr int C = D / 8;
  constexpr int kRowB = 2 * D;
  constexpr int kTok = D <= 128 ? 64 : 32;
  constexpr int kSub = kTok / 32;
  constexpr int kTileB = kTok * kRowB;
  constexpr int kCopies = kTileB / 1024 / kLWaves;
  constexpr int kRowsPerCopy = 1024 / kRowB;
  constexpr int kKSteps = D / 16;
  constexpr int kDimTiles = D / 32;
  static_assert(kCopies * kLWaves * 1024 == kTileB, "whole copies per wave");
  // [K, V][tile parity]
  __shared__ __attribute__((aligned(16))) unsigned char bufs[4 * kTileB];
  __shared__ int odd_v[2][kLWaves];  // [tile parity][wave]: see below
  __shared__ float few_m[kLWaves][32], few_l[kLWaves][32];

  const int group = static_cast<int>(plan.group.by);
  const int item = divide(blockIdx.x, plan.h_kv);
  const int hk = blockIdx.x - item * a.h_kv;
  const Item it = plan.round > 0 ? find_by_cost(a, group, item, plan.shift, plan.round,
                                                reinterpret_cast<int*>(bufs + 512 * wave_id()))
                                 : find_in_order(a, group, item);
  if (it.block < 0) return;  // uniform
  barrier();  // the tables are read: the buffers are free
  const int split = blockIdx.y;
  const int m = it.m;

  const int wave = wave_id();
  const int lane = threadIdx.x & 63;
  const int g = lane >> 5, c32 = lane & 31;

  const int t0 = split * a.split_tokens;
  const int t1 = split + 1 == a.num_splits ? it.n : min(t0 + a.split_tokens, it.n);
  const float ninf = -__builtin_inff();
  // The scale is applied inside the exponent, after the mask and the maximum.  That needs a
  // positive one: otherwise the scores are scaled before either.
  const bool prescale = !(a.scale > 0.f);  // uniform
  const float scale_log2 = prescale ? 1.f : a.scale * kLog2e;

  const unsigned char* const kp = static_cast<const unsigned char*>(a.k) +
                                  2 * (it.k0 * a.k_stride_t + hk * a.k_stride_h);
  const unsigned char* const vp = static_cast<const unsigned char*>(a.v) +
                                  2 * (it.k0 * a.v_stride_t + hk * a.v_stride_h);
  // 32-bit lane offsets inside a tile (host check)
  const unsigned int k_tb = static_cast<unsigned int>(2 * a.k_stride_t);
  const unsigned int v_tb = static_cast<unsigned int>(2 * a.v_stride_t);
  const int crow = lane / C, cslot = lane % C;
  unsigned int koff[kCopies], voff[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    const int r = (kCopies * wave + i) * kRowsPerCopy + crow;
    koff[i] = r * k_tb + 16 * (cslot ^ fk<C>(r));
    voff[i] = r * v_tb + 16 * (cslot ^ (fv<C>(r) << 1));
  }
  auto issue = [&](int u, int buf) {
    const int start = t0 + kTok * u;
    const unsigned char* const ks = kp + static_cast<long long>(start) * k_tb;
    const unsigned char* const vs = vp + static_cast<long long>(start) * v_tb;
    unsigned char* const kd = bufs + buf * kTileB + kCopies * wave * 1024;
    unsigned char* const vd = bufs + (2 + buf) * kTileB + kCopies * wave * 1024;
    if (start + kTok <= t1) {  // uniform
#pragma unroll
      for (int i = 0; i < kCopies; ++i) lds_dma16_off(ks, koff[i], (FA_LDS void*)(kd + 1024 * i));
#pragma unroll
      for (int i = 0; i < kCopies; ++i) lds_dma16_off(vs, voff[i], (FA_LDS void*)(vd + 1024 * i));
    } else {  // rows past the end repeat the last one (masked)
      const int last = t1 - 1 - start;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int r = (kCopies * wave + i) * kRowsPerCopy + crow;
        const unsigned int back = r > last ? r - last : 0;
        lds_dma16_off(ks, koff[i] - back * k_tb, (FA_LDS void*)(kd + 1024 * i));
        lds_dma16_off(vs, voff[i] - back * v_tb, (FA_LDS void*)(vd + 1024 * i));
      }
    }
  };

  const int row0 = it.block * kLRows;
  const int left = min(m * group - row0, kLRows);  // the work-group's rows
  // One wave's rows and several tiles of keys: the keys are dealt out to the waves.
  const bool few = left <= kLWaveRows && t1 - t0 > kFewKeys;  // uniform
  unsigned char* const quarter = bufs + wave * kTileB;
  // the first tile is on its way from here on
  if (few) {
    const int first = t0 + 32 * wave;
    if (first < t1) {
      copy32<D, false>(kp, k_tb, first, t1, quarter);
      if (D <= 128) copy32<D, true>(vp, v_tb, first, t1, quarter + 64 * D);
    }
  } else if (t1 > t0) {
    issue(0, 0);
  }

  // Position and query head of the work-group's row r, counted from its first: rows are few, so a
  // reciprocal and a correction divide them by the group.
  const int pos0 = divide(row0, plan.group), rem0 = row0 - pos0 * group;
  const float group_inv = __builtin_amdgcn_rcpf(static_cast<float>(group));
  auto pos_of = [&](int r) -> int {  // counted from pos0
    const int x = rem0 + r;
    int q = static_cast<int>(static_cast<float>(x) * group_inv);
    q += x - q * group >= group ? 1 : 0;
    q -= x - q * group < 0 ? 1 : 0;
    return q;
  };
  auto head_of = [&](int r, int pos) -> int { return rem0 + r - pos * group; };
  // keys visible to a position: [0, n - m + 1 + position) causal, all otherwise
  const int first_lim = it.n - m + 1 + pos0;
  auto limit_of = [&](int pos) -> int { return a.causal ? min(first_lim + pos, t1) : t1; };
  const int wg_min = limit_of(0);
  const int wg_lim = limit_of(pos_of(left - 1));
  const int ntiles = wg_lim > t0 ? cdiv(wg_lim - t0, kTok) : 0;
  const int wrow0 = few ? 0 : kLWaveRows * wave;
  const int wave_min = limit_of(pos_of(min(wrow0, left - 1)));
  const int wave_max = limit_of(pos_of(min(wrow0 + kLWaveRows, left) - 1));
  const bool wave_on = wrow0 < left;
  const int row = min(wrow0 + c32, left - 1);  // past the end: the last row, not stored
  const int mm = pos_of(row), jj = head_of(row, mm);
  const int lim = limit_of(mm);

  // Q^T operand: row c32, dims 16kk + 8g..+7
  RowState<T, D> r;
  {
    // a uniform base and 32-bit row offsets (host check), as for the output below
    const T* const qbase = static_cast<const T*>(a.q) + (it.q0 + pos0) * a.q_stride_t +
                           hk * group * a.q_stride_h;
    const unsigned int off = mm * static_cast<unsigned int>(a.q_stride_t) +
                             jj * static_cast<unsigned int>(a.q_stride_h) + 8 * g;
#pragma unroll
    for (int kk = 0; kk < kKSteps; ++kk)
      r.qf[kk] = *reinterpret_cast<const T8*>(qbase + off + 16 * kk);
  }

#pragma unroll
  for (int dt = 0; dt < kDimTiles; ++dt) r.acc[dt] = floatx16{};
  r.mref = ninf;
  r.lsum = 0.f;
  const LaneReads<D> at(lane);

  if (few) {  // uniform
    walk_few<T, D>(r, at, quarter, kp, k_tb, vp, v_tb, t0 + 32 * wave, t1, wg_lim, wg_min, lim,
                   prescale, a.scale * kLog2e, scale_log2);
    wait_vmem<0>();  // a first tile that no row sees
    const float l = sum_xor32(r.lsum);
    if (g == 0) {
      few_m[wave][c32] = r.mref;
      few_l[wave][c32] = l;
    }
    barrier();
    auto top_of = [&](int row) -> float {
      return fmaxf(fmaxf(few_m[0][row], few_m[1][row]), fmaxf(few_m[2][row], few_m[3][row]));
    };
    auto part_of = [&](float ref, float top) -> float {
      return ref == top ? 1.f : __builtin_amdgcn_exp2f(ref - top);
    };
    const float mul = part_of(r.mref, top_of(c32));
    // 128 dims at a time: every wave's rows as fp32, 16-byte chunks in another order in each row
    constexpr int kDims = D <= 128 ? D : 128, kChunks = kDims / 4;
    static_assert(kLWaves * 32 * kDims * 4 <= 4 * kTileB, "the rows fit the tile buffers");
    float* const rows = reinterpret_cast<float*>(bufs);
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += kDims) {
      if (d0 > 0) barrier();  // the ones before are read
#pragma unroll
      for (int dt = 0; dt < kDims / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          floatx4 w;
#pragma unroll
          for (int x = 0; x < 4; ++x) w[x] = r.acc[d0 / 32 + dt][4 * i + x] * mul;
          const int chunk = (8 * dt + 2 * i + g) ^ (c32 & (kChunks - 1));
          *reinterpret_cast<floatx4*>(rows + (32 * wave + c32) * kDims + 4 * chunk) = w;
        }
      barrier();
#pragma unroll
      for (int j = 0; j < 32 * kChunks / kLThreads; ++j) {
        const int at_row = (threadIdx.x + kLThreads * j) / kChunks;
        const int at_chunk = (threadIdx.x + kLThreads * j) % kChunks;
        if (at_row >= left) break;
        const float top = top_of(at_row);
        float sum = 0.f;
        floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kLWaves; ++w) {
          sum += few_l[w][at_row] * part_of(few_m[w][at_row], top);
          o += *reinterpret_cast<const floatx4*>(
              rows + (32 * w + at_row) * kDims + 4 * (at_chunk ^ (at_row & (kChunks - 1))));
        }
        const bool some = !(sum == 0.f);  // else no visible key: out 0, lse -inf
        const float inv = some ? 1.f / sum : 0.f;
        const float lse = some ? (top + log2f(sum)) * kLn2 : ninf;
        const int pos = pos_of(at_row), j2 = head_of(at_row, pos);
        const long long orow =
            static_cast<long long>(hk * group + j2) * a.total_q + it.q0 + pos0 + pos;
#pragma unroll
        for (int x = 0; x < 4; ++x) o[x] = some ? o[x] * inv : 0.f;
        const bool heads_row = d0 == 0 && at_chunk == 0;  // one lane per row
        if (a.num_splits > 1) {
          const long long prow = orow * a.num_splits + split;
          if (some) *reinterpret_cast<floatx4*>(a.o_part + prow * D + d0 + 4 * at_chunk) = o;
          if (heads_row) a.lse_part[prow] = lse == lse ? lse : -ninf;
        } else {
          T4 w;
#pragma unroll
          for (int x = 0; x < 4; ++x) w[x] = static_cast<T>(o[x]);
          *reinterpret_cast<T4*>(static_cast<T*>(a.out) + (it.q0 + pos0 + pos) * a.o_stride_t +
                                 (hk * group + j2) * a.o_stride_h + d0 + 4 * at_chunk) = w;
          if (heads_row && a.lse) a.lse[orow] = lse;
        }
      }
    }
    return;
  }

  for (int u = 0; u < ntiles; ++u) {
    // The accumulators as whole registers: without this each of their elements is copied in every
    // step, for its uses behind the loop (6 x 8,192 at head dim 128: 779 -> 744 us).
#pragma unroll
    for (int dt = 0; dt < kDimTiles; ++dt) asm volatile("" : "+v"(r.acc[dt]));
    const int buf = u & 1;
    const int start = t0 + kTok * u;
    wait_vmem<0>();  // this wave's copies of tile u (requested one step ago)
    // A weight of 0 does not hide an infinity or a NaN in V: 0 times either is NaN.  A tile that
    // some row sees in part (or that ends behind the last key) is looked through for them (each wave its own copies).
    const bool part_seen = start + kTok > wg_min;  // uniform
    if (part_seen) {
      unsigned int best = 0u;
#pragma unroll
      for (int i = 0; i < kCopies; ++i)
        fold_bits(best, *reinterpret_cast<const uintx4*>(bufs + (2 + buf) * kTileB +
                                                         (kCopies * wave + i) * 1024 + 16 * lane));
      const bool any = __ballot(is_odd<T>(best)) != 0ull;
      if (lane == 0) odd_v[buf][wave] = any;
    }
    barrier();  // everyone's copies; and everyone is done with tile u-1
    if (u + 1 < ntiles) issue(u + 1, buf ^ 1);
    const bool odd = part_seen && (odd_v[buf][0] | odd_v[buf][1] | odd_v[buf][2] | odd_v[buf][3]) != 0;
    // every wave takes its odd values out of its own copies once all have used them
    auto clean_tile = [&] {
      barrier();
#pragma unroll
      for (int i = 0; i < kCopies; ++i)
        clean16<T>(bufs + (2 + buf) * kTileB + (kCopies * wave + i) * 1024 + 16 * lane);
      barrier();
    };
    if (!wave_on || start >= wave_max) {  // uniform: no row of the wave sees a key here
      if (odd) clean_tile();              // uniform over the work-group
      continue;
    }
    const unsigned char* const kb = bufs + buf * kTileB;
    const unsigned char* const vb = bufs + (2 + buf) * kTileB;

    T8 pb[2 * kSub];
    // masked: some row does not see the whole tile (uniform)
    weigh<T, D, kSub, false>(r, kb, at, start + kTok > wave_min, lim - start - 4 * g, prescale,
                      a.scale * kLog2e, scale_log2, pb);
    if (odd) {
      add_odd_values<T, D>(r, vb, g, kTok, lim - start);
      clean_tile();
    }
    add_values<T, D, kSub>(r, vb, at, pb);
  }
  wait_vmem<0>();  // a first tile that no row sees
  if (!wave_on) return;

  const float l = sum_xor32(r.lsum);
  const bool some = !(l == 0.f);  // else no visible key: out 0, lse -inf (NaN sums stay NaN)
  const float inv = some ? 1.f / l : 0.f;
  const float lse = some ? (r.mref + log2f(l)) * kLn2 : ninf;
  const int h = hk * group + jj;
  const long long orow = static_cast<long long>(h) * a.total_q + it.q0 + pos0 + mm;
  const bool mine = wrow0 + c32 < left;
  if (a.num_splits > 1) {
    if (mine) {
      const long long prow = orow * a.num_splits + split;
      float* const op = a.o_part + prow * D + 4 * g;
#pragma unroll
      for (int dt = 0; dt < kDimTiles; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          floatx4 w;
#pragma unroll
          for (int x = 0; x < 4; ++x) w[x] = r.acc[dt][4 * i + x] * inv;
          if (some) *reinterpret_cast<floatx4*>(op + 32 * dt + 8 * i) = w;
        }
      // the merge takes the largest lse, which a NaN would not be
      if (g == 0) a.lse_part[prow] = lse == lse ? lse : -ninf;
    }
    return;
  }
  if (mine && g == 0 && a.lse) a.lse[orow] = lse;
  // Lanes c32 and c32 + 32 share a row; a swap of halves leaves each with 16 bytes of it in a row
  // (through LDS, whole rows to a store: three prompts of up to 48 tokens 5.38 instead of 5.16 us, 64 of
  // up to 256 37.2 instead of 36.5, longer ones the same).
  T* const orow_p = static_cast<T*>(a.out) + (it.q0 + pos0) * a.o_stride_t +
                    hk * group * a.o_stride_h +
                    (mm * static_cast<unsigned int>(a.o_stride_t) +
                     jj * static_cast<unsigned int>(a.o_stride_h) + 8 * g);
#pragma unroll
  for (int dt = 0; dt < kDimTiles; ++dt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      T4 w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          w[i][x] = static_cast<T>(some ? r.acc[dt][8 * j + 4 * i + x] * inv : 0.f);
      typedef unsigned int uintx2 __attribute__((ext_vector_type(2)));
      const uintx2 lo = __builtin_bit_cast(uintx2, w[0]), hi = __builtin_bit_cast(uintx2, w[1]);
      const auto p = __builtin_amdgcn_permlane32_swap(lo[0], hi[0], false, false);
      const auto q = __builtin_amdgcn_permlane32_swap(lo[1], hi[1], false, false);
      const uintx4 v = {p[0], q[0], p[1], q[1]};
      if (mine) *reinterpret_cast<uintx4*>(orow_p + 32 * dt + 16 * j) = v;
    }
}

// Row blocks per KV head at most: each sequence, and the rows behind the last and before the
// first, rounds up once.
long long row_blocks(const fa_varlen_args* a) {
  return static_cast<long long>(a->total_q) * (a->h_q / a->h_kv) / kLRows + a->num_seqs + 2;
}

template <typename T>
void launch_varlen(const fa_varlen_args* a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(row_blocks(a) * a->h_kv),
                  static_cast<unsigned>(a->num_splits));
  // More work-groups than run at once (2 per CU; 3 at head dim 64): the longest go first.  Under
  // that their order is all the same and finding it costs a little more than finding the next.
  const bool by_cost = a->num_seqs + 2 <= 64 && grid.x * grid.y > (a->d == 64 ? 768u : 512u);
  const int group = a->h_q / a->h_kv;
  const Plan plan{divisor(group), divisor(a->h_kv),
                  31 - __builtin_clz(static_cast<unsigned int>(std::max(kLRows / group, 1))),
                  by_cost ? std::max(kCus / a->h_kv, 1) : 0};
  if (a->d == 64)
    hipLaunchKernelGGL((varlen_kernel<T, 64>), grid, dim3(kLThreads), 0, stream, *a, plan);
  else if (a->d == 128)
    hipLaunchKernelGGL((varlen_kernel<T, 128>), grid, dim3(kLThreads), 0, stream, *a, plan);
  else
    hipLaunchKernelGGL((varlen_kernel<T, 256>), grid, dim3(kLThreads), 0, stream, *a, plan);
}

// Splits along the keys: the cheapest by a model of the launch, in us.  A work-group takes `step`
// for a tile of keys by itself, and `shared` times as many as a CU has (two at least once the grid
// comes near the CUs, for the dispatcher then doubles some up); the merge costs 3.5 and the partial
// rows written and read at 4 TB/s, of which a causal batch leaves some empty.  Measured / model, 8 KV
// heads, group 4, D = 128: 256 tokens behind 8,192 keys in 1 / 2 / 4 / 8 / 12 splits 168 / 96 / 77 /
// 57 / 61 against 170 / 95 / 76 / 56 / 63, 700 tokens 20.9 / 33.4 / 32.2 in 1 / 2 / 4 against 19 / 25 /
// 34 (two splits per CU whatever their rows took 32.3), D = 256, 4 KV heads, 1,200 tokens 57 / 49 / 48 /
// 51 in 1 / 2 / 3 / 4 against 58 / 54 / 48 / 51.  Blocks of few rows are bound by their keys' bytes
// and want four work-groups per CU also where every CU has one: 32 tokens over up to 7,218 keys
// 103 / 82 / 83 / 92 in 1 / 4 / 8 / 16, but 64 over up to 2,000 37 / 41 in 1 / 2.
int choose_splits(const fa_varlen_args* a, int64_t max_q, int64_t max_k, int64_t cus) {
  const int64_t group = a->h_q / a->h_kv;
  const int64_t blocks =
      a->h_kv * std::max<int64_t>({std::min(a->num_seqs, a->total_q),
                                   (a->total_q * group + kLRows - 1) / kLRows, 1});
  const bool few = max_q * group <= kLWaveRows;
  int64_t pick = 1;
  if (blocks < cus) {
    const int keys = a->d == 256 ? 32 : 64;  // of a tile
    const int64_t tiles = (max_k + keys - 1) / keys;
    const double step = few ? (a->d == 64 ? 0.33 : 0.65) : a->d == 64 ? 0.87 : a->d == 128 ? 1.25 : 1.4;
    const double shared = few ? (a->d == 64 ? 0.28 : 0.55) : a->d == 64 ? 0.47 : a->d == 128 ? 0.9 : 0.95;
    const double full = a->causal ? 1 - 0.5 * a->total_q / std::max(a->total_k, a->total_q) : 1;
    const double part = full * a->h_q * a->total_q * a->d * 8.0 / 4e6;
    double best = 0;
    for (int64_t s : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 16, 20, 24, 32, 48, 64, 96, 128}) {
      if (s > 1 && tiles < 2 * s) break;
      const double per_cu = static_cast<double>(blocks * s) / static_cast<double>(cus);
      const double load = few || per_cu <= 0.7 ? per_cu : std::max(per_cu, 2.0);
      const double t = static_cast<double>((tiles + s - 1) / s) * std::max(step, shared * load) +
                       (s > 1 ? 3.5 + 0.06 * s + part * s : 0);
      if (s == 1 || t < best) {
        best = t;
        pick = s;
      }
    }
  }
  if (few) pick = std::max(pick, std::min((4 * cus + blocks - 1) / blocks, max_k / 1024));
  return static_cast<int>(std::min<int64_t>(std::max<int64_t>(pick, 1), 128));
}

bool rows16(const void* p, int64_t s0, int64_t s1) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s0 % 8 == 0 && s1 % 8 == 0;
}

int check_varlen(const fa_varlen_args* a) {
  FA_CHECK_ARG(a != nullptr, "args is NULL");
  FA_CHECK_ARG(a->num_seqs >= 0 && a->total_q >= 1 && a->total_k >= 0,
               "num_seqs %d / total_q %d / total_k %d invalid", a->num_seqs, a->total_q, a->total_k);
  // positions of the tile after the last one stay in 32 bits
  FA_CHECK_ARG(a->total_k <= INT32_MAX - 256, "total_k %d is more than 2^31 - 257", a->total_k);
  FA_CHECK_ARG(a->h_q >= 1 && a->h_kv >= 1 && a->h_q % a->h_kv == 0,
               "h_q %d is not a multiple of h_kv %d", a->h_q, a->h_kv);
  FA_CHECK_ARG(a->d == 64 || a->d == 128 || a->d == 256, "head dim %d not in {64, 128, 256}", a->d);
  FA_CHECK_ARG(a->dtype == 0 || a->dtype == 1, "dtype %d is not 0 (fp16) or 1 (bf16)", a->dtype);
  FA_CHECK_ARG(a->q && a->out && a->cu_seqlens_q && a->cu_seqlens_k &&
                   (a->total_k == 0 || (a->k && a->v)),
               "NULL q / k / v / out / cu_seqlens");
  FA_CHECK_ARG(rows16(a->q, a->q_stride_t, a->q_stride_h) &&
                   rows16(a->k, a->k_stride_t, a->k_stride_h) &&
                   rows16(a->v, a->v_stride_t, a->v_stride_h) &&
                   rows16(a->out, a->o_stride_t, a->o_stride_h),
               "q / k / v / out rows must be 16-byte aligned");
  // 32-bit lane offsets inside a tile
  FA_CHECK_ARG(a->k_stride_t >= 0 && a->v_stride_t >= 0 && a->k_stride_t < (1ll << 23) &&
                   a->v_stride_t < (1ll << 23),
               "k / v token strides must be in [0, 2^23)");
  // and inside a row block
  const long long group = a->h_q / a->h_kv;
  FA_CHECK_ARG(a->q_stride_t >= 0 && a->o_stride_t >= 0 && a->q_stride_t < (1ll << 23) &&
                   a->o_stride_t < (1ll << 23) && a->q_stride_h >= 0 && a->o_stride_h >= 0 &&
                   group * a->q_stride_h < (1ll << 29) && group * a->o_stride_h < (1ll << 29),
               "q / out token strides must be in [0, 2^23), a group's heads within 2^29 elements");
  // every work-group goes through the starts, and each sequence may have one
  FA_CHECK_ARG(a->num_seqs <= 65535, "num_seqs %d is more than 65535, too many sequences",
               a->num_seqs);
  FA_CHECK_ARG(static_cast<long long>(a->total_q) * (a->h_q / a->h_kv) < (1ll << 30) &&
                   row_blocks(a) * a->h_kv < (1ll << 24),
               "too many query rows or row blocks");  // a grid holds less than 2^32 lanes
  FA_CHECK_ARG(a->num_splits >= 1 && a->num_splits <= 65535 && a->split_tokens >= 1 &&
                   static_cast<int64_t>(a->num_splits - 1) * a->split_tokens <= INT32_MAX,
               "num_splits %d of %d tokens invalid", a->num_splits, a->split_tokens);
  FA_CHECK_ARG(a->num_splits == 1 || (a->o_part && a->lse_part),
               "num_splits %d > 1 needs o_part and lse_part", a->num_splits);
  FA_CHECK_ARG(a->num_splits == 1 ||
                   static_cast<long long>(a->h_q) * a->total_q <= max_merge_rows(a->num_splits),
               "too many query rows for splits");
  return FA_OK;
}

}  // namespace
}  // namespace fa

extern "C" int64_t fa_varlen_args_size(void) { return static_cast<int64_t>(sizeof(fa_varlen_args)); }

extern "C" int fa_varlen_plan(fa_varlen_args* a, int32_t max_q, int32_t max_k, int32_t cu_count) {
  FA_CHECK_ARG(a != nullptr, "args is NULL");
  FA_CHECK_ARG(a->num_seqs >= 0 && a->total_q >= 1 && a->total_k >= 0 && a->h_q >= 1 &&
                   a->h_kv >= 1 && a->h_q % a->h_kv == 0 && a->d >= 1 && max_q >= 0 && max_k >= 0 &&
                   cu_count >= 1,
               "num_seqs %d / total_q %d / total_k %d / h_q %d / h_kv %d / max_q %d / max_k %d / "
               "cu_count %d invalid",
               a->num_seqs, a->total_q, a->total_k, a->h_q, a->h_kv, max_q, max_k, cu_count);
  const int64_t longest = std::min(max_k, a->total_k);
  const int64_t s = fa::choose_splits(a, max_q, longest, cu_count);
  const int64_t each = ((longest + s - 1) / s + 63) / 64 * 64;  // whole tiles
  a->split_tokens = static_cast<int32_t>(std::max<int64_t>(std::min<int64_t>(each, INT32_MAX - 63), 64));
  a->num_splits = s == 1 ? 1 : static_cast<int32_t>((longest + a->split_tokens - 1) / a->split_tokens);
  return FA_OK;
}

extern "C" int fa_varlen_attention(const fa_varlen_args* a, void* stream) {
  const int rc = fa::check_varlen(a);
  if (rc != FA_OK) return rc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == 1)
    fa::launch_varlen<__bf16>(a, s);
  else
    fa::launch_varlen<_Float16>(a, s);
  FA_CHECK_HIP(hipGetLastError());
  return FA_OK;
}

extern "C" int fa_varlen_combine(const fa_varlen_args* a, void* stream) {
  const int rc = fa::check_varlen(a);
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(a->o_part && a->lse_part, "combine needs o_part and lse_part");
  FA_CHECK_ARG(static_cast<int64_t>(a->h_q) * a->total_q <= fa::max_merge_rows(a->num_splits),
               "too many query rows for splits");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const fa::MergeArgs m{a->o_part, a->lse_part, a->out, a->lse, a->o_stride_h, a->o_stride_t,
                        static_cast<int>(static_cast<int64_t>(a->h_q) * a->total_q), a->total_q,
                        a->num_splits};
  if (a->dtype == 1)
    fa::launch_merge<__bf16>(m, a->d, s);
  else
    fa::launch_merge<_Float16>(m, a->d, s);
  FA_CHECK_HIP(hipGetLastError());
  return FA_OK;
}
