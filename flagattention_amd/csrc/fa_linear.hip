// Linear attention with a decay per head over packed sequences for gfx950: fp16 or bf16, head dim 64,
// 128, 256.  Per KV head with log decay a, S_t = e^a S_{t-1} + k_t v_t^T, o_t = scale q_t S_t.
//
// A work-group takes one (sequence, KV head) through its tokens, 32 at a time.  For such a chunk of c
// tokens, counted from 0, with S the state before it:
//   O^T = (S^T Q^T) diag(scale e^{a (i+1)}) + V^T P^T,  P^T[j, i] = scale e^{a (i-j)} (K Q^T)[j, i], j <= i
//   S'  = e^{a c} S + K^T diag(e^{a (c-1-j)}) V
// No weight is above 1 for a decay (a <= 0), however long the chunk or fast the decay; S is kept by what
// it has fallen since it was last brought up, at most 16, and what meets it is taken that much larger.
//
// Wave w owns columns 32w .. 32w + 31 of S, in fp32 in its accumulators for the whole sequence, and the
// same dims of the output; D / 32 waves.  Products are MFMA 32x32x16.  S leaves the accumulators as the
// operands of the next products (the rows of a state tile are dealt to dims so that a lane's 8 registers
// are the 8 dims of its part of a step).  Every wave needs the whole of P^T.  At head dim 256, and at 128
// without groups, four waves work out 16 x 16 of it each and hand it round in LDS; each wave for itself
// would make it a fifth of its products and read K and Q whole again (16 x 1,024 tokens of 16 heads,
// D = 256: 200 us so, 179 shared, when it was made so; 32 heads, D = 128, fp16: 143 / 137; a lone sequence
// of one head waits for the exchange, 410 / 441 at 8,192 tokens; two heads at once at D = 128: 227 / 233,
// so not there).
//
// Bound by q, k, v and out where the card is full (16 x 1,024 tokens of 32 heads, D = 128: 132 us, 117
// at the rate of a copy; of 64, D = 64: 145, 111), by a chunk's chain of products where it is not: 1.3,
// 1.8 and 3.7 us in bf16 at D = 64, 128, 256 for a lone sequence of one head.  At D = 256 one work-group
// fits a CU and the chain shows in full launches too (of 16: 190, 131).  Inputs come three chunks deep
// into LDS, so that no chunk waits for memory.
//
// Rounding: scores, sums and states are fp32.  P and the state's copy are rounded to the input type to
// meet V and Q, which costs as much as rounding the output does: 2.1e-3 from 64 bits in bf16 and 2.5e-4 to
// 2.9e-4 in fp16, 1.7e-3 and 2.1e-4 without.  (Two numbers of the type for each would save that: 10 to
// 14% more time at D = 128, 20 to 26% at 256, where the state's are 360 instructions of a lane and chunk
// more; for P alone 1 to 4%.)  The weighted values that a state takes in are split in three bf16 or two
// fp16 numbers, which hold 24 and 22 bits: the state is an output in fp32 (two bf16 numbers left it 2e-6
// from 64 bits, three 2e-7).  fp16 operands are taken relative to a power of two by the largest (a
// column's of the state, of the weighted values, of P^T), since states, scores and products of tiny inputs
// leave its range.
#include <algorithm>
#include <cmath>

#include "fa_common.h"
#include "fa_divide.h"
#include "fa_linear.h"
#include "fa_rows_tile.h"
#include "fa_wave.h"
#include "flagattention_amd_linear.h"

namespace fa {

int check_linear_shape(const fa_linear_args& a) {
  FA_CHECK_ARG(a.d == 64 || a.d == 128 || a.d == 256, "head dim %d is not 64, 128 or 256", a.d);
  FA_CHECK_ARG(a.dtype == 0 || a.dtype == 1, "dtype %d", a.dtype);
  FA_CHECK_ARG(a.h_kv >= 1 && a.h_q >= 1 && a.h_q % a.h_kv == 0,
               "%d query heads are no multiple of %d", a.h_q, a.h_kv);
  FA_CHECK_ARG(static_cast<int64_t>(a.h_q) * a.d < 1 << 23, "too many heads");
  FA_CHECK_ARG(a.num_seqs >= 0 && a.num_seqs <= 65535 && a.total >= 0,
               "%d sequences, %d tokens out of range", a.num_seqs, a.total);
  return FA_OK;
}

int check_linear(const fa_linear_args& a) {
  const int rc = check_linear_shape(a);
  if (rc != FA_OK) return rc;
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
// fp16: weighted values and scores are below 2^kHalfBits of the power of two that they are relative to: its
// whole range holds what is small beside them (2^-25 of that power is lost, 2^-39 of the largest).
constexpr int kHalfBits = 15;
// The least power of two that they are relative to.  What is below it by 2^-25 is below half
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

__device__ inline floatx4 mfma_16x16x32(PVec<__bf16>::v8 a, PVec<__bf16>::v8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline floatx4 mfma_16x16x32(PVec<_Float16>::v8 a, PVec<_Float16>::v8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A barrier that no access to memory passes.
__device__ inline void sync() {
  asm volatile("" ::: "memory");
  barrier();
  asm volatile("" ::: "memory");
}

// 16 bytes per lane from base + off into LDS at `to`, lane after lane.
__device__ inline void lds_dma16_at(const unsigned char* base, unsigned int off, unsigned int to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(base), "s"(uniform(static_cast<int>(to)))
               : "memory", "m0");
}

// Largest |x| of packed 16-bit values as unsigned bit patterns, folded into best.
__device__ inline void fold_bits(unsigned int& best, uintx4 w) {
  typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    best = __builtin_bit_cast(
        unsigned int, __builtin_elementwise_max(__builtin_bit_cast(ushortx2, best),
                                                __builtin_bit_cast(ushortx2, w[i] & 0x7FFF7FFFu)));
}
// Whether an infinity or a NaN is among them.
template <typename T>
__device__ inline bool is_odd(unsigned int best) {
  constexpr unsigned int kInf = __is_same(T, __bf16) ? 0x7F80u : 0x7C00u;
  return (best & 0xFFFFu) >= kInf || (best >> 16) >= kInf;
}

// The upper 8 bits of a float's 24 as a float, and those of two as bf16.
__device__ inline float upper_of(float x) {
  return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
}
__device__ inline unsigned int upper_halves(float x, float y) {
  return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
}

// Power of two above |x|, 0 for 0, infinities and NaN.
__device__ inline int power_of(float x) { return __builtin_amdgcn_frexp_expf(x); }
__device__ inline float two_to(int e) { return __builtin_amdgcn_ldexpf(1.f, e); }

// A run of tokens that a work-group takes: a sequence, or a segment of one.
struct Run {
  int seq;       // -1: none
  int part;      // segment of the sequence
  int place;     // of its state in the workspace
  int start, n;  // first packed token, tokens
  bool last;     // of its sequence
  int slot;      // of the sequence's state, as given
  bool has;      // whether it starts from it
};

// The slot and the has_state of sequence s, where there are states.
__device__ inline int slot_of(const fa_linear_args& a, int s) {
  return !a.state ? -1 : a.state_indices ? a.state_indices[s] : s;
}
__device__ inline bool has_of(const fa_linear_args& a, int s) {
  return a.has_state == nullptr || a.has_state[s] != 0;
}

// Run `index` of the launch.  With segments of L tokens those of sequence s have the places start_s / L + s
// and on: a sequence of n tokens has ceil(n / L) of them, and the next one's start is at least that
// far on.
//
// Sorted (up to 64 sequences, a lane each): whole segments first, then what is left of each sequence, the
// longest first, so that the work-groups that run longest do not start last (64 sequences of up to
// 1,000 tokens, 16 heads, D = 128: 131 -> 108 us; up to 3,900, 8 heads, D = 256: 814 -> 567; 60 single
// tokens 23.5 -> 24.9, so not for short ones; the 65th sequence costs such a batch what the order gives).
// Otherwise in packed order, by their places; the sequence is the last one whose first place
// is not past `index`, and a wave looks at 64 at a time.
__device__ inline Run find_run(const fa_linear_args& a, int index) {
  Run run = {-1, 0, 0, 0, 0, true, -1, false};
  const int lane = threadIdx.x & 63;
  int seq, start, n;
  if (a.sorted) {
    int start_of = 0, n_of = 0, slot = -1;
    bool has = false;
    if (lane < a.num_seqs) {
      start_of = min(max(a.cu_seqlens[lane], 0), a.total);
      n_of = min(max(a.cu_seqlens[lane + 1], start_of), a.total) - start_of;
      slot = slot_of(a, lane);
      has = has_of(a, lane);
    }
    const int whole = a.segment > 0 ? n_of / a.segment : 0;
    const int rest = n_of - whole * a.segment;
    const int upto = wave_incl_scan(whole);
    const int wholes = __builtin_amdgcn_readlane(upto, 63);
    unsigned long long found;
    if (index < wholes) {
      found = __ballot(upto > index);
    } else {
      // by the upper bits of what is left as a float: the sequences that have more, or as much and come
      // before
      const unsigned int key = __float_as_uint(static_cast<float>(rest)) >> 20;
      unsigned long long same = ~0ull;
      int longer = 0;
#pragma unroll
      for (int bit = 10; bit >= 0; --bit) {
        const unsigned long long set = __ballot(key >> bit & 1u);
        const bool mine = key >> bit & 1u;
        longer += mine ? 0 : __popcll(same & set);
        same &= mine ? set : ~set;
      }
      longer += __popcll(same & ((1ull << lane) - 1ull));
      found = __ballot(rest > 0 && longer == index - wholes);
    }
    if (found == 0ull) return run;
    seq = uniform(__ffsll(found) - 1);
    start = __builtin_amdgcn_readlane(start_of, seq);
    n = __builtin_amdgcn_readlane(n_of, seq);
    run.slot = __builtin_amdgcn_readlane(slot, seq);
    run.has = __builtin_amdgcn_readlane(static_cast<int>(has), seq) != 0;
    const int mine = __builtin_amdgcn_readlane(whole, seq);
    run.part = index < wholes ? index - (__builtin_amdgcn_readlane(upto, seq) - mine) : mine;
    run.place = a.segment > 0 ? start / a.segment + seq + run.part : seq;
  } else {
    seq = index;
    if (a.segment > 0) {
      int lo = 0, hi = a.num_seqs;
      while (true) {
        const int step = cdiv(hi - lo, 64);
        const int s = lo + lane * step;
        const bool before =
            s < hi && min(max(a.cu_seqlens[s], 0), a.total) / a.segment + s <= index;
        const int count = __popcll(__ballot(before));
        if (count == 0) return run;  // in front of the first
        lo += (count - 1) * step;
        hi = min(lo + step, hi);
        if (step == 1) break;
      }
      seq = uniform(lo);
    }
    if (seq >= a.num_seqs) return run;
    const int begins = a.cu_seqlens[seq], ends = a.cu_seqlens[seq + 1];  // one trip to memory for all
    const int slot = slot_of(a, seq);
    const bool has = has_of(a, seq);
    start = uniform(min(max(begins, 0), a.total));
    n = uniform(min(max(ends, start), a.total) - start);
    run.slot = uniform(slot);
    run.has = uniform(static_cast<int>(has)) != 0;
    if (n == 0) return run;
    run.place = index;
    if (a.segment > 0) {
      run.part = index - (start / a.segment + seq);
      if (run.part < 0 || run.part > (n - 1) / a.segment) return run;  // (< 0: starts that fall)
    }
  }
  const int from = run.part * a.segment;
  run.seq = seq;
  run.start = start + from;
  run.n = a.segment > 0 ? min(n - from, a.segment) : n;
  run.last = from + run.n == n;
  return run;
}

// Whether the waves share a chunk's scores, or each works all of them out for itself.
constexpr bool shares(int d, bool one) { return d == 256 || (d == 128 && one); }
constexpr int kScoreRow = 36;  // floats of a row of shared scores: 16 rows lie in different banks

// LDS of a work-group: tiles of k, v and of q's kHeads heads, kStages of each, P of each head, and weights
// by the place m of a token before the chunk's last: at 1 + m scale e^{a (31 - m)}, 0 past 31 (tokens to
// come); and e^{a (31 - m)}, 1 past 31.
template <int D, int kHeads, bool kShare>
struct Lds {
  unsigned char bufs[(2 + kHeads) * kStages * kChunk * 2 * D];
  float scores[kShare ? kHeads * kChunk * kScoreRow : 4];  // P by [head][query][key]
  float scales[kHeads > 0 ? kHeads : 1][D];  // of the state's columns, by wave: fp16
  float seen[1 + 2 * kChunk], left_of[2 * kChunk];
};

// bf16: s is kept times 2^-kLift.  Values are taken up to 16 times into it (by what s has yet to fall), and
// the largest finite ones stay within fp32 so.
constexpr int kLift = 5;

// A run of one KV head, from its state through its chunks.  kStates: only the state that it makes, from
// zeros, or the first run's from its sequence's.  kOne: groups of one query head.  kSplit: heads that
// are attended at once, by D / 32 waves each, which all keep the state.
template <typename T, int D, bool kStates, bool kOne, int kSplit>
__device__ inline void walk(const fa_linear_args& a, const Run run, int hk,
                            Lds<D, kStates ? 0 : kSplit, !kStates && shares(D, kOne)>& shared) {
  typedef typename PVec<T>::v8 T8;
  typedef typename PVec<T>::v4 T4;
  constexpr bool kHalf = !__is_same(T, __bf16);
  constexpr int C = D / 8;
  constexpr int kRowB = 2 * D;
  constexpr int kTileB = kChunk * kRowB;
  constexpr int kThreads = 2 * D * kSplit;
  constexpr int kCopies = 2;               // of 1 KiB a wave, of its head's q tile
  constexpr int kKvCopies = 4 / kSplit;    // of the k and v tiles
  constexpr int kRowsPerCopy = 512 / D;
  constexpr int kKSteps = D / 16;
  constexpr int kTiles = D / 32;
  constexpr int kTerms = kHalf ? 2 : 3;  // 22 and 24 bits
  constexpr int kGroupSteps = D == 256 ? 2 : 4;  // of a product of rows, read at once
  constexpr bool kEarly = kOne && D <= 128;  // values are split beside the scores' products
  constexpr bool kKeepQ = D == 64;  // from the scores to S^T Q^T, else it is read twice
  constexpr bool kShare = !kStates && shares(D, kOne);
  static_assert(kCopies * kTiles * 1024 == kTileB, "whole copies per wave");
  static_assert(!kShare || kSplit == 1, "the waves that share scores meet at a barrier in each item");
  unsigned char* const bufs = shared.bufs;  // [k, v, q][stage]
  float* const seen = shared.seen;
  float* const left_of = shared.left_of;

  const int wave = uniform(wave_id() % kTiles);     // 32 columns of the state
  const int part_of = uniform(wave_id() / kTiles);  // of the heads at once
  // At head dim 256 the state leaves few registers: what follows from the lane is worked out where it is
  // used, and not kept (a wait for a register that comes back from memory waits for every copy too).
  auto lane_id = [&]() -> int { return D == 256 ? fresh_lane() : threadIdx.x & 63; };
  const int group = kStates || kOne ? 1 : a.h_q / a.h_kv;

  const int n = run.n;
  const float log_decay = sload(a.log_decay + hk);
  float* const slot_state =  // the sequence's
      run.slot >= 0 && run.slot < a.num_slots
          ? a.state + run.slot * a.state_stride_s + hk * a.state_stride_h
          : nullptr;

  // Of a sequence of several runs, part has what each makes at the place of the next, and at the first's
  // a copy of what that starts from: the last run may write the sequence's state while the first
  // has not read it yet.
  const long long part_step = static_cast<long long>(a.h_kv) * (D * D);
  float* const part = a.part + run.place * part_step + hk * (D * D);
  float* const to_state = kStates ? part + part_step : run.last ? slot_state : nullptr;

  // Items are (chunk, kSplit query heads of the group), heads innermost; k and v come with the first.
  // States alone go through the chunks from the last one back: what they read last is what the next
  // launch reads first.  They end where e^{a n} is 0 in fp32 (below 2^-149): what lies before adds zeros
  // (a third of the work at |a| = 0.1 and segments of 4,096: 131,001 tokens of 16 heads,
  // D = 128: 702 -> 638 us when it was made so).
  const float log2_decay = log_decay * kLog2e;
  int chunks = cdiv(n, kChunk);
  const int begin = run.start + (kStates ? (chunks - 1) * kChunk : 0);
  if (kStates && log2_decay < 0.f)
    chunks = min(chunks, static_cast<int>(min(150.f / (-log2_decay * kChunk), 1e9f)) + 1);
  // The next chunk's rows, and q's of its next head.
  const unsigned char* k_next = static_cast<const unsigned char*>(a.k) +
                                2 * (begin * a.k_stride_t + hk * a.k_stride_h);
  const unsigned char* v_next = static_cast<const unsigned char*>(a.v) +
                                2 * (begin * a.v_stride_t + hk * a.v_stride_h);
  const unsigned char* q_next =
      static_cast<const unsigned char*>(a.q) +
      2 * (begin * a.q_stride_t + static_cast<long long>(hk) * group * a.q_stride_h);
  const unsigned int q_tb = 2 * a.q_stride_t, k_tb = 2 * a.k_stride_t, v_tb = 2 * a.v_stride_t;
  const long long q_hb = 2 * a.q_stride_h;
  // A tile is 2 kTiles copies of 1 KiB; a wave's are number 2 wave and 2 wave + 1.  Rows past the end
  // repeat the last one.
  auto copy = [&](const unsigned char* from, unsigned int row_b, int rows, unsigned int to, int i) {
    const int lane = lane_id();
    int r = (kCopies * wave + i) * kRowsPerCopy + lane / C;
    const int piece = 16 * ((lane % C) ^ swizzle<C>(r));
    asm volatile("" : "+v"(r));  // no offsets are kept for three tensors
    lds_dma16_at(from, __umul24(min(r, rows - 1), row_b) + piece,
                 to + 1024 * (kCopies * wave + i));
  };
  const unsigned int lds = uniform(static_cast<int>(
      reinterpret_cast<__SIZE_TYPE__>((FA_LDS unsigned char*)bufs)));
  // (segments whose states are made alone are whole chunks)
  auto rows_of = [&](int chunk) { return kStates ? kChunk : n - chunk * kChunk; };
  int next_chunk = 0, next_head = 0;
  int next_q = 0, next_kv = 0;     // bytes of its stages
  // Returns the copies that it issues.
  auto fetch = [&]() -> int {
    if (next_chunk == chunks) return 0;
    const int rows = rows_of(next_chunk);
    int issued = 0;
    if (!kStates) {
      const int mine = kSplit == 1 ? next_head : min(next_head + part_of, group - 1);
#pragma unroll
      for (int i = 0; i < kCopies; ++i)
        copy(q_next + mine * q_hb, q_tb, rows, lds + (2 * kStages + part_of) * kTileB + next_q, i);
      next_q = next_q == (kStages - 1) * kSplit * kTileB ? 0 : next_q + kSplit * kTileB;
      issued += kCopies;
    }
    if (next_head == 0) {
      // the heads' waves share them: all of k and v, k or v, or half of one
      const unsigned int to_k = lds + next_kv, to_v = to_k + kStages * kTileB;
      if constexpr (kSplit == 1) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) copy(k_next, k_tb, rows, to_k, i);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) copy(v_next, v_tb, rows, to_v, i);
      } else {
        const bool takes_v = part_of >= kSplit / 2;  // uniform
        const unsigned char* const from = takes_v ? v_next : k_next;
        const unsigned int row_b = takes_v ? v_tb : k_tb, to = takes_v ? to_v : to_k;
        if (kSplit == 2 || part_of % 2 == 0) copy(from, row_b, rows, to, 0);
        if (kSplit == 2 || part_of % 2 == 1) copy(from, row_b, rows, to, 1);
      }
      next_kv = next_kv == (kStages - 1) * kTileB ? 0 : next_kv + kTileB;
      k_next += (kStates ? -kChunk : kChunk) * static_cast<long long>(k_tb);
      v_next += (kStates ? -kChunk : kChunk) * static_cast<long long>(v_tb);
      issued += kKvCopies;
    }
    next_head += kSplit;
    if (next_head >= group) {
      next_head = 0;
      ++next_chunk;
      q_next += kChunk * static_cast<long long>(q_tb);
    }
    return issued;
  };
  fetch();
  int ahead = fetch();  // copies on their way after those of the item at hand
  int stored = 0;       // stores of the last item

  // Row rho of a 32-row tile of the state (or of O^T) is dim 16 (rho / 16) + 8 ((rho / 4) % 2) +
  // 4 ((rho / 8) % 2) + rho % 4: accumulator register r of half h is then dim 16 (r / 8) + 8h + r % 8.
  auto state_place = [&]() -> int {
    const int lane = lane_id(), c32 = lane & 31;
    const int pi = (c32 & 16) + 8 * ((c32 >> 2) & 1) + 4 * ((c32 >> 3) & 1) + (c32 & 3);
    return 8 * (lane >> 5) * D + 32 * wave + pi;
  };
  floatx16 s[kTiles] = {};
  constexpr float kInit = kHalf || kStates ? 1.f : 1.f / (1 << kLift);
  // What the run starts from: its sequence's state, the joined state in front of it, or what every run
  // before it made.
  const float* from = part;
  int states = 0;
  if (run.part == 0) {
    states = slot_state && run.has;
    if (kStates || run.last) from = slot_state;
  } else if (!kStates) {
    states = a.joined ? 1 : run.part;
    from -= (states - 1) * part_step;
  }
  const bool from_state = states > 0;
  if (from_state) {
    const int state_at = state_place();
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[t][r] = kInit * from[state_at + (32 * t + 16 * (r >> 3) + (r & 7)) * D];
  }
  if (states > 1) {
    constexpr int kAtOnce = D == 256 ? 1 : kTiles;  // tiles: more would be spilled
    const Fall fall = fall_of(log_decay, a.segment);
    const int state_at = state_place();
#pragma unroll
    for (int t0 = 0; t0 < kTiles; t0 += kAtOnce) {
      const float* next = from;
      for (int i = 1; i < states; ++i) {
        next += part_step;
#pragma unroll
        for (int t = t0; t < t0 + kAtOnce; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[t][r] = add_fallen(s[t][r], fall,
                                 kInit * next[state_at + (32 * t + 16 * (r >> 3) + (r & 7)) * D]);
      }
    }
  }
  // s is kept times 2^-s_power.  fp16: a power for each column (a lane's), kLowest or more; states alone
  // have no copies in fp16, and 0.
  constexpr int kLowest = -126;
  int s_power = kHalf || kStates ? 0 : kLift;
  // The largest of the lane's column that is finite.
  auto most_of = [&]() -> float {
    float most = 0.f;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(s[t][r]));
    if (__ballot(most == __builtin_inff()) != 0ull) {  // uniform
      most = 0.f;
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          most = fabsf(s[t][r]) < __builtin_inff() ? fmaxf(most, fabsf(s[t][r])) : most;
    }
    return max_xor32(most);
  };
  auto scale_down = [&](int by) {
    const float x = two_to(-by);
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] *= x;
    s_power += by;
  };
  if constexpr (kStates) {
    if (from_state) {
      const int state_at = state_place();
      const float fall = decay(log_decay, n);
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          part[state_at + (32 * t + 16 * (r >> 3) + (r & 7)) * D] = s[t][r];
          s[t][r] *= fall;
        }
    }
  }

  if (threadIdx.x < 2 * kChunk) {
    const int m = threadIdx.x;
    const float e = decay(log_decay, max(kChunk - 1 - m, 0));
    seen[1 + m] = m < kChunk ? a.scale * e : 0.f;
    if (m == 0) seen[0] = a.scale * decay(log_decay, kChunk);
    left_of[m] = kInit * e;
  }
  // The state is s times sigma = e^{a reset}, reset the tokens since s was last brought up: a product
  // of a whole state only where sigma has fallen by 16 (or grown, for a > 0), and no rounding of a
  // factor next to 1 at every chunk.
  int reset = 0;
  float sigma = 1.f, sigma_then = 1.f;
  // States alone have their weights counted to the run's end instead, and are never brought up.
  int after = 0;

  // fp16: a column's largest is 2^7 to 2^12 when it was last looked at: there is room for a growth by 2^4
  // (past it an output is not finite, and the chunk is taken again) and a fall by 2^kFall (counted below),
  // before which 2^-32 of it or less is lost in its copies, and 2^-20 behind it.
  constexpr int kFall = 12;
  int looked = -1;  // tokens since, -1: to be looked at behind this chunk
  float* const scales = shared.scales[kStates ? 0 : part_of] + 32 * wave;
  auto look = [&]() {
    const float most = most_of();
    // |s| 2^s_power is at most 2^128: both factors stay in range
    const int by = most > 0.f ? max(power_of(most) - 10, -100 - s_power) : 0;
    if (__ballot(by < -2 || by > 2) != 0ull) scale_down(by);  // uniform
    // A column of zeros is far below its first values, which have it looked at again.  (One that stays so,
    // as the dims that a head is padded by, costs nothing: 8,192 tokens of one head, 96 of D = 128 filled,
    // 539 us where such a column was looked at behind every chunk, 504 now.)
    if (most == 0.f) s_power = kLowest;
    looked = 0;
    scales[lane_id() & 31] = two_to(min(s_power, 127));
  };
  if (kHalf && !kStates) {
    scales[lane_id() & 31] = 1.f;
    if (from_state) look();
  }

  // Token of register r in P^T's rows, and of element r of the values' operands, less 4h.
  auto token = [&](int r) { return 8 * (r >> 2) + (r & 3); };
  // dims 32t .. 32t + 31 of tokens token(8 ss) .. token(8 ss + 7), transposed
  // (from: the tile's first byte plus tr_at)
  auto transposed = [&](int from, int t, int ss) -> T8 {
    const unsigned char* const p = bufs + 16 * ss * kRowB;
    const T4 lo = lds_tr_read4<T>(p + (from ^ (64 * t)));
    const T4 hi = lds_tr_read4<T>(p + 8 * kRowB + (from ^ (64 * t + 16)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  int q_stage = 0, kv_stage = 0, head = 0;
  int chunk = 0;
  bool first = true;
  int turn = 0;  // the waves whose scores are next, at head dim 256
  T8 va[2];
  // the chunk's first row of the output
  unsigned char* out = static_cast<unsigned char*>(a.out) +
                       2 * (static_cast<long long>(run.start) * a.h_q + hk * group) * D;
  while (true) {
    // all but what was issued after this item's copies: the next item's, and the last one's stores
    const int pending = first || ahead == 0 ? 0 : ahead + stored;
    if (pending >= 8)
      wait_vmem<8>();
    else if (pending >= 6)
      wait_vmem<6>();
    else if (pending >= 4)
      wait_vmem<4>();
    else if (pending >= 2)
      wait_vmem<2>();
    else
      wait_vmem<0>();
    first = false;
    sync();
    ahead = fetch();
    unsigned char* const kb = bufs + kv_stage;
    unsigned char* const vb = bufs + kStages * kTileB + kv_stage;
    const int taken = min(rows_of(chunk), kChunk);
    if (taken < kChunk && head == 0) {  // uniform: rows past the end become zeros
      for (int i = taken * kRowB / 16 + threadIdx.x; i < kTileB / 16; i += kThreads) {
        reinterpret_cast<uintx4*>(kb)[i] = uintx4{0, 0, 0, 0};
        reinterpret_cast<uintx4*>(vb)[i] = uintx4{0, 0, 0, 0};
      }
      sync();
    }
    if (!kStates && head == 0) {  // the state after this chunk is s times sigma_then
      sigma_then = __builtin_amdgcn_exp2f(log2_decay * static_cast<float>(reset + taken));
      if (!(sigma_then >= 0.0625f && sigma_then <= 16.f)) {  // uniform
        if (reset > 0) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[t][r] *= sigma;
          reset = 0;
          sigma = 1.f;
        }
        sigma_then = __builtin_amdgcn_exp2f(log2_decay * static_cast<float>(taken));
      }
    }
    // A chunk whose own fall is past the range is taken into s before its values are.
    const bool steep = !kStates && !(sigma_then >= 0.0625f && sigma_then <= 16.f);  // uniform
    // Addresses of this chunk, worked out afresh: kept, each of their many forms would be a register.
    const int lane = lane_id(), h = lane >> 5, c32 = lane & 31;
    const int row_at = c32 * kRowB + 16 * (h ^ swizzle<C>(c32));
    // transposed reads: lanes 4e + x of 16 point at 4 dims of token row e
    const int e = (lane & 15) >> 2, x4 = lane & 3, p16 = (lane >> 4) & 1;
    const int tr_at = (4 * h + e) * kRowB +
                      16 * ((2 * p16 + (x4 & 1)) ^ swizzle<C>(4 * h + e)) + 8 * (x4 >> 1);
    int k_row = kv_stage + row_at, k_tr = kv_stage + tr_at;
    asm volatile("" : "+v"(k_row), "+v"(k_tr));
    va[0] = transposed(kStages * kTileB + k_tr, wave, 0);
    va[1] = transposed(kStages * kTileB + k_tr, wave, 1);

    // The weighted values, each as a sum of kTerms numbers of the type (fp16: relative to 2^v_power, which
    // their column's largest is 2^14 of, so that what an infinity does to s elsewhere changes no bit of them).
    T8 terms[kTerms][2];
    int v_power = 0;
    auto split = [&]() {
      const float* const weight = left_of + kChunk - taken + 4 * h;
      float against = 1.f;
      if (kStates ? after > 0 : !steep)
        against = __builtin_amdgcn_exp2f(
            log2_decay * static_cast<float>(kStates ? after : -(reset + taken)));
      float f[16];
#pragma unroll
      for (int r = 0; r < 16; ++r)
        f[r] = static_cast<float>(va[r >> 3][r & 7]) * (weight[token(r)] * against);
      if constexpr (kHalf) {
        float top = two_to(kLowest);
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(f[r]));
        v_power = min(max(power_of(max_xor32(top)) - kHalfBits, kLowest + kHalfBits), 100);
        const float by = two_to(-v_power);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float x = f[r] * by;
          terms[0][r >> 3][r & 7] = static_cast<T>(x);
          terms[1][r >> 3][r & 7] = static_cast<T>(x - static_cast<float>(terms[0][r >> 3][r & 7]));
        }
      } else {  // the upper 8 bits, the next 8, the rest
#pragma unroll
        for (int ss = 0; ss < 2; ++ss) {
          uintx4 upper, next, rest;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float y = f[8 * ss + 2 * x], z = f[8 * ss + 2 * x + 1];
            upper[x] = upper_halves(y, z);
            y -= upper_of(y), z -= upper_of(z);
            next[x] = upper_halves(y, z);
            y -= upper_of(y), z -= upper_of(z);
            rest[x] = upper_halves(y, z);
          }
          terms[0][ss] = __builtin_bit_cast(T8, upper);
          terms[1][ss] = __builtin_bit_cast(T8, next);
          terms[2][ss] = __builtin_bit_cast(T8, rest);
        }
      }
    };

    const bool mine = kSplit == 1 || head + part_of < group;  // uniform
    bool odd = false;  // something is not finite
    floatx16 o = {};
    if constexpr (kStates) {
      unsigned int best = 0u;
#pragma unroll
      for (int ss = 0; ss < 2; ++ss) fold_bits(best, __builtin_bit_cast(uintx4, va[ss]));
      odd = __ballot(is_odd<T>(best)) != 0ull;
    } else {
      const int q_row_of_tile = (2 * kStages + part_of) * kTileB + q_stage;
      int q_row = q_row_of_tile + row_at;
      asm volatile("" : "+v"(q_row));
      q_stage = q_stage == (kStages - 1) * kSplit * kTileB ? 0 : q_stage + kSplit * kTileB;
      // A quarter of P^T for the head's waves, 16 keys by 16 queries; at head dim 256 those of four waves
      // and of the other four in turn.
      float* const scores = shared.scores + (kShare ? part_of * kChunk * kScoreRow : 0);
      const bool sharing = kShare && mine && (D < 256 || (wave >> 2) == turn);  // uniform
      turn ^= 1;
      int quarter_at = 0;
      floatx4 quarter = {};
      auto share = [&]() {
        const int in = lane_id(), row = in & 15, piece = in >> 4;
        const int query = 16 * (wave & 1) + row, key = 16 * (wave >> 1 & 1) + row;
        int key_at = kv_stage + key * kRowB + 16 * (piece ^ swizzle<C>(key));
        int query_at = q_row_of_tile + query * kRowB + 16 * (piece ^ swizzle<C>(query));
        asm volatile("" : "+v"(key_at), "+v"(query_at));
        floatx4 p[2] = {};
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
          p[x & 1] = mfma_16x16x32(*reinterpret_cast<const T8*>(bufs + (key_at ^ (64 * x))),
                                   *reinterpret_cast<const T8*>(bufs + (query_at ^ (64 * x))), p[x & 1]);
        const int key0 = key - row + 4 * piece;
#pragma unroll
        for (int r = 0; r < 4; ++r) quarter[r] = (p[0][r] + p[1][r]) * seen[kChunk - query + key0 + r];
        quarter_at = query * kScoreRow + key0;
      };
      // O^T of the item.  kOdd: with weights of 0 for what is not finite and yet to come.
      auto attend = [&](auto tag) {
        constexpr bool kOdd = decltype(tag)::value != 0;
        int p_power = 0;
        // A group of steps is read while the last one is multiplied.
        floatx16 p = {};
        T8 qa[kKeepQ ? kKSteps : 2 * kGroupSteps], ka[2 * kGroupSteps];
        auto read = [&](int i, bool keys) {
#pragma unroll
          for (int x = kGroupSteps * i; x < kGroupSteps * (i + 1); ++x) {
            if (keys)
              ka[x % (2 * kGroupSteps)] = *reinterpret_cast<const T8*>(bufs + (k_row ^ (32 * x)));
            if (keys || !kKeepQ)
              qa[kKeepQ ? x : x % (2 * kGroupSteps)] =
                  *reinterpret_cast<const T8*>(bufs + (q_row ^ (32 * x)));
          }
        };
        if constexpr (!kShare) {
          read(0, true);
#pragma unroll
          for (int i = 0; i < kKSteps / kGroupSteps; ++i) {
            if (i + 1 < kKSteps / kGroupSteps) read(i + 1, true);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = kGroupSteps * i; x < kGroupSteps * (i + 1); ++x)
              p = mfma_32x32x16(ka[x % (2 * kGroupSteps)], qa[kKeepQ ? x : x % (2 * kGroupSteps)], p);
          }
        }
        if (!kKeepQ) read(0, false);
        if constexpr (kShare && !kOdd) {
          if (sharing) share();
        }
        if (kEarly && !kOdd) split();  // beside those products
#pragma unroll
        for (int i = 0; i < kKSteps / kGroupSteps; ++i) {
          if (!kKeepQ && i + 1 < kKSteps / kGroupSteps) read(i + 1, false);
          if (D == 256) __builtin_amdgcn_sched_barrier(0);  // few of s's copies at once
#pragma unroll
          for (int x = kGroupSteps * i; x < kGroupSteps * (i + 1); ++x) {
            T8 sa;
#pragma unroll
            for (int y = 0; y < 8; ++y) sa[y] = static_cast<T>(s[x >> 1][8 * (x & 1) + y]);
            o = mfma_32x32x16(sa, qa[kKeepQ ? x : x % (2 * kGroupSteps)], o);
          }
        }
        const float* const weight = seen + kChunk - c32 + 4 * h;
        const float since = seen[kChunk - 1 - c32] * sigma;  // scale e^{a (i + 1)} of the state
        if constexpr (kShare) {
          if (!kOdd) {
            if (sharing) *reinterpret_cast<floatx4*>(scores + quarter_at) = quarter;
            sync();
          }
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const floatx4 four =
                *reinterpret_cast<const floatx4*>(scores + c32 * kScoreRow + 8 * y + 4 * h);
#pragma unroll
            for (int x = 0; x < 4; ++x) p[4 * y + x] = four[x];
          }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (!kShare) p[r] *= weight[token(r)];
          if (kOdd) p[r] = token(r) + 4 * h <= c32 ? p[r] : 0.f;
        }
        if constexpr (kHalf) {
          float top = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(p[r]));
          p_power = min(max(power_of(max_xor32(top)) - kHalfBits, kLeastPower), 100);
        }
        // O^T, relative to 2^p_power
        const float by = kHalf ? __builtin_amdgcn_ldexpf(since, -p_power) : since * (1 << kLift);
        const float p_by = two_to(-p_power), p_back = two_to(p_power);
#pragma unroll
        for (int r = 0; r < 16; ++r) {  // token(r) + 4h is the column too
          if (kHalf) o[r] *= scales[token(r) + 4 * h];
          o[r] *= by;
        }
#pragma unroll
        for (int ss = 0; ss < 2; ++ss) {
          T8 pb, v8 = va[ss];
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            pb[x] = static_cast<T>(kHalf ? p[8 * ss + x] * p_by : p[8 * ss + x]);
            if (kOdd)
              v8[x] = fabsf(static_cast<float>(v8[x])) < __builtin_inff() ? v8[x]
                                                                         : static_cast<T>(0.f);
          }
          o = mfma_32x32x16(v8, pb, o);
        }
        if constexpr (kHalf) {
#pragma unroll
          for (int r = 0; r < 16; ++r) o[r] *= p_back;
        }
        if constexpr (kOdd) {  // those values, for the tokens that see them
          for (int j = 0; j < taken; ++j) {
            float w = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) w = token(r) == (j & ~4) ? p[r] : w;
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
      };
      if (mine) attend(IntTag<0>{});  // (the waves that share scores are of one head)
      // An infinity or a NaN among the scores or in v reaches the tokens before its own, through
      // weights of 0, and the outputs of its own: such a chunk is taken again.
      floatx4 trace = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 16; ++r) trace[r & 3] = __builtin_fmaf(o[r], 0.f, trace[r & 3]);
      odd = __ballot((trace[0] + trace[1]) + (trace[2] + trace[3]) != 0.f) != 0ull;  // uniform
      if (odd) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int t = 0; t < kTiles; ++t) asm volatile("" : "+v"(s[t]));  // nothing is kept for it
        if (kHalf) look();
        o = floatx16{};
        attend(IntTag<1>{});
      }
    }

    T8 kt[2][2];  // K^T of a tile of the state, the next one on its way
    if (kStates || kOne) {
      kt[0][0] = transposed(k_tr, 0, 0);
      kt[0][1] = transposed(k_tr, 0, 1);
    }
    if constexpr (!kStates) {
      stored = 0;
      if (mine) {
        if (c32 < taken) {
          unsigned char* const to =
              out + 2 * D * (head + part_of) +
              2 * (c32 * static_cast<unsigned int>(a.h_q * D) + 32 * wave + 8 * h);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            T8 y;
#pragma unroll
            for (int x = 0; x < 8; ++x) y[x] = static_cast<T>(o[8 * half + x]);
            *reinterpret_cast<T8*>(to + 32 * half) = y;
          }
        }
        stored = 2;
      }
      head += kSplit;
      if (head < group) continue;
      head = 0;
      out += 2 * D * static_cast<long long>(kChunk) * a.h_q;
      if (chunk + 1 == chunks && to_state == nullptr) break;
    }

    if (!(kStates || kOne)) {
      kt[0][0] = transposed(k_tr, 0, 0);
      kt[0][1] = transposed(k_tr, 0, 1);
    }
    if (!kEarly) split();
    if (odd) {  // what is not finite has no rest
      asm volatile("" ::: "memory");
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!(fabsf(static_cast<float>(terms[0][r >> 3][r & 7])) < __builtin_inff()))
#pragma unroll
          for (int x = 1; x < kTerms; ++x) terms[x][r >> 3][r & 7] = static_cast<T>(0.f);
    }
    if (steep) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] *= sigma_then;
      reset = 0;
      sigma = 1.f;
    } else {
      reset += taken;
      sigma = sigma_then;
    }
    after += taken;
    if constexpr (kHalf && !kStates) {
      // A column that was next to nothing when it was last looked at, or nothing, may be far below the unit
      // of these products (of at most 2^37 units): s takes it then, or they would leave fp32.
      if (__ballot(v_power - s_power > 64) != 0ull) {  // uniform
        scale_down(v_power - s_power > 64 ? v_power - s_power : 0);
        looked = -1;
      }
    }
    // of the products in units of s
    const float add_by = kHalf ? two_to(min(max(v_power - s_power, -126), 127)) : 1.f;
    // A chunk's products are summed by themselves, the least terms first: each added to s alone, what is
    // below its last bit would be lost, and always the same way (bf16, values of one sign behind a state of
    // 1e6, 131,001 tokens: 1.5e-4 of it).  A tile's sums are added while the next tile's are made.
    floatx16 add[2];
    auto take = [&](int t) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[t][r] = kHalf ? __builtin_fmaf(add[t & 1][r], add_by, s[t][r]) : s[t][r] + add[t & 1][r];
    };
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      if (t + 1 < kTiles) {
        kt[(t + 1) & 1][0] = transposed(k_tr, t + 1, 0);
        kt[(t + 1) & 1][1] = transposed(k_tr, t + 1, 1);
      }
      __builtin_amdgcn_sched_barrier(0);
      add[t & 1] = floatx16{};
#pragma unroll
      for (int x = kTerms - 1; x >= 0; --x)
#pragma unroll
        for (int ss = 0; ss < 2; ++ss)
          add[t & 1] = mfma_32x32x16(kt[t & 1][ss], terms[x][ss], add[t & 1]);
      if (kStates)
        take(t);
      else if (t > 0)
        take(t - 1);
    }
    if (!kStates) take(kTiles - 1);
    kv_stage = kv_stage == (kStages - 1) * kTileB ? 0 : kv_stage + kTileB;
    if (++chunk == chunks) break;
    if constexpr (kHalf && !kStates) {
      if (looked >= 0) looked += taken;
      if (looked < 0 || !(log2_decay * static_cast<float>(looked) > -kFall)) look();  // uniform
    }
  }

  if (kSplit > 1) {  // the heads' waves read the state that those of the first write
    sync();
    if (part_of > 0) return;
  }
  if (to_state != nullptr) {
    const int state_at = state_place();
    const float back = __builtin_amdgcn_ldexpf(sigma, s_power);
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        to_state[state_at + (32 * t + 16 * (r >> 3) + (r & 7)) * D] = s[t][r] * back;
  }
}

template <typename T, int D, bool kOne, int kSplit>
__global__ __launch_bounds__(2 * D * kSplit, 2) void linear_kernel(const fa_linear_args a,
                                                                   const Divisor h_kv) {
  __shared__ __attribute__((aligned(1024))) Lds<D, kSplit, shares(D, kOne)> shared;
  const int begins = sload(a.cu_seqlens), ends = sload(a.cu_seqlens + a.num_seqs);
  const int index = divide(blockIdx.x, h_kv);
  const int hk = blockIdx.x - index * a.h_kv;
  const Run run = find_run(a, index);
  {  // rows of no sequence: everybody takes a share of their 16 bytes
    const int first = min(max(begins, 0), a.total);
    const int behind = max(first, min(max(ends, 0), a.total));
    const long long row16 = static_cast<long long>(a.h_q) * (D / 8);
    const long long head = first * row16, all = a.total * row16, tail = behind * row16;
    uintx4* const out16 = static_cast<uintx4*>(a.out);
    const long long step = static_cast<long long>(gridDim.x) * (2 * D * kSplit);
    const long long me = static_cast<long long>(blockIdx.x) * (2 * D * kSplit) + threadIdx.x;
    for (long long i = me; i < head; i += step) out16[i] = uintx4{0, 0, 0, 0};
    for (long long i = tail + me; i < all; i += step) out16[i] = uintx4{0, 0, 0, 0};
  }
  if (run.seq < 0) return;  // uniform
  walk<T, D, false, kOne, kSplit>(a, run, hk, shared);
}

// What every run but a sequence's last makes.  Without tiles of q three work-groups fit a CU at D = 128
// (the first runs' outputs in the same launch leave two: 131,001 tokens of 16 heads 638 -> 710 us; not
// measured for ragged batches, where first runs are half of the launch).  That sequence: 207 us here, for
// the half of k and v that is not skipped, then 458 for the outputs, 4.7 TB/s.
template <typename T, int D>
__global__ __launch_bounds__(2 * D, 2) void states_kernel(const fa_linear_args a,
                                                          const Divisor h_kv) {
  __shared__ __attribute__((aligned(1024))) Lds<D, 0, false> shared;
  const int index = divide(blockIdx.x, h_kv);
  const int hk = blockIdx.x - index * a.h_kv;
  const Run run = find_run(a, index);
  if (run.seq < 0 || run.last) return;  // uniform
  walk<T, D, true, false, 1>(a, run, hk, shared);
}

// The states that runs start from, but for the first two: each what its predecessor made on top of what
// that one started from, part[i] += e^{a L} part[i - 1].
template <int D>
__global__ __launch_bounds__(256) void join_kernel(const fa_linear_args a, const Divisor h_kv) {
  constexpr int kAhead = 8;
  const int seq = divide(blockIdx.x, h_kv);
  const int hk = blockIdx.x - seq * a.h_kv;
  const int start = min(max(sload(a.cu_seqlens + seq), 0), a.total);
  const int n = min(max(sload(a.cu_seqlens + seq + 1), start), a.total) - start;
  const int states = n == 0 ? 0 : (n - 1) / a.segment;  // those that the others start from
  if (states < 2) return;
  const long long step = static_cast<long long>(a.h_kv) * (D * D) / 4;
  floatx4* at = reinterpret_cast<floatx4*>(a.part) +
                (static_cast<long long>(start / a.segment + seq + 1) * a.h_kv + hk) * (D * D / 4) +
                blockIdx.y * 256 + threadIdx.x;
  const Fall fall = fall_of(sload(a.log_decay + hk), a.segment);
  if (fall.by == 0.f && fall.keep == 0.f) return;
  floatx4 sum = *at;
  for (int i = 1; i < states; i += kAhead) {
    floatx4 next[kAhead] = {};
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j < states) next[j] = at[(j + 1) * step];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
#pragma unroll
      for (int x = 0; x < 4; ++x) next[j][x] = add_fallen(j > 0 ? next[j - 1][x] : sum[x], fall, next[j][x]);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j < states) at[(j + 1) * step] = next[j];
    sum = next[kAhead - 1];  // (another round follows only if all were there)
    at += kAhead * step;
  }
}

// Indices of runs in a launch (find_run).
int runs_of(const fa_linear_args& a) {
  const int seqs = a.num_seqs > 0 ? a.num_seqs : 1;  // rows of no sequence are there too
  return a.segment > 0 ? a.total / a.segment + seqs : seqs;
}

// Runs of a sequence from which on their states are joined in a launch of their own, which takes 6 to 24
// us; below, each run adds up what those before it made (one sequence of 16 heads, D = 128, in three
// segments of 512 59.0 us so, 60.5 joined, in five 62.3 / 61.9, in seven 64.8 / 62.8, 131,001 tokens in
// segments of 4,096 710 / 661; D = 256 in three 121 / 124, in four 128 / 126, 8 prompts of up to 2,048
// in segments of 416 197 / 194).
int join_runs(int d) { return d == 256 ? 3 : 5; }

// Heads that a work-group attends at once: as many as the registers of two waves per SIMD keep the state
// for (8 sequences of 1,024 tokens, 64 heads of 8, D = 128: 136 us with one, 97 with two; three of up to
// 48, 8 heads of 2, D = 64: 10.8 with one, 8.1 with four).
int heads_at_once(int group, int d) {
  return group == 1 || d == 256 ? 1 : d == 128 || group == 2 ? 2 : 4;
}

// What a launch takes, in us, by segments of L tokens (0: whole sequences), from times of 12 shapes per
// head dim (one sequence of 1,000 to 131,001 tokens, 3 to 40 of up to 8,000, groups of 1, 4 and 8), off by
// a tenth on average.  Of another 12 its choice is within 4% of the best of the powers of two in ten, 8% off
// in three of 8,000, 64 heads of 8, D = 128, and 11% in 12 of 4,000, 16 of 4, D = 64; lengths that it does
// not try can be better still (8 prompts at D = 256: 416 or 448 194 us, 480 182).
//
// The longest run's chunks or a slot's share of all, whichever is more; starts and ends of the
// work-groups; the segments' states; no less than the bytes.
struct Cost {
  float chunk_one;          // a chunk, groups of one head
  float item, chunk_group;  // heads at once, a chunk beside them
  float chunk_state;        // a chunk of the states alone
  float state;              // a segment's state, written, read and joined
  float start;              // a work-group's start and end
  int slots;                // work-groups per CU
};
double cost_of(const fa_linear_args& a, int segment, int max_seqlen, int cus) {
  static const Cost kCost[3] = {{1.29f, 1.12f, .7f, .56f, .0109f, 5.4f, 4},
                                {1.98f, 1.4f, .31f, .63f, .056f, 5.4f, 2},
                                {3.53f, 1.62f, 2.57f, 2.f, .165f, 21.f, 1}};
  constexpr double kBytesPerUs = 5.1e6;
  const Cost& c = kCost[a.d == 64 ? 0 : a.d == 128 ? 1 : 2];
  const int group = a.h_q / a.h_kv, split = heads_at_once(group, a.d);
  const double slots = cus * std::max(1, c.slots / split);
  const double chunk = group == 1 ? c.chunk_one : cdiv(group, split) * c.item + c.chunk_group;
  const double share = static_cast<double>(a.total) * a.h_kv / kChunk / slots;
  double runs = a.num_seqs, longest = cdiv(max_seqlen, kChunk), each = chunk, states = 0.;
  if (segment > 0) {
    runs = static_cast<double>(a.total) / segment + .6 * a.num_seqs;
    longest = segment / kChunk;
    each += c.chunk_state;
    // about half a segment of a sequence hands nothing on, or less where some are short
    states = std::max(0., static_cast<double>(a.total) / segment - .3 * a.num_seqs) * a.h_kv * c.state;
  }
  const double starts = c.start * std::ceil(runs * a.h_kv / slots) * (segment > 0 ? 1. : .5);
  const double bytes = 4. * a.total * a.d * (a.h_q + a.h_kv * (segment > 0 ? 2. : 1.));
  return (segment > 0 ? 8. : 3.) +
         std::max(std::max(longest, share) * each + starts, bytes / kBytesPerUs) + states;
}

constexpr int64_t kMaxWorkspace = int64_t{1} << 32;  // bytes

// Tokens of a segment, 0 for whole sequences: the cheapest of powers of two and of what gives every slot
// one segment.
int choose_segment(const fa_linear_args& a, int max_seqlen, int cus) {
  if (a.num_seqs == 0 || max_seqlen <= 2 * kChunk) return 0;
  int best = 0;
  double least = cost_of(a, 0, max_seqlen, cus);
  auto consider = [&](int64_t segment) {
    const int64_t states = (a.total / segment + a.num_seqs) * static_cast<int64_t>(a.h_kv);
    if (segment >= max_seqlen || states * a.d * a.d > kMaxWorkspace / 4) return;
    const double c = cost_of(a, static_cast<int>(segment), max_seqlen, cus);
    if (c < least) least = c, best = static_cast<int>(segment);
  };
  for (int64_t segment = 2 * kChunk; segment <= 1 << 16; segment *= 2) consider(segment);
  const int64_t slots = static_cast<int64_t>(cus) * (a.d == 64 ? 4 : a.d == 128 ? 2 : 1) /
                        heads_at_once(a.h_q / a.h_kv, a.d);
  const int64_t fit = static_cast<int64_t>(a.total) * a.h_kv / std::max<int64_t>(slots, 1);
  consider(std::max<int64_t>((fit + kChunk - 1) / kChunk, 2) * kChunk);
  return best;
}

template <typename T, int D, bool kOne, int kSplit>
void launch_split(const fa_linear_args& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(runs_of(a) * a.h_kv)), block(2 * D * kSplit);
  const Divisor h_kv = divisor(a.h_kv);
  if (a.segment > 0) {
    hipLaunchKernelGGL((states_kernel<T, D>), grid, dim3(2 * D), 0, stream, a, h_kv);
    if (a.joined)
      hipLaunchKernelGGL((join_kernel<D>),
                         dim3(static_cast<unsigned>(a.num_seqs * a.h_kv), D * D / 1024), dim3(256), 0,
                         stream, a, h_kv);
  }
  hipLaunchKernelGGL((linear_kernel<T, D, kOne, kSplit>), grid, block, 0, stream, a, h_kv);
}

template <typename T, int D>
void launch(const fa_linear_args& a, hipStream_t stream) {
  constexpr int kTwo = D == 256 ? 1 : 2, kMany = D == 64 ? 4 : kTwo;
  const int group = a.h_q / a.h_kv;
  if (group == 1)
    launch_split<T, D, true, 1>(a, stream);
  else if (heads_at_once(group, D) == kMany)
    launch_split<T, D, false, kMany>(a, stream);
  else
    launch_split<T, D, false, kTwo>(a, stream);
}

}  // namespace
}  // namespace fa

extern "C" int64_t fa_linear_args_size(void) {
  return static_cast<int64_t>(sizeof(fa_linear_args));
}

extern "C" int64_t fa_linear_plan(fa_linear_args* args, int32_t max_seqlen, int32_t cu_count) {
  FA_CHECK_ARG(args != nullptr, "args is NULL");
  fa_linear_args& a = *args;
  const int rc = fa::check_linear_shape(a);
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(max_seqlen >= 0 && cu_count >= 1, "max_seqlen %d, %d CUs", max_seqlen, cu_count);
  a.segment = fa::choose_segment(a, max_seqlen, cu_count);
  a.joined = a.segment > 0 && fa::cdiv(max_seqlen, a.segment) >= fa::join_runs(a.d);
  a.sorted = a.num_seqs >= 2 && a.num_seqs <= 64 && max_seqlen > 4 * fa::kChunk;
  return a.segment > 0 ? static_cast<int64_t>(fa::runs_of(a)) * a.h_kv * a.d * a.d : 0;
}

extern "C" int fa_linear_prompt(const fa_linear_args* args, void* stream) {
  FA_CHECK_ARG(args != nullptr, "args is NULL");
  const fa_linear_args& a = *args;
  const int rc = fa::check_linear(a);
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(a.segment >= 0 && a.segment % fa::kChunk == 0, "segments of %d tokens", a.segment);
  FA_CHECK_ARG(a.segment == 0 || a.num_seqs == 0 ||
                   (a.part && (reinterpret_cast<uintptr_t>(a.part) & 15) == 0),
               "part is NULL or not 16-byte aligned");
  FA_CHECK_ARG(!a.sorted || a.num_seqs <= 64, "%d sequences are not sorted", a.num_seqs);
  FA_CHECK_ARG(a.total <= INT32_MAX - 256, "too many tokens");
  FA_CHECK_ARG((static_cast<int64_t>(a.segment > 0 ? a.total / a.segment : 0) + a.num_seqs) * a.h_kv <
                   1 << 22, "too many sequences or heads");
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
