// A paged K/V cache in 4 bits for gfx950: its writer, its reader and one-token decode over it.
//
// Rows hold e2m1 codes (dim 2i in the low half of byte i) and one power-of-two scale byte for 32
// dims, 4.25 bits a value.  These are the operands of the hardware's conversions, which take two
// codes and a scale to two fp16 or bf16 values (or back) in one instruction, exactly: a code has
// two significant bits, and with a power of two as the scale the quotient x / scale is exact,
// so a code depends on nothing but the value.
#include "fa_common.h"
#include "fa_divide.h"
#include "fa_merge.h"
#include "fa_rows_tile.h"
#include "fa_wave.h"
#include "flagattention_amd_packed.h"

namespace fa {
namespace {

__device__ inline floatx4 mfma_16x16x32(PVec<__bf16>::v8 a, PVec<__bf16>::v8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline floatx4 mfma_16x16x32(PVec<_Float16>::v8 a, PVec<_Float16>::v8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The scale 2^(byte - 127) as the conversions take it: they read the exponent bits alone, 0 as
// 2^-127 and 255 as NaN.
__device__ inline float scale_of(unsigned int byte) { return __uint_as_float(byte << 23); }

template <typename T, int kByte>
__device__ inline typename PVec<T>::v2 codes2(unsigned int w, float scale) {
  if constexpr (__is_same(T, __bf16))
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, kByte);
  else
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, kByte);
}
// The eight values of a word of codes.
template <typename T>
__device__ inline typename PVec<T>::v8 codes8(unsigned int w, float scale) {
  const auto a = codes2<T, 0>(w, scale), b = codes2<T, 1>(w, scale);
  const auto c = codes2<T, 2>(w, scale), d = codes2<T, 3>(w, scale);
  const auto lo = __builtin_shufflevector(a, b, 0, 1, 2, 3);
  const auto hi = __builtin_shufflevector(c, d, 0, 1, 2, 3);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <typename T, int kByte>
__device__ inline unsigned int to_codes2(unsigned int old, typename PVec<T>::v2 x, float scale) {
  if constexpr (__is_same(T, __bf16))
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, x, scale, kByte);
  else
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, x, scale, kByte);
}

// ---- cache write ----

template <int kCtrl>
__device__ inline unsigned int dpp_u32(unsigned int v) {
  return static_cast<unsigned int>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xF, 0xF, false));
}

constexpr int kWThreads = 256;
constexpr int kWTokens = 16;  // tokens per work-group at most

// Rows of a work-group's tokens in the cache: byte offsets of their codes and scales, -1: none.
struct RowSlots {
  long long code[kWTokens], scale[kWTokens];
};

__device__ inline void set_row(RowSlots& rows, int t, const fa_mxfp4_cache& cache, bool in,
                               long long block, long long row) {
  rows.code[t] = in ? block * cache.code_stride_0 + row * cache.code_stride_t : -1;
  rows.scale[t] = in ? block * cache.scale_stride_0 + row * cache.scale_stride_t : -1;
}

// The n-th 8-dim piece of a work-group's rows [token][head][piece].  Heads divide by a reciprocal
// and a correction: n / pieces is below 2^20.
struct Piece {
  int token, head, piece;
};
__device__ inline Piece piece_of(int n, int log_pieces, int h_kv, float h_inv) {
  Piece p;
  p.piece = n & ((1 << log_pieces) - 1);
  const int th = n >> log_pieces;
  p.token = static_cast<int>(static_cast<float>(th) * h_inv);
  p.token += th - p.token * h_kv >= h_kv ? 1 : 0;
  p.token -= th - p.token * h_kv < 0 ? 1 : 0;
  p.head = th - p.token * h_kv;
  return p;
}

// A lane holds 8 dims of a row (16 bytes in, 4 out), four neighbouring lanes a group of 32, whose
// amax they find with two lane exchanges.  blockIdx.y: K or V.  Bound by memory: it reads
// 2 bytes and writes 0.53 a value.
template <typename T>
__global__ __launch_bounds__(kWThreads) void mxfp4_write_kernel(
    const fa_mxfp4_cache cache, const T* __restrict__ key, long long key_st, long long key_sh,
    const T* __restrict__ value, long long value_st, long long value_sh, const void* slots,
    int slots64, int num_tokens, int tokens) {
  typedef typename PVec<T>::v8 T8;
  constexpr int kItems = 4;  // requested before the first is stored
  __shared__ RowSlots rows;
  const bool is_v = blockIdx.y != 0;
  const long long st = is_v ? value_st : key_st, sh = is_v ? value_sh : key_sh;
  const int tok0 = blockIdx.x * tokens;
  const T* const src = (is_v ? value : key) + tok0 * st;
  unsigned char* const codes = static_cast<unsigned char*>(is_v ? cache.v_codes : cache.k_codes);
  unsigned char* const scales = static_cast<unsigned char*>(is_v ? cache.v_scales : cache.k_scales);
  const int log_pieces = __builtin_ctz(cache.d / 8);
  const int mine = min(tokens, num_tokens - tok0);
  const int n = (mine * cache.h_kv) << log_pieces;
  const float h_inv = __builtin_amdgcn_rcpf(static_cast<float>(cache.h_kv));
  if (static_cast<int>(threadIdx.x) < mine) {
    const int t = tok0 + threadIdx.x;
    const long long slot =
        slots64 ? static_cast<const long long*>(slots)[t] : static_cast<const int*>(slots)[t];
    const long long block = slot >> __builtin_ctz(static_cast<unsigned int>(cache.block_size));
    set_row(rows, threadIdx.x, cache, slot >= 0 && block < cache.num_blocks, block,
            slot & (cache.block_size - 1));
  }
  for (int base = 0; base < n; base += kWThreads * kItems) {
    const int i0 = base + threadIdx.x;
    T8 x[kItems];
    Piece p[kItems];
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      p[j] = piece_of(min(i0 + kWThreads * j, n - 1), log_pieces, cache.h_kv, h_inv);
      x[j] = __builtin_nontemporal_load(
          reinterpret_cast<const T8*>(src + p[j].token * st + p[j].head * sh + 8 * p[j].piece));
    }
    if (base == 0) __syncthreads();  // the rows, whose slots came beside the first values
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      // bit patterns of |x|: their unsigned order is the order of the values, and NaN lies above all
      unsigned int amax = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        amax = max(amax, __float_as_uint(static_cast<float>(x[j][i])) & 0x7FFFFFFFu);
      amax = max(amax, dpp_u32<0xB1>(amax));  // quad_perm [1, 0, 3, 2]
      amax = max(amax, dpp_u32<0x4E>(amax));  // quad_perm [2, 3, 0, 1]
      // smallest e with amax <= 7 * 2^(e - 127): 7 = 1.75 * 4, so amax's own exponent less 2, and
      // one more where its fraction is above 1.75 (the addition then carries into the exponent)
      const int field = static_cast<int>((amax + 0x1FFFFFu) >> 23) - 2;
      const bool finite = amax < 0x7F800000u;
      const unsigned int e = finite ? static_cast<unsigned int>(max(field, 0)) : 255u;
      const float scale = scale_of(e);
      unsigned int w = 0u;
      if (finite) {
        w = to_codes2<T, 0>(w, __builtin_shufflevector(x[j], x[j], 0, 1), scale);
        w = to_codes2<T, 1>(w, __builtin_shufflevector(x[j], x[j], 2, 3), scale);
        w = to_codes2<T, 2>(w, __builtin_shufflevector(x[j], x[j], 4, 5), scale);
        w = to_codes2<T, 3>(w, __builtin_shufflevector(x[j], x[j], 6, 7), scale);
      }
      const long long code = rows.code[p[j].token];
      if (i0 + kWThreads * j >= n || code < 0) continue;
      *reinterpret_cast<unsigned int*>(codes + code + p[j].head * cache.code_stride_h +
                                       4 * p[j].piece) = w;
      if ((p[j].piece & 3) == 0)
        scales[rows.scale[p[j].token] + p[j].head * cache.scale_stride_h + (p[j].piece >> 2)] =
            static_cast<unsigned char>(e);
    }
  }
}

// ---- read back ----

// A lane takes 8 dims of a packed row: 4 bytes of codes in, 16 bytes out.  A wave finds the
// sequences of a quarter of the work-group's tokens, 64 starts at a time.
template <typename T>
__global__ __launch_bounds__(kWThreads) void mxfp4_gather_kernel(
    const fa_mxfp4_cache cache, const int32_t* __restrict__ block_table, long long bt_stride,
    int max_blocks, const int32_t* __restrict__ cu, int num_seqs, int total, int tokens,
    T* __restrict__ k_out, T* __restrict__ v_out) {
  typedef typename PVec<T>::v8 T8;
  constexpr int kItems = 4;
  __shared__ RowSlots rows;
  const bool is_v = blockIdx.y != 0;
  const unsigned char* const codes =
      static_cast<const unsigned char*>(is_v ? cache.v_codes : cache.k_codes);
  const unsigned char* const scales =
      static_cast<const unsigned char*>(is_v ? cache.v_scales : cache.k_scales);
  const int tok0 = blockIdx.x * tokens;
  const int mine = min(tokens, total - tok0);
  const int log_pieces = __builtin_ctz(cache.d / 8);
  const int n = (mine * cache.h_kv) << log_pieces;
  const float h_inv = __builtin_amdgcn_rcpf(static_cast<float>(cache.h_kv));
  {
    constexpr int kEach = kWTokens / (kWThreads / 64);
    const int lane = threadIdx.x & 63;
    const int first = tok0 + kEach * wave_id();
    int starts[kEach] = {};  // starts at or before the wave's tokens
    for (int base = 0; base <= num_seqs; base += 64) {
      const int c = base + lane <= num_seqs ? cu[base + lane] : 0x7FFFFFFF;
#pragma unroll
      for (int i = 0; i < kEach; ++i) starts[i] += __builtin_popcountll(__ballot(c <= first + i));
    }
    int s = -1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) s = lane == i ? starts[i] - 1 : s;
    const int t = kEach * wave_id() + lane;
    if (lane < kEach && t < mine) {
      bool in = s >= 0 && s < num_seqs;
      const int pos = in ? tok0 + t - cu[s] : -1;
      const int blk = pos >> __builtin_ctz(static_cast<unsigned int>(cache.block_size));
      in = pos >= 0 && blk < max_blocks;
      const int page = in ? block_table[s * bt_stride + blk] : -1;
      set_row(rows, t, cache, page >= 0 && page < cache.num_blocks, page,
              pos & (cache.block_size - 1));
    }
  }
  __syncthreads();
  T* const out = (is_v ? v_out : k_out) + ((static_cast<long long>(tok0) * cache.h_kv) << log_pieces) * 8;
  for (int i0 = threadIdx.x; i0 < n; i0 += kWThreads * kItems) {
    unsigned int w[kItems], e[kItems];
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const Piece p = piece_of(min(i0 + kWThreads * j, n - 1), log_pieces, cache.h_kv, h_inv);
      const long long code = rows.code[p.token], scale = rows.scale[p.token];
      w[j] = e[j] = 0u;
      if (code >= 0) {
        w[j] = __builtin_nontemporal_load(reinterpret_cast<const unsigned int*>(
            codes + code + p.head * cache.code_stride_h + 4 * p.piece));
        e[j] = scales[scale + p.head * cache.scale_stride_h + (p.piece >> 2)];
      }
    }
#pragma unroll
    for (int j = 0; j < kItems; ++j)
      if (i0 + kWThreads * j < n)
        *reinterpret_cast<T8*>(out + 8ll * (i0 + kWThreads * j)) = codes8<T>(w[j], scale_of(e[j]));
  }
}

constexpr int kMaxTokens = (1 << 28) - kWTokens;  // a grid holds less than 2^32 lanes per dimension

// Tokens per work-group of the two: fewer where they would not give every CU work.
int tokens_per_group(int64_t tokens) {
  int t = kWTokens;
  while (t > 1 && tokens < 512 * static_cast<int64_t>(t)) t /= 2;
  return t;
}

// ---- decode ----
//
// The layout of the 16-bit decode (gqa_decode_kernel): one work-group = 4 waves = one (sequence,
// KV head, block of 16 query heads, split), the split's 32-token tiles dealt round-robin to the
// waves, each with its own online softmax.  What differs is the way of a tile into the MFMAs:
//   a lane loads a quarter of one token's row (of K, and of V) for each 16-token half, D / 8
//   bytes of codes and their scale bytes, straight into registers;
//   K: the eight dims of a word are one k-step of S^T = K Q^T (the k order only has to agree
//   between the operands: k-step kk takes dims (D / 4) G + 8 kk .. + 7 of lane group G);
//   V: the values are written to a tile in LDS, private to the wave, and read back transposed.
// fp16 values are halved on the way (its largest codes, 4 * 2^14, would not fit otherwise) and
// the scores and the output doubled.
constexpr int kWaves = 4;
constexpr int kDTile = 32;
constexpr int kDRows = 16;
// P is relative to a row's running maximum.  From the first bf16 tile with a scale byte of kHuge on
// (values of 6 * 2^97 and more) it is 2^-kAbove of that: the sums of 2^16 keys of the largest finite V
// then stay within fp32.  P ends at 2^-126: weights below 2^-126 of the largest are 0, with such values
// those below 2^-110.
//
// The largest P is a power of two, whose rounding to 16 bits costs nothing.  A reference that lags up to
// 2^6 behind rescales less often, but its error against 64 bits was 2.23 / 2.26e-3 in bf16 at 512 /
// 4,096 keys where this has 2.03 / 2.03e-3, 2.77 / 2.81e-4 in fp16 where this has 2.51 / 2.52e-4; 32 ragged
// contexts of up to 4,096 keys took 20.5 us with it and take 20.7, 32 of up to 3,000 at head dim 256 23.9
// and 24.3 (0.3 less without a look at the scales), long ones the same.
constexpr float kAbove = 16.f;
constexpr unsigned int kHuge = 224;

template <int kBytes>
struct CodeWords {
  typedef unsigned int v __attribute__((ext_vector_type(kBytes / 4)));
};

// scale bytes of a lane's words of a token
template <int D>
struct ScaleOf {
  typedef unsigned char type;
};
template <>
struct ScaleOf<256> {
  typedef unsigned short type;
};

#define FA_GLOBAL __attribute__((address_space(1)))

// What a launch works out once for its work-groups.
struct DecodePlan {
  int group, turn;          // query heads per KV head; sequences that a split starts on from the last
  Divisor row_blocks, batch;  // blocks of heads per KV head; sequences
};

template <typename T, int D, bool kSmallBlocks>
__global__ __launch_bounds__(64 * kWaves, D == 64 ? 4 : D == 128 ? 3 : 2) void mxfp4_decode_kernel(
    const fa_mxfp4_decode_args a, const DecodePlan plan) {
  typedef typename PVec<T>::v8 T8;
  typedef typename PVec<T>::v4 T4;
  // Bytes per token row of the V tile: 32 more than its values, so that the 8 rows x 32 bytes of a
  // transposing read's half wave, and the 8 x 16 of a write's, lie in different banks.
  constexpr int kRowB = 2 * D + 32;
  constexpr int kTileB = kDTile * kRowB;
  constexpr int kWords = D / 32;          // words of codes per lane and token = k-steps of QK
  constexpr int kDimTiles = D / 16;
  constexpr bool kHalved = __is_same(T, _Float16);
  typedef typename CodeWords<4 * kWords>::v Words;
  typedef typename ScaleOf<D>::type ScaleBytes;
  __shared__ __attribute__((aligned(16))) unsigned char vbuf[kWaves * kTileB];
  __shared__ float ml[2 * kWaves * kDRows];
  constexpr int kMergeRow = D + 4;  // floats: 16 rows of a write lie in different banks
  static_assert(kTileB >= kDRows * kMergeRow * 4, "merge area must fit in the tile buffers");
  // At head dim 256 two tiles of loads spill, and K alone two tiles ahead was 2 .. 16% slower.
  constexpr bool kTwoTiles = D <= 128;

  const fa_mxfp4_cache& cache = a.cache;
  const int group = plan.group;
  const int hk = divide(blockIdx.x, plan.row_blocks);
  const int rb = blockIdx.x - hk * plan.row_blocks.by;
  const int split = blockIdx.z;
  // the splits of a long context start away from each other (see launch_decode_d)
  const int turned = blockIdx.y + split * plan.turn;
  const int b = turned - divide(turned, plan.batch) * a.batch;
  const int wave = wave_id();
  const int lane = threadIdx.x & 63;
  const int G = lane >> 4, c16 = lane & 15;
  const float ninf = -__builtin_inff();

  const int t0 = split * a.split_tokens;
  const int rows = min(group - rb * kDRows, kDRows);
  const int h0 = hk * group + rb * kDRows;  // query head of row 0
  // The scale is applied inside the exponent, after the maximum, so it has to be positive: a
  // negative one turns Q's signs instead, and zero makes Q zero.
  const float mag = fabsf(a.scale) * kLog2e * (kHalved ? 2.f : 1.f);
  const float scale_log2 = a.scale == 0.f ? 1.f : mag;
  uintx4 q_raw[kWords];
  {
    const T* const qrow = static_cast<const T*>(a.q) + b * a.q_stride_b +
                          (h0 + (c16 < rows ? c16 : 0)) * a.q_stride_h + (D / 4) * G;
#pragma unroll
    for (int kk = 0; kk < kWords; ++kk) q_raw[kk] = *reinterpret_cast<const uintx4*>(qrow + 8 * kk);
  }

  // ---- loads of a tile ----
  // A tile lies in one block, or in two of 16 tokens (kSmallBlocks).  Where a block's rows are is
  // worked out for 64 of the wave's blocks at once, a lane each; a tile then takes its scalars
  // from there, and its loads are a uniform base plus 32-bit lane offsets that never change.
  // (With scalar page lookups and address arithmetic per tile a step was 430 instructions.)
  constexpr int kBlocks = kSmallBlocks ? 2 : 1;  // per tile
  constexpr int kBlockKeys = kDTile / kBlocks;
  constexpr int kBatch = 64 / kBlocks;           // tiles worked out at once
  const FA_GLOBAL unsigned char* const kc =
      (const FA_GLOBAL unsigned char*)cache.k_codes + hk * cache.code_stride_h;
  const FA_GLOBAL unsigned char* const vc =
      (const FA_GLOBAL unsigned char*)cache.v_codes + hk * cache.code_stride_h;
  const FA_GLOBAL unsigned char* const ks =
      (const FA_GLOBAL unsigned char*)cache.k_scales + hk * cache.scale_stride_h;
  const FA_GLOBAL unsigned char* const vs =
      (const FA_GLOBAL unsigned char*)cache.v_scales + hk * cache.scale_stride_h;
  const int32_t* const bt_row = a.block_table + static_cast<long long>(b) * a.bt_stride_b;
  const unsigned int code_t = static_cast<unsigned int>(cache.code_stride_t);
  const unsigned int scale_t = static_cast<unsigned int>(cache.scale_stride_t);
  unsigned int code_lane[2], scale_lane[2];  // of a block's first and second 16 tokens
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = c16 + (kSmallBlocks ? 0 : 16 * h);
    code_lane[h] = r * code_t + (D / 8) * G;
    scale_lane[h] = r * scale_t + (D / 4) * G / FA_MXFP4_GROUP;
  }
  unsigned int at_c[2], at_s[2];  // this lane's block: offsets of its codes and scales
  int at_keys = 0;                // and how many keys it has
  const int bs_shift = __builtin_ctz(static_cast<unsigned int>(cache.block_size));
  auto start_of = [&](int i0) -> int {  // this lane's block among those of the wave's tiles i0, ...
    return t0 + kDTile * (wave + kWaves * (i0 + lane / kBlocks)) + kBlockKeys * (lane % kBlocks);
  };
  auto block_id = [&](int i0) -> int {
    const int blk = start_of(i0) >> bs_shift;
    return blk < a.max_blocks_per_seq ? bt_row[blk] : -1;
  };
  // The length, the first block ids and Q are requested together; only the tiles wait for them.
  int next_id = block_id(0);
  const int seqlen = min(sload(a.seqlens + b), 1 << 30);  // positions stay in 32 bits
  const int t1 = split + 1 == a.num_splits ? seqlen : min(t0 + a.split_tokens, seqlen);
  const int ntok = max(0, t1 - t0);
  const int ntiles = cdiv(ntok, kDTile);
  if (ntiles == 0 && a.num_splits > 1) {    // the merge does not look at an empty split's rows
    if (threadIdx.x < rows)
      a.lse_part[(static_cast<long long>(b) * a.h_q + h0 + threadIdx.x) * a.num_splits + split] =
          ninf;
    return;
  }

  auto work_out = [&](int i0, int block) {
    const int start = start_of(i0);
    const int id = start < t1 ? block : -1;
    const bool in = id >= 0 && id < cache.num_blocks;
    // a block outside the cache: the first one instead, all masked
    const long long page = in ? id : 0;
    const int row = in ? start & (cache.block_size - 1) : 0;
    const long long c = page * cache.code_stride_0 + row * cache.code_stride_t;
    const long long sc = page * cache.scale_stride_0 + row * cache.scale_stride_t;
    at_c[0] = static_cast<unsigned int>(c);
    at_c[1] = static_cast<unsigned int>(c >> 32);
    at_s[0] = static_cast<unsigned int>(sc);
    at_s[1] = static_cast<unsigned int>(sc >> 32);
    at_keys = in ? min(t1 - start, kBlockKeys) : 0;
  };
  auto lane_of = [&](unsigned int v, int l) -> unsigned int {
    return static_cast<unsigned int>(__builtin_amdgcn_readlane(static_cast<int>(v), l));
  };
  struct Tile {
    Words k[2], v[2];
    ScaleBytes ks[2], vs[2];
    int keys[kBlocks];  // keys of each block, from its first token on (uniform)
  };
  auto base_of = [&](unsigned int (&at)[2], int l) -> unsigned long long {
    return (static_cast<unsigned long long>(lane_of(at[1], l)) << 32) | lane_of(at[0], l);
  };
  // Seen afresh, a lane offset stays 32 bits beside a scalar base: hoisted as 64 bits it costs an
  // addition per load and twice the registers.
  auto afresh = [](unsigned int v) -> unsigned int {
    asm volatile("" : "+v"(v));
    return v;
  };
  auto issue_k = [&](Tile& x, int i) {  // i: tile of the batch
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int l = kBlocks * i + (kSmallBlocks ? h : 0);
      const FA_GLOBAL unsigned char *const c = kc + base_of(at_c, l), *const sc = ks + base_of(at_s, l);
      x.k[h] = __builtin_nontemporal_load((const FA_GLOBAL Words*)(c + afresh(code_lane[h])));
      x.ks[h] = *(const FA_GLOBAL ScaleBytes*)(sc + afresh(scale_lane[h]));
    }
  };
  auto issue_v = [&](Tile& x, int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int l = kBlocks * i + (kSmallBlocks ? h : 0);
      const FA_GLOBAL unsigned char *const c = vc + base_of(at_c, l), *const sc = vs + base_of(at_s, l);
      x.v[h] = __builtin_nontemporal_load((const FA_GLOBAL Words*)(c + afresh(code_lane[h])));
      x.vs[h] = *(const FA_GLOBAL ScaleBytes*)(sc + afresh(scale_lane[h]));
    }
  };
  auto keys_of = [&](Tile& x, int i) {
#pragma unroll
    for (int j = 0; j < kBlocks; ++j) x.keys[j] = __builtin_amdgcn_readlane(at_keys, kBlocks * i + j);
  };
  auto issue = [&](Tile& x, int i) {
    keys_of(x, i);
    issue_k(x, i);
    issue_v(x, i);
  };
  // the scale of word kk of a lane, from its scale bytes
  auto word_scale = [&](ScaleBytes bytes, int kk) -> float {
    unsigned int e = D == 256 && kk >= 4 ? bytes >> 8 : bytes & 255;
    if (kHalved) e = e == 255u ? e : max(e, 1u) - 1u;
    return scale_of(e);
  };

  auto largest = [](ScaleBytes bytes) -> unsigned int {
    return D == 256 ? max(bytes & 255u, static_cast<unsigned int>(bytes) >> 8) : bytes;
  };

  // Q^T operand: row c16, dims (D / 4) G + 8 kk ..; rows past the last are zeros
  T8 qf[kWords];
  auto take_q = [&] {
    const bool row_ok = c16 < rows && a.scale != 0.f;
    const unsigned int sign = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int kk = 0; kk < kWords; ++kk) {
      uintx4 w = q_raw[kk];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = row_ok ? w[i] ^ sign : 0u;
      qf[kk] = __builtin_bit_cast(T8, w);
    }
  };
  float m_run = ninf, l_run = 0.f, above = 0.f;  // see kAbove
  floatx4 acc[kDimTiles];
#pragma unroll
  for (int dt = 0; dt < kDimTiles; ++dt) acc[dt] = floatx4{};
  unsigned char* const vb = vbuf + wave * kTileB;

  // A tile is taken out of its registers, which the wave's tile after the next is then requested
  // into: one tile of loads is in flight during all of a step, two during most of it.
  auto step = [&](Tile& x, int i, bool more) {
    // keys of the tile's halves (uniform)
    const int keys0 = kSmallBlocks ? x.keys[0] : min(x.keys[0], 16);
    const int keys1 = kSmallBlocks ? x.keys[kBlocks - 1] : x.keys[0] - 16;
    const bool whole = min(keys0, keys1) >= 16;
    floatx4 s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = floatx4{};
#pragma unroll
      for (int kk = 0; kk < kWords; ++kk)
        s[h] = mfma_16x16x32(codes8<T>(x.k[h][kk], word_scale(x.ks[h], kk)), qf[kk], s[h]);
      __builtin_amdgcn_sched_barrier(0);
    }
    constexpr int kAhead = kTwoTiles ? 2 : 1;
    if constexpr (!kTwoTiles) {
      if (more) issue_k(x, i + kAhead);
    }
    ScaleBytes vse[2] = {x.vs[0], x.vs[1]};
    if (!whole) {
      // a masked key's weight is 0, which does not hide a NaN: its scales become the smallest
      if (c16 >= keys0) vse[0] = 0;
      if (c16 >= keys1) vse[1] = 0;
    }
    bool huge = false;  // uniform
    if constexpr (!kHalved) huge = __ballot(max(largest(vse[0]), largest(vse[1])) >= kHuge) != 0ull;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int kk = 0; kk < kWords; ++kk)
        *reinterpret_cast<T8*>(vb + (16 * h + c16) * kRowB + 16 * (kWords * G + kk)) =
            codes8<T>(x.v[h][kk], word_scale(vse[h], kk));
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kTwoTiles) {
      if (more) issue(x, i + kAhead);
    } else {
      if (more) {
        keys_of(x, i + kAhead);
        issue_v(x, i + kAhead);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    // softmax down the column: keys 16h + 4G + i of the tile
    if (!whole) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int left = (h == 0 ? keys0 : keys1) - 4 * G;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[h][i] = i < left ? s[h][i] : ninf;
      }
    }
    float tmax = s[0][0];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) tmax = fmaxf(tmax, s[h][i]);
    tmax = max_xor32(max_xor16(tmax)) * scale_log2;
    const float up_by = huge ? kAbove : above;  // uniform
    const bool up = tmax + up_by > m_run || up_by != above;
    if (__ballot(up) != 0ull) {  // uniform
      // only the rows that are up move: a row's result does not depend on those beside it
      const float m_new = up ? fmaxf(m_run - above, tmax) + up_by : m_run;
      const float alpha = !up || m_new == ninf ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      above = up_by;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < kDimTiles; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[dt][i] *= alpha;
    }
    const float nm = m_run == ninf ? 0.f : -m_run;
    float c = scale_log2;
    // a fused multiply-add does not round the product that a large reference is made of
    const bool far = fabsf(nm) > 1024.f;
    if (__ballot(far) != 0ull) {  // uniform
      const float by = far ? c : 1.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[h][i] *= by;
      c = far ? 1.f : c;
    }
    float psum = 0.f;
    T8 pb;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][i], c, nm));
        psum += p;
        pb[4 * h + i] = static_cast<T>(p);
      }
    l_run += psum;
    __builtin_amdgcn_sched_barrier(0);
    const unsigned char* const vr = vb + (4 * G + (c16 >> 2)) * kRowB + 8 * (c16 & 3);
#pragma unroll
    for (int dt = 0; dt < kDimTiles; ++dt) {
      const T4 lo = lds_tr_read4<T>(vr + 32 * dt);
      const T4 hi = lds_tr_read4<T>(vr + 16 * kRowB + 32 * dt);
      const T8 va = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      acc[dt] = mfma_16x16x32(va, pb, acc[dt]);
      if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  };

  const int mine = wave < ntiles ? (ntiles - wave + kWaves - 1) / kWaves : 0;  // tiles dealt in turn
  for (int i0 = 0; i0 < mine; i0 += kBatch) {
    const int n = min(mine - i0, kBatch);
    Tile x;
    work_out(i0, next_id);
    issue(x, 0);
    if (i0 + kBatch < mine) next_id = block_id(i0 + kBatch);
    if (i0 == 0) take_q();
    int i = 0;
    if constexpr (!kTwoTiles) {
      for (; i + 1 < n; ++i) step(x, i, true);
      step(x, i, false);
    } else {
      Tile y;
      if (n > 3) {
        // Without a condition in front of a request the compiler knows how many are in flight, and
        // waits for a tile without waiting for the one behind it.
        issue(y, 1);
        do {
          step(x, i, true);
          step(y, i + 1, true);
          i += 2;
        } while (i + 3 < n);
      } else if (n > 1) {
        issue(y, 1);
      }
      for (;;) {
        step(x, i, i + 2 < n);
        if (++i >= n) break;
        step(y, i, false);
        if (++i >= n) break;
      }
    }
  }

  // ---- merge the waves' states ----
  const float l_col = sum_xor32(sum_xor16(l_run));
  __syncthreads();
  float* const om = reinterpret_cast<float*>(vbuf);  // [wave][16][kMergeRow]
  if (G == 0) {
    ml[wave * kDRows + c16] = m_run;
    ml[(kWaves + wave) * kDRows + c16] = l_col;
  }
  if (c16 < rows) {
#pragma unroll
    for (int dt = 0; dt < kDimTiles; ++dt)
      *reinterpret_cast<floatx4*>(om + (wave * kDRows + c16) * kMergeRow + 16 * dt + 4 * G) = acc[dt];
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < rows * (D / 4); idx += 64 * kWaves) {
    const int r = idx / (D / 4), d = 4 * (idx - r * (D / 4));
    float mw[kWaves], M = ninf;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      mw[w] = ml[w * kDRows + r];
      M = fmaxf(M, mw[w]);
    }
    // no visible key: every weight and sum is 0; NaN sums stay NaN.  In bf16 the waves' sums are taken at
    // a quarter: each may be as large as fp32 holds (see kAbove).
    const float m_use = M == ninf ? 0.f : M + (kHalved ? 0.f : 2.f);
    float L = 0.f;
    floatx4 O = floatx4{};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(mw[w] - m_use);
      L += ml[(kWaves + w) * kDRows + r] * f;
      const floatx4 o = *reinterpret_cast<const floatx4*>(om + (w * kDRows + r) * kMergeRow + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) O[i] += o[i] * f;
    }
    const float inv = L == 0.f ? 0.f : (kHalved ? 2.f : 1.f) / L;
#pragma unroll
    for (int i = 0; i < 4; ++i) O[i] *= inv;
    const int h = h0 + r;
    if (a.num_splits == 1) {
      T4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = static_cast<T>(O[i]);
      *reinterpret_cast<T4*>(static_cast<T*>(a.out) + b * a.o_stride_b + h * a.o_stride_h + d) = w;
    } else {
      const long long prow = (static_cast<long long>(b) * a.h_q + h) * a.num_splits + split;
      *reinterpret_cast<floatx4*>(a.o_part + prow * D + d) = O;
      // the merge takes the largest lse, which a NaN would not be
      if (d == 0)
        a.lse_part[prow] = L == 0.f ? ninf : L == L ? (m_use + log2f(L)) * kLn2 : -ninf;
    }
  }
}

template <typename T, int D>
void launch_decode_d(const fa_mxfp4_decode_args* a, hipStream_t stream) {
  const int group = a->h_q / a->cache.h_kv;
  // Heads vary fastest and splits slowest: work-groups are dealt round-robin over 8 XCDs, and the
  // late splits of ragged contexts are empty (with splits fastest, 8 of them, one XCD had all the
  // last ones: 33.7 us instead of 27.3 at 32 sequences of 97 .. 4,096 keys).
  const dim3 grid(a->cache.h_kv * cdiv(group, kDRows), a->batch, a->num_splits);
  const DecodePlan plan{group, cdiv(a->batch, a->num_splits), divisor(cdiv(group, kDRows)),
                        divisor(a->batch)};
  if (a->cache.block_size < kDTile)
    hipLaunchKernelGGL((mxfp4_decode_kernel<T, D, true>), grid, dim3(64 * kWaves), 0, stream, *a, plan);
  else
    hipLaunchKernelGGL((mxfp4_decode_kernel<T, D, false>), grid, dim3(64 * kWaves), 0, stream, *a,
                       plan);
}

template <typename T>
int launch_decode(const fa_mxfp4_decode_args* a, hipStream_t stream) {
  if (a->cache.d == 64)
    launch_decode_d<T, 64>(a, stream);
  else if (a->cache.d == 128)
    launch_decode_d<T, 128>(a, stream);
  else
    launch_decode_d<T, 256>(a, stream);
  FA_CHECK_HIP(hipGetLastError());
  return FA_OK;
}

// Splits of `groups` (sequence, KV head, block of heads) triples of up to max_len keys: the cheapest
// by a model of the launch, in us.  By itself a work-group takes `step` for 128 keys; together they
// take the time of their bytes, contexts being three quarters of the longest on average, and then
// some of the last one's steps (fewer where a CU has two or more unsplit ones, which fill each
// other's ends); past the first on a CU a work-group costs 1.0 for its start and end, the merge 3.5
// and a little per split.  CUs hold a whole number of work-groups: the count per CU is taken halfway
// to the next whole one.  Measured: 1,024 work-groups of one key take 7.0 a call, 256 of them 3.9; a
// call in 1 / 2 / 3 / 4 / 5 / 8 splits at D = 128, 8 KV heads: 32 ragged contexts of up to 4,096 keys
// 26.9 / 23.8 / 22.4 / 21.4 / 19.5 / 23.4, 64 x 8,192 95.7 / 103.5 / 104.4 / 105.8 / 108.9 / 116; at
// D = 256, 4 KV heads, 32 of up to 3,000 33.0 / 23.0 / 28.8 / 24.5 / 22.2 / 26.2.  The constants are a
// fit to 33 such calls in up to 48 splits each (D 64 .. 256, 1 .. 1,024 triples, 800 .. 131,001 keys):
// the pick takes 4% longer than the best count on average and 12% at most; for 12 other calls 5% and
// 23% (40 x 2,000 keys, D = 256).
int choose_splits(int64_t groups, int d, int64_t max_len, int64_t cus) {
  const double step = d == 64 ? 0.46 : d == 128 ? 0.89 : 0.87;
  const double per_cu = static_cast<double>(groups) / static_cast<double>(cus);
  const double bytes = 0.48 * d / 128 * per_cu * static_cast<double>(max_len) / 128 * 0.75;
  double best = 0;
  int pick = 1;
  for (int s : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 16, 20, 24, 32, 48, 64, 96, 128}) {
    if (s > 1 && max_len < 128 * static_cast<int64_t>(s)) break;
    const double alone = step * static_cast<double>((max_len + 128 * s - 1) / (128 * s));
    const double even = per_cu * s, whole = static_cast<double>((groups * s + cus - 1) / cus);
    const double k = even + 0.51 * (whole - even);
    const double shared = bytes * (k > 1 ? k / even : 1) + alone * (per_cu < 2 ? 0.44 : 0.19);
    const double t = (alone > shared ? alone : shared) + (k > 1 ? k - 1 : 0) +
                     (s > 1 ? 3.5 + 0.03 * s : 0);
    if (s == 1 || t < best) {
      best = t;
      pick = s;
    }
  }
  return pick;
}

bool aligned(const void* p, int64_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0;
}

int check_cache(const fa_mxfp4_cache* c) {
  FA_CHECK_ARG(c != nullptr, "cache is NULL");
  FA_CHECK_ARG(c->d == 64 || c->d == 128 || c->d == 256, "head dim %d not in {64, 128, 256}", c->d);
  FA_CHECK_ARG(c->h_kv >= 1 && c->h_kv <= 65535, "h_kv %d not in [1, 65535]", c->h_kv);
  FA_CHECK_ARG(c->block_size >= 16 && (c->block_size & (c->block_size - 1)) == 0,
               "block_size %d is not a power of two of at least 16", c->block_size);
  FA_CHECK_ARG(c->num_blocks >= 1 && c->num_blocks <= INT32_MAX, "num_blocks %lld invalid",
               static_cast<long long>(c->num_blocks));
  FA_CHECK_ARG(c->k_codes && c->k_scales && c->v_codes && c->v_scales, "NULL cache pointer");
  const int64_t ca = c->d / 8 < 16 ? c->d / 8 : 16, sa = c->d == 256 ? 2 : 1;
  FA_CHECK_ARG(aligned(c->k_codes, ca) && aligned(c->v_codes, ca) && c->code_stride_0 % ca == 0 &&
                   c->code_stride_h % ca == 0 && c->code_stride_t % ca == 0,
               "rows of codes must be %d-byte aligned", static_cast<int>(ca));
  FA_CHECK_ARG(aligned(c->k_scales, sa) && aligned(c->v_scales, sa) && c->scale_stride_0 % sa == 0 &&
                   c->scale_stride_h % sa == 0 && c->scale_stride_t % sa == 0,
               "rows of scales must be %d-byte aligned", static_cast<int>(sa));
  // 32-bit lane offsets inside 16 tokens
  FA_CHECK_ARG(c->code_stride_t >= 0 && c->code_stride_t < (1ll << 27) && c->scale_stride_t >= 0 &&
                   c->scale_stride_t < (1ll << 27),
               "token strides of the cache must be in [0, 2^27)");
  return FA_OK;
}

int check_decode(const fa_mxfp4_decode_args* a) {
  FA_CHECK_ARG(a != nullptr, "args is NULL");
  const int rc = check_cache(&a->cache);
  if (rc != FA_OK) return rc;
  const int h_kv = a->cache.h_kv;
  FA_CHECK_ARG(a->batch >= 1 && a->batch <= 65535 && a->h_q >= 1, "batch %d / h_q %d invalid",
               a->batch, a->h_q);
  FA_CHECK_ARG(a->h_q % h_kv == 0, "h_q %d is not a multiple of h_kv %d", a->h_q, h_kv);
  FA_CHECK_ARG(static_cast<long long>(h_kv) * cdiv(a->h_q / h_kv, kDRows) <= 65535,
               "grid too large: h_kv x ceil(group / 16) must be <= 65535");
  FA_CHECK_ARG(a->dtype == 0 || a->dtype == 1, "dtype %d is not 0 (fp16) or 1 (bf16)", a->dtype);
  FA_CHECK_ARG(a->num_splits >= 1 && a->num_splits <= 65535 && a->split_tokens >= 1 &&
                   (a->num_splits == 1 || a->split_tokens % kDTile == 0) &&
                   static_cast<int64_t>(a->num_splits - 1) * a->split_tokens <= (1 << 30),
               "num_splits %d of %d tokens invalid", a->num_splits, a->split_tokens);
  FA_CHECK_ARG(a->num_splits == 1 || (a->o_part && a->lse_part),
               "num_splits %d > 1 needs o_part and lse_part", a->num_splits);
  // the merge takes up to a work-group of 256 lanes for a row
  FA_CHECK_ARG(a->num_splits == 1 || static_cast<int64_t>(a->batch) * a->h_q < (1 << 24),
               "batch %d x h_q %d is 2^24 or more, too many rows for splits", a->batch, a->h_q);
  FA_CHECK_ARG(a->q && a->out && a->block_table && a->seqlens && a->max_blocks_per_seq >= 1,
               "NULL q / out / block_table / seqlens or no block per sequence");
  FA_CHECK_ARG(aligned(a->q, 16) && a->q_stride_b % 8 == 0 && a->q_stride_h % 8 == 0,
               "q rows must be 16-byte aligned");
  FA_CHECK_ARG(aligned(a->out, 8) && a->o_stride_b % 4 == 0 && a->o_stride_h % 4 == 0,
               "out rows must be 8-byte aligned");
  return FA_OK;
}

}  // namespace
}  // namespace fa

extern "C" int64_t fa_mxfp4_cache_size(void) { return static_cast<int64_t>(sizeof(fa_mxfp4_cache)); }

extern "C" int64_t fa_mxfp4_decode_args_size(void) {
  return static_cast<int64_t>(sizeof(fa_mxfp4_decode_args));
}

extern "C" int fa_mxfp4_cache_write(const fa_mxfp4_cache* cache, const void* key,
                                    int64_t key_stride_t, int64_t key_stride_h, const void* value,
                                    int64_t value_stride_t, int64_t value_stride_h,
                                    const void* slots, int32_t slots64, int32_t num_tokens,
                                    int32_t dtype, void* stream) {
  const int rc = fa::check_cache(cache);
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(num_tokens >= 0, "num_tokens %d < 0", num_tokens);
  FA_CHECK_ARG(dtype == 0 || dtype == 1, "dtype %d is not 0 (fp16) or 1 (bf16)", dtype);
  if (num_tokens == 0) return FA_OK;
  FA_CHECK_ARG(key && value && slots, "NULL pointer");
  FA_CHECK_ARG(fa::aligned(key, 16) && fa::aligned(value, 16) && key_stride_t % 8 == 0 &&
                   key_stride_h % 8 == 0 && value_stride_t % 8 == 0 && value_stride_h % 8 == 0,
               "key / value rows must be 16-byte aligned");
  FA_CHECK_ARG(static_cast<int64_t>(num_tokens) * cache->h_kv <= INT32_MAX,
               "num_tokens %d x h_kv %d is 2^31 or more", num_tokens, cache->h_kv);
  FA_CHECK_ARG(num_tokens <= fa::kMaxTokens, "num_tokens %d is more than 2^28 - 16", num_tokens);
  const int tokens = fa::tokens_per_group(num_tokens);
  const dim3 grid(static_cast<unsigned>(fa::cdiv(num_tokens, tokens)), 2);
  const hipStream_t s = static_cast<hipStream_t>(stream);
#define FA_WRITE(T)                                                                            \
  hipLaunchKernelGGL(fa::mxfp4_write_kernel<T>, grid, dim3(fa::kWThreads), 0, s, *cache,        \
                     static_cast<const T*>(key), static_cast<long long>(key_stride_t),          \
                     static_cast<long long>(key_stride_h), static_cast<const T*>(value),        \
                     static_cast<long long>(value_stride_t),                                    \
                     static_cast<long long>(value_stride_h), slots, slots64, num_tokens, tokens)
  if (dtype == 1)
    FA_WRITE(__bf16);
  else
    FA_WRITE(_Float16);
#undef FA_WRITE
  FA_CHECK_HIP(hipGetLastError());
  return FA_OK;
}

extern "C" int fa_mxfp4_gather(const fa_mxfp4_cache* cache, const int32_t* block_table,
                               int64_t bt_stride_b, int32_t max_blocks_per_seq,
                               const int32_t* cu_seqlens, int32_t num_seqs, int32_t total,
                               void* k_out, void* v_out, int32_t dtype, void* stream) {
  const int rc = fa::check_cache(cache);
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(total >= 0 && num_seqs >= 0, "total %d / num_seqs %d < 0", total, num_seqs);
  FA_CHECK_ARG(dtype == 0 || dtype == 1, "dtype %d is not 0 (fp16) or 1 (bf16)", dtype);
  if (total == 0) return FA_OK;
  FA_CHECK_ARG(max_blocks_per_seq >= 0, "max_blocks_per_seq %d < 0", max_blocks_per_seq);
  FA_CHECK_ARG(cu_seqlens && k_out && v_out &&
                   (num_seqs == 0 || max_blocks_per_seq == 0 || block_table),
               "NULL pointer");
  FA_CHECK_ARG(fa::aligned(k_out, 16) && fa::aligned(v_out, 16), "outputs must be 16-byte aligned");
  FA_CHECK_ARG(static_cast<int64_t>(total) * cache->h_kv <= INT32_MAX,
               "total %d x h_kv %d is 2^31 or more", total, cache->h_kv);
  FA_CHECK_ARG(total <= fa::kMaxTokens, "total %d is more than 2^28 - 16", total);
  // every wave goes through the starts
  FA_CHECK_ARG(num_seqs <= 65535, "num_seqs %d is more than 65535, too many sequences", num_seqs);
  const int tokens = fa::tokens_per_group(total);
  const dim3 grid(static_cast<unsigned>(fa::cdiv(total, tokens)), 2);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == 1)
    hipLaunchKernelGGL(fa::mxfp4_gather_kernel<__bf16>, grid, dim3(fa::kWThreads), 0, s, *cache,
                       block_table, static_cast<long long>(bt_stride_b), max_blocks_per_seq,
                       cu_seqlens, num_seqs, total, tokens, static_cast<__bf16*>(k_out),
                       static_cast<__bf16*>(v_out));
  else
    hipLaunchKernelGGL(fa::mxfp4_gather_kernel<_Float16>, grid, dim3(fa::kWThreads), 0, s, *cache,
                       block_table, static_cast<long long>(bt_stride_b), max_blocks_per_seq,
                       cu_seqlens, num_seqs, total, tokens, static_cast<_Float16*>(k_out),
                       static_cast<_Float16*>(v_out));
  FA_CHECK_HIP(hipGetLastError());
  return FA_OK;
}

extern "C" int fa_mxfp4_decode_plan(int32_t batch, int32_t h_q, int32_t h_kv, int32_t d,
                                    int32_t max_len, int32_t cu_count, fa_mxfp4_decode_args* a) {
  FA_CHECK_ARG(a != nullptr, "args is NULL");
  FA_CHECK_ARG(batch >= 1 && h_q >= 1 && h_kv >= 1 && h_q % h_kv == 0 && max_len >= 1 &&
                   cu_count >= 1 && (d == 64 || d == 128 || d == 256),
               "batch %d / h_q %d / h_kv %d / d %d / max_len %d / cu_count %d invalid", batch, h_q,
               h_kv, d, max_len, cu_count);
  const int s = fa::choose_splits(
      static_cast<int64_t>(batch) * h_kv * fa::cdiv(h_q / h_kv, fa::kDRows), d, max_len, cu_count);
  const int64_t each = (static_cast<int64_t>(max_len) + s - 1) / s;
  a->split_tokens = static_cast<int32_t>((each + fa::kDTile - 1) / fa::kDTile * fa::kDTile);
  a->num_splits = static_cast<int32_t>((static_cast<int64_t>(max_len) + a->split_tokens - 1) /
                                       a->split_tokens);
  return FA_OK;
}

extern "C" int fa_mxfp4_decode(const fa_mxfp4_decode_args* a, void* stream) {
  const int rc = fa::check_decode(a);
  if (rc != FA_OK) return rc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == 1 ? fa::launch_decode<__bf16>(a, s) : fa::launch_decode<_Float16>(a, s);
}

extern "C" int fa_mxfp4_combine(const fa_mxfp4_decode_args* a, void* stream) {
  const int rc = fa::check_decode(a);
  if (rc != FA_OK) return rc;
  FA_CHECK_ARG(a->o_part && a->lse_part, "combine needs o_part and lse_part");
  FA_CHECK_ARG(static_cast<int64_t>(a->batch) * a->h_q < (1 << 24),
               "batch %d x h_q %d is 2^24 or more, too many rows for splits", a->batch, a->h_q);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const fa::MergeArgs m{a->o_part, a->lse_part, a->out, nullptr, a->o_stride_b, a->o_stride_h,
                        static_cast<int>(static_cast<int64_t>(a->batch) * a->h_q), a->h_q,
                        a->num_splits};
  if (a->dtype == 1)
    fa::launch_merge<__bf16>(m, a->cache.d, s);
  else
    fa::launch_merge<_Float16>(m, a->cache.d, s);
  FA_CHECK_HIP(hipGetLastError());
  return FA_OK;
}
