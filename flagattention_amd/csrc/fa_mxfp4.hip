// A paged K/V cache in 4 bits for gfx950: its writer, its reader and one-token decode over it.
//
// Rows hold e2m1 codes (dim 2i in the low half of byte i) and one power-of-two scale byte for 32
// dims, 4.25 bits a value.  These are the operands of the hardware's conversions, which take two
// codes and a scale to two fp16 or bf16 values (or back) in one instruction, exactly: a code has
// two significant bits, and with a power of two as the scale the quotient x / scale is exact,
// so a code depends on nothing but the value.
#include "fa_common.h"
#include "fa_wave.h"
#include "flagattention_amd_packed.h"

namespace fa {
namespace {

template <typename T>
struct FVec {
  typedef T v8 __attribute__((ext_vector_type(8)));
  typedef T v4 __attribute__((ext_vector_type(4)));
  typedef T v2 __attribute__((ext_vector_type(2)));
};

__device__ inline floatx4 mfma_16x16x32(FVec<__bf16>::v8 a, FVec<__bf16>::v8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline floatx4 mfma_16x16x32(FVec<_Float16>::v8 a, FVec<_Float16>::v8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <typename T>
__device__ inline typename FVec<T>::v4 lds_tr4(const unsigned char* p) {
  typedef short shortx4 __attribute__((ext_vector_type(4)));
  const shortx4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((FA_LDS shortx4*)(p));
  return __builtin_bit_cast(typename FVec<T>::v4, v);
}

// The scale 2^(byte - 127) as the conversions take it: they read the exponent bits alone, 0 as
// 2^-127 and 255 as NaN.
__device__ inline float scale_of(unsigned int byte) { return __uint_as_float(byte << 23); }

template <typename T, int kByte>
__device__ inline typename FVec<T>::v2 codes2(unsigned int w, float scale) {
  if constexpr (__is_same(T, __bf16))
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, kByte);
  else
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, kByte);
}
// The eight values of a word of codes.
template <typename T>
__device__ inline typename FVec<T>::v8 codes8(unsigned int w, float scale) {
  const auto a = codes2<T, 0>(w, scale), b = codes2<T, 1>(w, scale);
  const auto c = codes2<T, 2>(w, scale), d = codes2<T, 3>(w, scale);
  const auto lo = __builtin_shufflevector(a, b, 0, 1, 2, 3);
  const auto hi = __builtin_shufflevector(c, d, 0, 1, 2, 3);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <typename T, int kByte>
__device__ inline unsigned int to_codes2(unsigned int old, typename FVec<T>::v2 x, float scale) {
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
constexpr int kWItems = 4;  // 8-dim pieces per thread, all requested before the first is stored

// A lane holds 8 dims of a row (16 bytes in, 4 out), four neighbouring lanes a group of 32, whose
// amax they find with two lane exchanges.  blockIdx.y: K or V.  Bound by memory: it reads
// 2 bytes and writes 0.53 a value.
template <typename T>
__global__ __launch_bounds__(kWThreads) void mxfp4_write_kernel(
    const fa_mxfp4_cache cache, const T* __restrict__ key, long long key_st, long long key_sh,
    const T* __restrict__ value, long long value_st, long long value_sh, const void* slots,
    int slots64, int num_tokens) {
  typedef typename FVec<T>::v8 T8;
  const bool is_v = blockIdx.y != 0;
  const T* const src = is_v ? value : key;
  const long long st = is_v ? value_st : key_st, sh = is_v ? value_sh : key_sh;
  unsigned char* const codes = static_cast<unsigned char*>(is_v ? cache.v_codes : cache.k_codes);
  unsigned char* const scales = static_cast<unsigned char*>(is_v ? cache.v_scales : cache.k_scales);
  const int pieces = cache.d / 8;
  const int log_pieces = __builtin_ctz(pieces);
  const long long total = static_cast<long long>(num_tokens) * cache.h_kv * pieces;
  const long long first = static_cast<long long>(blockIdx.x) * (kWThreads * kWItems) + threadIdx.x;
  T8 x[kWItems];
  long long slot[kWItems];
  int head[kWItems], piece[kWItems];
#pragma unroll
  for (int j = 0; j < kWItems; ++j) {
    const long long i = min(first + j * kWThreads, total - 1);
    piece[j] = static_cast<int>(i) & (pieces - 1);
    const unsigned int th = static_cast<unsigned int>(i >> log_pieces);  // below 2^31 (host)
    const unsigned int tok = th / static_cast<unsigned int>(cache.h_kv);
    head[j] = static_cast<int>(th - tok * cache.h_kv);
    slot[j] = slots64 ? static_cast<const long long*>(slots)[tok]
                      : static_cast<const int*>(slots)[tok];
    x[j] = __builtin_nontemporal_load(
        reinterpret_cast<const T8*>(src + tok * st + head[j] * sh + 8 * piece[j]));
  }
#pragma unroll
  for (int j = 0; j < kWItems; ++j) {
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
    const long long blk = slot[j] >= 0 ? slot[j] / cache.block_size : -1;
    if (first + j * kWThreads >= total || blk < 0 || blk >= cache.num_blocks) continue;
    const long long row = slot[j] - blk * cache.block_size;
    *reinterpret_cast<unsigned int*>(codes + blk * cache.code_stride_0 +
                                     head[j] * cache.code_stride_h + row * cache.code_stride_t +
                                     4 * piece[j]) = w;
    if ((piece[j] & 3) == 0)
      scales[blk * cache.scale_stride_0 + head[j] * cache.scale_stride_h +
             row * cache.scale_stride_t + (piece[j] >> 2)] = static_cast<unsigned char>(e);
  }
}

// ---- read back ----

// A lane takes 8 dims of a packed row: 4 bytes of codes in, 16 bytes out.
template <typename T>
__global__ __launch_bounds__(kWThreads) void mxfp4_gather_kernel(
    const fa_mxfp4_cache cache, const int32_t* __restrict__ block_table, long long bt_stride,
    int max_blocks, const int32_t* __restrict__ cu, int num_seqs, int total, T* __restrict__ k_out,
    T* __restrict__ v_out) {
  typedef typename FVec<T>::v8 T8;
  const bool is_v = blockIdx.y != 0;
  const unsigned char* const codes =
      static_cast<const unsigned char*>(is_v ? cache.v_codes : cache.k_codes);
  const unsigned char* const scales =
      static_cast<const unsigned char*>(is_v ? cache.v_scales : cache.k_scales);
  T* const out = is_v ? v_out : k_out;
  const int pieces = cache.d / 8;
  const int log_pieces = __builtin_ctz(pieces);
  const long long items = static_cast<long long>(total) * cache.h_kv * pieces;
  const long long i = static_cast<long long>(blockIdx.x) * kWThreads + threadIdx.x;
  if (i >= items) return;
  const int piece = static_cast<int>(i) & (pieces - 1);
  const unsigned int th = static_cast<unsigned int>(i >> log_pieces);
  const int tok = static_cast<int>(th / static_cast<unsigned int>(cache.h_kv));
  const int head = static_cast<int>(th - static_cast<unsigned int>(tok) * cache.h_kv);
  // the last sequence that starts at or before the row
  int lo = -1, hi = num_seqs;  // cu[lo] <= tok < cu[hi], as far as looked at
  if (cu[num_seqs] > tok) {
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= tok)
        lo = mid;
      else
        hi = mid;
    }
  }
  T8 w = T8{};
  if (lo >= 0) {
    const int pos = tok - cu[lo];
    const int blk = pos / cache.block_size;
    const int page = blk < max_blocks ? block_table[lo * bt_stride + blk] : -1;
    if (page >= 0 && page < cache.num_blocks) {
      const long long row = pos - blk * cache.block_size;
      const unsigned int c = *reinterpret_cast<const unsigned int*>(
          codes + page * cache.code_stride_0 + head * cache.code_stride_h +
          row * cache.code_stride_t + 4 * piece);
      const unsigned int e = scales[page * cache.scale_stride_0 + head * cache.scale_stride_h +
                                    row * cache.scale_stride_t + (piece >> 2)];
      w = codes8<T>(c, scale_of(e));
    }
  }
  *reinterpret_cast<T8*>(out + 8 * i) = w;
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
constexpr int kDThreads = 256;
constexpr int kDTile = 32;
constexpr int kDRows = 16;

__device__ __attribute__((aligned(16))) unsigned char g_mxfp4_zero[32];

template <int D>
__device__ inline int vslot(int r) {  // swizzle of the V tile's 16-byte chunks
  constexpr int C = D / 8;
  constexpr int L = C >= 16 ? 1 : 16 / C;
  constexpr int H = (C < 16 ? C : 16) / 2;
  return 2 * ((r / L) % H);
}

template <int kBytes>
struct CodeWords {
  typedef unsigned int v __attribute__((ext_vector_type(kBytes / 4)));
};

template <typename T, int D>
__global__ __launch_bounds__(kDThreads, 2) void mxfp4_decode_kernel(const fa_mxfp4_decode_args a) {
  typedef typename FVec<T>::v8 T8;
  typedef typename FVec<T>::v4 T4;
  constexpr int kRowB = 2 * D;            // bytes per token row of the V tile
  constexpr int kTileB = kDTile * kRowB;
  constexpr int kWords = D / 32;          // words of codes per lane and token = k-steps of QK
  constexpr int kDimTiles = D / 16;
  constexpr bool kHalved = __is_same(T, _Float16);
  typedef typename CodeWords<4 * kWords>::v Words;
  __shared__ __attribute__((aligned(16))) unsigned char vbuf[4 * kTileB];
  __shared__ float ml[8 * kDRows];
  static_assert(4 * kTileB >= 4 * kDRows * D * 4, "merge area must fit in the tile buffers");

  const fa_mxfp4_cache& cache = a.cache;
  const int split = blockIdx.x;
  const int group = a.h_q / cache.h_kv;
  const int n_rb = cdiv(group, kDRows);
  const int hk = blockIdx.y / n_rb;
  const int rb = blockIdx.y - hk * n_rb;
  const int b = blockIdx.z;
  const int wave = wave_id();
  const int lane = threadIdx.x & 63;
  const int G = lane >> 4, c16 = lane & 15;

  const int seqlen = sload(a.seqlens + b);
  const int t0 = split * a.split_tokens;
  const int t1 = split + 1 == a.num_splits ? seqlen : min(t0 + a.split_tokens, seqlen);
  const int ntok = max(0, t1 - t0);
  const int ntiles = cdiv(ntok, kDTile);
  const int last = t1 - 1;

  const int rho = rb * kDRows + c16;
  const bool row_ok = rho < group;
  const int hq = hk * group + (row_ok ? rho : 0);
  const float scale_log2 = a.scale * kLog2e * (kHalved ? 2.f : 1.f);
  const float ninf = -__builtin_inff();

  T8 qf[kWords];
#pragma unroll
  for (int kk = 0; kk < kWords; ++kk)
    qf[kk] = row_ok ? *reinterpret_cast<const T8*>(static_cast<const T*>(a.q) + b * a.q_stride_b +
                                                   hq * a.q_stride_h + (D / 4) * G + 8 * kk)
                    : T8{};

  // ---- loads of a tile ----
  const unsigned char* const kc = static_cast<const unsigned char*>(cache.k_codes);
  const unsigned char* const vc = static_cast<const unsigned char*>(cache.v_codes);
  const unsigned char* const ks = static_cast<const unsigned char*>(cache.k_scales);
  const unsigned char* const vs = static_cast<const unsigned char*>(cache.v_scales);
  const int32_t* const bt_row = a.block_table + static_cast<long long>(b) * a.bt_stride_b;
  const int bs_shift = (cache.block_size & (cache.block_size - 1)) == 0
                           ? __builtin_ctz(static_cast<unsigned int>(cache.block_size))
                           : -1;
  Words kw[2], vw[2];
  unsigned int kse[2], vse[2];
  bool seen[2];  // the half's page is inside the cache
  auto issue = [&](int u) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int start = t0 + kDTile * u + 16 * h;
      const int first = min(start, last);  // uniform; a half's 16 tokens lie in one block
      const int blk = bs_shift >= 0 ? first >> bs_shift : first / cache.block_size;
      const int page = blk < a.max_blocks_per_seq ? sload(bt_row + blk) : -1;
      seen[h] = page >= 0 && page < cache.num_blocks;
      const long long row = min(start + c16, last) - blk * cache.block_size;
      const long long code = page * cache.code_stride_0 + hk * cache.code_stride_h +
                             row * cache.code_stride_t + (D / 8) * G;
      const long long sc = page * cache.scale_stride_0 + hk * cache.scale_stride_h +
                           row * cache.scale_stride_t + (D / 4) * G / FA_MXFP4_GROUP;
      kw[h] = *reinterpret_cast<const Words*>(seen[h] ? kc + code : g_mxfp4_zero);
      vw[h] = *reinterpret_cast<const Words*>(seen[h] ? vc + code : g_mxfp4_zero);
      const unsigned char* const kp = seen[h] ? ks + sc : g_mxfp4_zero;
      const unsigned char* const vp = seen[h] ? vs + sc : g_mxfp4_zero;
      if constexpr (D == 256) {
        kse[h] = *reinterpret_cast<const unsigned short*>(kp);
        vse[h] = *reinterpret_cast<const unsigned short*>(vp);
      } else {
        kse[h] = *kp;
        vse[h] = *vp;
      }
    }
  };
  // the scale of word kk of a lane, from its scale bytes
  auto word_scale = [&](unsigned int bytes, int kk) -> float {
    unsigned int e = D == 256 && kk >= 4 ? bytes >> 8 : bytes & 255u;
    if (kHalved) e = e == 255u ? e : max(e, 1u) - 1u;
    return scale_of(e);
  };

  float m_run = ninf, l_run = 0.f;
  floatx4 acc[kDimTiles];
#pragma unroll
  for (int dt = 0; dt < kDimTiles; ++dt) acc[dt] = floatx4{};
  unsigned char* const vb = vbuf + wave * kTileB;

  if (wave < ntiles) issue(wave);
  for (int u = wave; u < ntiles; u += 4) {
    const int tile_start = t0 + kDTile * u;
    floatx4 s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = floatx4{};
#pragma unroll
      for (int kk = 0; kk < kWords; ++kk)
        s[h] = mfma_16x16x32(codes8<T>(kw[h][kk], word_scale(kse[h], kk)), qf[kk], s[h]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 16 * h + c16;
#pragma unroll
      for (int kk = 0; kk < kWords; ++kk)
        *reinterpret_cast<T8*>(vb + r * kRowB + 16 * ((kWords * G + kk) ^ vslot<D>(r))) =
            codes8<T>(vw[h][kk], word_scale(vse[h], kk));
    }
    const bool seen0 = seen[0], seen1 = seen[1];
    if (u + 4 < ntiles) issue(u + 4);
    // softmax down the column: tokens tile_start + 16h + 4G + i
    float sv[2][4];
    float tmax = ninf;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool ok = tile_start + 16 * h + 4 * G + i < t1 && (h == 0 ? seen0 : seen1);
        sv[h][i] = ok ? s[h][i] * scale_log2 : ninf;
        tmax = fmaxf(tmax, sv[h][i]);
      }
    tmax = max_xor32(max_xor16(tmax));
    const float m_new = fmaxf(m_run, tmax);
    const float m_use = m_new == ninf ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
    float psum = 0.f;
    T8 pb;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(sv[h][i] - m_use);
        psum += p;
        pb[4 * h + i] = static_cast<T>(p);
      }
    l_run = l_run * alpha + psum;
    m_run = m_new;
    const int e = c16 >> 2, qd = c16 & 3;
    const int r0 = 4 * G + e, r1 = 16 + 4 * G + e;
#pragma unroll
    for (int dt = 0; dt < kDimTiles; ++dt) {
      const int chunk = 2 * dt + (qd >> 1);
      const T4 lo = lds_tr4<T>(vb + r0 * kRowB + 16 * (chunk ^ vslot<D>(r0)) + 8 * (qd & 1));
      const T4 hi = lds_tr4<T>(vb + r1 * kRowB + 16 * (chunk ^ vslot<D>(r1)) + 8 * (qd & 1));
      const T8 va = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      floatx4 o = acc[dt];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= alpha;
      acc[dt] = mfma_16x16x32(va, pb, o);
    }
  }

  // ---- merge the four waves' states ----
  const float l_col = sum_xor32(sum_xor16(l_run));
  __syncthreads();
  float* const om = reinterpret_cast<float*>(vbuf);  // [wave][16][D]
  if (G == 0) {
    ml[wave * kDRows + c16] = m_run;
    ml[(4 + wave) * kDRows + c16] = l_col;
  }
#pragma unroll
  for (int dt = 0; dt < kDimTiles; ++dt)
    *reinterpret_cast<floatx4*>(om + (wave * kDRows + c16) * D + 16 * dt + 4 * G) = acc[dt];
  __syncthreads();
  for (int idx = threadIdx.x; idx < kDRows * D; idx += kDThreads) {
    const int r = idx / D, d = idx - r * D;
    const int rr = rb * kDRows + r;
    if (rr >= group) break;  // rows are in order: the rest are past the end too
    float mw[4], M = ninf;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      mw[w] = ml[w * kDRows + r];
      M = fmaxf(M, mw[w]);
    }
    // no visible key: every weight and sum is 0; NaN sums stay NaN
    const float m_use = M == ninf ? 0.f : M;
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(mw[w] - m_use);
      L += ml[(4 + w) * kDRows + r] * f;
      O += om[(w * kDRows + r) * D + d] * f;
    }
    const int h = hk * group + rr;
    const float o = L == 0.f ? 0.f : O / L * (kHalved ? 2.f : 1.f);
    if (a.num_splits == 1) {
      static_cast<T*>(a.out)[b * a.o_stride_b + h * a.o_stride_h + d] = static_cast<T>(o);
    } else {
      const long long prow = (static_cast<long long>(b) * a.h_q + h) * a.num_splits + split;
      a.o_part[prow * D + d] = o;
      // the merge takes the largest lse, which a NaN would not be
      if (d == 0)
        a.lse_part[prow] = L == 0.f ? ninf : L == L ? (M + log2f(L)) * kLn2 : -ninf;
    }
  }
}

template <typename T>
int launch_decode(const fa_mxfp4_decode_args* a, hipStream_t stream) {
  const int group = a->h_q / a->cache.h_kv;
  const dim3 grid(a->num_splits, a->cache.h_kv * cdiv(group, kDRows), a->batch);
  if (a->cache.d == 64)
    hipLaunchKernelGGL((mxfp4_decode_kernel<T, 64>), grid, dim3(kDThreads), 0, stream, *a);
  else if (a->cache.d == 128)
    hipLaunchKernelGGL((mxfp4_decode_kernel<T, 128>), grid, dim3(kDThreads), 0, stream, *a);
  else
    hipLaunchKernelGGL((mxfp4_decode_kernel<T, 256>), grid, dim3(kDThreads), 0, stream, *a);
  FA_CHECK_HIP(hipGetLastError());
  return FA_OK;
}

bool aligned(const void* p, int64_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0;
}

int check_cache(const fa_mxfp4_cache* c) {
  FA_CHECK_ARG(c != nullptr, "cache is NULL");
  FA_CHECK_ARG(c->d == 64 || c->d == 128 || c->d == 256, "head dim %d not in {64, 128, 256}", c->d);
  FA_CHECK_ARG(c->h_kv >= 1 && c->h_kv <= 65535, "h_kv %d not in [1, 65535]", c->h_kv);
  FA_CHECK_ARG(c->block_size >= 16 && c->block_size % 16 == 0,
               "block_size %d is not a multiple of 16", c->block_size);
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
                   (a->num_splits == 1 || a->split_tokens % 16 == 0) &&
                   static_cast<int64_t>(a->num_splits - 1) * a->split_tokens <= INT32_MAX,
               "num_splits %d of %d tokens invalid", a->num_splits, a->split_tokens);
  FA_CHECK_ARG(a->num_splits == 1 || (a->o_part && a->lse_part),
               "num_splits %d > 1 needs o_part and lse_part", a->num_splits);
  FA_CHECK_ARG(a->q && a->out && a->block_table && a->seqlens && a->max_blocks_per_seq >= 1,
               "NULL q / out / block_table / seqlens or no block per sequence");
  FA_CHECK_ARG(aligned(a->q, 16) && a->q_stride_b % 8 == 0 && a->q_stride_h % 8 == 0,
               "q rows must be 16-byte aligned");
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
  const int64_t items = static_cast<int64_t>(num_tokens) * cache->h_kv * (cache->d / 8);
  const dim3 grid(static_cast<unsigned>((items + fa::kWThreads * fa::kWItems - 1) /
                                        (fa::kWThreads * fa::kWItems)), 2);
  const hipStream_t s = static_cast<hipStream_t>(stream);
#define FA_WRITE(T)                                                                            \
  hipLaunchKernelGGL(fa::mxfp4_write_kernel<T>, grid, dim3(fa::kWThreads), 0, s, *cache,        \
                     static_cast<const T*>(key), static_cast<long long>(key_stride_t),          \
                     static_cast<long long>(key_stride_h), static_cast<const T*>(value),        \
                     static_cast<long long>(value_stride_t),                                    \
                     static_cast<long long>(value_stride_h), slots, slots64, num_tokens)
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
  FA_CHECK_ARG(cu_seqlens && k_out && v_out && (num_seqs == 0 || block_table), "NULL pointer");
  FA_CHECK_ARG(max_blocks_per_seq >= 0, "max_blocks_per_seq %d < 0", max_blocks_per_seq);
  FA_CHECK_ARG(fa::aligned(k_out, 16) && fa::aligned(v_out, 16), "outputs must be 16-byte aligned");
  FA_CHECK_ARG(static_cast<int64_t>(total) * cache->h_kv <= INT32_MAX,
               "total %d x h_kv %d is 2^31 or more", total, cache->h_kv);
  const int64_t items = static_cast<int64_t>(total) * cache->h_kv * (cache->d / 8);
  const dim3 grid(static_cast<unsigned>((items + fa::kWThreads - 1) / fa::kWThreads), 2);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == 1)
    hipLaunchKernelGGL(fa::mxfp4_gather_kernel<__bf16>, grid, dim3(fa::kWThreads), 0, s, *cache,
                       block_table, static_cast<long long>(bt_stride_b), max_blocks_per_seq,
                       cu_seqlens, num_seqs, total, static_cast<__bf16*>(k_out),
                       static_cast<__bf16*>(v_out));
  else
    hipLaunchKernelGGL(fa::mxfp4_gather_kernel<_Float16>, grid, dim3(fa::kWThreads), 0, s, *cache,
                       block_table, static_cast<long long>(bt_stride_b), max_blocks_per_seq,
                       cu_seqlens, num_seqs, total, static_cast<_Float16*>(k_out),
                       static_cast<_Float16*>(v_out));
  FA_CHECK_HIP(hipGetLastError());
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
  fa_gqa_decode_args g = {};  // the merge reads the partial rows alone
  g.q = g.k = g.v = a->q;
  g.out = a->out;
  g.o_stride_b = a->o_stride_b;
  g.o_stride_h = a->o_stride_h;
  g.o_part = a->o_part;
  g.lse_part = a->lse_part;
  g.batch = a->batch;
  g.h_q = a->h_q;
  g.h_kv = a->cache.h_kv;
  g.m = 1;
  g.d = a->cache.d;
  g.num_splits = a->num_splits;
  g.split_tokens = a->split_tokens;
  g.dtype = a->dtype;
  return fa_gqa_combine(&g, stream);
}
