// Products in 8-bit floating point with one power-of-two scale per block of 128 along the contracted axis, and the quantisers that feed them
// (no counterpart in the reference: its semantic heads, autolabel/models.py:117-136, run in fp16 through tinycudann).
//
// A row x[0, K) is cut into blocks of 128; a block is held as q (e4m3 or e5m2) and ONE exponent e, x ~ q 2^e:
//     e = the smallest e >= -126 with max |x| 2^-e <= 448 (e4m3) or 57344 (e5m2);   0 for a block of zeros
//     q = x 2^-e rounded to the nearest 8-bit value, ties to even
// Both types' largest value is 1.75 2^EMAX (EMAX = 8, 15), so e = exponent(max) - EMAX, plus one where max's mantissa is above 1.75: nothing is
// clipped, and since 2^-e x is exact, q is one rounding of x whatever the order of the arithmetic.  A power of two costs a floating type no
// precision against an fp32 scale (only the top fraction of a binade of range), and it is what v_mfma_scale_f32_32x32x64_f8f6f4 takes as an
// operand: y = sum_b 2^(ex_b + ew_b) sum_{k in b} qx qw costs no instruction beside the matrix instructions.
// That instruction accumulates in fp32, but aligns the 64 products of a step to the largest of them and drops what lies 13 binades below it
// (measured; the older v_mfma_f32_32x32x16_fp8_fp8 does the same): 1.3e-5 of the result for Gaussian operands, 7e-5 for values spread over 12
// binades.  That is under the half step of a 16-bit result (4.9e-4, 3.9e-3) where the sum does not cancel: the half step goes with the sum, what is
// dropped with its largest term (up to 2^-13 of it a term, K of them).  It is far above the half step of an fp32 result: such products turn the 8-bit
// values back into bf16, which holds q 2^e exactly but at the ends of the exponents (WIDE_LO), and use the bf16 instruction (5e-8, at half the rate).
// A block that holds an infinity or a NaN is NaN throughout (its row of the product would be non-finite in every column anyway).
//
// Layout: q [rows, ldq] bytes, columns [K, 128 ceil(K / 128)) zero; scale [rows, lds] bytes e + 127, lds a multiple of 4, so that the four
// scales of 512 columns are one aligned 4-byte word.
#include "common.h"
#include "fp8_pieces.h"
#include <type_traits>

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

enum { F8_E4M3 = 0, F8_E5M2 = 1 };                       // also the format codes of the matrix instruction
enum { FT_F16 = 0, FT_BF16 = 1, FT_F32 = 2 };
static inline int64_t ceil128(int64_t n) { return (n + 127) / 128 * 128; }

// ---------------------------------------------------------------------------------------------------------- block arithmetic
template <int CTRL> __device__ inline uint32_t dpp_umax(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
  return v > o ? v : o;
}
// the maximum over the 16 lanes of a row of the wave, in every one of them
__device__ inline uint32_t umax16(uint32_t v) {
  v = dpp_umax<0xB1>(v);    // quad_perm 1,0,3,2
  v = dpp_umax<0x4E>(v);    // quad_perm 2,3,0,1
  v = dpp_umax<0x141>(v);   // row_half_mirror
  return dpp_umax<0x140>(v);  // row_mirror
}

// A block's power of two 2^e from the bits of max |x| as fp32 (NaN and infinity compare above every finite value)
struct BlockScale { uint8_t byte; bool finite; float scale, factor; };    // e + 127; 2^e; 2^-e, or NaN for a block that is not finite
template <int FMT> __device__ inline BlockScale block_scale(uint32_t amax_bits) {
  constexpr int EMAX = FMT == F8_E4M3 ? 8 : 15;
  // exponent + 127 of the maximum, one more above 1.75 (a carry out of the mantissa), less EMAX; not under 2^-126
  int e = (int)((amax_bits + 0x1fffffu) >> 23) - EMAX;
  e = e < 1 ? 1 : e;
  e = amax_bits == 0 ? 127 : e;
  const bool finite = amax_bits < 0x7f800000u;
  return {(uint8_t)e, finite, __uint_as_float((uint32_t)e << 23), __uint_as_float(finite ? (uint32_t)(254 - e) << 23 : 0x7fc00000u)};
}

template <int FMT> __device__ inline uint32_t pack4(float a, float b, float c, float d) {
  int w = 0;
  if constexpr (FMT == F8_E4M3) { w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false); w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true); }
  else { w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false); w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true); }
  return (uint32_t)w;
}

// Eight consecutive values of a row as they are stored, the bits of their largest |x| as fp32, and their fp32 values.  Loads go through
// memcpy: a row of an odd number of columns is only aligned to its element.
template <int T> struct Eight;
template <> struct Eight<FT_F16> {
  u16x8 v;
  __device__ void load(const void* p, int64_t at, int n) {
    const uint16_t* s = (const uint16_t*)p + at;
    if (n >= 8) __builtin_memcpy(&v, s, 16);
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < n ? s[j] : (uint16_t)0;
    }
  }
  __device__ uint32_t amax() const {
    const u16x8 a = v & (uint16_t)0x7fff;
    uint16_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = a[j] > m ? a[j] : m;
    return __float_as_uint((float)__builtin_bit_cast(h16, m));
  }
  __device__ float get(int j) const { return (float)__builtin_bit_cast(h16, (uint16_t)v[j]); }
};
template <> struct Eight<FT_BF16> {
  u16x8 v;
  __device__ void load(const void* p, int64_t at, int n) {
    const uint16_t* s = (const uint16_t*)p + at;
    if (n >= 8) __builtin_memcpy(&v, s, 16);
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < n ? s[j] : (uint16_t)0;
    }
  }
  __device__ uint32_t amax() const {
    const u16x8 a = v & (uint16_t)0x7fff;
    uint16_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = a[j] > m ? a[j] : m;
    return (uint32_t)m << 16;
  }
  __device__ float get(int j) const { return __uint_as_float((uint32_t)v[j] << 16); }
};
template <> struct Eight<FT_F32> {
  float v[8];
  __device__ void load(const void* p, int64_t at, int n) {
    const float* s = (const float*)p + at;
    if (n >= 8) __builtin_memcpy(v, s, 32);
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < n ? s[j] : 0.f;
    }
  }
  __device__ uint32_t amax() const {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) { const uint32_t a = __float_as_uint(v[j]) & 0x7fffffffu; m = a > m ? a : m; }
    return m;
  }
  __device__ float get(int j) const { return v[j]; }
};

// Four of eight values as 8-bit ones, x 2^-e.  16-bit values are converted in pairs by the instruction that scales on the way (it divides by
// the power of two of `scale` exactly and rounds once); a block with a NaN or an infinity becomes NaN through its fp32 factor, or here.
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
template <int T, int FMT> __device__ inline uint32_t cvt4(uint32_t lo, uint32_t hi, float scale) {
  s16x2 w = {0, 0};
  if constexpr (T == FT_F16 && FMT == F8_E4M3) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(h16x2, lo), scale, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(h16x2, hi), scale, true);
  } else if constexpr (T == FT_F16) {
    w = __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(w, __builtin_bit_cast(h16x2, lo), scale, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(w, __builtin_bit_cast(h16x2, hi), scale, true);
  } else if constexpr (FMT == F8_E4M3) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(b16x2, lo), scale, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(b16x2, hi), scale, true);
  } else {
    w = __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(w, __builtin_bit_cast(b16x2, lo), scale, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(w, __builtin_bit_cast(b16x2, hi), scale, true);
  }
  return __builtin_bit_cast(uint32_t, w);
}
template <int T, int FMT> __device__ inline uint2 quant8(const Eight<T>& x, const BlockScale& s) {
  if constexpr (T == FT_F32) {
    const float f = s.factor;
    return make_uint2(pack4<FMT>(x.v[0] * f, x.v[1] * f, x.v[2] * f, x.v[3] * f), pack4<FMT>(x.v[4] * f, x.v[5] * f, x.v[6] * f, x.v[7] * f));
  } else {
    const i32x4 w = __builtin_bit_cast(i32x4, x.v);
    const uint2 q = make_uint2(cvt4<T, FMT>(w[0], w[1], s.scale), cvt4<T, FMT>(w[2], w[3], s.scale));
    return s.finite ? q : make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);       // (0x7f: a NaN of both formats)
  }
}

// ------------------------------------------------------------------------------------------------------------ quantisers
// Rows: 16 lanes hold a block (8 values each), its maximum goes round them with four DPP steps; one read of x, one write of q.  Bound by memory:
// 8192 x 4096 fp16 17.7 us (5.7 TB/s, its input in the memory-side cache), 262144 x 512 79 us (5.1 TB/s; a large copy reaches 4.6).
template <int T, int FMT>
__global__ __launch_bounds__(256) void k_fp8_quant(const void* __restrict__ x, int64_t ldx, int64_t M, int K, int nb, uint8_t* __restrict__ q,
                                                   int64_t ldq, uint8_t* __restrict__ scale, int64_t lds) {
  const int sub = threadIdx.x & 15;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4; i < M * nb; i += (int64_t)gridDim.x * 16) {
    const int64_t row = i / nb;
    const int b = (int)(i - row * nb), k = b * 128 + sub * 8;
    Eight<T> v;
    v.load(x, row * ldx + k, K - k);
    const BlockScale bs = block_scale<FMT>(umax16(v.amax()));
    *(uint2*)(q + row * ldq + k) = quant8<T, FMT>(v, bs);
    if (sub == 0) scale[row * lds + b] = bs.byte;
    else if (sub < 4 && b == nb - 1 && nb + sub - 1 < (nb + 3) / 4 * 4) scale[row * lds + nb + sub - 1] = 127;   // the rest of the last word
  }
}

// Columns: q of x^T with blocks of 128 along the rows of x.  A block of threads turns a tile of 128 rows x 64 columns round: a thread reads
// eight columns of four rows, the maxima of a column meet through three shuffles and LDS, the 8-bit values cross in LDS and leave as whole
// 128-byte lines.  262144 x 512 fp16 101 us, 4.0 TB/s: the two barriers of a tile, with nothing of the next one in flight, are what is left.
template <int T, int FMT>
__global__ __launch_bounds__(256) void k_fp8_quant_t(const void* __restrict__ x, int64_t ldx, int64_t M, int C, int nb, uint8_t* __restrict__ q,
                                                     int64_t ldq, uint8_t* __restrict__ scale, int64_t lds) {
  __shared__ uint32_t amax[4][64];
  __shared__ __attribute__((aligned(16))) uint8_t tile[64][144];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c8 = (tid & 7) * 8, r0 = tid >> 3;   // rows r0 + 32 i
  const int nct = (C + 63) / 64;
  const int64_t b = blockIdx.x / nct;
  const int c0 = (int)(blockIdx.x % nct) * 64;
  Eight<T> v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = b * 128 + r0 + 32 * i;
    v[i].load(x, row * ldx + c0 + c8, row < M ? C - c0 - c8 : 0);
  }
  uint32_t m[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    m[j] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) { const uint32_t a = __float_as_uint(v[i].get(j)) & 0x7fffffffu; m[j] = a > m[j] ? a : m[j]; }
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) { const uint32_t a = (uint32_t)__shfl_xor((int)m[j], o); m[j] = a > m[j] ? a : m[j]; }
  }
  if (lane < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) amax[wave][c8 + j] = m[j];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint32_t a = amax[0][c8 + j];
#pragma unroll
    for (int w = 1; w < 4; ++w) a = amax[w][c8 + j] > a ? amax[w][c8 + j] : a;
    const BlockScale bs = block_scale<FMT>(a);
    const float f = bs.factor;
    const uint32_t p = pack4<FMT>(v[0].get(j) * f, v[1].get(j) * f, v[2].get(j) * f, v[3].get(j) * f);
#pragma unroll
    for (int i = 0; i < 4; ++i) tile[c8 + j][r0 + 32 * i] = (uint8_t)(p >> (8 * i));
    if (tid < 8 && c0 + c8 + j < C) {
      scale[(c0 + c8 + j) * lds + b] = bs.byte;
      if (b == nb - 1) for (int k = nb; k < (nb + 3) / 4 * 4; ++k) scale[(c0 + c8 + j) * lds + k] = 127;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = (tid >> 3) + 32 * i;
    if (c0 + c < C) *(uint4*)(q + (c0 + c) * ldq + b * 128 + (tid & 7) * 16) = *(const uint4*)&tile[c][(tid & 7) * 16];
  }
}

// -------------------------------------------------------------------------------------------------------------- products
// SA, SB: which byte of the words of scales
template <int FA, int FB, int SA = 0, int SB = 0> __device__ inline f32x16 mfma8(i32x8 a, i32x8 b, f32x16 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, FA, FB, SA, sa, SB, sb);
}

// two 8-bit values (the upper two of the word with HI) times a power of two, exact in bf16 between WIDE_LO and WIDE_HI
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
template <int FMT, bool HI> __device__ inline b16x2 widen2(uint32_t w, float s) {
  if constexpr (FMT == F8_E4M3) return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, HI);
  else return __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, s, HI);
}
template <int FMT> __device__ inline b16x8 widen8(uint32_t w0, uint32_t w1, float s) {
  const b16x2 a = widen2<FMT, false>(w0, s), b = widen2<FMT, true>(w0, s), c = widen2<FMT, false>(w1, s), d = widen2<FMT, true>(w1, s);
  return (b16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// bf16 holds q 2^e exactly from 2^-133 up and under 2^128: for every q of a block with e between these (as e + 127).  The few scales outside, where a value
// may be as small as 2^-135 (e4m3; e5m2 2^-142) or be 2^128, would lose bits, or become infinite and with a zero NaN.  Their powers of two are moved by
// 2^16 from one operand to the other, which then holds what it can hold of the product: below 2^-149 there is nothing to lose.
template <int FMT> constexpr uint32_t WIDE_LO = FMT == F8_E4M3 ? 3 : 10;
template <int FMT> constexpr uint32_t WIDE_HI = FMT == F8_E4M3 ? 246 : 239;
template <int FMT> __device__ inline int wide_end(uint32_t e) { return e < WIDE_LO<FMT> ? 1 : e > WIDE_HI<FMT> ? 2 : 0; }     // 1: small, 2: large
// how an operand of kind c is moved beside one of kind d.  Two small ones' product is 0 however they are moved; two large ones', where it is not 0,
// is infinite also 2^32 lower
__device__ inline int wide_shift(int c, int d) { return c == 2 ? -16 : c == 1 ? 16 : d == 2 ? 16 : d == 1 ? -16 : 0; }
// (at the ends of the range the product is infinite, or 0, all the same)
template <int FMT> __device__ inline uint32_t wide_moved(uint32_t e, int by) { return (uint32_t)min(max((int)e + by, 1), (int)WIDE_HI<FMT>); }

__device__ inline float relu_nan(float v) { return __builtin_elementwise_maximum(v, 0.f); }     // a NaN stays one

struct Fp8Out { void* y; int64_t ldy; int type, relu; };   // type: FT_*

// One wave's 32 x 64 block of the result.  The accumulators hold D[n][m]: lane = row m of y (lane % 32), register r = column
// 8 (r / 4) + 4 (lane / 32) + r % 4 -- stores from there would touch 32 rows per instruction with 8 bytes each, so the block, already rounded
// to its type, goes round through LDS (`buf`, the wave's own 4 KB, fp32 8 KB; 16-byte pieces turned by the row against bank conflicts) and
// leaves row by row, 16 bytes a lane.
template <bool F32>
__device__ inline void store_block(const Fp8Out& o, const f32x16& c0, const f32x16& c1, uint8_t* buf, int64_t m0, int64_t M, int n0, int N, int lane) {
  constexpr int ES = F32 ? 4 : 2, PIECES = 4 * ES, PER = 16 / ES;      // pieces of 16 bytes per row of 64, values per piece
  const int r = lane & 31, h = lane >> 5;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 v = s ? (f32x4){c1[4 * g], c1[4 * g + 1], c1[4 * g + 2], c1[4 * g + 3]} : (f32x4){c0[4 * g], c0[4 * g + 1], c0[4 * g + 2], c0[4 * g + 3]};
      if (o.relu) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = relu_nan(v[j]);
      }
      if constexpr (F32) *(f32x4*)(buf + r * 256 + (((8 * s + 2 * g + h) ^ (r & 15)) * 16)) = v;
      else {
        uint8_t* q = buf + r * 128 + (((4 * s + g) ^ (r & 7)) * 16) + 8 * h;
        if (o.type == FT_F16) *(h16x4*)q = __builtin_convertvector(v, h16x4);
        else *(b16x4*)q = __builtin_convertvector(v, b16x4);
      }
    }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int it = 0; it < PIECES / 2; ++it) {
    const int row = it * (64 / PIECES) + lane / PIECES, piece = lane % PIECES, c = piece * PER;
    const int64_t m = m0 + row;
    const uint4 w = *(const uint4*)(buf + row * 16 * PIECES + ((piece ^ (row & (F32 ? 15 : 7))) * 16));
    if (m >= M || n0 + c >= N) continue;
    uint8_t* p = (uint8_t*)o.y + (m * o.ldy + n0 + c) * ES;
    if (n0 + c + PER <= N) __builtin_memcpy(p, &w, 16);
    else {
      const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < PER - 1; ++j) {
        if (n0 + c + j >= N) continue;
        if constexpr (F32) ((uint32_t*)p)[j] = d[j];
        else ((uint16_t*)p)[j] = (uint16_t)(d[j / 2] >> (16 * (j & 1)));
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
}

// Blocks b and b + 8 run on the same XCD.  Each XCD takes a run of consecutive work items, so that those that share rows find them in its L2, and
// all eight have the same number, however few there are.  With the row tiles going round the XCDs instead, one row tile is work for 32 of the 256 CUs: blocks
// of x and their product for 64 x 4096 x 4096 take 15.0 us this way and 40.6 that way, the 128 parts of 64 x 512 x 4096 5.6 and 18.7.  -1: none left for this
// block of a grid of xcd_grid(items).
__device__ inline int xcd_item(int items) {
  const int each = (items + 7) / 8, i = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
  return i < items ? i : -1;
}
static inline uint32_t xcd_grid(int64_t items) { return (uint32_t)((items + 7) / 8 * 8); }

// The slot of piece c of row r in a tile of 128-byte rows is c ^ turn(r)
__device__ inline int turn(int row) { return (row >> 1) & 7; }

struct Fp8NT {
  const uint8_t* a; int64_t lda; const uint8_t* sa; int64_t ldsa;   // [M, K] rows of y
  const uint8_t* b; int64_t ldb; const uint8_t* sb; int64_t ldsb;   // [N, K] columns of y
  int64_t M; int N, nkb;                                            // nkb: blocks of 128 along K
  int splits, per;                                                  // K in `splits` parts of `per` blocks; part s writes slab s of y (fp32, M x N each)
  Fp8Out o;
};

// y = A B^T.  A tile of 128-byte rows lies in LDS with its 16-byte pieces turned by the row number (turn), on both sides of the direct
// global -> LDS copy: reads of 32 rows then meet every bank evenly (4% of the reads' cycles are conflicts).  Which bytes of a 128-block meet in
// which lane of the matrix instruction is free (both operands use the same order and the block has one scale), so a lane takes pieces 4 h .. 4 h + 3.
// Two buffers, one barrier per 128 columns: the next step's copies are sent before this one is multiplied.
// WIDE: the fp32 results' form, 16-bit operands out of the same tiles.
// Tiles: 256 x 256 by eight waves, or 128 x 128 by four (nt_type), and the contraction in parts where there are few (nt_plan).
// 8192 x 4096 x 4096 with 16-bit results: 122 .. 134 us by the card's temperature, 2.05 .. 2.25 PFLOP/s (the library's product of unscaled 8-bit
// values 112); with fp32 results 220 .. 242 us, bound by the bf16 matrix instructions (the library's bf16 product 202; 1345 TFLOP/s at 8192^3 would be 204);
// 256 x 512 x 4096 13 us with the joining of its parts.
// What bounds the large ones, in clocks of a CU per 256 x 256 x 128 step: 2050 for the 32 matrix instructions of a SIMD, 170 for the scales, 490 for
// waves that wait for each other at the barrier, 450 .. 1000 for the 64 KB copied (with the fragments that is 256 KB through LDS, all that 128 bytes
// a clock give in 2050): the barrier waits for every copy, which has to land inside its own step.  Other schedules, timed in the same runs, in which this one
// took 145 us (a warm card): the fragments of a half step read ahead across the barrier 144 .. 146, copies spread between the matrix instructions (through
// buffer descriptors, without a branch in the loop) 148, 128 x 128 results a wave with one wave per SIMD 170 .. 178, 4 x 8 groups of tiles per XCD 145.
template <int FA, int FB, bool WIDE, int WM, int WN, int MI, int NI>
__global__ __launch_bounds__(64 * WM * WN) void k_fp8_nt(Fp8NT p) {
  constexpr int BM = WM * MI * 32, BN = WN * NI * 32, NW = WM * WN, ROWS = BM + BN;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem8[];    // [2][ROWS][128]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const int wm = wave % WM, wn = wave / WM;
  const int ntn = (p.N + BN - 1) / BN, tile = xcd_item((int)((p.M + BM - 1) / BM) * ntn);      // the column tiles of a row tile follow each other
  if (tile < 0) return;
  const int64_t m0 = (int64_t)(tile / ntn) * BM;
  const int n0 = (tile % ntn) * BN;
  const int kb0 = blockIdx.y * p.per, kb1 = min(p.nkb, kb0 + p.per);
  f32x16 acc[NI][MI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  constexpr int PIECES = ROWS / 8 / NW;                   // direct copies of a wave per step, eight rows each
  const int sub = lane >> 3, slot = lane & 7;
  const uint8_t* src[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int row = (wave + i * NW) * 8 + sub;            // row of the tile: A's first, then B's (a wave's eight rows are all of one kind)
    src[i] = (row < BM ? p.a + min(m0 + row, p.M - 1) * p.lda : p.b + (int64_t)min(n0 + row - BM, p.N - 1) * p.ldb) + (int64_t)kb0 * 128 + ((slot ^ turn(row)) * 16);
  }
  auto fetch = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src[i],
                                       (__attribute__((address_space(3))) void*)(smem8 + buf * ROWS * 128 + (wave + i * NW) * 1024), 16, 0, 0);
      src[i] += 128;
    }
  };
  // scales: a word holds four blocks of a row; the next word is sent for when the current one is begun (parts begin at multiples of four)
  const uint8_t *pa[MI], *pb[NI];
  uint32_t sa[MI], sb[NI], na[MI], nb[NI];
#pragma unroll
  for (int j = 0; j < MI; ++j) { pa[j] = p.sa + min(m0 + (wm * MI + j) * 32 + r, p.M - 1) * p.ldsa + kb0; na[j] = *(const uint32_t*)pa[j]; }
#pragma unroll
  for (int i = 0; i < NI; ++i) { pb[i] = p.sb + (int64_t)min(n0 + (wn * NI + i) * 32 + r, p.N - 1) * p.ldsb + kb0; nb[i] = *(const uint32_t*)pb[i]; }
  int off[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) off[c] = r * 128 + (((4 * h + c) ^ turn(r)) * 16);
  fetch(0);
  __syncthreads();
  auto words = [&](int kb) __attribute__((always_inline)) {
    if (((kb - kb0) & 3) == 0) {
      const bool more = kb + 4 < kb1;
#pragma unroll
      for (int j = 0; j < MI; ++j) { sa[j] = na[j]; if (more) { pa[j] += 4; na[j] = *(const uint32_t*)pa[j]; } }
#pragma unroll
      for (int i = 0; i < NI; ++i) { sb[i] = nb[i]; if (more) { pb[i] += 4; nb[i] = *(const uint32_t*)pb[i]; } }
    }
  };
  auto fragments = [&](int buf, int ks, i32x8 (&fa)[MI], i32x8 (&fb)[NI]) __attribute__((always_inline)) {
    const uint8_t *ta = smem8 + buf * ROWS * 128 + wm * MI * 4096, *tb = smem8 + buf * ROWS * 128 + BM * 128 + wn * NI * 4096;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      fb[i] = __builtin_shufflevector(*(const i32x4*)(tb + i * 4096 + off[2 * ks]), *(const i32x4*)(tb + i * 4096 + off[2 * ks + 1]), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
    for (int j = 0; j < MI; ++j)
      fa[j] = __builtin_shufflevector(*(const i32x4*)(ta + j * 4096 + off[2 * ks]), *(const i32x4*)(ta + j * 4096 + off[2 * ks + 1]), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto widened = [&](const i32x8 (&fa)[MI], const i32x8 (&fb)[NI], const uint32_t (&ea)[MI], const uint32_t (&eb)[NI]) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      b16x8 xa[MI];
#pragma unroll
      for (int j = 0; j < MI; ++j) xa[j] = widen8<FA>(fa[j][2 * q], fa[j][2 * q + 1], __uint_as_float(ea[j] << 23));
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const b16x8 xb = widen8<FB>(fb[i][2 * q], fb[i][2 * q + 1], __uint_as_float(eb[i] << 23));
#pragma unroll
        for (int j = 0; j < MI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xb, xa[j], acc[i][j], 0, 0, 0);
      }
    }
  };
  auto finish = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < MI; ++j) sa[j] >>= 8;
#pragma unroll
    for (int i = 0; i < NI; ++i) sb[i] >>= 8;
    __syncthreads();            // the tile has been read, the next one has landed
  };
  int kb = kb0;
  for (; kb < kb1; ++kb) {
    const int buf = (kb - kb0) & 1;
    words(kb);
    uint32_t ea[MI], eb[NI];
    if constexpr (WIDE) {
      bool ends = false;
#pragma unroll
      for (int j = 0; j < MI; ++j) { ea[j] = sa[j] & 255u; ends |= wide_end<FA>(ea[j]) != 0; }
#pragma unroll
      for (int i = 0; i < NI; ++i) { eb[i] = sb[i] & 255u; ends |= wide_end<FB>(eb[i]) != 0; }
      if (__any(ends)) break;
    }
    if (kb + 1 < kb1) fetch(buf ^ 1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      i32x8 fa[MI], fb[NI];
      fragments(buf, ks, fa, fb);
      if constexpr (WIDE) widened(fa, fb, ea, eb);
      else {
#pragma unroll
        for (int j = 0; j < MI; ++j)
#pragma unroll
          for (int i = 0; i < NI; ++i) acc[i][j] = mfma8<FB, FA>(fb[i], fa[j], acc[i][j], (int)sb[i], (int)sa[j]);
      }
    }
    finish();
  }
  // from a wave's first step with a scale at the ends of the exponents on: each kind of row with each kind of column in turn, the others as zeros (one
  // barrier to a step here too: the waves of a block need not be in the same loop).  8192 x 4096 x 4096 with such a row in every 256: 441 us instead of 229;
  // with one in all 279.  (Its addresses do not fit beside 256 x 256 results: 44 bytes a lane lie in scratch, in this loop alone.)
  if constexpr (WIDE)
    for (bool first = true; kb < kb1; ++kb, first = false) {
      const int buf = (kb - kb0) & 1;
      if (!first) words(kb);
      if (kb + 1 < kb1) fetch(buf ^ 1);
#pragma unroll 1
      for (int pass = 0; pass < 9; ++pass) {
        const int ca = pass / 3, cb = pass % 3, da = wide_shift(ca, cb), db = wide_shift(cb, ca);
        uint32_t ea[MI], eb[NI];
        bool ka[MI], kc[NI], any_a = false, any_b = false;
#pragma unroll
        for (int j = 0; j < MI; ++j) { ka[j] = wide_end<FA>(sa[j] & 255u) == ca; any_a |= ka[j]; ea[j] = wide_moved<FA>(sa[j] & 255u, da); }
#pragma unroll
        for (int i = 0; i < NI; ++i) { kc[i] = wide_end<FB>(sb[i] & 255u) == cb; any_b |= kc[i]; eb[i] = wide_moved<FB>(sb[i] & 255u, db); }
        if (!__any(any_a) || !__any(any_b)) continue;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          i32x8 fa[MI], fb[NI];
          fragments(buf, ks, fa, fb);
#pragma unroll
          for (int j = 0; j < MI; ++j) fa[j] = ka[j] ? fa[j] : (i32x8)0;
#pragma unroll
          for (int i = 0; i < NI; ++i) fb[i] = kc[i] ? fb[i] : (i32x8)0;
          widened(fa, fb, ea, eb);
          __builtin_amdgcn_sched_barrier(0);     // (or the second half's fragments are read ahead, and registers spill)
        }
      }
      finish();
    }
  Fp8Out o = p.o;
  if (p.splits > 1) { o.y = (float*)o.y + (int64_t)blockIdx.y * p.M * p.N; o.ldy = p.N; o.type = FT_F32; o.relu = 0; }
  uint8_t* buf = smem8 + wave * 8192;
#pragma unroll
  for (int j = 0; j < MI; ++j)
#pragma unroll
    for (int i = 0; i < NI; i += 2) {
      if (o.type == FT_F32) store_block<true>(o, acc[i][j], acc[i + 1][j], buf, m0 + (wm * MI + j) * 32, p.M, n0 + (wn * NI + i) * 32, p.N, lane);
      else store_block<false>(o, acc[i][j], acc[i + 1][j], buf, m0 + (wm * MI + j) * 32, p.M, n0 + (wn * NI + i) * 32, p.N, lane);
    }
}

// y = x W^T with the rows of x cut into blocks on the way; the values of x never exist in 8 bits in memory, and the weights never in LDS: a wave
// keeps the 32 rows of W that it multiplies by -- all of their up to 1024 columns -- in registers (16 NKB of them) and lets x stream past.
// Sixteen waves hold 512 x 512 weights (half of a CU's registers); above 512 columns eight waves hold 256 x 1024.  A block of threads owns a
// range of rows and goes through it in tiles of up to 64: a tile's rows are cut into 8-bit blocks in one LDS buffer (four lanes to a block, its
// power of two worked out once for 32 values) while the tile before it is multiplied out of the other and the loads of the one after it are in
// flight.  One barrier per tile.
// Bound by memory where there are many rows: 2^20 x 512 x 512 fp16 479 us, 4.5 TB/s (a large copy reaches 4.6).  50000 rows are four tiles to a block
// and take 34 us (3.0 TB/s): the first tile's loads and the last one's results have nothing beside them, and tiles of 32 .. 48 rows instead of 64
// cost more than they hide (36 .. 37.5 us; 2^20 rows 561 .. 634).  4096 rows 10 us (one tile a block: a launch, the block's weights and its rows one
// after the other, and eight of the sixteen waves only cut), one row 5 us (a launch, and 256 KB of weights over all blocks).  The cut rows go to LDS in
// 8-byte pieces: a quarter of the kernel's LDS cycles are bank conflicts, 5% of its time.
// At NKB 4, 7 and 8 the registers do not quite hold everything: 12 .. 84 bytes a lane lie in scratch and are read once per tile.
struct Fp8Linear {
  const void* x; int64_t ldx;
  const uint8_t* w; int64_t ldw; const uint8_t* sw; int64_t ldsw;
  int64_t M; int N, K;
  int wn, parts;                  // waves side by side along the columns of y (a power of two); blocks of threads side by side
  int ranges, rows, bm;           // ranges of rows; rows of a range, of a tile (<= 64)
  Fp8Out o;
};
template <int NKB> constexpr int lin_threads() { return NKB <= 4 ? 1024 : 512; }

template <int FX, int NKB, int KB = 0> __device__ inline void lin_chain(f32x16& acc, const i32x8 (&w)[NKB][2], const uint32_t* sw, const uint32_t* sx, const uint8_t* x, const int (&off)[4]) {
  if constexpr (KB < NKB) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const uint8_t* t = x + KB * 64 * 128;
      const i32x8 f = __builtin_shufflevector(*(const i32x4*)(t + off[2 * ks]), *(const i32x4*)(t + off[2 * ks + 1]), 0, 1, 2, 3, 4, 5, 6, 7);
      acc = mfma8<F8_E4M3, FX, KB & 3, KB & 3>(w[KB][ks], f, acc, (int)sw[KB / 4], (int)sx[KB / 4]);
    }
    lin_chain<FX, NKB, KB + 1>(acc, w, sw, sx, x, off);
  }
}

template <int T, int FX, int NKB>
__global__ __launch_bounds__(lin_threads<NKB>()) void k_fp8_linear(Fp8Linear p) {
  constexpr int NT = lin_threads<NKB>(), NW = NT / 64, TASKS = 64 * NKB * 4, ROUNDS = (TASKS + NT - 1) / NT, WORDS = (NKB + 3) / 4;
  __shared__ __attribute__((aligned(16))) uint8_t xs[2][NKB][64][128];         // 16-byte pieces turned by the row
  __shared__ __attribute__((aligned(16))) uint8_t se[2][64][4 * WORDS];        // exponents + 127
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const int item = xcd_item(p.ranges * p.parts), part = item % p.parts;       // the parts of a row range follow each other
  if (item < 0) return;
  const int64_t lo = (int64_t)(item / p.parts) * p.rows, hi = lo + p.rows < p.M ? lo + p.rows : p.M;
  const int wn = wave % p.wn, wm = wave / p.wn, step = NW / p.wn, n0 = (part * p.wn + wn) * 32;
  Eight<T> v[ROUNDS][4];
  // (a uniform base and a 32-bit offset of the lane in bytes: pitches are under 2^25.  Rows behind the tile's last are read as that one: what is
  // made of them is never stored.)
  auto load = [&](int64_t m) __attribute__((always_inline)) {
    const uint8_t* base = (const uint8_t*)p.x + 2 * m * p.ldx;
    const int last = (int)(hi - m < p.bm ? hi - m : p.bm) - 1;
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q) {
      const int task = tid + q * NT, l = task & 3, b = (task >> 2) % NKB, row = min((task >> 2) / NKB, last);
      const uint32_t at = 2 * (uint32_t)row * (uint32_t)p.ldx;
      const int k = b * 128 + l * 8;
      if (p.K == NKB * 128) {
#pragma unroll
        for (int j = 0; j < 4; ++j) __builtin_memcpy(&v[q][j].v, base + (at + 2 * k) + 64 * j, 16);
      } else if (p.K % 8 == 0) {         // pieces behind the last column: read where the last one is, zero
#pragma unroll
        for (int j = 0; j < 4; ++j) __builtin_memcpy(&v[q][j].v, base + (at + 2 * min(k + 32 * j, p.K - 8)), 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) if (k + 32 * j >= p.K) v[q][j].v = (u16x8)(uint16_t)0;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[q][j].load(base + (at + 2 * k) + 64 * j, 0, p.K - (k + 32 * j));
      }
    }
  };
  auto cut = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q) {
      const int task = tid + q * NT, l = task & 3, b = (task >> 2) % NKB, row = (task >> 2) / NKB;
      if (TASKS % NT != 0 && task >= TASKS) continue;
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) { const uint32_t a = v[q][j].amax(); m = a > m ? a : m; }
      const BlockScale bs = block_scale<FX>(dpp_umax<0x4E>(dpp_umax<0xB1>(m)));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *(uint2*)&xs[buf][b][row][((2 * j + (l >> 1)) ^ turn(row)) * 16 + (l & 1) * 8] = quant8<T, FX>(v[q][j], bs);
      if (l == 0) se[buf][row][b] = bs.byte;
    }
  };
  load(lo);
  i32x8 w[NKB][2];
  uint32_t sw[WORDS];
  const bool busy = n0 < p.N && wm * 32 < p.bm;           // (others only cut)
  if (busy) {
    const int n = min(n0 + r, p.N - 1);
    const uint8_t* row = p.w + (int64_t)n * p.ldw + h * 64;
#pragma unroll
    for (int b = 0; b < NKB; ++b)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        w[b][ks] = __builtin_shufflevector(*(const i32x4*)(row + b * 128 + ks * 32), *(const i32x4*)(row + b * 128 + ks * 32 + 16), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
    for (int b = 0; b < WORDS; ++b) sw[b] = *(const uint32_t*)(p.sw + (int64_t)n * p.ldsw + 4 * b);
  }
  cut(0);
  if (lo + p.bm < hi) load(lo + p.bm);
  __syncthreads();
  int off[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) off[c] = r * 128 + ((4 * h + c) ^ turn(r)) * 16;
  int buf = 0;
  for (int64_t m = lo; m < hi; m += p.bm, buf ^= 1) {
    const int rows = (int)(hi - m < p.bm ? hi - m : p.bm);
    if (busy)
      for (int sub = wm; sub * 32 < rows; sub += step) {
        f32x16 acc;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] = 0.f;
        uint32_t sx[WORDS];
#pragma unroll
        for (int b = 0; b < WORDS; ++b) sx[b] = *(const uint32_t*)&se[buf][sub * 32 + r][4 * b];
        lin_chain<FX, NKB>(acc, w, sw, sx, &xs[buf][0][sub * 32][0], off);
        // lane = row r of y, register e = column 8 (e / 4) + 4 h + e % 4: two groups of eight columns trade halves between the halves of the
        // wave, and every lane holds 16 bytes of its row
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          f32x4 a = {acc[8 * g], acc[8 * g + 1], acc[8 * g + 2], acc[8 * g + 3]}, b = {acc[8 * g + 4], acc[8 * g + 5], acc[8 * g + 6], acc[8 * g + 7]};
          if (p.o.relu) {
#pragma unroll
            for (int j = 0; j < 4; ++j) { a[j] = relu_nan(a[j]); b[j] = relu_nan(b[j]); }
          }
          typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
          u32x2 ua, ub;
          if (p.o.type == FT_F16) { ua = __builtin_bit_cast(u32x2, __builtin_convertvector(a, h16x4)); ub = __builtin_bit_cast(u32x2, __builtin_convertvector(b, h16x4)); }
          else { ua = __builtin_bit_cast(u32x2, __builtin_convertvector(a, b16x4)); ub = __builtin_bit_cast(u32x2, __builtin_convertvector(b, b16x4)); }
          const auto s0 = __builtin_amdgcn_permlane32_swap(ua[0], ub[0], false, false), s1 = __builtin_amdgcn_permlane32_swap(ua[1], ub[1], false, false);
          const i32x4 out = {(int)s0[0], (int)s1[0], (int)s0[1], (int)s1[1]};
          const int n = n0 + 16 * g + 8 * h, row = sub * 32 + r;
          if (row < rows && n < p.N) {
            uint16_t* y = (uint16_t*)((uint8_t*)p.o.y + 2 * m * p.o.ldy + 2 * ((uint32_t)row * (uint32_t)p.o.ldy + (uint32_t)n));
            if (n + 8 <= p.N) __builtin_memcpy(y, &out, 16);
            else {
#pragma unroll
              for (int j = 0; j < 7; ++j) if (n + j < p.N) y[j] = (uint16_t)((uint32_t)out[j / 2] >> (16 * (j & 1)));
            }
          }
        }
      }
    if (m + p.bm < hi) {
      cut(buf ^ 1);
      if (m + 2 * p.bm < hi) load(m + 2 * p.bm);
    }
    __syncthreads();            // this tile has been read, the next one is written
  }
}

// ... and for more columns than registers hold: the tiles of k_fp8_nt (128 x 128, four waves) with the rows of x cut into blocks on the way into LDS.
// While a step is multiplied the 32 KB of x and 16 KB of W of the next one are on their way to registers (not straight to LDS: the wait for such
// copies would wait for x as well).  Every column tile cuts the rows again.  444219 x 1203 x 40 bound by memory: 266 .. 283 us, 3.9 TB/s; 1 x 4096 x 4096
// 13.6 us with the joining of its parts, 16 MB of weights.
struct Fp8Cut {
  const void* x; int64_t ldx;
  const uint8_t* w; int64_t ldw; const uint8_t* sw; int64_t ldsw;
  int64_t M; int N, K, nkb, splits, per;         // as in Fp8NT
  Fp8Out o;
};
template <int T, int FX>
__global__ __launch_bounds__(256, 2) void k_fp8_cut(Fp8Cut p) {
  __shared__ __attribute__((aligned(16))) uint8_t tiles[2][256][128];      // rows of x, rows of W; 16-byte pieces turned by the row
  __shared__ uint8_t se[2][128];                                           // exponents + 127 of x
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5, wm = wave & 1, wn = wave >> 1;
  const int ntn = (p.N + 127) / 128, item = xcd_item((int)((p.M + 127) / 128) * ntn);       // the column tiles of a row tile follow each other
  if (item < 0) return;
  const int64_t m0 = (int64_t)(item / ntn) * 128;
  const int n0 = item % ntn * 128, kb0 = blockIdx.y * p.per, kb1 = min(p.nkb, kb0 + p.per);
  // rows behind the last are read as that one: what is made of them is never stored
  const int l = tid & 3, row = tid >> 2, piece = tid & 7, wrow = tid >> 3;                  // rows of x: row + 64 q, of W: wrow + 32 i
  const uint16_t* px[2];
  const uint8_t* pw[4];
#pragma unroll
  for (int q = 0; q < 2; ++q) px[q] = (const uint16_t*)p.x + min(m0 + row + 64 * q, p.M - 1) * p.ldx;
#pragma unroll
  for (int i = 0; i < 4; ++i) pw[i] = p.w + (int64_t)min(n0 + wrow + 32 * i, p.N - 1) * p.ldw + piece * 16;
  Eight<T> v[2][4];
  i32x4 w[4];
  auto load = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *(const i32x4*)(pw[i] + (int64_t)kb * 128);
    // (pieces that reach over the row's end are read where the last whole one is, and shifted down when they are cut)
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) __builtin_memcpy(&v[q][j].v, px[q] + min(kb * 128 + l * 8 + 32 * j, p.K - 8), 16);
  };
  auto cut = [&](int buf, int kb) __attribute__((always_inline)) {
    if ((kb + 1) * 128 > p.K) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int over = kb * 128 + l * 8 + 32 * j - (p.K - 8);      // columns behind the last
#pragma unroll
        for (int q = 0; q < 2; ++q)
          if (over > 0) {
            typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
            u64x2 t = __builtin_bit_cast(u64x2, v[q][j].v);
            const int bits = 16 * over;
            if (bits >= 128) t = (u64x2)0;
            else if (bits >= 64) { t[0] = t[1] >> (bits - 64); t[1] = 0; }
            else { t[0] = (t[0] >> bits) | (t[1] << (64 - bits)); t[1] >>= bits; }
            v[q][j].v = __builtin_bit_cast(u16x8, t);
          }
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) { const uint32_t a = v[q][j].amax(); m = a > m ? a : m; }
      const BlockScale bs = block_scale<FX>(dpp_umax<0x4E>(dpp_umax<0xB1>(m)));
      const int at = row + 64 * q;
#pragma unroll
      for (int j = 0; j < 4; ++j) *(uint2*)&tiles[buf][at][((2 * j + (l >> 1)) ^ turn(at)) * 16 + (l & 1) * 8] = quant8<T, FX>(v[q][j], bs);
      if (l == 0) se[buf][at] = bs.byte;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) *(i32x4*)&tiles[buf][128 + wrow + 32 * i][(piece ^ turn(wrow + 32 * i)) * 16] = w[i];
  };
  // scales of W as in k_fp8_nt
  const uint8_t* pb[2];
  uint32_t sb[2], nb[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) { pb[i] = p.sw + (int64_t)min(n0 + (wn * 2 + i) * 32 + r, p.N - 1) * p.ldsw + kb0; nb[i] = *(const uint32_t*)pb[i]; }
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  int off[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) off[c] = r * 128 + (((4 * h + c) ^ turn(r)) * 16);
  load(kb0);
  cut(0, kb0);
  if (kb0 + 1 < kb1) load(kb0 + 1);
  __syncthreads();
  for (int kb = kb0; kb < kb1; ++kb) {
    const int buf = (kb - kb0) & 1;
    if (((kb - kb0) & 3) == 0) {
      const bool more = kb + 4 < kb1;
#pragma unroll
      for (int i = 0; i < 2; ++i) { sb[i] = nb[i]; pb[i] += 4; if (more) nb[i] = *(const uint32_t*)pb[i]; }
    }
    const uint8_t *ta = &tiles[buf][wm * 64][0], *tb = &tiles[buf][128 + wn * 64][0];
    int sa[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) sa[j] = se[buf][wm * 64 + 32 * j + r];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      i32x8 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fb[i] = __builtin_shufflevector(*(const i32x4*)(tb + i * 4096 + off[2 * ks]), *(const i32x4*)(tb + i * 4096 + off[2 * ks + 1]), 0, 1, 2, 3, 4, 5, 6, 7);
        fa[i] = __builtin_shufflevector(*(const i32x4*)(ta + i * 4096 + off[2 * ks]), *(const i32x4*)(ta + i * 4096 + off[2 * ks + 1]), 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[i][j] = mfma8<F8_E4M3, FX>(fb[i], fa[j], acc[i][j], (int)sb[i], sa[j]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) sb[i] >>= 8;
    if (kb + 1 < kb1) {
      cut(buf ^ 1, kb + 1);
      if (kb + 2 < kb1) load(kb + 2);
    }
    __syncthreads();            // this tile has been read, the next one is written
  }
  Fp8Out o = p.o;
  if (p.splits > 1) { o.y = (float*)o.y + (int64_t)blockIdx.y * p.M * p.N; o.ldy = p.N; o.type = FT_F32; o.relu = 0; }
  uint8_t* buf = &tiles[0][0][0] + wave * 8192;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t m = m0 + (wm * 2 + j) * 32;
    if (o.type == FT_F32) store_block<true>(o, acc[0][j], acc[1][j], buf, m, p.M, n0 + wn * 64, p.N, lane);
    else store_block<false>(o, acc[0][j], acc[1][j], buf, m, p.M, n0 + wn * 64, p.N, lane);
  }
}

// ------------------------------------------------------------------------------------------------------ weight gradients
// dW = G^T X over the rows of g and x, both cut into blocks of 128 ROWS per column on the way.  The result is fp32 and the sum long, so the
// 8-bit values go back to bf16 for the bf16 matrix instruction, exactly: 16-bit operands have nothing under 2^-133 that rounding could keep (fp16 2^-24),
// and what would round up to 2^128 takes the value below (tn_max).  A block of 8 waves owns 64 NI x 256 results and a range of
// 128-row steps.  Per step every wave turns strips of 128 rows x 32 columns round: a lane holds 8 rows x 8 columns (rows rg, rg + 16, ...: a
// load instruction reads 64 bytes of 16 rows), pairs up its rows (v_perm), the column's maximum crosses the 16 lanes of a DPP row, and each
// column leaves as 128 bytes of 8-bit values.  Both operands carry the same order of the rows, whatever it is.
// Two LDS buffers: while a step is multiplied the strips of the next one are cut into blocks, and the loads of the strip after that are in flight.
// 2^19 x 512 x 512 fp16: 393 .. 405 us (0.69 PFLOP/s, and 1.07 GB at 2.7 TB/s), with g in e5m2 the same.  Every value is read by two blocks (of the same XCD) and cut by both; the
// matrix instructions of a SIMD take 35% of the time, the vector ones that cut and widen most of the rest, and this pattern of loads alone 300 us.
// Strips of 64 columns by pairs of waves (128-byte pieces of 8 rows, 214 us alone) need a third barrier and took 417 us, two strips on their way per
// wave 395, sixteen waves or half strips in turn more registers than there are.
struct Fp8TN {
  const void* g; int64_t ldg; const void* x; int64_t ldx;
  int64_t M; int N, K;
  int tn, tk, parts, per;         // tiles of the result, parts of the rows, steps of a part
  float* y;                       // [parts][N][K]
};

__device__ inline uint32_t pk_max16(uint32_t a, uint32_t b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ inline uint32_t pk_min16(uint32_t a, uint32_t b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <int CTRL> __device__ inline uint32_t dpp_pk_max16(uint32_t v) {
  return pk_max16(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false));
}

// one strip: v[i] = eight columns of row i * 16 + rg; m: maxima of the eight columns, two to a word.  edge: the least bf16 magnitude that would round up
// to 2^128 in 8 bits, which the products' bf16 does not hold; it and what lies above become the 8-bit value below, `under`.
template <int T> __device__ inline void tn_max(u16x8 (&v)[8], uint32_t (&m)[4], uint32_t edge, uint32_t under) {
  constexpr uint32_t INF = T == FT_F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    m[k] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m[k] = pk_max16(m[k], __builtin_bit_cast(i32x4, v[i])[k] & 0x7fff7fff);
    m[k] = dpp_pk_max16<0xB1>(m[k]);
    m[k] = dpp_pk_max16<0x4E>(m[k]);
    m[k] = dpp_pk_max16<0x141>(m[k]);
    m[k] = dpp_pk_max16<0x140>(m[k]);
  }
  const uint32_t most = pk_max16(pk_max16(m[0], m[1]), pk_max16(m[2], m[3]));
  if (T == FT_F16) edge = INF;
  if (__any((most >> 16) >= edge || (most & 0xffffu) >= edge)) {
    if constexpr (T == FT_BF16) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        i32x4 w = __builtin_bit_cast(i32x4, v[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = (int)(pk_min16((uint32_t)w[k] & 0x7fff7fffu, under * 0x10001u) | ((uint32_t)w[k] & 0x80008000u));
        v[i] = __builtin_bit_cast(u16x8, w);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)        // a column with a NaN or an infinity becomes NaN throughout
      if (((m[j / 2] >> (16 * (j & 1))) & 0xffffu) >= INF) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i][j] = 0x7fff;
      }
  }
}
// ... in 8 bits: tile: [32 columns][128 bytes], scale: their powers of two
template <int T, int FMT> __device__ inline void tn_quant(const u16x8 (&v)[8], const uint32_t (&m)[4], uint8_t* tile, float* scale, int lane) {
  constexpr int EMAX = FMT == F8_E4M3 ? 8 : 15;
  const int rg = lane & 15, c8 = (lane >> 4) * 8;
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t a = (j & 1) ? m[j / 2] >> 16 : m[j / 2] & 0xffffu;
    const uint32_t bits = T == FT_F16 ? __float_as_uint((float)__builtin_bit_cast(h16, (uint16_t)a)) : a << 16;
    // block_scale's power of two (a column of zeros may have any)
    const int e = (int)(bits + 0x1fffffu) - (EMAX << 23);
    s[j] = __uint_as_float((uint32_t)(e < 1 << 23 ? 1 << 23 : e) & 0x7f800000u);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)        // column j of two rows in one word
      w[i] = __builtin_amdgcn_perm(__builtin_bit_cast(i32x4, v[2 * i + 1])[j / 2], __builtin_bit_cast(i32x4, v[2 * i])[j / 2], (j & 1) ? 0x07060302u : 0x05040100u);
    *(uint2*)(tile + (c8 + j) * 128 + ((((rg >> 1) ^ turn(c8 + j)) * 16) | ((rg & 1) * 8))) = make_uint2(cvt4<T, FMT>(w[0], w[1], s[j]), cvt4<T, FMT>(w[2], w[3], s[j]));
  }
  if (rg == 0) { *(f32x4*)(scale + c8) = (f32x4){s[0], s[1], s[2], s[3]}; *(f32x4*)(scale + c8 + 4) = (f32x4){s[4], s[5], s[6], s[7]}; }
}

// TAIL: the last step is not whole or its pieces would reach over the tensors' end; the code for that costs the others registers (with dx, 630 us
// -> 660 at 2^19 x 512 x 512, where there is none).
template <int T, int FG, int NI, bool TAIL>
__global__ __launch_bounds__(512, 2) void k_fp8_tn(Fp8TN p) {
  constexpr int TN = 64 * NI, TK = 256, COLS = TN + TK, STRIPS = COLS / 32;      // 8 < STRIPS <= 16
  extern __shared__ __attribute__((aligned(16))) uint8_t smem8[];     // [2][COLS][128], then [2][COLS] powers of two
  float* scales = (float*)(smem8 + 2 * COLS * 128);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
  const int wn = wave & 1, wk = wave >> 1;                // waves: 2 along n (32 NI columns each), 4 along k (64 each)
  const int tiles = p.tn * p.tk, item = xcd_item(p.parts * tiles), part = item / tiles, tile = item % tiles;     // the tiles of a part follow each other
  if (item < 0) return;
  const int64_t nsteps = (p.M + 127) / 128, s0 = (int64_t)part * p.per, s1 = s0 + p.per < nsteps ? s0 + p.per : nsteps;
  const int n0 = tile / p.tk * TN, k0 = tile % p.tk * TK;
  f32x16 acc[NI][2];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  u16x8 v[8];                                             // one strip on its way
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (u16x8)(uint16_t)0;
  const int rg = lane & 15, c8 = (lane >> 4) * 8;
  auto load = [&](int64_t step, int strip) __attribute__((always_inline)) {
    if (step >= s1 || strip >= STRIPS) return;
    // a uniform base and a 32-bit offset of the lane (ld < 2^24): no 64-bit arithmetic per lane
    const bool isg = strip < TN / 32;
    const int64_t ld = isg ? p.ldg : p.ldx;
    const int C = isg ? p.N : p.K, col = isg ? n0 + strip * 32 : k0 + (strip - TN / 32) * 32;
    if (col >= C) return;                                 // (whole strips behind the last column: cut from what is there, never stored)
    const uint16_t* base = (const uint16_t*)(isg ? p.g : p.x) + step * 128 * ld + col;
    const int c = tn_column(C, col, c8);
    if (!TAIL || tn_whole(p.M, ld, C, step, col)) {
      const uint32_t off = 2 * ((uint32_t)rg * (uint32_t)ld + (uint32_t)c);       // bytes
#pragma unroll
      for (int i = 0; i < 8; ++i) __builtin_memcpy(&v[i], (const uint8_t*)(base + i * 16 * ld) + off, 16);
    } else {
      const TnEnd e = tn_end(p.M, ld, C, step, col);
      int over[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const TnPiece q = tn_piece(e, (int)ld, rg + 16 * i, c);
        over[i] = q.over;
        __builtin_memcpy(&v[i], base + q.at, 16);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
        u64x2 w = __builtin_bit_cast(u64x2, v[i]);
        const int bits = 16 * over[i];
        if (bits >= 64) { w[0] = w[1] >> (bits - 64); w[1] = 0; }
        else if (bits > 0) { w[0] = (w[0] >> bits) | (w[1] << (64 - bits)); w[1] >>= bits; }
        if (rg + 16 * i > e.last) w = (u64x2)0;
        v[i] = __builtin_bit_cast(u16x8, w);
      }
    }
  };
  auto cut = [&](int64_t step, int strip) __attribute__((always_inline)) {
    if (step >= s1 || strip >= STRIPS) return;
    const int buf = (int)(step - s0) & 1;
    uint8_t* t = smem8 + (buf * COLS + strip * 32) * 128;
    float* sc = scales + buf * COLS + strip * 32;
    const bool other = FG != F8_E4M3 && strip < TN / 32;      // (1.9375 2^127 becomes 1.875 2^127 in e4m3, 1.875 2^127 becomes 1.75 2^127 in e5m2)
    uint32_t m[4];
    tn_max<T>(v, m, other ? 0x7f70u : 0x7f78u, other ? 0x7f60u : 0x7f70u);
    if (other) tn_quant<T, FG>(v, m, t, sc, lane);
    else tn_quant<T, F8_E4M3>(v, m, t, sc, lane);
  };
  const bool busy = n0 + wn * 32 * NI < p.N && k0 + wk * 64 < p.K;      // (waves without results only cut)
  load(s0, wave);
  const int64_t halves = 2 * (s1 - s0 + 1);
  for (int64_t u = 0; u < halves; ++u) {     // two halves to a step: half of step s0 + u / 2 - 1 is multiplied, a strip of step s0 + u / 2 cut
    const int half = (int)u & 1;
    const int64_t next = s0 + (u >> 1);
    if (u >= 2 && busy) {
      const int buf = (int)(next - 1 - s0) & 1;
      const uint8_t* gt = smem8 + (buf * COLS + wn * 32 * NI + r) * 128;
      const uint8_t* xt = smem8 + (buf * COLS + TN + wk * 64 + r) * 128;
      const float* sc = scales + buf * COLS;
      float sg[NI], sx[2];
#pragma unroll
      for (int i = 0; i < NI; ++i) sg[i] = sc[wn * 32 * NI + 32 * i + r];
#pragma unroll
      for (int j = 0; j < 2; ++j) sx[j] = sc[TN + wk * 64 + 32 * j + r];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int off = ((4 * h + 2 * half + c) ^ turn(r)) * 16;
        i32x4 fg[NI], fx[2];
#pragma unroll
        for (int i = 0; i < NI; ++i) fg[i] = *(const i32x4*)(gt + i * 4096 + off);
#pragma unroll
        for (int j = 0; j < 2; ++j) fx[j] = *(const i32x4*)(xt + j * 4096 + off);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          b16x8 bx[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) bx[j] = widen8<F8_E4M3>(fx[j][2 * q], fx[j][2 * q + 1], sx[j]);
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const b16x8 bg = widen8<FG>(fg[i][2 * q], fg[i][2 * q + 1], sg[i]);
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bg, bx[j], acc[i][j], 0, 0, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);     // (or every fragment of the half is read ahead, and registers spill)
      }
    }
    cut(next, wave + 8 * half);
    load(next + half, wave + 8 - 8 * half);
    if (half) __syncthreads();            // the step has been read, the next one is written
  }
  // lane = column k, register e = row 8 (e / 4) + 4 h + e % 4 of a 32 x 32 block: a uniform row and a 32-bit offset of the lane
  if (!busy || k0 + wk * 64 + r >= p.K) return;
  const int nw = n0 + wn * 32 * NI;
  float* y = p.y + ((int64_t)part * p.N + nw) * p.K + k0 + wk * 64;
  const bool second = k0 + wk * 64 + 32 + r < p.K;
  const uint32_t off = 4u * h * (uint32_t)p.K + r;        // (K < 2^24)
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int n = 32 * i + 8 * (e / 4) + e % 4;         // + 4 h
      if (nw + n + 4 * h < p.N) {
        float* row = y + (int64_t)n * p.K;
        row[off] = acc[i][0][e];
        if (second) row[off + 32] = acc[i][1][e];
      }
    }
}

// The slabs of a split contraction, added in a fixed order and rounded once.  Eight threads share four results (their slabs' sums meet through
// shuffles): 85 slabs of 128 x 512 6.8 us, and 22 with a result's slabs read by one thread alone; 64 slabs of 512 x 512 15 us, 4.5 TB/s.
__global__ __launch_bounds__(256) void k_fp8_join(const float* __restrict__ slabs, int splits, int64_t M, int N, Fp8Out o) {
  const int64_t n = M * N;
  for (int64_t q = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 3; q < (n + 3) / 4; q += (int64_t)gridDim.x * 32) {
    const int sub = threadIdx.x & 7;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    const bool whole = 4 * q + 4 <= n;
#pragma unroll 4
    for (int k = sub; k < splits; k += 8) {
      const float* p = slabs + k * n + 4 * q;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (whole) __builtin_memcpy(&v, p, 16);
      else for (int j = 0; j < 3; ++j) if (4 * q + j < n) v[j] = p[j];
      s += v;
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += __shfl_xor(s[j], d);
    const int64_t i = 4 * q + sub;
    if (sub >= 4 || i >= n) continue;
    float r = sub == 0 ? s[0] : sub == 1 ? s[1] : sub == 2 ? s[2] : s[3];
    if (o.relu) r = relu_nan(r);
    const int64_t at = i / N * o.ldy + i % N;
    if (o.type == FT_F32) ((float*)o.y)[at] = r;
    else if (o.type == FT_F16) ((h16*)o.y)[at] = (h16)r;
    else ((__bf16*)o.y)[at] = (__bf16)r;
  }
}

// ------------------------------------------------------------------------------------------------------------ entry points
#define MOST32 (((int64_t)1 << 31) - 256)      // sizes that are counted in 32 bits, in tiles of up to 256
static bool is_ft(int t) { return t >= FT_F16 && t <= FT_F32; }
static bool is_f8(int f) { return f == F8_E4M3 || f == F8_E5M2; }
static bool blocks_ok(const void* q, int64_t ldq, const void* s, int64_t lds, int64_t K) {
  return q && s && ldq >= ceil128(K) && ldq % 16 == 0 && ((uintptr_t)q & 15) == 0 && lds >= ceil128(K) / 128 && lds % 4 == 0 && ((uintptr_t)s & 3) == 0;
}
#define FP8_BAD_BLOCKS "%s: 8-bit blocks need 16-byte aligned values with a pitch that is a multiple of 16 and holds whole blocks of 128, and 4-byte aligned scales with a pitch that is a multiple of 4"

template <int T, int FMT>
static int quant_launch(bool t, const void* x, int64_t ldx, int64_t M, int K, void* q, int64_t ldq, uint8_t* scale, int64_t lds, hipStream_t st) {
  if (!t) {
    const int nb = (int)(ceil128(K) / 128);
    hipLaunchKernelGGL((k_fp8_quant<T, FMT>), dim3(aln_grid_for(M * nb, 16, 256 * 16)), dim3(256), 0, st, x, ldx, M, K, nb, (uint8_t*)q, ldq, scale, lds);
  } else {
    const int64_t nb = ceil128(M) / 128, g = nb * ((K + 63) / 64);
    ALN_REQUIRE(g < (int64_t)1 << 24, "fp8_quantize: %lld x %d values are too many for one launch", (long long)M, K);
    hipLaunchKernelGGL((k_fp8_quant_t<T, FMT>), dim3((uint32_t)g), dim3(256), 0, st, x, ldx, M, K, (int)nb, (uint8_t*)q, ldq, scale, lds);
  }
  ALN_CHECK_LAUNCH("fp8_quantize");
  return 0;
}
template <int T>
static int quant_fmt(int fmt, bool t, const void* x, int64_t ldx, int64_t M, int K, void* q, int64_t ldq, uint8_t* scale, int64_t lds, hipStream_t st) {
  return fmt == F8_E4M3 ? quant_launch<T, F8_E4M3>(t, x, ldx, M, K, q, ldq, scale, lds, st) : quant_launch<T, F8_E5M2>(t, x, ldx, M, K, q, ldq, scale, lds, st);
}
static int quantize(const char* name, bool t, const void* x, int x_type, int64_t ldx, int64_t M, int K, int fmt, void* q, int64_t ldq, uint8_t* scale, int64_t lds,
                    hipStream_t st) {
  ALN_REQUIRE(is_ft(x_type) && is_f8(fmt), "%s: unknown type %d or format %d", name, x_type, fmt);
  ALN_REQUIRE(M >= 0 && M <= MOST32 && K >= 1 && K <= MOST32 && ldx >= 0, "%s: %lld x %d values with pitch %lld", name, (long long)M, K, (long long)ldx);
  if (M == 0) return 0;
  ALN_REQUIRE(x, "%s: NULL pointer", name);
  ALN_REQUIRE(((uintptr_t)x & (x_type == FT_F32 ? 3 : 1)) == 0, "%s: x is not aligned to its type", name);
  ALN_REQUIRE(blocks_ok(q, ldq, scale, lds, t ? M : K), FP8_BAD_BLOCKS, name);
  return x_type == FT_F16 ? quant_fmt<FT_F16>(fmt, t, x, ldx, M, K, q, ldq, scale, lds, st) : x_type == FT_BF16 ? quant_fmt<FT_BF16>(fmt, t, x, ldx, M, K, q, ldq, scale, lds, st)
                                                                                                : quant_fmt<FT_F32>(fmt, t, x, ldx, M, K, q, ldq, scale, lds, st);
}
extern "C" int aln_fp8_quantize(const void* x, int32_t x_type, int64_t ldx, int64_t M, int32_t K, int32_t fmt, void* q, int64_t ldq, uint8_t* scale, int64_t lds,
                                void* stream) {
  return quantize("fp8_quantize", false, x, x_type, ldx, M, K, fmt, q, ldq, scale, lds, (hipStream_t)stream);
}
extern "C" int aln_fp8_quantize_t(const void* x, int32_t x_type, int64_t ldx, int64_t M, int32_t C, int32_t fmt, void* q, int64_t ldq, uint8_t* scale, int64_t lds,
                                  void* stream) {
  return quantize("fp8_quantize_t", true, x, x_type, ldx, M, C, fmt, q, ldq, scale, lds, (hipStream_t)stream);
}

// How a product is cut: tiles of y, and parts of the contraction where the tiles alone leave CUs without work.  A step of 128 x 128 x 128 takes a
// lone block on its CU about 0.8 us; joining the parts costs a launch (4 us) and their slabs' way through the memory-side cache and back.  With
// and without parts: 256 x 512 x 4096 12.7 us and 24.2, 64 x 1024 x 4096 11.0 and 28.2, 1024 x 1024 x 4096 22.6 and 29.8; but 1920 x 1024 x 2048 in
// four parts 26.4 and 15.6 in one.
struct NtPlan { int splits, per; };
static NtPlan nt_plan(int64_t M, int N, int64_t K, double step = 0.8) {
  const int64_t tiles = (M + 127) / 128 * ((N + 127) / 128), nkb = ceil128(K) / 128;
  NtPlan best{1, (int)((nkb + 3) / 4 * 4)};
  double least = step * nkb;
  for (int64_t per = 4; per < nkb; per += 4) {            // (whole words of scales)
    const int64_t parts = (nkb + per - 1) / per;
    const double t = step * per + 4.0 + 2e-6 * parts * M * N;
    if (parts * tiles <= 256 && t < least) { least = t; best = {(int)parts, (int)per}; }
  }
  return best;
}
static int64_t slab_bytes(const NtPlan& pl, int64_t M, int N) { return pl.splits > 1 ? (int64_t)pl.splits * M * N * 4 : 0; }
extern "C" int64_t aln_fp8_nt_ws_bytes(int64_t M, int32_t N, int64_t K) { return M <= 0 || N <= 0 || K <= 0 ? 0 : slab_bytes(nt_plan(M, N, K), M, N); }
template <int FA, int FB, bool WIDE, int WM, int WN, int MI, int NI> static int nt_launch(const Fp8NT& p, hipStream_t st) {
  constexpr int BM = WM * MI * 32, BN = WN * NI * 32, LDS = 2 * (BM + BN) * 128;
  // (at every call: it holds for the current device)
  const hipError_t big = hipFuncSetAttribute((const void*)k_fp8_nt<FA, FB, WIDE, WM, WN, MI, NI>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  ALN_REQUIRE(big == hipSuccess, "fp8_nt: %s", hipGetErrorString(big));
  const int64_t g = (p.M + BM - 1) / BM * ((p.N + BN - 1) / BN);
  ALN_REQUIRE(g < (int64_t)1 << 22, "fp8_nt: %lld x %d results are too many for one launch", (long long)p.M, p.N);
  hipLaunchKernelGGL((k_fp8_nt<FA, FB, WIDE, WM, WN, MI, NI>), dim3(xcd_grid(g), p.splits), dim3(64 * WM * WN), LDS, st, p);
  ALN_CHECK_LAUNCH("fp8_nt");
  return 0;
}
template <int FA, int FB> static int nt_type(const Fp8NT& p, int y_type, hipStream_t st) {
  // rounds of the 256 CUs: one 256 x 256 tile at a time takes 4 / 3 of the time of two 128 x 128 ones.  Large and small tiles: 4096 x 4096 x 4096 65.5 us and
  // 88.5, 3840 x 3840 x 2048 33.6 and 44.7, 8192 x 4096 x 1024 40.6 and 52.4, but 2048 x 4096 x 4096 57.0 and 43.7
  const int64_t large = (p.M + 255) / 256 * ((p.N + 255) / 256), small = (p.M + 127) / 128 * ((p.N + 127) / 128);
  const bool big = 4 * ((large + 255) / 256) <= 3 * ((small + 511) / 512);
  if (y_type == FT_F32) return big ? nt_launch<FA, FB, true, 2, 4, 4, 2>(p, st) : nt_launch<FA, FB, true, 2, 2, 2, 2>(p, st);
  return big ? nt_launch<FA, FB, false, 2, 4, 4, 2>(p, st) : nt_launch<FA, FB, false, 2, 2, 2, 2>(p, st);
}
extern "C" int aln_fp8_nt(const void* a, int64_t lda, const uint8_t* sa, int64_t ldsa, int32_t fmt_a, const void* b, int64_t ldb, const uint8_t* sb, int64_t ldsb,
                          int32_t fmt_b, int64_t M, int32_t N, int64_t K, void* y, int64_t ldy, int32_t y_type, int32_t relu, void* ws, int64_t ws_bytes,
                          void* stream) {
  ALN_REQUIRE(is_f8(fmt_a) && is_f8(fmt_b) && is_ft(y_type), "fp8_nt: unknown format %d, %d or type %d", fmt_a, fmt_b, y_type);
  ALN_REQUIRE(M >= 0 && M <= MOST32 && N >= 1 && N <= MOST32 && K >= 1 && K <= MOST32 && ldy >= N, "fp8_nt: sizes %lld x %d x %lld, pitch %lld", (long long)M, N, (long long)K,
              (long long)ldy);
  if (M == 0) return 0;
  ALN_REQUIRE(blocks_ok(a, lda, sa, ldsa, K) && blocks_ok(b, ldb, sb, ldsb, K), FP8_BAD_BLOCKS, "fp8_nt");
  ALN_REQUIRE(y && ((uintptr_t)y & (y_type == FT_F32 ? 3 : 1)) == 0, "fp8_nt: y is NULL or not aligned to its type");
  const NtPlan pl = nt_plan(M, N, K);
  ALN_REQUIRE(ws_bytes >= aln_fp8_nt_ws_bytes(M, N, K) && (pl.splits == 1 || (ws && ((uintptr_t)ws & 15) == 0)), "fp8_nt: the workspace needs %lld bytes, aligned to 16",
              (long long)aln_fp8_nt_ws_bytes(M, N, K));
  const Fp8Out o{y, ldy, y_type, relu};
  Fp8NT p{(const uint8_t*)a, lda, sa, ldsa, (const uint8_t*)b, ldb, sb, ldsb, M, N, (int)(ceil128(K) / 128), pl.splits, pl.per, o};
  if (pl.splits > 1) p.o.y = ws;
  hipStream_t st = (hipStream_t)stream;
  const int rc = fmt_a == F8_E4M3 ? (fmt_b == F8_E4M3 ? nt_type<F8_E4M3, F8_E4M3>(p, y_type, st) : nt_type<F8_E4M3, F8_E5M2>(p, y_type, st))
                                  : (fmt_b == F8_E4M3 ? nt_type<F8_E5M2, F8_E4M3>(p, y_type, st) : nt_type<F8_E5M2, F8_E5M2>(p, y_type, st));
  if (rc || pl.splits == 1) return rc;
  hipLaunchKernelGGL(k_fp8_join, dim3(aln_grid_for((M * N + 3) / 4, 32, 4096)), dim3(256), 0, st, (const float*)ws, pl.splits, M, N, o);
  ALN_CHECK_LAUNCH("fp8_nt");
  return 0;
}

// ---- x W^T for x as it is.  16-bit x and y, e4m3 weights, up to 512 columns (1024 with few rows or few columns of y): the one-launch kernel;
// otherwise, with few rows or few columns of y, the tiles that cut rows (lin_cut), or blocks of x in the workspace, then the product.
// (eight waves hold 256 columns of y at 513 .. 1024 columns of x, and every further part cuts the rows again.  In one launch and in two: 64 x 1024 x 4096
// 8.9 us and 14.0, 1024 x 1024 x 4096 16.9 and 16.6, 8192 x 1024 x 4096 62 and 50, 8192 x 640 x 4096 44 and 38, 8192 x 1024 x 1024 24 either way, 65537 x 1024
// x 512 80 and 95; up to 512 columns 131072 x 512 x 4096 482 and 557)
static bool lin_fused(int64_t M, int N, int64_t K, int x_type, int y_type, int fmt_w) {
  return (K <= 512 || (K <= 1024 && (N <= 1024 || M <= 512))) && x_type != FT_F32 && y_type != FT_F32 && fmt_w == F8_E4M3;
}
// Otherwise k_fp8_cut, where its column tiles are few or there is one row tile to cut again: 444219 x 1203 x 40 283 us and 499 in two launches, 65536 x 1280
// x 128 40 and 67, 200000 x 1100 x 300 251 and 294, 30000 x 4096 x 384 130 and 136, but x 512 154 and 143; 3 x 1844 x 3304 13.4 and 13.5 (a launch less on the
// host: 13.4 and 15.4 a call), 64 x 4096 x 4096 17.8 either way, 128 x 4096 x 4096 20.6 and 22.3, but 129 x 4096 x 4096 23.8 and 21.6, 257 x 4096 x 4096 37.1 and
// 29.6, 384 x 4096 x 4096 39.9 and 32.6, 384 x 2048 x 4096 28.3 and 19.5 (300 x 2048 x 2048 19.1 and 19.7).
#define CUT_STEP 1.4                 // us of a lone block's step (nt_plan)
static bool lin_cut(int64_t M, int N, int x_type, int y_type, int fmt_w) {
  return (N <= 384 || M <= 128) && x_type != FT_F32 && y_type != FT_F32 && fmt_w == F8_E4M3;
}
static inline int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
extern "C" int64_t aln_fp8_linear_ws_bytes(int64_t M, int32_t N, int32_t K, int32_t x_type, int32_t y_type, int32_t fmt_w) {
  if (M <= 0 || N <= 0 || K <= 0 || lin_fused(M, N, K, x_type, y_type, fmt_w)) return 0;
  if (lin_cut(M, N, x_type, y_type, fmt_w)) return slab_bytes(nt_plan(M, N, K, CUT_STEP), M, N);
  const int64_t nb = ceil128(K) / 128;
  return M * nb * 128 + up16(M * ((nb + 3) / 4 * 4)) + aln_fp8_nt_ws_bytes(M, N, K);
}
template <int T, int FX> static int cut_launch(const Fp8Cut& p, hipStream_t st) {
  const int64_t g = (p.M + 127) / 128 * ((p.N + 127) / 128);
  ALN_REQUIRE(g < (int64_t)1 << 22, "fp8_linear: %lld x %d results are too many for one launch", (long long)p.M, p.N);
  hipLaunchKernelGGL((k_fp8_cut<T, FX>), dim3(xcd_grid(g), p.splits), dim3(256), 0, st, p);
  ALN_CHECK_LAUNCH("fp8_linear");
  return 0;
}
template <int T, int FX, int NKB> static int lin_launch(const Fp8Linear& p, hipStream_t st) {
  const int64_t g = (int64_t)p.ranges * p.parts;
  ALN_REQUIRE(g < (int64_t)1 << 22, "fp8_linear: %lld x %d results are too many for one launch", (long long)p.M, p.N);
  hipLaunchKernelGGL((k_fp8_linear<T, FX, NKB>), dim3(xcd_grid(g)), dim3(lin_threads<NKB>()), 0, st, p);
  ALN_CHECK_LAUNCH("fp8_linear");
  return 0;
}
template <int T, int FX> static int lin_pick(const Fp8Linear& p, int nkb, hipStream_t st) {
  switch (nkb) {
    case 1: return lin_launch<T, FX, 1>(p, st);
    case 2: return lin_launch<T, FX, 2>(p, st);
    case 3: return lin_launch<T, FX, 3>(p, st);
    case 4: return lin_launch<T, FX, 4>(p, st);
    case 5: return lin_launch<T, FX, 5>(p, st);
    case 6: return lin_launch<T, FX, 6>(p, st);
    case 7: return lin_launch<T, FX, 7>(p, st);
    default: return lin_launch<T, FX, 8>(p, st);
  }
}
extern "C" int aln_fp8_linear(const void* x, int32_t x_type, int64_t ldx, int32_t fmt_x, const void* w, int64_t ldw, const uint8_t* sw, int64_t ldsw, int32_t fmt_w,
                              int64_t M, int32_t N, int32_t K, void* y, int64_t ldy, int32_t y_type, int32_t relu, void* ws, int64_t ws_bytes, void* stream) {
  ALN_REQUIRE(is_ft(x_type) && is_ft(y_type) && is_f8(fmt_x) && is_f8(fmt_w), "fp8_linear: unknown type %d, %d or format %d, %d", x_type, y_type, fmt_x, fmt_w);
  ALN_REQUIRE(M >= 0 && M <= MOST32 && N >= 1 && K >= 1 && K <= MOST32 && ldx >= 0 && ldy >= N && ldx < 1 << 25 && ldy < 1 << 25,
              "fp8_linear: sizes %lld x %d x %d, pitches %lld, %lld (under 2^25)", (long long)M, N, K, (long long)ldx, (long long)ldy);
  if (M == 0) return 0;
  ALN_REQUIRE(blocks_ok(w, ldw, sw, ldsw, K), FP8_BAD_BLOCKS, "fp8_linear");
  ALN_REQUIRE(x && ((uintptr_t)x & (x_type == FT_F32 ? 3 : 1)) == 0 && y && ((uintptr_t)y & (y_type == FT_F32 ? 3 : 1)) == 0, "fp8_linear: x or y is NULL or not aligned to its type");
  const int64_t need = aln_fp8_linear_ws_bytes(M, N, K, x_type, y_type, fmt_w);
  ALN_REQUIRE(ws_bytes >= need && (need == 0 || (ws && ((uintptr_t)ws & 15) == 0)), "fp8_linear: the workspace needs %lld bytes, aligned to 16", (long long)need);
  const int nkb = (int)(ceil128(K) / 128);
  if (!lin_fused(M, N, K, x_type, y_type, fmt_w) && lin_cut(M, N, x_type, y_type, fmt_w)) {
    const NtPlan pl = nt_plan(M, N, K, CUT_STEP);
    const Fp8Out o{y, ldy, y_type, relu};
    Fp8Cut p{x, ldx, (const uint8_t*)w, ldw, sw, ldsw, M, N, K, nkb, pl.splits, pl.per, o};
    if (pl.splits > 1) p.o.y = ws;
    hipStream_t st = (hipStream_t)stream;
    const int rc = x_type == FT_F16 ? (fmt_x == F8_E4M3 ? cut_launch<FT_F16, F8_E4M3>(p, st) : cut_launch<FT_F16, F8_E5M2>(p, st))
                                    : (fmt_x == F8_E4M3 ? cut_launch<FT_BF16, F8_E4M3>(p, st) : cut_launch<FT_BF16, F8_E5M2>(p, st));
    if (rc || pl.splits == 1) return rc;
    hipLaunchKernelGGL(k_fp8_join, dim3(aln_grid_for((M * N + 3) / 4, 32, 4096)), dim3(256), 0, st, (const float*)ws, pl.splits, M, N, o);
    ALN_CHECK_LAUNCH("fp8_linear");
    return 0;
  }
  if (!lin_fused(M, N, K, x_type, y_type, fmt_w)) {
    uint8_t* q = (uint8_t*)ws, *sc = q + M * nkb * 128, *rest = sc + up16(M * ((nkb + 3) / 4 * 4));
    const int rc = aln_fp8_quantize(x, x_type, ldx, M, K, fmt_x, q, (int64_t)nkb * 128, sc, (nkb + 3) / 4 * 4, stream);
    if (rc) return rc;
    return aln_fp8_nt(q, (int64_t)nkb * 128, sc, (nkb + 3) / 4 * 4, fmt_x, w, ldw, sw, ldsw, fmt_w, M, N, K, y, ldy, y_type, relu, rest, ws_bytes - (rest - q), stream);
  }
  // One block of threads per CU.  While there are fewer 64-row tiles than CUs the columns of y are cut into more parts (each cuts the rows
  // into blocks again); the rows then go round evenly, in tiles of one size.  512 x 512 weights with these parts and with one part: 64 rows 5.4 us and
  // 12.3, 4096 rows 10.0 and 13.5, 8192 rows 14.3 and 14.9, the same from 16384 rows on.
  const int waves = nkb <= 4 ? 16 : 8, need_wn = (N + 31) / 32;
  const int64_t mt = (M + 63) / 64;
  int wn = 1;
  while (wn < waves && wn < need_wn && ((need_wn + wn - 1) / wn) * mt > 256) wn *= 2;
  const int parts = (need_wn + wn - 1) / wn;
  int64_t blocks = parts >= 256 ? 1 : 256 / parts;
  if (blocks > mt) blocks = mt;
  const int64_t rows = (M + blocks - 1) / blocks, tiles = (rows + 63) / 64;
  ALN_REQUIRE(rows < (int64_t)1 << 31, "fp8_linear: too many rows");
  const Fp8Linear p{x, ldx, (const uint8_t*)w, ldw, sw, ldsw, M, N, K, wn, parts, (int)((M + rows - 1) / rows), (int)rows, (int)((rows + tiles - 1) / tiles), Fp8Out{y, ldy, y_type, relu}};
  hipStream_t st = (hipStream_t)stream;
  return x_type == FT_F16 ? (fmt_x == F8_E4M3 ? lin_pick<FT_F16, F8_E4M3>(p, nkb, st) : lin_pick<FT_F16, F8_E5M2>(p, nkb, st))
                          : (fmt_x == F8_E4M3 ? lin_pick<FT_BF16, F8_E4M3>(p, nkb, st) : lin_pick<FT_BF16, F8_E5M2>(p, nkb, st));
}

// ---- dW [N, K] (fp32, contiguous) = G^T X over M rows.  16-bit g and x of one type (eight values each): the one-launch kernel (and the addition of its parts);
// otherwise both transposed into blocks in the workspace, then the product.
static bool tn_fused(int64_t M, int N, int K, int g_type, int x_type) { return g_type == x_type && g_type != FT_F32 && M * N >= 8 && M * K >= 8; }
struct TnPlan { int ni, tn, tk, parts, per; };
static TnPlan tn_plan(int64_t M, int N, int K) {
  TnPlan t;
  // 256 x 256 results to a block cut every value of g and x half as often as 128 x 256 do, where there are blocks enough for every CU: 2^19 x 512 x 512
  // 470 us against 609, 16384 x 1024 x 1024 75 against 84, but 8192 x 512 x 512 32.1 against 27.6 and 4096 x 512 x 512 29.1 against 24.2
  t.ni = N > 128 && (N + 255) / 256 * (int64_t)((K + 255) / 256) * ((M + 127) / 128) >= 512 ? 4 : 2;
  t.tn = (N + 64 * t.ni - 1) / (64 * t.ni); t.tk = (K + 255) / 256;
  const int64_t tiles = (int64_t)t.tn * t.tk, steps = (M + 127) / 128;
  int64_t parts = tiles >= 256 ? 1 : 256 / tiles;         // one block per CU
  if (parts > steps) parts = steps;
  // two steps at least, where the parts' slabs are more than small change.  With one step to a part and with two: 1003 x 77 x 130 11.9 us and 16.3,
  // 1000 x 256 x 256 13.6 and 17.9, 600 x 600 x 600 15.3 and 17.0, but 4096 x 256 x 512 21.2 and 19.4, 4096 x 512 x 512 25.9 and 24.2
  if (parts * N * K > 1 << 21 && parts > (steps + 1) / 2) parts = (steps + 1) / 2;
  t.per = (int)((steps + parts - 1) / parts);
  t.parts = (int)((steps + t.per - 1) / t.per);
  return t;
}
extern "C" int64_t aln_fp8_grad_weight_ws_bytes(int64_t M, int32_t N, int32_t K, int32_t g_type, int32_t x_type) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (tn_fused(M, N, K, g_type, x_type)) { const TnPlan t = tn_plan(M, N, K); return t.parts > 1 ? (int64_t)t.parts * N * K * 4 : 0; }
  const int64_t nb = ceil128(M) / 128, per_row = nb * 128 + (nb + 3) / 4 * 4;
  return up16(((int64_t)N + K) * per_row) + 16 * 4 + aln_fp8_nt_ws_bytes(N, K, M);
}
template <int T, int FG, int NI, bool TAIL> static int tn_launch(const Fp8TN& p, hipStream_t st) {
  constexpr int COLS = 64 * NI + 256, LDS = 2 * COLS * 132;
  const hipError_t big = hipFuncSetAttribute((const void*)k_fp8_tn<T, FG, NI, TAIL>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  ALN_REQUIRE(big == hipSuccess, "fp8_grad_weight: %s", hipGetErrorString(big));
  const int64_t g = (int64_t)p.parts * p.tn * p.tk;
  ALN_REQUIRE(g < (int64_t)1 << 22, "fp8_grad_weight: %d x %d results are too many for one launch", p.N, p.K);
  hipLaunchKernelGGL((k_fp8_tn<T, FG, NI, TAIL>), dim3(xcd_grid(g)), dim3(512), LDS, st, p);
  ALN_CHECK_LAUNCH("fp8_grad_weight");
  return 0;
}
template <int T, int FG, int NI> static int tn_tail(const Fp8TN& p, hipStream_t st) {
  return tn_has_tail(p.M, p.N, p.K) ? tn_launch<T, FG, NI, true>(p, st) : tn_launch<T, FG, NI, false>(p, st);
}
template <int T> static int tn_pick(const Fp8TN& p, const TnPlan& t, int fmt_g, hipStream_t st) {
  if (fmt_g == F8_E4M3) return t.ni == 4 ? tn_tail<T, F8_E4M3, 4>(p, st) : tn_tail<T, F8_E4M3, 2>(p, st);
  return t.ni == 4 ? tn_tail<T, F8_E5M2, 4>(p, st) : tn_tail<T, F8_E5M2, 2>(p, st);
}
extern "C" int aln_fp8_grad_weight(const void* g, int32_t g_type, int64_t ldg, int32_t fmt_g, const void* x, int32_t x_type, int64_t ldx, int64_t M, int32_t N, int32_t K,
                                   float* dw, void* ws, int64_t ws_bytes, void* stream) {
  ALN_REQUIRE(is_ft(g_type) && is_ft(x_type) && is_f8(fmt_g), "fp8_grad_weight: unknown type %d, %d or format %d", g_type, x_type, fmt_g);
  ALN_REQUIRE(M >= 1 && M <= MOST32 && N >= 1 && K >= 1 && ldg >= N && ldx >= K && ldg < 1 << 24 && ldx < 1 << 24,
              "fp8_grad_weight: sizes %lld x %d x %d, pitches %lld, %lld (at least the columns, under 2^24)", (long long)M, N, K, (long long)ldg, (long long)ldx);
  ALN_REQUIRE(g && ((uintptr_t)g & (g_type == FT_F32 ? 3 : 1)) == 0 && x && ((uintptr_t)x & (x_type == FT_F32 ? 3 : 1)) == 0 && dw && ((uintptr_t)dw & 3) == 0,
              "fp8_grad_weight: g, x or dw is NULL or not aligned to its type");
  const int64_t need = aln_fp8_grad_weight_ws_bytes(M, N, K, g_type, x_type);
  ALN_REQUIRE(ws_bytes >= need && (need == 0 || (ws && ((uintptr_t)ws & 15) == 0)), "fp8_grad_weight: the workspace needs %lld bytes, aligned to 16", (long long)need);
  hipStream_t st = (hipStream_t)stream;
  if (!tn_fused(M, N, K, g_type, x_type)) {
    const int64_t nb = ceil128(M) / 128, ld = nb * 128, lds = (nb + 3) / 4 * 4;
    uint8_t *qg = (uint8_t*)ws, *qx = qg + N * ld, *sg = qx + K * ld, *sx = sg + up16(N * lds), *rest = sx + up16(K * lds);
    int rc = aln_fp8_quantize_t(g, g_type, ldg, M, N, fmt_g, qg, ld, sg, lds, stream);
    if (rc == 0) rc = aln_fp8_quantize_t(x, x_type, ldx, M, K, F8_E4M3, qx, ld, sx, lds, stream);
    if (rc) return rc;
    return aln_fp8_nt(qg, ld, sg, lds, fmt_g, qx, ld, sx, lds, F8_E4M3, N, K, M, dw, K, FT_F32, 0, rest, ws_bytes - (rest - qg), stream);
  }
  const TnPlan t = tn_plan(M, N, K);
  const Fp8TN p{g, ldg, x, ldx, M, N, K, t.tn, t.tk, t.parts, t.per, t.parts > 1 ? (float*)ws : dw};
  const int rc = g_type == FT_F16 ? tn_pick<FT_F16>(p, t, fmt_g, st) : tn_pick<FT_BF16>(p, t, fmt_g, st);
  if (rc || t.parts == 1) return rc;
  hipLaunchKernelGGL(k_fp8_join, dim3(aln_grid_for(((int64_t)N * K + 3) / 4, 32, 4096)), dim3(256), 0, st, (const float*)ws, t.parts, (int64_t)N, K, Fp8Out{dw, K, FT_F32, 0});
  ALN_CHECK_LAUNCH("fp8_grad_weight");
  return 0;
}
