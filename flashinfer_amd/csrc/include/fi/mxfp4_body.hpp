// Products with MXFP4 weights for gfx950, plain and gated:
//   out = a @ dequant(b)^T
//   out = act(a @ dequant(b_gate)^T) * (a @ dequant(b_up)^T)
// a: bf16 or fp16 rows, or MXFP8 (e4m3 with a scale byte for 32 neighbours);
// b: [rows, K/2] packed e2m1, b_scale [rows, K/32]; the gated form holds the
// N gate rows first, then the N up rows.
//
// Operand map, in 16x16 tiles (weights are the rows, tokens the columns):
// lane l holds weight row l & 15 and, with g = l >> 4, the 32 values of block
// g of a chunk of 128 - one load of 16 bytes and one scale byte.
//   MXFP8 a: one v_mfma_scale_f32_16x16x128_f8f6f4 takes both operands as they
//     lie in memory. Its fp8 operand holds k = 16g..16g+15 in the first four
//     registers and 64+16g.. in the last four, its fp4 operand k = 32g..32g+31,
//     and lane group g supplies the scale of block g for either.
//   16-bit a: the block becomes bf16 (two values an instruction, the scale
//     applied by it, exact below 2^128: 4 and 6 times 2^126, and 2 to 6 times
//     2^127, become infinite) and feeds four 16x16x32 products; product i takes
//     k = 32g + 8i .. 32g + 8i + 7 from lane group g.
//   fp16 a: the same in fp16 where every scale of the wave's chunk keeps the
//     weights exact in fp16 (2^-23 .. 2^13); elsewhere a is split into two
//     bf16 parts, high and low, which hold its 11 bits exactly (a tile of many
//     tokens is then taken once more from the start). The scale alone is looked
//     at: a block of zeros with the scale byte 0 counts as not exact. One such
//     block in 128 weight rows takes 2048 x 14336 x 4096 from 234 to 1080 us and
//     256 x 6144 x 4096 from 23 to 103, few tokens (64 x 6144 x 4096) from 11 to 24.
// Sums are held in 32 bits, but the block-scaled instruction aligns its 64 or 128
// 8-bit products to the largest of them and keeps 18 bits below it: at most 2^-11
// of the magnitudes that a sum is made of, 2e-5 of the results' size on normal data.
// An output in 16 bits rounds to 4e-3 or 5e-4 and hides that (14336 products: an
// error against 64 bits of 0.001653 with either sum, 1 % of the roundings differ). An MXFP8 output has
// scales, and one block in 50,000 would get the neighbour of its own: there, for
// any number of tokens, both operands become bf16 (exactly, from 2^-133 to below
// 2^128) and the error is that of 32 bits. Where the matrix unit bounds the time it costs the rate of 8-bit
// products (gated 4096 x 4096 x 7680: 377 us for 233).
#pragma once
#include <type_traits>

#include "fi/common.hpp"
#include "fi/mfma.hpp"
#include "fi/mx.hpp"

namespace fi {
namespace mx4 {

struct Params {
  const void* a;
  const uint8_t* a_scale;
  const uint8_t* b;
  const uint8_t* b_scale;
  void* out;
  uint8_t* out_scale;
  int M, N, K;
  int64_t lda, ldo;
  int act, out_fp16;
  float* sums;  // of the parts of K, where a product is split over it
};

enum { kBf16 = 0, kFp16 = 1, kFp8 = 2 };  // types of a
// Outputs are OUT8 (MXFP8, with their scales) or 16 bits wide; bf16 or fp16 is
// a choice at run time, so that the kernels are compiled once for both.
__device__ __forceinline__ uint16_t to16(float x, bool fp16_out) {
  return fp16_out ? __builtin_bit_cast(uint16_t, (_Float16)x)
                  : __builtin_bit_cast(uint16_t, (__bf16)x);
}

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;

// g / (1 + 2^t): the exponential and the reciprocal of the hardware are off by
// an ulp, and by |t| 2^-24 through t - far below a rounding to 16 bits. Where
// 2^t overflows the reciprocal is 0.
__device__ __forceinline__ float times_logistic(float g, float t) {
  return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(t));
}

// erfc(x) within 1.2e-7 of its value, the rounding of the exponent apart: the
// Chebyshev fit of W. H. Press et al., Numerical Recipes (2nd ed., 6.2), where
// erfc(z) = t exp(-z^2 + P(t)), t = 1 / (1 + z / 2), z = |x|. It keeps the small
// negative tail of the activation, which 1 + erf rounds away.
__device__ __forceinline__ float erfc_close(float x) {
  const float z = __builtin_fabsf(x);
  const float t = __builtin_amdgcn_rcpf(1.f + 0.5f * z);
  float q = 0.17087277f;
  q = q * t - 0.82215223f;
  q = q * t + 1.48851587f;
  q = q * t - 1.13520398f;
  q = q * t + 0.27886807f;
  q = q * t - 0.18628806f;
  q = q * t + 0.09678418f;
  q = q * t + 0.37409196f;
  q = q * t + 1.00002368f;
  q = q * t - 1.26551223f;
  const float r = t * __builtin_amdgcn_exp2f((q - z * z) * 1.4426950408889634f);
  return x < 0.f ? 2.f - r : r;
}

template <int kAct>
__device__ __forceinline__ float activate(float g) {
  if constexpr (kAct == 0) {
    return times_logistic(g, g * -1.4426950408889634f);
  } else if constexpr (kAct == 1) {
    return 0.5f * g * erfc_close(g * -0.70710678118654752f);
  } else {
    // 0.5 (1 + tanh(u)) = 1 / (1 + exp(-2u)), u = sqrt(2 / pi) (g + 0.044715 g^3)
    return times_logistic(g, g * (-2.3022081985f - 0.1029432397f * g * g));
  }
}

__device__ __forceinline__ float activate(int act, float g) {
  return act == 0 ? activate<0>(g) : act == 1 ? activate<1>(g) : activate<2>(g);
}

__device__ __forceinline__ float scale_value(uint32_t byte) {
  // the conversions read the exponent bits alone: 0 is 2^-127, 255 is NaN
  return __uint_as_float(byte << 23);
}

// Eight weights of one dword as bf16 or fp16, scaled.
__device__ __forceinline__ bf16x8_t widen_bf16(uint32_t q, float s) {
  union { bf16x8_t v; bf16x2_t p[4]; } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 0);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 1);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 2);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 3);
  return u.v;
}
__device__ __forceinline__ f16x8_t widen_f16(uint32_t q, float s) {
  union { f16x8_t v; f16x2_t p[4]; } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, s, 0);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, s, 1);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, s, 2);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, s, 3);
  return u.v;
}

// Eight e4m3 values of two dwords as bf16, scaled.
__device__ __forceinline__ bf16x8_t widen_fp8(uint32_t lo, uint32_t hi, float s) {
  union { bf16x8_t v; bf16x2_t p[4]; } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
  return u.v;
}

// fp16 as the sum of two bf16: 8 bits, then the remaining 3.
__device__ __forceinline__ void split_f16(uint4 x, bf16x8_t& hi, bf16x8_t& lo) {
  union { uint4 q; _Float16 h[8]; } u;
  u.q = x;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float f = (float)u.h[j];
    const __bf16 h = (__bf16)f;
    hi[j] = h;
    // an infinity has no remainder: inf - inf would make it a NaN
    const float rest = f - (float)h;
    lo[j] = (__bf16)(abs_bits(f) < 0x7f800000u ? rest : 0.f);
  }
}

__device__ __forceinline__ bool f16_exact(uint32_t byte) {
  return byte >= 104u && byte <= 140u;
}

// ---------------------------------------------------------------------------
// Loads to shared memory, and the waits for them.

// 16 bytes a lane to the wave's 1024 at `dst` (a wave's own, uniform address).
// In assembly, for the compiler holds every read of shared memory behind such
// a load, also where the two go to different buffers: with the builtin the
// next step's loads were waited for before this step's products. Nothing waits
// for it here: the callers count these loads. m0 is the compiler's own register,
// of which it warns; that it is written has to be said all the same.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds16(const uint8_t* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(dst), "v"(src)
               : "memory", "m0");
}
__device__ __forceinline__ void load_lds16(const uint8_t* base, uint32_t at, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(dst), "v"(at), "s"(base)
               : "memory", "m0");
}
#pragma clang diagnostic pop

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// s_waitcnt for at most `vm` loads, and for shared memory too where `lds`
constexpr int wait_code(int vm, bool lds) {
  return (vm & 15) | (vm >> 4) << 14 | 7 << 4 | (lds ? 0 : 15) << 8;
}

// until all but the newest `stages` of a wave's stages, kOps loads each, are in
template <int kOps, int kMost>
__device__ __forceinline__ void wait_stages(int stages) {
  static_assert(kOps * kMost < 64, "");
  if constexpr (kMost > 0) {
    if (stages >= kMost) __builtin_amdgcn_s_waitcnt(wait_code(kOps * kMost, false));
    else wait_stages<kOps, kMost - 1>(stages);
  } else {
    __builtin_amdgcn_s_waitcnt(wait_code(0, false));
  }
}

// 16-byte units spread over the banks: of rows of 32 to 256 bytes, a column of
// 16 or 32 rows is then read without conflicts
__device__ __forceinline__ uint32_t spread(uint32_t off) {
  return off ^ (((off >> 8) & 15) << 4);
}

// Scales at .. at + 15 of a row's `count`: 16 unaligned bytes, or what is left
// of them and 127 (the scale 1) behind the end.
__device__ __forceinline__ void load_scales(uint32_t (&v)[4], const uint8_t* row, int at,
                                            int count) {
  if (at + 16 <= count) {
    __builtin_memcpy(v, row + at, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = at + j * 4 + k;
        const uint32_t byte = row[i < count ? i : count - 1];
        v[j] |= (i < count ? byte : 127u) << (8 * k);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Few tokens (64 at most): the weights' bytes are what the time goes to, and
// how many of them are on their way at once decides how fast they come. (From
// 17 tokens on it is the tokens' way from L2 to every CU.) A
// workgroup of WAVES waves takes RT * 16 outputs and shares K among its waves
// in chunks of 128. Each wave has D chunks of weights (AT KB) and tokens (XI
// KB) on their way to its own part of shared memory, by loads that bypass the
// registers, and waits for the oldest alone: there is no barrier in the loop.
// The scales of a slab of K are read ahead of it. The waves' sums are joined
// in a fixed order.
template <int ACT, bool GATED, int RT, int XI, int WAVES, int D>
struct Rows {
  static constexpr int AT = GATED ? 2 * RT : RT;             // tiles of 16 weight rows
  static constexpr int kXRow = ACT == kFp8 ? 128 : 256;      // bytes of a token in a chunk
  static constexpr int MR = XI * 1024 / kXRow;               // tokens held, 64 at most
  static constexpr int MT = (MR + 15) / 16;                  // tiles of 16 tokens
  static constexpr int kStage = (AT + XI) * 1024;
  static constexpr int kSlab = 192;                          // blocks of K with resident scales
  static constexpr int kSRow = kSlab + 16;                   // one unit more: rows in unlike banks
  static constexpr int kSRows = AT * 16 + (ACT == kFp8 ? MR : 0);
  static constexpr int LD = AT * 16 + 4;                     // of the sums to be joined
  static constexpr int kRing = WAVES * D * kStage;
  static constexpr int kJoin = WAVES * MT * 16 * LD * 4;
  static constexpr int kLds = kRing + kSRows * kSRow > kJoin ? kRing + kSRows * kSRow : kJoin;
  static constexpr int kFit = kLdsBytes / kLds;              // workgroups that a CU has room for
  static constexpr int kWavesPerSimd = WAVES / 4 * kFit < 4 ? WAVES / 4 * kFit : 4;
  static_assert(MR <= 64 && kLds <= kLdsBytes, "");
};

template <int ACT, bool GATED, bool OUT8, int RT, int XI, int WAVES, int D>
__global__ __launch_bounds__(WAVES * 64, (Rows<ACT, GATED, RT, XI, WAVES, D>::kWavesPerSimd))
void rows_kernel(Params p) {
  using C = Rows<ACT, GATED, RT, XI, WAVES, D>;
  constexpr int AT = C::AT, MT = C::MT;
  constexpr bool kWiden = ACT == kFp8 && OUT8;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[C::kLds];
  uint8_t* const lds_s = lds + C::kRing;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * RT * 16;
  const int blocks = p.K / kMxBlock;

  auto weight_at = [&](int r) {  // the weight row of row r of the AT tiles
    const int n = n0 + r % (RT * 16);
    return (n < p.N ? n : p.N - 1) + (r >= RT * 16 ? (int64_t)p.N : 0);
  };
  // lane l brings unit l of a kilobyte: the place is linear, the source permuted
  const uint32_t b_unit = spread(lane * 16);
  const uint8_t* b_src[AT];
#pragma unroll
  for (int t = 0; t < AT; ++t)
    b_src[t] = p.b + weight_at(t * 16 + (int)(b_unit / 64)) * (p.K / 2);
  const uint8_t* x_src[XI];
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int r = (int)(spread(i * 1024 + lane * 16) / C::kXRow);
    x_src[i] = (const uint8_t*)p.a +
               (int64_t)(r < p.M ? r : p.M - 1) * p.lda * (ACT == kFp8 ? 1 : 2);
  }
  const uint32_t ring = lds_address(lds) + wave * D * C::kStage;
  const uint8_t* const ring_p = lds + wave * D * C::kStage;

  // chunk c of K to place `slot` of the wave's ring. Behind the end of a row
  // its last unit comes again: those values are cleared where they are used.
  auto stage = [&](int c, int slot) {
    const uint32_t to = ring + slot * C::kStage;
    const int b_last = p.K / 2 - 16, x_last = p.K * (ACT == kFp8 ? 1 : 2) - 16;
    const int b_off = c * 64 + (int)(b_unit % 64);
#pragma unroll
    for (int t = 0; t < AT; ++t)
      load_lds16(b_src[t] + (b_off < b_last ? b_off : b_last), to + t * 1024);
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const int x_off = c * C::kXRow + (int)(spread(i * 1024 + lane * 16) % C::kXRow);
      load_lds16(x_src[i] + (x_off < x_last ? x_off : x_last), to + (AT + i) * 1024);
    }
  };

  // where a lane reads: its weights' block, and its token's values. A column
  // of no token reads some other token; its sums are not used.
  const uint32_t read_b = spread(lr * 64 + g * 16);
  auto token = [&](int j) { return (j * 16 + lr) & (C::MR - 1); };

  floatx4 acc[AT][MT];
#pragma unroll
  for (int t = 0; t < AT; ++t)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[t][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  for (int s0 = 0; s0 < blocks; s0 += C::kSlab) {
    const int width = blocks - s0 < C::kSlab ? blocks - s0 : C::kSlab;
    const int c0 = s0 / 4, chunks = (width + 3) / 4;
    // this wave's chunks of the slab: c0 + wave, and every WAVES further
    const int mine = chunks > wave ? (chunks - wave - 1) / WAVES + 1 : 0;
    // The slab's scales, 16 to a load: they are asked for before they are
    // written, all at once. Behind the slab's end lies 127, which is 1.
    constexpr int kUnits = C::kSRows * (C::kSlab / 16);
    constexpr int kEach = (kUnits + WAVES * 64 - 1) / (WAVES * 64);
    uint32_t sv[kEach][4];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = tid + j * WAVES * 64;
      const int r = i / (C::kSlab / 16), at = i % (C::kSlab / 16) * 16;
      if (i >= kUnits || at >= width) continue;
      const uint8_t* src =
          r < AT * 16 ? p.b_scale + weight_at(r) * blocks + s0
                      : p.a_scale + (int64_t)(r - AT * 16 < p.M ? r - AT * 16 : p.M - 1) * blocks + s0;
      load_scales(sv[j], src, at, width);
    }
#pragma unroll
    for (int i = 0; i < D; ++i)
      if (i < mine) stage(c0 + wave + i * WAVES, i);
    if (s0) __syncthreads();  // the slab before this one is done with its scales
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = tid + j * WAVES * 64;
      const int r = i / (C::kSlab / 16), at = i % (C::kSlab / 16) * 16;
      if (i >= kUnits || at >= width) continue;
      *(uint4*)(lds_s + r * C::kSRow + at) = make_uint4(sv[j][0], sv[j][1], sv[j][2], sv[j][3]);
    }
    __syncthreads();

    int slot = 0;
    for (int i = 0; i < mine; ++i) {
      const int c = wave + i * WAVES;  // in the slab
      wait_stages<AT + XI, D - 1>(mine - 1 - i);
      asm volatile("" ::: "memory");  // no read moves before the wait
      const uint8_t* from = ring_p + slot * C::kStage;
      uint4 w[AT];
      uint32_t ws[AT];
#pragma unroll
      for (int t = 0; t < AT; ++t) {
        w[t] = *(const uint4*)(from + t * 1024 + read_b);
        ws[t] = lds_s[(t * 16 + lr) * C::kSRow + c * 4 + g];
      }
      constexpr int XU = ACT == kFp8 ? 2 : 4;  // 16-byte units of a token a lane takes
      uint4 x[MT][XU];
      uint32_t xs[MT];
#pragma unroll
      for (int j = 0; j < MT; ++j) {
#pragma unroll
        for (int k = 0; k < XU; ++k) {
          const int byte = kWiden ? g * 32 + k * 16 : ACT == kFp8 ? g * 16 + k * 64 : g * 64 + k * 16;
          x[j][k] = *(const uint4*)(from + AT * 1024 + spread(token(j) * C::kXRow + byte));
        }
        if constexpr (ACT == kFp8) xs[j] = lds_s[(AT * 16 + token(j)) * C::kSRow + c * 4 + g];
      }
      // all read: the place may be filled again
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (i + D < mine) stage(c0 + c + D * WAVES, slot);
      slot = slot == D - 1 ? 0 : slot + 1;

      if (c * 4 + 4 > width) {  // the last chunk of a K that 128 does not divide
        const int left = width - c * 4;
#pragma unroll
        for (int t = 0; t < AT; ++t)
          if (g >= left) w[t] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < XU; ++k)
          if ((ACT == kFp8 && !kWiden ? k * 2 + g / 2 : g) >= left) {
#pragma unroll
            for (int j = 0; j < MT; ++j) x[j][k] = make_uint4(0, 0, 0, 0);
          }
      }
      auto weights = [&](int t, int k) {
        return k == 0 ? w[t].x : k == 1 ? w[t].y : k == 2 ? w[t].z : w[t].w;
      };
      if constexpr (kWiden) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          bf16x8_t xv[MT];
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            const uint4 h = x[j][k / 2];
            xv[j] = widen_fp8(k % 2 ? h.z : h.x, k % 2 ? h.w : h.y, scale_value(xs[j]));
          }
#pragma unroll
          for (int t = 0; t < AT; ++t) {
            const bf16x8_t wv = widen_bf16(weights(t, k), scale_value(ws[t]));
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[t][j] = mfma_16x16x32_bf16(wv, xv[j], acc[t][j]);
          }
        }
      } else if constexpr (ACT == kFp8) {
#pragma unroll
        for (int t = 0; t < AT; ++t) {
          const intx8 wv = {(int)w[t].x, (int)w[t].y, (int)w[t].z, (int)w[t].w, 0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            const uint4 u = x[j][0], v = x[j][1];
            const intx8 xv = {(int)u.x, (int)u.y, (int)u.z, (int)u.w,
                              (int)v.x, (int)v.y, (int)v.z, (int)v.w};
            acc[t][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                wv, xv, acc[t][j], 4, 0, 0, (int)ws[t], 0, (int)xs[j]);
          }
        }
      } else {
        bool exact = true;
#pragma unroll
        for (int t = 0; t < AT; ++t) exact = exact && f16_exact(ws[t]);
        if (ACT == kFp16 && __all(exact)) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int t = 0; t < AT; ++t) {
              const f16x8_t wv = widen_f16(weights(t, k), scale_value(ws[t]));
#pragma unroll
              for (int j = 0; j < MT; ++j)
                acc[t][j] =
                    mfma_16x16x32_f16(wv, __builtin_bit_cast(f16x8_t, x[j][k]), acc[t][j]);
            }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              bf16x8_t hi = __builtin_bit_cast(bf16x8_t, x[j][k]), lo;
              if constexpr (ACT == kFp16) {
                __builtin_amdgcn_sched_barrier(0);  // one split's registers at a time
                split_f16(x[j][k], hi, lo);
              }
#pragma unroll
              for (int t = 0; t < AT; ++t) {
                const bf16x8_t wv = widen_bf16(weights(t, k), scale_value(ws[t]));
                acc[t][j] = mfma_16x16x32_bf16(wv, hi, acc[t][j]);
                if constexpr (ACT == kFp16) acc[t][j] = mfma_16x16x32_bf16(wv, lo, acc[t][j]);
              }
            }
          }
        }
      }
    }
  }

  // Join the waves' sums. Every lane writes its own, also where its column is
  // no token: an operand of a product may not sink into a branch.
  __syncthreads();
  float* const join = (float*)lds;
#pragma unroll
  for (int t = 0; t < AT; ++t)
#pragma unroll
    for (int j = 0; j < MT; ++j)
      *(floatx4*)(join + ((wave * MT + j) * 16 + lr) * C::LD + t * 16 + g * 4) = acc[t][j];
  __syncthreads();

  auto joined = [&](int m, int nl) {
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      s += join[(w * MT * 16 + m) * C::LD + nl];
      if constexpr (GATED) u += join[(w * MT * 16 + m) * C::LD + RT * 16 + nl];
    }
    return GATED ? activate(p.act, s) * u : s;
  };
  if constexpr (OUT8) {
    // an output to a lane: 32 of them hold one block. N is a multiple of 32 here.
    static_assert(RT == 2, "");
    for (int i = tid; i < MT * 512; i += WAVES * 64) {
      const int m = i / 32, nl = i % 32, n = n0 + nl;
      if (m >= p.M) continue;
      const float y = joined(m, nl);
      const uint32_t byte = mxfp8_scale_byte(max32(abs_bits(y)));
      const float q = y * mx_inverse_scale(byte);
      const uint32_t e4m3 = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q, q, 0, false);
      ((uint8_t*)p.out)[(int64_t)m * p.ldo + n] = byte == 255u ? 0x7f : (uint8_t)e4m3;
      if (nl == 0) p.out_scale[(int64_t)m * (p.N / kMxBlock) + n / kMxBlock] = (uint8_t)byte;
    }
  } else {
    for (int i = tid; i < MT * 16 * RT * 16; i += WAVES * 64) {
      const int m = i / (RT * 16), nl = i % (RT * 16), n = n0 + nl;
      if (m < p.M && n < p.N)
        ((uint16_t*)p.out)[(int64_t)m * p.ldo + n] = to16(joined(m, nl), p.out_fp16);
    }
  }
}

template <int ACT, bool GATED, bool OUT8, int RT, int XI, int WAVES, int D>
hipError_t launch_rows(const Params& p, hipStream_t stream) {
  hipLaunchKernelGGL((rows_kernel<ACT, GATED, OUT8, RT, XI, WAVES, D>),
                     dim3(ceil_div(p.N, RT * 16)), dim3(WAVES * 64), 0, stream, p);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Many tokens: a workgroup of GN x GM waves computes a tile of GN * WN * 32
// weight rows by GM * WM * 32 tokens in 32x32 products. Steps of 128 bytes of
// a token row (128 values in 8 bits, 64 in 16) go to shared memory with their
// weights, several buffers in turn, by loads that bypass the registers; the
// scales of 512 values of a row come as 16 bytes once per 512.
//
// 256 x 128, two on a CU: 4096 x 4096 x 14336 with 8-bit tokens takes 200 to 209 us
// from card to card, 2.3 to 2.4 PFLOP/s (a library product of 8-bit matrices of that
// size reaches 3.2); a gated block of 2047 x 14336 x 4096 with bf16 tokens 391 to
// 405 us, 1.2 (1.42). Staging a
// quarter of the tokens only would save a fifth of that, of the weights a
// twelfth: what is left is the way of the operands from the L2 cache. Three
// buffers and counted waits brought 311 -> 229 us, outputs through shared
// memory 239 -> 197. Eight waves at 256 x 256 and waves of higher priority
// during their products brought nothing.
// Small tiles are bound by their tokens' way from L2 as well (47 to 59 bytes a
// nanosecond for a CU), or, with less than 256 of them, by the latency of a step.
//
// Operand map of 32x32: lane l holds row (token) l & 31 and, with g = l >> 5,
//   8-bit a, 32x32x64: fp4 k = 32g..32g+31; fp8 k = 16g..16g+15 and 32+16g..;
//     lane group g supplies the scale of block g.
//   16-bit a, 32x32x16, product i of 4 in a step: k = 32g + 8i .. 32g + 8i + 7,
//     so that a lane's weights are one block of one scale here as well.

template <int ACT, bool GATED, int WN, int WM, int GN, int GM, int GK>
struct Tile {
  static constexpr int kGroup = GN * GM * 64;            // threads of one part of K
  static constexpr int kThreads = kGroup * GK;
  // Small tiles wait for memory rather than for the matrix unit: a wave more
  // brings the scales, so that no other wave's wait for its scales is a wait
  // for all the steps that it has asked for since.
  static constexpr bool kHelper = WN * WM <= 2 || GK > 1;
  static constexpr int kLaunch = kThreads + (kHelper ? 64 : 0);
  static constexpr int kScaleThreads = kHelper ? 64 : kThreads;
  static constexpr int TN = GN * WN * 32, TM = GM * WM * 32;
  static constexpr int kOut = GATED ? TN / 2 : TN;       // outputs of a tile along N
  static constexpr int KS = ACT == kFp8 ? 128 : 64;      // values of a step
  static constexpr int WB = KS / 2;                      // bytes of a weight row in a step
  static constexpr int kSteps = 512 / KS;                // steps of one load of scales
  static constexpr int kABytes = TM * 128, kBBytes = TN * WB;
  static constexpr int kSRows = TN + (ACT == kFp8 ? TM : 0);
  static constexpr int kStage = kABytes + kBBytes, kScales = 2 * 16 * kSRows;
  // a workgroup of four waves shares a CU with another
  static constexpr int kMost = kThreads <= 256 ? kLdsBytes / 2 : kLdsBytes;
  static constexpr int kFit = (kMost - kScales - (ACT == kFp16 ? 16 : 0)) / (kStage * GK);
  static constexpr int kBufs = kFit < 6 ? kFit : 6;
  static constexpr int kAhead = kBufs - 1;               // steps on their way
  static constexpr int kRing = GK * kBufs * kStage;
  static constexpr int kJoin = (GK - 1) * GN * GM * WN * WM * 4096;
  static constexpr int kLds = kRing + kScales > kJoin ? kRing + kScales : kJoin;
  static_assert(kBufs >= 2 && kSteps % GK == 0, "");
  static constexpr int AU = kABytes / 16 / kGroup, BU = kBBytes / 16 / kGroup;
  static constexpr int kWavesPerSimd = !kHelper ? 2 : ceil_div(kLaunch / 64 * (kLds <= kLdsBytes / 2 ? 2 : 1), 4);
  static constexpr int kInFlight = AU + BU;              // loads a wave issues for a step
  static constexpr int SU = (kSRows + kScaleThreads - 1) / kScaleThreads;
  static_assert(AU * 16 * kGroup == kABytes && BU * 16 * kGroup == kBBytes, "");
};

// Row r of a tile of weights: a wave holds WN tiles of 32, where gated half of
// them gate rows and half the up rows of the same outputs.
template <bool GATED, int WN>
__device__ __forceinline__ bool is_up(int r) {
  return GATED && r / 32 % WN >= WN / 2;
}
// its output, counted from n0 and held inside N
template <bool GATED, int WN>
__device__ __forceinline__ int weight_row(int n0, int r, int N) {
  if constexpr (GATED) r = (r / (WN * 32) * (WN / 2) + r / 32 % (WN / 2)) * 32 + r % 32;
  return n0 + r < N ? r : N - 1 - n0;
}

template <int ACT, bool GATED, bool OUT8, int WN, int WM, int GN, int GM, int GK>
__global__ __launch_bounds__((Tile<ACT, GATED, WN, WM, GN, GM, GK>::kLaunch),
                             (Tile<ACT, GATED, WN, WM, GN, GM, GK>::kWavesPerSimd))
void tile_kernel(Params p, int tiles_n, int tiles_m) {
  using C = Tile<ACT, GATED, WN, WM, GN, GM, GK>;
  constexpr bool kWiden = ACT == kFp8 && OUT8;
  constexpr int kSize = OUT8 ? 1 : 2;
  constexpr int kRow = C::kOut * kSize + 16;  // of the outputs; the odd piece spreads the banks
  constexpr int kShared = C::TM * kRow > C::kLds ? C::TM * kRow : C::kLds;
  __shared__ __attribute__((aligned(256))) uint8_t lds[kShared];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave_all = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave = wave_all % (GN * GM), part = wave_all / (GN * GM);  // of K: step part of GK
  const int gid = tid % C::kGroup;                                     // in the part
  const int wn = wave % GN, wm = wave / GN;
  const int lr = lane & 31, g = lane >> 5;
  uint8_t* const lds_a = lds + part * C::kBufs * C::kStage;  // a part's own buffers
  uint8_t* const lds_b = lds_a + C::kBufs * C::kABytes;
  uint32_t* const lds_s = (uint32_t*)(lds + C::kRing);       // [2][4][kSRows], everybody's

  // neighbouring tiles run on one XCD, in bands of eight tiles of tokens
  const int id = (int)xcd_swizzle(blockIdx.x, gridDim.x);
  const int band = id / (8 * tiles_n), first = band * 8;
  const int high = tiles_m - first < 8 ? tiles_m - first : 8;
  const int in_band = id - band * 8 * tiles_n;
  const int m0 = (first + in_band % high) * C::TM, n0 = in_band / high * C::kOut;

  const int blocks = p.K / kMxBlock;
  const int steps = (p.K + C::KS - 1) / C::KS;
  const int64_t a_row_bytes = p.lda * (ACT == kFp8 ? 1 : 2);

  // where this thread's 16-byte units come from: dst is linear, src permuted.
  // A wave's unit lies in one 32-row tile of weights, so gate or up is uniform.
  // The offsets fit 32 bits: the host holds 256 rows of either to 4 GB.
  const uint8_t* const a_tile = (const uint8_t*)p.a + (int64_t)m0 * a_row_bytes;
  const uint8_t* const b_tile = p.b + (int64_t)n0 * (p.K / 2);
  uint32_t a_at[C::AU], b_at[C::BU];
  const uint8_t* b_from[C::BU];
#pragma unroll
  for (int i = 0; i < C::AU; ++i) {
    const uint32_t dst = (uint32_t)(gid + i * C::kGroup) * 16;
    const uint32_t off = spread(dst);
    const int r = (int)(off / 128);
    a_at[i] = (uint32_t)(m0 + r < p.M ? r : p.M - 1 - m0) * (uint32_t)a_row_bytes + off % 128;
  }
#pragma unroll
  for (int i = 0; i < C::BU; ++i) {
    const uint32_t dst = (uint32_t)(gid + i * C::kGroup) * 16;
    const uint32_t off = spread(dst);
    const int r = weight_row<GATED, WN>(n0, (int)(off / C::WB), p.N);
    b_at[i] = (uint32_t)r * (uint32_t)(p.K / 2) + off % C::WB;
    const int first = (wave * 64 + i * C::kGroup) * 16 / C::WB;
    b_from[i] = b_tile + (is_up<GATED, WN>(first) ? (int64_t)p.N * (p.K / 2) : 0);
  }
  const uint32_t a_base = lds_address(lds_a);
  const uint32_t b_base = lds_address(lds_b);

  auto stage = [&](int t, int buf) {
    if ((t + 1) * C::KS <= p.K) {
#pragma unroll
      for (int i = 0; i < C::AU; ++i)
        load_lds16(a_tile + (int64_t)t * 128, a_at[i],
                   a_base + buf * C::kABytes + (wave * 64 + i * C::kGroup) * 16);
#pragma unroll
      for (int i = 0; i < C::BU; ++i)
        load_lds16(b_from[i] + (int64_t)t * C::WB, b_at[i],
                   b_base + buf * C::kBBytes + (wave * 64 + i * C::kGroup) * 16);
    } else {
      // the last step of a K that is no multiple of it: zeros behind the end
      const int left = p.K - t * C::KS;  // values
#pragma unroll
      for (int i = 0; i < C::AU; ++i) {
        const uint32_t dst = (uint32_t)(gid + i * C::kGroup) * 16;
        const uint32_t off = spread(dst);
        const bool in = (int)(off % 128) < left * (ACT == kFp8 ? 1 : 2);
        *(uint4*)(lds_a + buf * C::kABytes + dst) =
            in ? *(const uint4*)(a_tile + a_at[i] + (int64_t)t * 128) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < C::BU; ++i) {
        const uint32_t dst = (uint32_t)(gid + i * C::kGroup) * 16;
        const uint32_t off = spread(dst);
        const bool in = (int)(off % C::WB) < left / 2;
        *(uint4*)(lds_b + buf * C::kBBytes + dst) =
            in ? *(const uint4*)(b_from[i] + b_at[i] + (int64_t)t * C::WB) : make_uint4(0, 0, 0, 0);
      }
    }
  };

  // scales of blocks 16u .. 16u + 15 of every row of the tile
  auto scales = [&](int u, uint32_t (&v)[C::SU][4]) {
#pragma unroll
    for (int i = 0; i < C::SU; ++i) {
      const int r = tid % C::kScaleThreads + i * C::kScaleThreads;
      if (r >= C::kSRows) break;
      const uint8_t* src;
      if (r < C::TN) {
        src = p.b_scale + (n0 + weight_row<GATED, WN>(n0, r, p.N) +
                           (is_up<GATED, WN>(r) ? (int64_t)p.N : 0)) * blocks;
      } else {
        const int m = m0 + r - C::TN;
        src = p.a_scale + (int64_t)(m < p.M ? m : p.M - 1) * blocks;
      }
      load_scales(v[i], src, u * 16, blocks);
    }
  };
  auto put_scales = [&](int buf, const uint32_t (&v)[C::SU][4]) {
#pragma unroll
    for (int i = 0; i < C::SU; ++i) {
      const int r = tid % C::kScaleThreads + i * C::kScaleThreads;
      if (r >= C::kSRows) break;
#pragma unroll
      for (int j = 0; j < 4; ++j) lds_s[(buf * 4 + j) * C::kSRows + r] = v[i][j];
    }
  };

  floatx16 acc[WN][WM];

  // this workgroup's part of K, in loads of scales and in steps
  const int u_all = ceil_div(blocks, 16), u_part = ceil_div(u_all, (int)gridDim.y);
  const int u0 = blockIdx.y * u_part, u1 = u0 + u_part < u_all ? u0 + u_part : u_all;
  const int t0 = u0 * C::kSteps, t1 = u1 * C::kSteps < steps ? u1 * C::kSteps : steps;

  const int rounds = t0 < t1 ? (t1 - t0 + GK - 1) / GK : 0;

  uint32_t sv[C::SU][4];
  // What the helping wave does during a pass. Barriers as the others have
  // them: one ahead of the rounds and one a round. During load u of the scales
  // it writes load u + 1 and asks for load u + 4: every eighth load of a row
  // meets a new line of memory, which takes longer than the rounds of one load.
  auto bring_scales = [&]() {
    constexpr int kRounds = C::kSteps / GK, kSets = 4;
    uint32_t set[kSets][C::SU][4];
#pragma unroll
    for (int i = 0; i < kSets; ++i)
      if (u0 + i < u1) scales(u0 + i, set[i]);
    if (u0 < u1) put_scales(u0 & 1, set[0]);
    __syncthreads();
    for (int first = u0; first < u1; first += kSets) {
#pragma unroll
      for (int i = 0; i < kSets; ++i) {
        const int u = first + i;
        if (u >= u1) break;
        if (u + kSets < u1) scales(u + kSets, set[i]);
        const int to = u + 1 < u1 ? kRounds : rounds - (u - u0) * kRounds;
        for (int r = 1; r < to; ++r) __syncthreads();
        if (u + 1 < u1) put_scales((u + 1) & 1, set[(i + 1) % kSets]);
        __syncthreads();
      }
    }
  };

  // Where a lane reads. Rows 32 apart have one permutation (tokens), so a byte
  // of the row is flipped into the address and the tile of 32 is an offset.
  const int b_row = wn * WN * 32 + lr, a_row = wm * WM * 32 + lr;
  const uint32_t read_a = spread(a_row * 128);
  uint32_t read_b[WN];
#pragma unroll
  for (int i = 0; i < WN; ++i) read_b[i] = spread((b_row + i * 32) * C::WB) ^ (g * 16);
  const int first_t = t0 + part;
  bool inexact = false;  // a weight of this lane is not exact in fp16
  auto pass = [&](auto wide) {
    constexpr bool kWide = decltype(wide)::value;
#pragma unroll
    for (int i = 0; i < WN; ++i)
#pragma unroll
      for (int j = 0; j < WM; ++j) acc[i][j] = {};
    if (first_t < t1) {
      if (!C::kHelper) {
        scales(u0, sv);
        put_scales(u0 & 1, sv);
      }
#pragma unroll
      for (int i = 0; i < C::kAhead; ++i)
        if (first_t + i * GK < t1) stage(first_t + i * GK, i);
    }
    wait_stages<C::kInFlight, C::kAhead - 1>(first_t + (C::kAhead - 1) * GK < t1 ? C::kAhead - 1
                                                                                 : 0);
    if (ACT == kFp16 && !kWide && tid == 0) flag = 0;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();
    int buf = 0;
    for (int round = 0; round < rounds; ++round) {
      const int t = first_t + round * GK;
      const int u = t / C::kSteps, s = t % C::kSteps;
      const bool more = u + 1 < u1;
      // Scales are written before the loads of a step: what the compiler waits
      // for then is due at this step's end anyway.
      if (!C::kHelper && s == C::kSteps - 1 && more) put_scales((u + 1) & 1, sv);
      if (!C::kHelper && s == 0 && more) scales(u + 1, sv);
      __builtin_amdgcn_sched_barrier(0);
      if (t + C::kAhead * GK < t1)
        stage(t + C::kAhead * GK, buf == 0 ? C::kBufs - 1 : buf - 1);

      // a part whose last step is behind the end waits for the others
      if (GK == 1 || t < t1) {
        const uint32_t at_a = read_a + buf * C::kABytes, at_b = buf * C::kBBytes;
        const uint32_t* ls = lds_s + ((u & 1) * 4 + s * 4 / C::kSteps) * C::kSRows;
        uint32_t ws[WN];
#pragma unroll
        for (int i = 0; i < WN; ++i) ws[i] = ls[b_row + i * 32] >> (8 * g);
        if constexpr (kWiden) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4 w[WN], x[WM][2];
#pragma unroll
            for (int i = 0; i < WN; ++i)
              w[i] = *(const uint4*)(lds_b + at_b + (read_b[i] ^ (h * 32)));
#pragma unroll
            for (int j = 0; j < WM; ++j) {
              x[j][0] = *(const uint4*)(lds_a + (at_a ^ (h * 64 + g * 32)) + j * 4096);
              x[j][1] = *(const uint4*)(lds_a + (at_a ^ (h * 64 + g * 32 + 16)) + j * 4096);
            }
            float sw[WN], sx[WM];  // bytes 2h and 2h + 1 of the step's scales, by lane group
#pragma unroll
            for (int i = 0; i < WN; ++i) sw[i] = scale_value(ws[i] >> (16 * h) & 255u);
#pragma unroll
            for (int j = 0; j < WM; ++j)
              sx[j] = scale_value(ls[C::TN + a_row + j * 32] >> (8 * g + 16 * h) & 255u);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              bf16x8_t xv[WM];
#pragma unroll
              for (int j = 0; j < WM; ++j) {
                const uint4 q = x[j][k / 2];
                xv[j] = widen_fp8(k % 2 ? q.z : q.x, k % 2 ? q.w : q.y, sx[j]);
              }
#pragma unroll
              for (int i = 0; i < WN; ++i) {
                const uint32_t q = k == 0 ? w[i].x : k == 1 ? w[i].y : k == 2 ? w[i].z : w[i].w;
                const bf16x8_t wv = widen_bf16(q, sw[i]);
#pragma unroll
                for (int j = 0; j < WM; ++j) acc[i][j] = mfma_32x32x16_bf16(wv, xv[j], acc[i][j]);
              }
            }
          }
        } else if constexpr (ACT == kFp8) {
          uint32_t as[WM];
#pragma unroll
          for (int j = 0; j < WM; ++j) as[j] = ls[C::TN + a_row + j * 32] >> (8 * g);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            union { intx8 v; uint4 q[2]; } x[WM];
            uint4 w[WN];
#pragma unroll
            for (int i = 0; i < WN; ++i)
              w[i] = *(const uint4*)(lds_b + at_b + (read_b[i] ^ (k * 32)));
#pragma unroll
            for (int j = 0; j < WM; ++j) {
              x[j].q[0] = *(const uint4*)(lds_a + (at_a ^ (k * 64 + g * 16)) + j * 4096);
              x[j].q[1] = *(const uint4*)(lds_a + (at_a ^ (k * 64 + 32 + g * 16)) + j * 4096);
            }
#pragma unroll
            for (int i = 0; i < WN; ++i) {
              const intx8 wv = {(int)w[i].x, (int)w[i].y, (int)w[i].z, (int)w[i].w, 0, 0, 0, 0};
#pragma unroll
              for (int j = 0; j < WM; ++j) {
                // bytes 2k and 2k + 1 of the step's scales belong to this product
                if (k == 0)
                  acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                      wv, x[j].v, acc[i][j], 4, 0, 0, (int)ws[i], 0, (int)as[j]);
                else
                  acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                      wv, x[j].v, acc[i][j], 4, 0, 2, (int)ws[i], 2, (int)as[j]);
              }
            }
          }
        } else {
          uint4 w[WN];
#pragma unroll
          for (int i = 0; i < WN; ++i) {
            w[i] = *(const uint4*)(lds_b + at_b + read_b[i]);
            ws[i] = ws[i] >> (16 * (s & 1)) & 255u;  // two steps to a dword
          }
          if constexpr (ACT == kFp16 && !kWide) {
#pragma unroll
            for (int i = 0; i < WN; ++i) inexact |= !f16_exact(ws[i]);
          }
          if constexpr (!kWide) {
            // the next product's tokens are on their way while this one's multiply
            uint4 x[2][WM];
#pragma unroll
            for (int j = 0; j < WM; ++j)
              x[0][j] = *(const uint4*)(lds_a + (at_a ^ (g * 64)) + j * 4096);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (k < 3) {
#pragma unroll
                for (int j = 0; j < WM; ++j)
                  x[(k + 1) & 1][j] =
                      *(const uint4*)(lds_a + (at_a ^ (g * 64 + (k + 1) * 16)) + j * 4096);
              }
              __builtin_amdgcn_sched_barrier(0);
#pragma unroll
              for (int i = 0; i < WN; ++i) {
                const uint32_t q = k == 0 ? w[i].x : k == 1 ? w[i].y : k == 2 ? w[i].z : w[i].w;
                if constexpr (ACT == kFp16) {
                  const f16x8_t wv = widen_f16(q, scale_value(ws[i]));
#pragma unroll
                  for (int j = 0; j < WM; ++j)
                    acc[i][j] =
                        mfma_32x32x16_f16(wv, __builtin_bit_cast(f16x8_t, x[k & 1][j]), acc[i][j]);
                } else {
                  const bf16x8_t wv = widen_bf16(q, scale_value(ws[i]));
#pragma unroll
                  for (int j = 0; j < WM; ++j)
                    acc[i][j] =
                        mfma_32x32x16_bf16(wv, __builtin_bit_cast(bf16x8_t, x[k & 1][j]), acc[i][j]);
                }
              }
            }
          } else {
            // kept small rather than fast
#pragma unroll 1
            for (int k = 0; k < 4; ++k) {
#pragma unroll
              for (int j = 0; j < WM; ++j) {
                const uint4 x = *(const uint4*)(lds_a + (at_a ^ (g * 64 + k * 16)) + j * 4096);
                bf16x8_t hi, lo;
                split_f16(x, hi, lo);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < WN; ++i) {
                  const uint32_t q = k == 0 ? w[i].x : k == 1 ? w[i].y : k == 2 ? w[i].z : w[i].w;
                  const bf16x8_t wv = widen_bf16(q, scale_value(ws[i]));
                  acc[i][j] = mfma_32x32x16_bf16(wv, hi, acc[i][j]);
                  acc[i][j] = mfma_32x32x16_bf16(wv, lo, acc[i][j]);
                }
              }
            }
          }
        }
      }
      // Until the next step's buffer is full: the loads for the steps after it
      // stay in flight (the last step of a K that it does not divide has none).
      const int left = t < t1 ? (t1 - 1 - t) / GK : 0;  // steps of this part behind t
      const int ahead = left < C::kAhead ? left : C::kAhead;
      wait_stages<C::kInFlight, C::kAhead - 1>(ahead - 1 -
                                               ((t + ahead * GK + 1) * C::KS > p.K));
      if (ACT == kFp16 && !kWide && round == rounds - 1 && inexact) flag = 1;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __syncthreads();
      buf = buf == C::kBufs - 1 ? 0 : buf + 1;
    }
  };
  const bool helps = C::kHelper && wave_all == GN * GM * GK;
  if (helps) bring_scales();
  else pass(std::false_type());
  // fp16: where some weight of the tile is not exact in fp16 all of it is
  // computed again with a split in two. Every wave sees the same flag.
  if (ACT == kFp16 && __builtin_amdgcn_readfirstlane(*(volatile int*)&flag)) {
    __syncthreads();
    if (helps) bring_scales();
    else pass(std::integral_constant<bool, ACT == kFp16>());
  }
  if (helps) {
    // the barriers behind the passes
    if (GK > 1) __syncthreads(), __syncthreads();
    if (gridDim.y == 1) __syncthreads();
    return;
  }

  if constexpr (GK > 1) {
    // the parts together, in their order
    float* const join = (float*)lds + wave * WN * WM * 1024 + lane * 4;
    if (part > 0) {
#pragma unroll
      for (int i = 0; i < WN * WM * 4; ++i)
        *(float4*)(join + (part - 1) * GN * GM * WN * WM * 1024 + i * 256) =
            make_float4(acc[i / 4 / WM][i / 4 % WM][i % 4 * 4], acc[i / 4 / WM][i / 4 % WM][i % 4 * 4 + 1],
                        acc[i / 4 / WM][i / 4 % WM][i % 4 * 4 + 2], acc[i / 4 / WM][i / 4 % WM][i % 4 * 4 + 3]);
    }
    __syncthreads();
    if (part == 0) {
      for (int k = 0; k < GK - 1; ++k) {
#pragma unroll
        for (int i = 0; i < WN * WM * 4; ++i) {
          const float4 v = *(const float4*)(join + k * GN * GM * WN * WM * 1024 + i * 256);
          acc[i / 4 / WM][i / 4 % WM][i % 4 * 4] += v.x;
          acc[i / 4 / WM][i / 4 % WM][i % 4 * 4 + 1] += v.y;
          acc[i / 4 / WM][i / 4 % WM][i % 4 * 4 + 2] += v.z;
          acc[i / 4 / WM][i / 4 % WM][i % 4 * 4 + 3] += v.w;
        }
      }
    }
    __syncthreads();
  }

  if (gridDim.y > 1) {
    // as the registers lie: join_kernel reads them so
    if (part > 0) return;
    float* to = p.sums + (((int64_t)blockIdx.y * gridDim.x + id) * GN * GM + wave) * WN * WM * 1024;
#pragma unroll
    for (int i = 0; i < WN; ++i)
#pragma unroll
      for (int j = 0; j < WM; ++j)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          *(float4*)(to + ((i * WM + j) * 4 + r / 4) * 256 + lane * 4) =
              make_float4(acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]);
    return;
  }

  // Through shared memory, so that a row of the tile leaves in 16-byte pieces.
  // Lane: token lr of 32; register r: output (r & 3) + 8 (r >> 2) + 4 g.
  constexpr int H = GATED ? WN / 2 : WN;
  if (GATED && part == 0) {
    auto gate = [&](auto kind) {
#pragma unroll
      for (int i = 0; i < H; ++i)
#pragma unroll
        for (int j = 0; j < WM; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            acc[i][j][r] = activate<decltype(kind)::value>(acc[i][j][r]) * acc[i + H * GATED][j][r];
    };
    if (p.act == 0) gate(std::integral_constant<int, 0>());
    else if (p.act == 1) gate(std::integral_constant<int, 1>());
    else gate(std::integral_constant<int, 2>());
  }
#pragma unroll
  for (int j = 0; j < WM; ++j) {
    if (part > 0) break;
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const int nl = (wn * H + i) * 32 + 4 * g;
      uint8_t* to = lds + (a_row + j * 32) * kRow + nl * kSize;
      if constexpr (OUT8) {
        float y[16];
        uint32_t most = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          y[r] = acc[i][j][r];
          most = abs_bits(y[r]) > most ? abs_bits(y[r]) : most;
        }
        uint32_t a, b;
        permlane32_pair(most, most, a, b);  // the other half of the block
        most = a > b ? a : b;
        const uint32_t byte = mxfp8_scale_byte(most);
        const float inv = mx_inverse_scale(byte);
#pragma unroll
        for (int r = 0; r < 16; r += 8) {
          const uint2 q = mxfp8_pack8(y + r, inv, byte == 255u);
          *(uint32_t*)(to + r * 2) = q.x;
          *(uint32_t*)(to + r * 2 + 8) = q.y;
        }
        const int m = m0 + a_row + j * 32, n = n0 + nl;
        if (g == 0 && m < p.M && n < p.N)
          p.out_scale[(int64_t)m * (p.N / kMxBlock) + n / kMxBlock] = (uint8_t)byte;
      } else {
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          union { uint16_t v[4]; uint2 q; } y;
#pragma unroll
          for (int k = 0; k < 4; ++k) y.v[k] = to16(acc[i][j][r + k], p.out_fp16);
          *(uint2*)(to + r * 4) = y.q;
        }
      }
    }
  }
  __syncthreads();
  constexpr int kPieces = C::kOut * kSize / 16, kEach = 16 / kSize;
  const bool whole = OUT8 ? ((uintptr_t)p.out % 16 | p.ldo % 16) == 0
                          : ((uintptr_t)p.out % 16 | p.ldo % 8 | p.N % 8) == 0;
  if (OUT8 || whole) {
    for (int i = tid; i < C::TM * kPieces; i += C::kThreads) {
      const int ml = i / kPieces, nl = i % kPieces * kEach;
      const int m = m0 + ml, n = n0 + nl;
      if (m >= p.M || n >= p.N) continue;
      const uint8_t* from = lds + ml * kRow + nl * kSize;
      uint8_t* to = (uint8_t*)p.out + ((int64_t)m * p.ldo + n) * kSize;
      if (whole) {
        *(uint4*)to = *(const uint4*)from;
      } else {  // MXFP8: rows at multiples of 8, N at one of 32
        ((uint2*)to)[0] = ((const uint2*)from)[0];
        ((uint2*)to)[1] = ((const uint2*)from)[1];
      }
    }
  } else {
    // odd rows: pieces at any address, the last of a row one by one
    for (int i = tid; i < C::TM * kPieces; i += C::kThreads) {
      const int ml = i / kPieces, nl = i % kPieces * kEach;
      const int m = m0 + ml, n = n0 + nl;
      if (m >= p.M || n >= p.N) continue;
      const uint16_t* from = (const uint16_t*)(lds + ml * kRow) + nl;
      uint16_t* to = (uint16_t*)p.out + (int64_t)m * p.ldo + n;
      if (n + kEach <= p.N) {
        const uint4 v = *(const uint4*)from;
        __builtin_memcpy(to, &v, 16);
      } else {
        for (int k = 0; k < p.N - n; ++k) to[k] = from[k];
      }
    }
  }
}

// The parts of K together: a workgroup for 32 outputs by 32 tokens. Each of its
// waves sums a quarter of the parts, the quarters follow in their order.
template <bool GATED, bool OUT8, int WN, int WM, int GN, int GM, int GK>
__global__ __launch_bounds__(256) void join_kernel(Params p, int tiles_n, int tiles_m, int parts) {
  constexpr int H = GATED ? WN / 2 : WN, kSums = GATED ? 32 : 16;
  __shared__ float quarter[3][kSums][64];
  const int lane = threadIdx.x & 63, lr = lane & 31, g = lane >> 5;
  const int q = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int at = blockIdx.x;
  const int j = at % WM, i = at / WM % H, wave = at / (WM * H) % (GN * GM);
  const int id = at / (WM * H * GN * GM);
  const int band = id / (8 * tiles_n), first = band * 8;
  const int high = tiles_m - first < 8 ? tiles_m - first : 8;
  const int in_band = id - band * 8 * tiles_n;
  const int m = (((first + in_band % high) * GM + wave / GN) * WM + j) * 32 + lr;
  const int n = ((in_band / high * GN + wave % GN) * H + i) * 32 + 4 * g;

  const int64_t part = (int64_t)tiles_n * tiles_m * GN * GM * WN * WM * 1024;
  const float* from = p.sums + (((int64_t)id * GN * GM + wave) * WN * WM + i * WM + j) * 1024 + lane * 4;
  float sum[kSums] = {};  // of the gate, then of up
  const int each = ceil_div(parts, 4);
  const int s1 = (q + 1) * each < parts ? (q + 1) * each : parts;
#pragma unroll 2
  for (int s = q * each; s < s1; ++s) {
#pragma unroll
    for (int r = 0; r < kSums; r += 4) {
      const float4 v = *(const float4*)(from + s * part + r / 16 * H * WM * 1024 + r % 16 / 4 * 256);
      sum[r] += v.x, sum[r + 1] += v.y, sum[r + 2] += v.z, sum[r + 3] += v.w;
    }
  }
  if (q > 0) {
#pragma unroll
    for (int r = 0; r < kSums; ++r) quarter[q - 1][r][lane] = sum[r];
  }
  __syncthreads();
  if (q > 0) return;
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int r = 0; r < kSums; ++r) sum[r] += quarter[k][r][lane];
  float y[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) y[r] = GATED ? activate(p.act, sum[r]) * sum[r + kSums - 16] : sum[r];
  if constexpr (OUT8) {
    uint32_t most = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) most = abs_bits(y[r]) > most ? abs_bits(y[r]) : most;
    uint32_t a, b;
    permlane32_pair(most, most, a, b);
    most = a > b ? a : b;
    const uint32_t byte = mxfp8_scale_byte(most);
    const float inv = mx_inverse_scale(byte);
    if (m < p.M && n < p.N) {
      uint8_t* o = (uint8_t*)p.out + (int64_t)m * p.ldo + n;
#pragma unroll
      for (int r = 0; r < 16; r += 8) {
        const uint2 q = mxfp8_pack8(y + r, inv, byte == 255u);
        *(uint32_t*)(o + r * 2) = q.x;
        *(uint32_t*)(o + r * 2 + 8) = q.y;
      }
      if (g == 0) p.out_scale[(int64_t)m * (p.N / kMxBlock) + n / kMxBlock] = (uint8_t)byte;
    }
  } else if (m < p.M) {
    uint16_t* o = (uint16_t*)p.out + (int64_t)m * p.ldo + n;
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      union { uint16_t v[4]; uint2 q; } t;
#pragma unroll
      for (int k = 0; k < 4; ++k) t.v[k] = to16(y[r + k], p.out_fp16);
      if (n + 2 * r + 4 <= p.N) {
        __builtin_memcpy(o + 2 * r, &t.q, 8);  // at any address
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n + 2 * r + k < p.N) o[2 * r + k] = t.v[k];
      }
    }
  }
}

template <int ACT, bool GATED, bool OUT8, int WN, int WM, int GN, int GM, int GK>
hipError_t launch_tile(const Params& all, int parts, hipStream_t stream) {
  using C = Tile<ACT, GATED, WN, WM, GN, GM, GK>;
  const int64_t tiles_n = ceil_div(all.N, C::kOut);
  // A launch has less than 2^32 threads: more tiles go some rows of them at a time.
  // (Parts of K are for few tiles.)
  const int64_t most = (((int64_t)1 << 32) - 1) / C::kLaunch / tiles_n;
  for (int64_t m = 0; m < all.M; m += most * C::TM) {
    Params p = all;
    p.a = (const char*)p.a + m * p.lda * (ACT == kFp8 ? 1 : 2);
    if (ACT == kFp8) p.a_scale += m * (p.K / kMxBlock);
    p.out = (char*)p.out + m * p.ldo * (OUT8 ? 1 : 2);
    if (OUT8) p.out_scale += m * (p.N / kMxBlock);
    p.M = (int)(all.M - m < most * C::TM ? all.M - m : most * C::TM);
    const int64_t tiles_m = ceil_div(p.M, C::TM);
    hipLaunchKernelGGL((tile_kernel<ACT, GATED, OUT8, WN, WM, GN, GM, GK>),
                       dim3((unsigned)(tiles_n * tiles_m), parts), dim3(C::kLaunch), 0, stream, p,
                       (int)tiles_n, (int)tiles_m);
    if (parts > 1) {
      const int64_t joins = tiles_n * tiles_m * GN * GM * WN * WM / (GATED ? 2 : 1);
      hipLaunchKernelGGL((join_kernel<GATED, OUT8, WN, WM, GN, GM, GK>), dim3((unsigned)joins),
                         dim3(256), 0, stream, p, (int)tiles_n, (int)tiles_m, parts);
    }
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Which kernel, tile and parts of K a product gets.

enum Shape {
  kRows,      // 64 tokens at most, 32 with an MXFP8 output
  k256x128,   // weight rows x tokens, one part of K in a workgroup
  k128x128,
  k128x128x2, // two parts of K in a workgroup
  k128x64,
  k64x64x4,
  k64x32x4,
  k128x32x4,
};

struct Plan {
  int shape, parts;  // parts of K over workgroups
  int64_t floats;    // of the sums that they leave
};

// How many rows a workgroup takes and how many waves share its K. Measured at
// one bf16 token, us for (tiles of 16 rows, waves, chunks ahead) = (1, 8, 2) /
// (2, 8, 1) / (2, 4, 1): 4096 x 14336 8.4 / 10.2 / 15.6, 6144 x 4096 5.6 / 5.0 /
// 6.2, 12288 x 8192 14.7 / 10.9 / 11.4, 32000 x 4096 14.5 / 13.2 / 12.4. Few
// workgroups need many waves each; many of them hide each other's start, and
// shared memory that is spent on chunks ahead keeps some of them out. Four
// tiles with an MXFP8 output, (2, 8, 1) / (2, 4, 2): 14336 x 4096 12.3 / 12.6, 28672
// x 8192 54.3 / 55.8; fp16 4096 x 4096 (2, 8, 2) / (2, 8, 1) 7.5 / 7.6, 16 tokens of
// 2560 x 8192 12.5 / 14.0. Sixteen waves lose everywhere (6144 x 4096 10.2), three
// chunks ahead as well (4096 x 14336 8.6).
// With 17 to 64 tokens a workgroup's time is its tokens' way from L2, and two tiles
// read them once for both as long as that leaves work for every CU: kFewPairs.
constexpr int kFewPairs = 129;

template <int ACT, bool GATED, bool OUT8, int XI>
hipError_t choose_rows(const Params& p, hipStream_t stream) {
  if constexpr (OUT8) {
    // a block of the output is 32 wide: four tiles
    if constexpr (ACT != kFp16 || XI == 8) {
      return launch_rows<ACT, GATED, OUT8, 2, XI, 8, 1>(p, stream);
    } else {
      // its two ways of widening want more registers than four waves a SIMD have
      if (p.N <= 256 * 32) return launch_rows<ACT, GATED, OUT8, 2, XI, 8, 2>(p, stream);
      return launch_rows<ACT, GATED, OUT8, 2, XI, 4, 2>(p, stream);
    }
  } else {
    constexpr int RT = GATED ? 1 : 2;
    constexpr bool kMany = XI * 1024 / Rows<ACT, GATED, RT, XI, 8, 1>::kXRow > 16;
    const int pairs = ceil_div(p.N, RT * 16);  // workgroups of two tiles
    // 32 tokens of 8 bits in rows apart keep eight waves: 32000 x 2080 14.3 for 16.5
    const bool eight = ACT == kFp8 && XI == 4 && p.K % 128 != 0;
    if (pairs >= 512 && !eight)
      return launch_rows<ACT, GATED, OUT8, RT, XI, 4, 1>(p, stream);
    if (pairs < (kMany ? kFewPairs : 192)) return launch_rows<ACT, GATED, OUT8, 1, XI, 8, XI < 8 ? 2 : 1>(p, stream);
    return launch_rows<ACT, GATED, OUT8, RT, XI, 8, 1>(p, stream);
  }
}

template <int ACT, bool GATED, bool OUT8>
hipError_t launch_out(const Plan& plan, const Params& p, hipStream_t stream) {
  switch (plan.shape) {
    case kRows: {
      constexpr int kFew = ACT == kFp8 ? 8 : 4;  // tokens in a kilobyte of a chunk
      if (p.M <= kFew) return choose_rows<ACT, GATED, OUT8, 1>(p, stream);
      if (p.M <= 2 * kFew) return choose_rows<ACT, GATED, OUT8, 2>(p, stream);
      if (p.M <= 16) return choose_rows<ACT, GATED, OUT8, 16 / kFew>(p, stream);
      if (p.M <= 32) return choose_rows<ACT, GATED, OUT8, 32 / kFew>(p, stream);
      if constexpr (!OUT8) {
        if (p.M <= 64) return choose_rows<ACT, GATED, OUT8, 64 / kFew>(p, stream);
      }
      return hipErrorInvalidValue;
    }
    case k256x128: return launch_tile<ACT, GATED, OUT8, 2, 4, 4, 1, 1>(p, plan.parts, stream);
    case k128x128: return launch_tile<ACT, GATED, OUT8, 2, 2, 2, 2, 1>(p, plan.parts, stream);
    case k128x128x2: return launch_tile<ACT, GATED, OUT8, 2, 2, 2, 2, 2>(p, plan.parts, stream);
    case k128x64:
      // 8-bit products leave time for two waves to read a token, in two parts
      // of K; where registers have to widen values, larger tiles of a wave
      // widen fewer of them. bf16 64 x 28672, K = 4096: 24.2 and 21.4 us.
      if constexpr (ACT == kFp8 && !OUT8)
        return launch_tile<ACT, GATED, OUT8, 2, 1, 2, 2, 2>(p, plan.parts, stream);
      else
        return launch_tile<ACT, GATED, OUT8, 2, 2, 2, 1, 4>(p, plan.parts, stream);
    case k64x64x4: return launch_tile<ACT, GATED, OUT8, 2, 1, 1, 2, 4>(p, plan.parts, stream);
    case k64x32x4: return launch_tile<ACT, GATED, OUT8, 2, 1, 1, 1, 4>(p, plan.parts, stream);
    case k128x32x4: return launch_tile<ACT, GATED, OUT8, 2, 1, 2, 1, 4>(p, plan.parts, stream);
  }
  return hipErrorInvalidValue;
}

// gated: 0 plain, 1 gated, 2 gated with an MXFP8 output
template <int ACT>
hipError_t launch_act(int gated, const Plan& plan, const Params& p, hipStream_t stream) {
  switch (gated) {
    case 0: return launch_out<ACT, false, false>(plan, p, stream);
    case 1: return launch_out<ACT, true, false>(plan, p, stream);
    case 2: return launch_out<ACT, true, true>(plan, p, stream);
  }
  return hipErrorInvalidValue;
}

// one translation unit each
hipError_t launch_bf16(int gated, const Plan& plan, const Params& p, hipStream_t stream);
hipError_t launch_fp16(int gated, const Plan& plan, const Params& p, hipStream_t stream);
hipError_t launch_fp8(int gated, const Plan& plan, const Params& p, hipStream_t stream);

}  // namespace mx4
}  // namespace fi
