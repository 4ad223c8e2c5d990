// MXFP8 output: an activation, or its RMSNorm (with or without the residual's
// addition), written as e4m3 values with one scale for 32 neighbours.
//
//   r = x (+ residual, which is stored back rounded to its type)
//   y = r / sqrt(mean(r^2) + eps) * w          (y = r without a weight)
//   2^e: the least with max|y_block| <= 448 * 2^e;   q = e4m3(y * 2^-e)
//
// One workgroup takes one row (short rows share a wave) and keeps it in
// registers, eight values to a lane, so every input is read once and every
// output written once. The four lanes of a quad hold one block of 32: its
// maximum needs two register exchanges and no shared memory. The sum of squares
// is held in 64 bits, which costs nothing: the bound is memory. 16384 x 8192 bf16
// with a residual takes 163 us, 5.8 TB/s, where a copy of a gigabyte reaches 5.1;
// an activation of 8191 x 14336 takes 60 us, 5.9 TB/s. Up to about 100 rows the
// launch is the time (5 us).
#include "fi/common.hpp"
#include "fi/mx.hpp"
#include "fi/vec.hpp"

namespace fi {
namespace mxq {

template <typename T, bool kAligned>
__device__ __forceinline__ void load8(float* v, const T* p) {
  vec_t<T, 8> t;
  if constexpr (kAligned) {
    t.load(p);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) t.data[j] = p[j];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = t.get(j);
}

// NV: groups of eight values a lane holds; 0: one group, and several rows to a
// wave, `lanes` (a power of two) for each. kAligned: 16-byte rows.
template <typename T, int NV, bool kNorm, bool kAdd, bool kAligned>
__global__ __launch_bounds__(NV ? 1024 : 256) void mx_quant_kernel(
    const T* __restrict__ x, T* __restrict__ residual, const T* __restrict__ w,
    uint8_t* __restrict__ out, uint8_t* __restrict__ scale, int rows, int k, int64_t stride_x,
    int64_t stride_r, double eps, int lanes) {
  constexpr bool kShort = NV == 0;
  constexpr int kGroups = kShort ? 1 : NV;
  __shared__ double sums[16];
  int64_t row = blockIdx.x;
  int t = threadIdx.x;
  if constexpr (kShort) {
    row = row * (blockDim.x / lanes) + t / lanes;
    t %= lanes;
    if (row >= rows) return;
  }
  const T* xr = x + row * stride_x;
  T* rr = kAdd ? residual + row * stride_r : nullptr;
  float v[kGroups][8];
  double ss = 0.;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int at = (i * blockDim.x + t) * 8;
    if (at < k) {
      load8<T, kAligned>(v[i], xr + at);
      if constexpr (kAdd) {
        float r[8];
        load8<T, kAligned>(r, rr + at);
        vec_t<T, 8> t;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          t.set(j, v[i][j] + r[j]);
          v[i][j] = t.get(j);  // the norm is that of the residual as it is stored
        }
        if constexpr (kAligned) {
          t.store(rr + at);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) rr[at + j] = t.data[j];
        }
      }
      if constexpr (kNorm) {
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)v[i][j], (double)v[i][j], ss);
      }
    }
  }
  double rrms = 1.;
  if constexpr (kNorm) {
    if constexpr (kShort) {
      for (int i = 1; i < lanes; i *= 2) ss += __shfl_xor(ss, i);
    } else {
#pragma unroll
      for (int i = 1; i < kWaveSize; i *= 2) ss += __shfl_xor(ss, i);
      const int waves = blockDim.x / kWaveSize;
      if (t % kWaveSize == 0) sums[t / kWaveSize] = ss;
      __syncthreads();
      ss = 0.;
      for (int i = 0; i < waves; ++i) ss += sums[i];
    }
    rrms = 1. / sqrt(ss / k + eps);
  }
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int at = (i * blockDim.x + t) * 8;
    if (at < k) {  // k is a multiple of 32: a quad is inside or outside as one
      uint32_t most = 0;
      float wv[8], y[8];
      if constexpr (kNorm) load8<T, kAligned>(wv, w + at);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = kNorm ? v[i][j] * (float)rrms * wv[j] : v[i][j];
        const uint32_t b = abs_bits(y[j]);
        most = b > most ? b : most;
      }
      most = quad_max(most);
      if constexpr (kNorm) {
        // Next to the border of two scales 32 bits could take the wrong one: there
        // (one block in a million) 64 bits decide, for the quad as one.
        if ((most & 0x7fffffu) - 0x5ffff0u <= 0x20u && most < 0x7f800000u) {
          const double border = (double)__uint_as_float((most & 0x7f800000u) | 0x600000u);
          uint32_t over = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            over |= __builtin_fabs((double)v[i][j] * rrms * (double)wv[j]) > border;
          most = (most & 0x7f800000u) | (0x600000u + quad_max(over));
        }
      }
      const uint32_t byte = mxfp8_scale_byte(most);
      const uint2 q = mxfp8_pack8(y, mx_inverse_scale(byte), byte == 255u);
      uint8_t* o = out + row * k + at;
      if constexpr (kAligned) {
        *reinterpret_cast<uint2*>(o) = q;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[j] = (uint8_t)(q.x >> (8 * j));
          o[4 + j] = (uint8_t)(q.y >> (8 * j));
        }
      }
      if (t % 4 == 0) scale[row * (k / kMxBlock) + at / kMxBlock] = (uint8_t)byte;
    }
  }
}

template <typename T, bool kNorm, bool kAdd, bool kAligned>
hipError_t launch(const void* x, void* residual, const void* w, void* out, void* scale,
                  int rows, int k, int64_t sx, int64_t sr, double eps, hipStream_t stream) {
  // Two groups to a lane from 4096 values on: 512 lanes with two wait for their
  // sum with half the waves of 1024 with one (16384 x 8192: 5.7 and 5.45 TB/s,
  // 4096 x 7168: 5.6 and 5.2), and 896 lanes with two beat 448 with four
  // (8191 x 14336: 5.55 and 5.4). Rows that leave half a wave idle share it:
  // 262144 x 128 with a residual takes 45 us for 104, 1048576 x 64 quantized 39
  // for 225.
  const int groups = k / 8;
  const int nv = groups <= kWaveSize / 2 ? 0
                 : groups <= 512         ? 1
                 : groups <= 2048        ? 2
                 : groups <= 4096        ? 4
                                         : 8;
  int lanes = 4;
  while (lanes < groups) lanes *= 2;
  const int threads = nv ? ceil_div(ceil_div(groups, nv), kWaveSize) * kWaveSize : 256;
  if (threads > 1024) return hipErrorInvalidValue;
  // a launch has less than 2^32 threads: 2^21 rows at a time
  constexpr int kRows = 1 << 21;
  for (int64_t r = 0; r < rows; r += kRows) {
    const int some = rows - r < kRows ? (int)(rows - r) : kRows;
    const int groups_of_rows = nv ? some : ceil_div(some, threads / lanes);
#define FI_GO(NV)                                                                       \
  hipLaunchKernelGGL((mx_quant_kernel<T, NV, kNorm, kAdd, kAligned>),                   \
                     dim3(groups_of_rows), dim3(threads), 0, stream, (const T*)x + r * sx, \
                     residual ? (T*)residual + r * sr : nullptr, (const T*)w,           \
                     (uint8_t*)out + r * k, (uint8_t*)scale + r * (k / kMxBlock), some, \
                     k, sx, sr, eps, lanes)
    switch (nv) {
      case 0: FI_GO(0); break;
      case 1: FI_GO(1); break;
      case 2: FI_GO(2); break;
      case 4: FI_GO(4); break;
      default: FI_GO(8); break;
    }
#undef FI_GO
  }
  return hipGetLastError();
}

template <typename T>
hipError_t dispatch(const void* x, void* residual, const void* w, void* out, void* scale,
                    int rows, int k, int64_t sx, int64_t sr, double eps, int aligned,
                    hipStream_t stream) {
#define FI_GO(NORM, ADD)                                                                  \
  (aligned ? launch<T, NORM, ADD, true>(x, residual, w, out, scale, rows, k, sx, sr, eps, \
                                        stream)                                           \
           : launch<T, NORM, ADD, false>(x, residual, w, out, scale, rows, k, sx, sr,     \
                                         eps, stream))
  if (!w) return FI_GO(false, false);
  return residual ? FI_GO(true, true) : FI_GO(true, false);
#undef FI_GO
}

}  // namespace mxq
}  // namespace fi

// dtype: 0 bf16, 1 fp16, 2 fp32. Without `w` the activation itself is written;
// with `residual` x is added to it in place first. k: a multiple of 32, at
// most 65536. `aligned`: x, residual and w have rows of whole 16 bytes, and
// out starts at a multiple of 8.
extern "C" hipError_t fi_mx_quant(int dtype, const void* x, void* residual, const void* w,
                                  void* out, void* scale, int rows, int k, int64_t sx,
                                  int64_t sr, double eps, int aligned, hipStream_t stream) {
  if (rows == 0) return hipSuccess;
  if (k <= 0 || k % fi::kMxBlock != 0 || k > 65536) return hipErrorInvalidValue;
  switch (dtype) {
    case 0: return fi::mxq::dispatch<fi::bf16>(x, residual, w, out, scale, rows, k, sx, sr, eps, aligned, stream);
    case 1: return fi::mxq::dispatch<fi::fp16>(x, residual, w, out, scale, rows, k, sx, sr, eps, aligned, stream);
    case 2: return fi::mxq::dispatch<float>(x, residual, w, out, scale, rows, k, sx, sr, eps, aligned, stream);
  }
  return hipErrorInvalidValue;
}
