// Products with MXFP4 weights: the choice of a kernel, and the entry. The
// kernels are in fi/mxfp4_body.hpp.
#include "fi/mxfp4_body.hpp"

namespace fi {
namespace mx4 {

// The largest tile that still gives the chip's 256 CUs something to do: tokens
// are read once for each tile of weight rows and weights once for each tile of
// tokens, so large tiles move less. Measured (us, K = 4096 unless said) where
// two of them meet, in the order of the enum:
//   8-bit tokens 4096 x 6144: 256x128 93, 128x128 104; 1024 x 6144: 39 and 32
//   bf16 1024 x 4096: 128x128 43, 128x128x2 37, 128x64x2 48
//   8-bit 512 x 4096, K = 14336: 128x128x2 43, 128x64x2 41, 64x64x4 53
//   bf16 128 x 4096: 64x64x4 14.4, 64x32x4 11.5; 256 x 4096: 15.7 and 20.9
//   bf16 24 x 28672: 128x32x4 16.0, 64x32x4 21.2, 128x64x2 23.4
// With a long K and few tiles K is split over workgroups too, and a second
// kernel joins the parts: 8-bit 64 x 4096, K = 14336, 64x64x4 in 1 / 2 / 4
// parts 27 / 18.9 / 14.7.
Plan make_plan(int M, int N, int K, bool gated) {
  if (M <= 16) return {kRows, 1, 0};
  const int64_t rows = gated ? 2 * (int64_t)N : N;
  auto tiles = [&](int r, int t) { return ceil_div64(rows, r) * ceil_div64(M, t); };
  if (M > 32 && tiles(256, 128) >= 512) return {k256x128, 1, 0};
  if (M > 64 && tiles(128, 128) > 256) return {k128x128, 1, 0};
  if (M <= 32 && tiles(128, 32) >= 192) return {k128x32x4, 1, 0};
  if (M > 64 && tiles(128, 128) >= 160) return {k128x128x2, 1, 0};
  if (M > 32 && tiles(128, 64) >= 160) return {k128x64x2, 1, 0};
  if (M > 32 && tiles(64, 64) >= 192) return {k64x64x4, 1, 0};
  const int loads = ceil_div(K, 512);  // of scales; a part holds whole ones
  if (loads < 16) return {k64x32x4, 1, 0};
  const int wide = M > 32 ? 64 : 32;
  int64_t parts = 256 / tiles(64, wide);
  if (parts > loads / 6) parts = loads / 6;
  if (parts <= 1) return {M > 32 ? k64x64x4 : k64x32x4, 1, 0};
  return {M > 32 ? k64x64x4 : k64x32x4, (int)parts, parts * tiles(64, wide) * 64 * wide};
}

}  // namespace mx4
}  // namespace fi

// How many floats of workspace fi_gemm_mxfp4 wants for this product.
extern "C" int64_t fi_gemm_mxfp4_floats(int gated, int M, int N, int K) {
  return M > 0 && N > 0 ? fi::mx4::make_plan(M, N, K, gated).floats : 0;
}

// a_type: 0 bf16, 1 fp16, 2 e4m3 with scale bytes; out_type the same, 2 for the
// gated form alone and N a multiple of 32. N counts outputs; the gated form
// reads 2 * N weight rows. act: 0 silu, 1 gelu, 2 gelu with tanh. K is a
// multiple of 32; the rows of a and b start at multiples of 16 bytes, those of
// an e4m3 out at multiples of 8. floats: fi_gemm_mxfp4_floats of them.
extern "C" hipError_t fi_gemm_mxfp4(int a_type, int out_type, int gated, int act,
                                    const void* a, const void* a_scale, const void* b,
                                    const void* b_scale, void* out, void* out_scale,
                                    float* floats, int M, int N, int K, int64_t lda,
                                    int64_t ldo, hipStream_t stream) {
  using namespace fi::mx4;
  if (M == 0 || N == 0) return hipSuccess;
  if (K <= 0 || K % fi::kMxBlock != 0) return hipErrorInvalidValue;
  if (out_type == kFp8 && (!gated || N % fi::kMxBlock != 0)) return hipErrorInvalidValue;
  const Params all{a,   (const uint8_t*)a_scale, (const uint8_t*)b, (const uint8_t*)b_scale,
                   out, (uint8_t*)out_scale,     M, N, K, lda, ldo, act, out_type == kFp16,
                   floats};
  const int form = gated ? (out_type == kFp8 ? 2 : 1) : 0;
  auto launch = [&](const Plan& plan, const Params& p) {
    switch (a_type) {
      case kBf16: return launch_bf16(form, plan, p, stream);
      case kFp16: return launch_fp16(form, plan, p, stream);
      case kFp8: return launch_fp8(form, plan, p, stream);
    }
    return hipErrorInvalidValue;
  };
  const Plan plan = make_plan(M, N, K, gated);
  if (plan.parts > 1 && !floats) return hipErrorInvalidValue;
  const int a_size = a_type == kFp8 ? 1 : 2, out_size = out_type == kFp8 ? 1 : 2;
  // A tile counts its bytes in 32 bits. Rows further apart than that allows go
  // 16 tokens at a time through the kernel that does not.
  const int64_t far = lda * a_size > (int64_t)K / 2 ? lda * a_size : (int64_t)K / 2;
  if (plan.shape == kRows || far < ((int64_t)1 << 32) / 256) return launch(plan, all);
  for (int m = 0; m < M; m += 16) {
    Params p = all;
    p.a = (const char*)a + (int64_t)m * lda * a_size;
    p.a_scale = p.a_scale ? p.a_scale + (int64_t)m * (K / fi::kMxBlock) : nullptr;
    p.out = (char*)out + (int64_t)m * ldo * out_size;
    p.out_scale = p.out_scale ? p.out_scale + (int64_t)m * (N / fi::kMxBlock) : nullptr;
    p.M = M - m < 16 ? M - m : 16;
    const hipError_t e = launch({kRows, 1, 0}, p);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
