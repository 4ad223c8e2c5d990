// Products with MXFP4 weights: the choice of a kernel, and the entry. The
// kernels are in fi/mxfp4_body.hpp.
#include "fi/mxfp4_body.hpp"

namespace fi {
namespace mx4 {

// What a tile costs: us to start and to finish, and us for 1024 of K where a CU
// holds one workgroup and where it holds two. Fitted to K = 1024, 2048 and 7680
// with 256, 512 and 1024 tiles (each time within 17 %; 25 % for 128 x 32). Over
// random products the time of the tile chosen is 0.1 % (bf16, MXFP8), 2.1 % (fp16,
// which shares the costs of bf16) and 2.4 % (8 bits in and out) over that of the
// best, at worst 1.34 times it (206 x 25714 x 13088 in fp16). Large tiles move fewer
// bytes for a product, small ones leave fewer CUs without work.
// `apart`: how much longer it takes where rows of a do not start at multiples of
// 128 bytes, so that every piece of one lies in two lines (K = 2080 to 7680).
struct Cost {
  int shape, rows, tokens;
  float start, one, two;  // two: 0 where a CU has room for one
  float apart;
};
constexpr Cost kCosts16[] = {
    {k256x128, 256, 128, 4.1f, 14.3f, 26.8f, 1.08f}, {k128x128, 128, 128, 2.6f, 8.8f, 14.9f, 1.06f},
    {k128x128x2, 128, 128, 3.1f, 7.5f, 0.f, 1.08f},  {k128x64, 128, 64, 2.6f, 4.1f, 0.f, 1.13f},
    {k64x64x4, 64, 64, 1.9f, 2.75f, 0.f, 1.15f},     {k64x32x4, 64, 32, 1.4f, 1.8f, 0.f, 1.17f},
    {k128x32x4, 128, 32, 1.9f, 3.f, 0.f, 1.25f},
};
constexpr Cost kCosts8[] = {
    {k256x128, 256, 128, 3.6f, 8.6f, 14.7f, 1.26f}, {k128x128, 128, 128, 2.2f, 4.6f, 8.1f, 1.16f},
    {k128x128x2, 128, 128, 3.2f, 4.2f, 0.f, 1.27f}, {k128x64, 128, 64, 1.9f, 2.7f, 0.f, 1.38f},
    {k64x64x4, 64, 64, 1.7f, 1.7f, 0.f, 1.28f},     {k64x32x4, 64, 32, 0.8f, 1.5f, 0.f, 1.22f},
    {k128x32x4, 128, 32, 1.3f, 2.2f, 0.f, 1.33f},
};

// 8 bits in and out, where every tile widens its operands (worst fit 15 %)
constexpr Cost kCosts8to8[] = {
    {k256x128, 256, 128, 4.1f, 13.f, 24.f, 1.11f},  {k128x128, 128, 128, 1.4f, 7.9f, 13.9f, 1.14f},
    {k128x128x2, 128, 128, 2.5f, 6.9f, 0.f, 1.15f}, {k128x64, 128, 64, 2.1f, 3.7f, 0.f, 1.25f},
    {k64x64x4, 64, 64, 1.7f, 2.1f, 0.f, 1.28f},     {k64x32x4, 64, 32, 0.8f, 1.6f, 0.f, 1.22f},
    {k128x32x4, 128, 32, 1.3f, 2.4f, 0.f, 1.33f},
};

// The same for rows_kernel with 17 to 32 tokens and with 33 to 64, for workgroups
// of one, two and four tiles of 16 weight rows: its time grows with the number of
// workgroups as well, `all` of them for 1024 of K, for all read the tokens from L2.
// Fitted to N = 512 to 28672, K = 4096 to 14336 (within 10 %). 6144 x 4096 with 32
// and 64 bf16 tokens takes 7.2 and 10.4 us where the best tile takes 11.3 and 11.6;
// 8-bit tokens 5.9 and 8.0 for 9.5 and 9.7. Larger products read their tokens too
// often (28672 x 4096 20 for 17 us).
struct FewCost {
  float start, one, all;
};
struct FewCosts {
  FewCost by1, by2;
  float start2, two;  // where a CU takes two of by2
  FewCost by4;        // an MXFP8 output
  float apart;
};
constexpr FewCosts kFew16[] = {
    {{0.6f, 0.48f, 0.0016f}, {1.7f, 0.4f, 0.0026f}, 2.f, 1.9f, {0.7f, 1.14f, 0.0042f}, 1.2f},
    {{1.7f, 0.72f, 0.003f}, {1.2f, 0.93f, 0.0032f}, 4.4f, 2.6f, {}, 1.2f}};
constexpr FewCosts kFew8[] = {
    {{0.7f, 0.49f, 0.0004f}, {0.f, 0.58f, 0.0016f}, 0.8f, 1.25f, {0.7f, 1.f, 0.0029f}, 1.35f},
    {{1.9f, 0.5f, 0.0016f}, {2.2f, 0.6f, 0.0018f}, 6.f, 1.f, {}, 1.35f}};

// The kernel and tile of the least cost, and in how many parts of K the tiles
// are computed. Parts cost a second kernel (3 us) and the way of their sums
// through memory.
Plan make_plan(int M, int N, int K, bool gated, bool act8, bool out8) {
  if (M <= 16) return {kRows, 1, 0};
  constexpr int kCus = kNumCU, kMostParts = 16;
  const int64_t rows = gated ? 2 * (int64_t)N : N;
  const int loads = ceil_div(K, 512);  // of scales; a part holds whole ones
  const bool odd = K % (act8 ? 128 : 64) != 0;
  Plan best{kRows, 1, 0};
  float least = -1.f;
  if (M <= (out8 ? 32 : 64)) {
    const FewCosts& f = (act8 ? kFew8 : kFew16)[M > 32];
    const int64_t pairs = ceil_div64(rows, 32), quads = ceil_div64(rows, 64);
    const float k = K / 1024.f * (odd ? f.apart : 1.f);
    auto cost = [&](const FewCost& c, int64_t all) { return c.start + (c.one + c.all * all) * k; };
    if (out8)
      least = ceil_div64(quads, kCus) * cost(f.by4, quads < kCus ? quads : kCus);
    else if (pairs < kFewPairs && !gated)
      least = cost(f.by1, 2 * pairs);
    else if (pairs <= kCus)
      least = cost(f.by2, pairs);
    else
      // a CU has room for more than two with 32 tokens, which evens out the end
      least = (M > 32 ? ceil_div64(pairs, 2 * kCus) : pairs > 2 * kCus ? pairs / (2.f * kCus) : 1.f) *
              (f.start2 + f.two * k);
  }
  const Cost* costs = !act8 ? kCosts16 : out8 ? kCosts8to8 : kCosts8;
  for (int i = 0; i < 7; ++i) {
    const Cost& c = costs[i];
    const int64_t tiles = ceil_div64(rows, c.rows) * ceil_div64(M, c.tokens);
    for (int parts = 1; parts <= kMostParts && parts <= loads; ++parts) {
      if (parts > 1 && tiles * parts > 2 * kCus) break;
      const float k = (parts > 1 ? 0.5f * ceil_div(loads, parts) : K / 1024.f) * (odd ? c.apart : 1.f);
      const int64_t each = ceil_div64(tiles * parts, kCus);  // workgroups of a CU
      float us = c.two > 0.f ? each / 2 * (c.start + c.two * k) + each % 2 * (c.start + c.one * k)
                             : each * (c.start + c.one * k);
      const int64_t floats = parts > 1 ? parts * tiles * c.rows * c.tokens : 0;
      if (parts > 1) us += 3.f + floats * 8 / 3e6f;
      if (least < 0.f || us < least) {
        least = us;
        best = {c.shape, parts, floats};
      }
    }
  }
  return best;
}

}  // namespace mx4
}  // namespace fi

// How many floats of workspace fi_gemm_mxfp4 wants for this product.
extern "C" int64_t fi_gemm_mxfp4_floats(int a_type, int out_type, int gated, int M, int N, int K) {
  using namespace fi::mx4;
  if (M <= 0 || N <= 0) return 0;
  return make_plan(M, N, K, gated, a_type == kFp8, out_type == kFp8).floats;
}

// Which kernel this product gets, and in how many parts of K over workgroups.
extern "C" const char* fi_gemm_mxfp4_plan(int a_type, int out_type, int gated, int M, int N,
                                          int K, int* parts) {
  using namespace fi::mx4;
  const Plan plan = make_plan(M, N, K, gated, a_type == kFp8, out_type == kFp8);
  *parts = plan.parts;
  switch (plan.shape) {
    case k256x128: return "256x128";
    case k128x128: return "128x128";
    case k128x128x2: return "128x128x2";
    case k128x64: return "128x64";
    case k64x64x4: return "64x64x4";
    case k64x32x4: return "64x32x4";
    case k128x32x4: return "128x32x4";
  }
  return "rows";
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
  const Plan plan = make_plan(M, N, K, gated, a_type == kFp8, out_type == kFp8);
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
