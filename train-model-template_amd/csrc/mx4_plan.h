// Which workgroup shape a product of mx4_gemm.hip takes: host code without HIP.
#pragma once

#include <stdint.h>

#include <algorithm>

enum Mx4Shape { kMx4Tall, kMx4Mid, kMx4Low, kMx4Thin };
constexpr int kMx4ThinRows = 64;

// Estimated us of a launch: with w = tiles a CU and rounds = ceil(w),
//   K tiles * (step * rounds + fill * w) + round * rounds + tile * w + base,
// fitted to 8 pairs (N, K) of 1024 to 12288 at 16 values of M from 32 to 14000, with a residual of 3-5% (standard
// deviation); over those the shape it picks takes 0.25% longer than the fastest one on average and 9% at the worst.
struct Mx4Cost {
  int bm;
  float step, fill, round, tile, base;
};
constexpr Mx4Cost kMx4CostE2m1[] = {{256, 0.2841f, 0.1367f, 0.2708f, 2.5179f, 4.4244f},
                                    {128, 0.1980f, 0.0471f, 0.6062f, 0.9878f, 3.5385f},
                                    {64, 0.1510f, 0.0068f, 0.0606f, 0.6905f, 3.9037f}};
constexpr Mx4Cost kMx4CostE4m3[] = {{256, 0.5079f, 0.1863f, 0.0f, 2.2064f, 4.7846f},
                                    {128, 0.2812f, 0.0811f, 0.7647f, 0.7549f, 3.4232f},
                                    {64, 0.2008f, 0.0213f, 0.5641f, 0.3903f, 3.1069f}};

// thin: the launch can take mx4_few.hip's kernel for few rows (16-bit output, weight rows in the PI order, nothing saved).
// It splits K over a workgroup's waves and has a workgroup for every 16 weight rows: us, Low / Thin, at 32 rows E4M3
// (N, K) = (2048, 6144) 13.0 / 7.4, (2048, 12288) 23.0 / 12.2, (6144, 2048) 7.2 / 6.5, (12288, 2048) 7.3 / 7.9; at 64 rows
// (2048, 6144) 13.3 / 11.7, (2048, 2048) 6.9 / 6.5, (6144, 2048) 7.0 / 9.4: it pays where K is no shorter than N.
inline Mx4Shape mx4_shape(int64_t M, int64_t rows_b, int64_t kt, bool e4m3, bool thin, int cus) {
  if (thin && M <= kMx4ThinRows && (kt * 128 >= rows_b || (M <= 32 && rows_b <= 8192))) return kMx4Thin;
  int best = kMx4Low;
  float t = 0.f;
  for (int s : {kMx4Low, kMx4Mid, kMx4Tall}) {
    const Mx4Cost& c = (e4m3 ? kMx4CostE4m3 : kMx4CostE2m1)[s];
    const int64_t tiles = (M + c.bm - 1) / c.bm * ((rows_b + 127) / 128);
    const float w = (float)tiles / cus, rounds = (float)((tiles + cus - 1) / cus);
    const float e = kt * (c.step * rounds + c.fill * w) + c.round * rounds + c.tile * w + c.base;
    if (s == kMx4Low || e < t) {
      best = s;
      t = e;
    }
  }
  return (Mx4Shape)best;
}
