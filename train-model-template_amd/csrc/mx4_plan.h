// Which workgroup shape a product of mx4_gemm.hip takes: host code without HIP.
#pragma once

#include <stdint.h>

#include <algorithm>

enum Mx4Shape { kMx4Tall, kMx4Mid, kMx4Low, kMx4Mini, kMx4Thin };
constexpr int kMx4ThinRows = 64;

// Estimated us of a launch of bm x bn tiles: with w = tiles a CU and rounds = ceil(w),
//   K tiles * (step * rounds + fill * w) + round * rounds + tile * w + base,
// fitted to 8 pairs (N, K) of 1024 to 12288 at 16 values of M from 32 to 14000, with a residual of 3-5% (standard
// deviation); over those the shape it picks takes 0.2% longer than the fastest one on average and 13% at the worst (5.3 us in
// place of 4.7).
struct Mx4Cost {
  int bm, bn;
  float step, fill, round, tile, base;
};
constexpr Mx4Cost kMx4CostE2m1[] = {{256, 128, 0.2893f, 0.1238f, 0.0000f, 3.2269f, 4.5370f},
                                    {128, 128, 0.1639f, 0.0698f, 0.3720f, 1.4199f, 3.5333f},
                                    {64, 128, 0.1319f, 0.0224f, 0.1588f, 0.7602f, 3.3331f},
                                    {64, 64, 0.1038f, 0.0000f, 0.2848f, 0.1300f, 3.3781f}};
constexpr Mx4Cost kMx4CostE4m3[] = {{256, 128, 0.5267f, 0.1732f, 0.0000f, 2.4730f, 4.7675f},
                                    {128, 128, 0.2673f, 0.0888f, 0.2432f, 1.3708f, 3.6692f},
                                    {64, 128, 0.1571f, 0.0614f, 0.7333f, 0.2474f, 2.9373f},
                                    {64, 64, 0.1465f, 0.0120f, 0.1349f, 0.2506f, 3.1320f}};

// gated: gate and up blocks lie beside each other in a wave's columns, which kMx4Mini's waves have no room for.
// thin: the launch can take mx4_few.hip's kernel for few rows (16-bit output, weight rows in the PI order, nothing saved).
// It splits K over a workgroup's waves and has a workgroup for every 16 weight rows, so it pays where the tiles' chain along
// K is long and the weight has few rows: us, tiles / Thin, at 32 rows (N, K) = (2048, 12288) E2M1 14.5 / 8.5, E4M3 17.8 / 12.4,
// (2048, 2048) 5.3 / 4.4 and 5.9 / 4.6, (12288, 2048) 5.3 / 6.0 and 5.7 / 7.9; at 64 rows (2048, 12288) 14.6 / 12.8 and
// 18.0 / 20.6, (2048, 2048) 5.0 / 4.8 and 5.7 / 5.9.
inline Mx4Shape mx4_shape(int64_t M, int64_t rows_b, int64_t kt, bool e4m3, bool gated, bool thin, int cus) {
  if (thin && M <= (e4m3 ? kMx4ThinRows / 2 : kMx4ThinRows) && kt * 128 >= rows_b) return kMx4Thin;
  int best = kMx4Low;
  float t = 0.f;
  for (int s : {kMx4Low, kMx4Mini, kMx4Mid, kMx4Tall}) {
    if (gated && s == kMx4Mini) continue;
    const Mx4Cost& c = (e4m3 ? kMx4CostE4m3 : kMx4CostE2m1)[s];
    const int64_t tiles = (M + c.bm - 1) / c.bm * ((rows_b + c.bn - 1) / c.bn);
    const float w = (float)tiles / cus, rounds = (float)((tiles + cus - 1) / cus);
    const float e = kt * (c.step * rounds + c.fill * w) + c.round * rounds + c.tile * w + c.base;
    if (s == kMx4Low || e < t) {
      best = s;
      t = e;
    }
  }
  return (Mx4Shape)best;
}
