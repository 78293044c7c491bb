// The products of mx4_gemm.hip for at most 16 rows (single tokens, a few conversations): the quantization of x, the
// product and the gate in one launch.
//
// What bounds it: the weight's bytes, read once (17/32 a code), and a launch's latency: 1 x 2048 x 6144 in E4M3 takes 4.3 us
// replayed from a graph, where 1 x 1024 x 1024 takes 2.6 and the weight's bytes at the rate of a large copy 1.3.  A workgroup takes 16 weight rows (gate and up: 16 of each); its waves split K and add their sums
// through LDS.  One v_mfma_scale_f32_16x16x128 takes a 1 KB weight block as it lies in memory, 16 bytes a lane, with the
// tokens as the other operand's rows; rows past M repeat the last one.  Its operand of x needs no exchange in E2M1 (lane l
// holds a whole 32-block of token l % 16) and two lane swaps in E4M3 (each block lies in two lanes), so every wave
// quantizes what it multiplies, from registers, while its weight blocks are under way.
//
// thin_kernel does the same for 17 to 64 rows of a quantized operand (32 in E4M3), which lies in memory as the instruction
// takes it: up to four 16-row blocks of tokens for each weight block.  Tiles of 64 rows leave most CUs without work there:
// mx4_plan.h has both sides' times.  32 x 2048 x 12288 takes 8.5 us in E2M1 and 12.4 in E4M3; every workgroup reads all of x.
#include "abi_common.h"
#include "mx4_device.h"
#include "mx4_plan.h"

using namespace mx4;

namespace {

struct FewArgs {
  const void* x;
  int64_t ld_x;
  const uint8_t* b;
  const uint8_t* sb;
  int M, N, K, kt;  // K: columns of x; kt: K tiles of 128 of B
  void* c;
  int64_t ldc;
  const void* add;
  int64_t ld_add;
  int fn, vec_x, vec_c;
  const uint8_t* sx;
};

// 16 values of columns k.. of a row, zeros past K
template <int kT, bool kFull>
__device__ __forceinline__ void load16p(const typename Elem<kT>::T* row, int k, int K, bool vec, Group<kT>* w) {
  if (kFull || (vec && k + 16 <= K)) {
    w[0] = load_group<kT>(row + k);
    w[1] = load_group<kT>(row + k + 8);
  } else {
    w[0] = load_group_edge<kT>(row, k, K);
    w[1] = load_group_edge<kT>(row, k + 8, K);
  }
}

// The lane's operand of one K tile from its 32 values w (E2M1: columns 32 g ..; E4M3: 16 g .. and 64 + 16 g ..), and the
// scale byte that the instruction reads from this lane (32-block g of its token)
template <int kT, int kFmt>
__device__ __forceinline__ v8i operand(const Group<kT>* w, int g, uint32_t& scale) {
  const uint32_t a0 = max(w[0].absmax(), w[1].absmax()), a1 = max(w[2].absmax(), w[3].absmax());
  uint32_t p, q, e0, e1;
  if constexpr (kFmt == MXFP4_E4M3) {
    pair16(a0, p, q);
    e0 = block_exponent<kFmt>(max(p, q));  // block g / 2
    pair16(a1, p, q);
    e1 = block_exponent<kFmt>(max(p, q));  // block 2 + g / 2
    const uint32_t mine = e0 | (e1 << 8);
    pair32(mine, p, q);
    const uint32_t other = p ^ q ^ mine;  // lane l ^ 32: blocks of g ^ 2
    scale = g == 0 ? e0 : g == 1 ? other & 255u : g == 2 ? other >> 8 : e1;
  } else {
    e0 = e1 = scale = block_exponent<kFmt>(max(a0, a1));
  }
  v8i r = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t c[2];
    encode_group<kT, kFmt>(w[i], i < 2 ? e0 : e1, c);
    if constexpr (kFmt == MXFP4_E4M3) {
      r[2 * i] = (int)c[0];
      r[2 * i + 1] = (int)c[1];
    } else {
      r[i] = (int)c[0];
    }
  }
  return r;
}

// The weight rows of a workgroup: 16-row block `blk` of B, or half blk % 2 of gate block and up block blk / 2
template <bool kGated>
struct Rows {
  static constexpr int kB = kGated ? 2 : 1;
  const uint8_t* w[kB];  // this lane's 16 bytes and scale byte of K tile 0
  const uint8_t* s[kB];
  __device__ __forceinline__ Rows(const uint8_t* b, const uint8_t* sb, int64_t blk, int64_t kt, int r16, int g) {
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      const int64_t rb = kGated ? (blk >> 1) * 64 + (blk & 1) * 16 + 32 * i : blk * 16, r = rb + r16;
      w[i] = b + (rb >> 4) * kt * 1024 + (g >> 1) * 512 + r16 * 32 + (((g & 1) ^ (r16 >> 3)) << 4);
      s[i] = sb + (r >> 7) * kt * 512 + (r & 31) * 16 + ((r & 127) >> 5) * 4 + g;
    }
  }
};
__device__ __forceinline__ v8i operand4(uint4 v) { return v8i{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0}; }
template <int kFmt>
__device__ __forceinline__ v4f mma(v8i w, uint32_t ws, v8i x, uint32_t xs, v4f acc) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc, 4, kFmt == MXFP4_E4M3 ? 0 : 4, 0, (int)ws, 0, (int)xs);
}

// Sums of a 16 x 16 block (gate and up): lane l holds token l % 16 and, of weight rows 4 (l / 16) + 0..3 of the 16, four
// consecutive columns (the PI order)
template <int kT, bool kGated>
__device__ __forceinline__ void finish(const FewArgs& a, int64_t blk, int lane, int m, const f32x4* s) {
  typedef typename Elem<kT>::T T;
  const int g = lane >> 4;
  const int64_t c = (blk >> 1) * 32 + (g & 1) * 16 + (2 * (int)(blk & 1) + (g >> 1)) * 4;
  if (m >= a.M) return;
  float v[4], u[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    v[q] = s[0][q];
    if constexpr (kGated) {
      u[q] = s[1][q];
      if (a.add && c + q < a.N) {
        const T* ad = reinterpret_cast<const T*>(a.add) + m * a.ld_add;
        v[q] += Elem<kT>::get(ad[c + q]);
        u[q] += Elem<kT>::get(ad[a.N + c + q]);
      }
      v[q] = (a.fn == MXFP4_SILU ? gate_fn<MXFP4_SILU>(v[q]) : gate_fn<MXFP4_GELU>(v[q])) * u[q];
    }
  }
  store_run<kT, 4>(reinterpret_cast<T*>(a.c) + m * a.ldc, c, a.N, a.vec_c, v);
}

// How a wave comes by the 32 values a lane of a K tile: kEdge element by element where rows are not aligned to 16 bytes or end
// inside a tile; kDirect from memory; kStaged through LDS, from where a lane's 64 bytes cost no more than their banks (from
// memory they lie in other lines than its neighbours', 64 lines an instruction).
enum Source { kEdge, kDirect, kStaged };

template <int kT, int kFmt, bool kGated, int kWaves, int kSrc>
__global__ __launch_bounds__(64 * kWaves) void few_kernel(const FewArgs a) {
  typedef typename Elem<kT>::T T;
  constexpr int kB = kGated ? 2 : 1;
  __shared__ __attribute__((aligned(16))) f32x4 part[kWaves][kB][64];
  __shared__ __attribute__((aligned(16))) uint8_t stage[kSrc == kStaged ? kWaves * 4096 : 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const Rows<kGated> rows(a.b, a.sb, blockIdx.x, a.kt, r16, g);
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* xrow = x + (int64_t)min(r16, a.M - 1) * a.ld_x;
  const int k0 = kFmt == MXFP4_E4M3 ? 16 * g : 32 * g, k1 = kFmt == MXFP4_E4M3 ? 64 + 16 * g : 32 * g + 16;
  // kStaged: 16 rows of 256 bytes; DMA j brings rows 4 j .. 4 j + 3 (lane l row 4 j + l / 16, the 16-byte chunk at place l % 16),
  // chunk c of row r at place c ^ r, so that 16 rows' reads of one chunk meet every bank.  Rows past M repeat the last one.
  uint8_t* const mine = stage + (kSrc == kStaged ? wave * 4096 : 0);
  const T* src[4];
  if constexpr (kSrc == kStaged) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = 4 * j + g;
      src[j] = x + (int64_t)min(r, a.M - 1) * a.ld_x + ((r16 ^ r) * 8);
    }
  }
  v4f acc[kB];
#pragma unroll
  for (int i = 0; i < kB; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int t = wave; t < a.kt; t += kWaves) {  // wave w takes K tiles w, w + kWaves, ..
    uint4 w[kB];
    uint32_t ws[kB], xs;
    Group<kT> v[4];
    if constexpr (kSrc == kStaged) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        dma16(src[j] + t * 128, lds_addr(mine) + j * 1024);
    }
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      w[i] = *reinterpret_cast<const uint4*>(rows.w[i] + (int64_t)t * 1024);
      ws[i] = rows.s[i][(int64_t)t * 512];
    }
    if constexpr (kSrc == kStaged) {
      wait_vmcnt<0>();  // this wave's own rows
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = ((i < 2 ? k0 : k1) >> 3) + (i & 1);
        v[i].w = *reinterpret_cast<const uint4*>(mine + r16 * 256 + ((c ^ r16) << 4));
      }
    } else {
      load16p<kT, kSrc == kDirect>(xrow, t * 128 + k0, a.K, a.vec_x, v);
      load16p<kT, kSrc == kDirect>(xrow, t * 128 + k1, a.K, a.vec_x, v + 2);
    }
    const v8i xo = operand<kT, kFmt>(v, g, xs);
#pragma unroll
    for (int i = 0; i < kB; ++i) acc[i] = mma<kFmt>(operand4(w[i]), ws[i], xo, xs, acc[i]);
    if constexpr (kSrc == kStaged) {
      __builtin_amdgcn_s_waitcnt(0xc07f);  // its reads, before the next tile's rows come
      asm volatile("" ::: "memory");
    }
  }
#pragma unroll
  for (int i = 0; i < kB; ++i) part[wave][i][lane] = f32x4{acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
  __syncthreads();
  if (wave) return;
  f32x4 s[kB];
#pragma unroll
  for (int i = 0; i < kB; ++i) {
    s[i] = part[0][i][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) s[i] += part[w][i][lane];
  }
  finish<kT, kGated>(a, blockIdx.x, lane, r16, s);
}

// kTB blocks of 16 rows of a quantized operand (a.x its codes, a.sx its scales)
template <int kT, int kFmt, bool kGated, int kTB>
__global__ __launch_bounds__(512) void thin_kernel(const FewArgs a) {
  constexpr int kB = kGated ? 2 : 1, kWaves = 8, kA = kFmt == MXFP4_E4M3 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) f32x4 part[kWaves][kB][kTB][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const Rows<kGated> rows(a.b, a.sb, blockIdx.x, a.kt, r16, g);
  const uint8_t* xp[kTB];
  const uint8_t* xsp[kTB];
#pragma unroll
  for (int b = 0; b < kTB; ++b) {  // blocks past the rows re-read the last one and are not stored
    const int blk = min(b, (a.M - 1) >> 4), r = blk * 16 + r16;
    xp[b] = reinterpret_cast<const uint8_t*>(a.x) + (int64_t)blk * a.kt * (1024 * kA) +
            (kA == 2 ? r16 * 64 + ((g ^ (r16 >> 2)) << 4) : (g >> 1) * 512 + r16 * 32 + (((g & 1) ^ (r16 >> 3)) << 4));
    xsp[b] = a.sx + (r & 31) * 16 + (r >> 5) * 4 + g;
  }
  v4f acc[kB][kTB];
#pragma unroll
  for (int i = 0; i < kB; ++i)
#pragma unroll
    for (int b = 0; b < kTB; ++b) acc[i][b] = v4f{0.f, 0.f, 0.f, 0.f};
  const int per = (a.kt + kWaves - 1) / kWaves, t0 = wave * per, t1 = min(a.kt, t0 + per);
  for (int t = t0; t < t1; ++t) {
    uint4 w[kB], x[kTB][kA];
    uint32_t ws[kB], xs[kTB];
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      w[i] = *reinterpret_cast<const uint4*>(rows.w[i] + (int64_t)t * 1024);
      ws[i] = rows.s[i][(int64_t)t * 512];
    }
#pragma unroll
    for (int b = 0; b < kTB; ++b) {
#pragma unroll
      for (int h = 0; h < kA; ++h) x[b][h] = *reinterpret_cast<const uint4*>(xp[b] + ((int64_t)t * kA + h) * 1024);
      xs[b] = xsp[b][(int64_t)t * 512];
    }
#pragma unroll
    for (int b = 0; b < kTB; ++b) {
      v8i xo = operand4(x[b][0]);
      if constexpr (kA == 2) {
        xo[4] = (int)x[b][1].x;
        xo[5] = (int)x[b][1].y;
        xo[6] = (int)x[b][1].z;
        xo[7] = (int)x[b][1].w;
      }
#pragma unroll
      for (int i = 0; i < kB; ++i) acc[i][b] = mma<kFmt>(operand4(w[i]), ws[i], xo, xs[b], acc[i][b]);
    }
  }
#pragma unroll
  for (int i = 0; i < kB; ++i)
#pragma unroll
    for (int b = 0; b < kTB; ++b) part[wave][i][b][lane] = f32x4{acc[i][b][0], acc[i][b][1], acc[i][b][2], acc[i][b][3]};
  __syncthreads();
  if (wave >= kTB) return;
  f32x4 s[kB];
#pragma unroll
  for (int i = 0; i < kB; ++i) {
    s[i] = part[0][i][wave][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) s[i] += part[w][i][wave][lane];
  }
  finish<kT, kGated>(a, blockIdx.x, lane, wave * 16 + r16, s);
}

template <int kT, int kFmt, bool kGated>
void launch(const FewArgs& a, unsigned blocks, hipStream_t st) {
  // us, 8 / 16 waves: one row E4M3, (N, K) = (2048, 6144) 5.9 / 5.3, (4096, 12288) 10.9 / 9.1, (6144, 2048) 4.3 / 4.3, gated
  // 4.9 / 5.8.  Direct / staged: 16 rows E2M1, (2048, 6144) 8.6 / 5.3, (6144, 2048) 6.3 / 4.3; 8 rows 6.8 / 5.6 and 5.2 / 5.0; 3
  // rows 5.4 / 6.2 and 4.2 / 4.9.
  const bool full = a.vec_x && a.K % 128 == 0, many = a.kt >= 32;
  if (!full) few_kernel<kT, kFmt, kGated, 8, kEdge><<<blocks, 512, 0, st>>>(a);
  else if (a.M >= 8 && many) few_kernel<kT, kFmt, kGated, 16, kStaged><<<blocks, 1024, 0, st>>>(a);
  else if (a.M >= 8) few_kernel<kT, kFmt, kGated, 8, kStaged><<<blocks, 512, 0, st>>>(a);
  else if (many) few_kernel<kT, kFmt, kGated, 16, kDirect><<<blocks, 1024, 0, st>>>(a);
  else few_kernel<kT, kFmt, kGated, 8, kDirect><<<blocks, 512, 0, st>>>(a);
}

template <bool kGated>
int run(FewArgs& a, int64_t fmt, int64_t type, const char* what, hipStream_t st) {
  const int64_t blocks = ((int64_t)a.N + 31) / 32 * 2;
  a.kt = (a.K + 127) / 128;
  a.vec_x = mx_aligned(a.x, 16) && a.ld_x % 8 == 0;
  a.vec_c = mx_aligned(a.c, 8) && a.ldc % 4 == 0;
  const bool f8 = fmt == MXFP4_E4M3;
  if (type == MXFP4_BF16)
    f8 ? launch<MXFP4_BF16, MXFP4_E4M3, kGated>(a, (unsigned)blocks, st) : launch<MXFP4_BF16, MXFP4_E2M1, kGated>(a, (unsigned)blocks, st);
  else
    f8 ? launch<MXFP4_F16, MXFP4_E4M3, kGated>(a, (unsigned)blocks, st) : launch<MXFP4_F16, MXFP4_E2M1, kGated>(a, (unsigned)blocks, st);
  MX_CHECK_LAUNCH(what);
  return MXFP8_OK;
}

template <int kT, int kFmt, bool kGated>
void launch_thin(const FewArgs& a, unsigned blocks, hipStream_t st) {
  if (kFmt == MXFP4_E4M3 || a.M <= 32) thin_kernel<kT, kFmt, kGated, 2><<<blocks, 512, 0, st>>>(a);  // 32 rows at most in E4M3
  else thin_kernel<kT, kFmt, kGated, kFmt == MXFP4_E4M3 ? 2 : 4><<<blocks, 512, 0, st>>>(a);
}
template <bool kGated>
void run_thin(const FewArgs& a, int64_t fmt, int64_t type, hipStream_t st) {
  const unsigned blocks = (unsigned)(((int64_t)a.N + 31) / 32 * 2);
  const bool f8 = fmt == MXFP4_E4M3;
  if (type == MXFP4_BF16)
    f8 ? launch_thin<MXFP4_BF16, MXFP4_E4M3, kGated>(a, blocks, st) : launch_thin<MXFP4_BF16, MXFP4_E2M1, kGated>(a, blocks, st);
  else
    f8 ? launch_thin<MXFP4_F16, MXFP4_E4M3, kGated>(a, blocks, st) : launch_thin<MXFP4_F16, MXFP4_E2M1, kGated>(a, blocks, st);
}

int check(const char* what, const void* x, int64_t ld_x, int64_t fmt, const void* b, const void* sb, int64_t M, int64_t N,
          int64_t K, const void* c, int64_t ldc, int64_t type) {
  MX_CHECK_ARG(M >= 0 && M <= MXFP4_FEW_ROWS && N > 0 && N < (1LL << 29) && K > 0 && K < (1LL << 26),
               "%s: bad shape (M=%lld N=%lld K=%lld; at most %d rows)", what, (long long)M, (long long)N, (long long)K,
               MXFP4_FEW_ROWS);
  MX_CHECK_ARG(fmt == MXFP4_E2M1 || fmt == MXFP4_E4M3, "%s: unknown format %lld", what, (long long)fmt);
  MX_CHECK_ARG(type == MXFP4_BF16 || type == MXFP4_F16, "%s: bf16 or f16 (type %lld)", what, (long long)type);
  if (M == 0) return MXFP8_OK;
  MX_CHECK_ARG(x && b && sb && c && ld_x >= 0 && ldc >= N, "%s: null pointer or bad stride", what);
  MX_CHECK_ARG(mx_aligned(x, 2) && mx_aligned(b, 16) && mx_aligned(sb, 16) && mx_aligned(c, 2), "%s: misaligned buffer",
               what);
  return MXFP8_OK;
}

}  // namespace

// mx4_gemm.hip's call for kMx4ThinRows rows at most (mx4_plan.h), its arguments checked there
void mx4_thin(bool gated, const void* q, const void* sq, int64_t fmt, const void* b, const void* sb, int M, int N, int kt,
              const void* add, int64_t ld_add, int fn, void* c, int64_t ldc, int64_t type, hipStream_t st) {
  const FewArgs a{q, 0, (const uint8_t*)b, (const uint8_t*)sb, M, N, kt * 128, kt, c, ldc, add, ld_add, fn, 0,
                  mx_aligned(c, 8) && ldc % 4 == 0, (const uint8_t*)sq};
  gated ? run_thin<true>(a, fmt, type, st) : run_thin<false>(a, fmt, type, st);
}

extern "C" int mxfp4_few(const void* x, int64_t ld_x, int64_t fmt, const void* b, const void* sb, int64_t M, int64_t N,
                         int64_t K, void* c, int64_t ldc, int64_t type, void* stream) {
  if (int rc = check("mxfp4_few", x, ld_x, fmt, b, sb, M, N, K, c, ldc, type)) return rc;
  if (M == 0) return MXFP8_OK;
  FewArgs a{x, ld_x, (const uint8_t*)b, (const uint8_t*)sb, (int)M, (int)N, (int)K, 0, c, ldc, nullptr, 0, 0, 0, 0, nullptr};
  return run<false>(a, fmt, type, "mxfp4_few", (hipStream_t)stream);
}

extern "C" int mxfp4_few_gated(const void* x, int64_t ld_x, int64_t fmt, const void* b, const void* sb, int64_t M,
                               int64_t N, int64_t K, const void* add, int64_t ld_add, int64_t fn, void* h, int64_t ldh,
                               int64_t type, void* stream) {
  if (int rc = check("mxfp4_few_gated", x, ld_x, fmt, b, sb, M, N, K, h, ldh, type)) return rc;
  MX_CHECK_ARG(fn == MXFP4_SILU || fn == MXFP4_GELU, "mxfp4_few_gated: unknown gate function %lld", (long long)fn);
  MX_CHECK_ARG(!add || ((ld_add == 0 || ld_add >= 2 * N) && mx_aligned(add, 2)), "mxfp4_few_gated: bad addend");
  if (M == 0) return MXFP8_OK;
  FewArgs a{x, ld_x, (const uint8_t*)b, (const uint8_t*)sb, (int)M, (int)N, (int)K, 0, h, ldh, add, ld_add, (int)fn, 0, 0, nullptr};
  return run<true>(a, fmt, type, "mxfp4_few_gated", (hipStream_t)stream);
}
