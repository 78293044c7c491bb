// Products of MX operands with MXFP4 weights for gfx950: C[M, N] = A[M, K] . B[N, K]^T, B in E2M1, A in E2M1 or E4M3, fp32
// sums on v_mfma_scale_f32_32x32x64_f8f6f4; and the gated block, whose epilogue takes [g | u] of the same tile and writes
// h = fn(g) u.
//
// A workgroup computes a kBM x kBN tile with kWM x kWN waves, each kMB x kNB blocks of 32 x 32.  Operands come straight
// from memory into a ring of LDS stages (global_load_lds) of kKS matrix steps of 64 codes: the 1 KB blocks of the tiled
// layouts, which are the LDS image already, and the 512-byte scale tiles of the K tile.  A step's LDS reads and DMAs stand
// between its matrix instructions; the fragments are read a step ahead of their use, or a whole K tile (kDeep) where
// registers allow.
// The matrix instruction takes B's fragment first, so a lane's accumulators are one row m and, with B's rows in the PI
// order, 16 contiguous columns.
//
// What bounds it (times from kernel traces of whole training steps, from box to box).  Large products: in E4M3 the matrix
// pipe, busy 59-64% of cycles at a clock that the power limit holds at 1.9 GHz (10752 x 2048 x 12288 228-245 us, 2.2-2.4
// PFLOP/s); in E2M1, at 3.0-3.5 PFLOP/s (10752 x 2048 x 6144 77-80 us, x 6144 x 2048 85-90), the pipe is busy 36-44% at 2.0 GHz
// and no other unit more (LDS 17-20%, reads of 340 cycles, 80% of them from L2): waves wait to issue, and a tile's fill and
// epilogue are 3 of its 10 us at K = 2048.  Small ones: the chain of a tile's K tiles, 0.10 (E2M1) to 0.15 us (E4M3) each.
#include <algorithm>
#include <type_traits>

#include "abi_common.h"
#include "mx4_device.h"
#include "mx4_plan.h"

using namespace mx4;

void mx4_thin(bool gated, const void* q, const void* sq, int64_t fmt, const void* b, const void* sb, int M, int N, int kt,
              const void* add, int64_t ld_add, int fn, void* c, int64_t ldc, int64_t type, hipStream_t st);  // mx4_few.hip

namespace {

template <int kAF_, int kMB_, int kNB_, int kWM_, int kWN_, int kKS_, int kStages_>
struct Shape {
  static constexpr int kAF = kAF_, kMB = kMB_, kNB = kNB_, kWM = kWM_, kWN = kWN_, kKS = kKS_, kStages = kStages_;
  static constexpr bool kDeep = kMB * kNB <= 4;  // registers for a whole K tile's fragments ahead
  static constexpr int kWaves = kWM * kWN, kThreads = 64 * kWaves;
  static constexpr int kBM = 32 * kMB * kWM, kBN = 32 * kNB * kWN;
  static constexpr int kGroupM = 1024 / kBM;                                      // M-tiles of a tile group
  static constexpr int kTilesA = (kBM + 127) / 128, kTilesB = (kBN + 127) / 128;  // scale tiles of a stage
  static constexpr int kRowA = kAF == MXFP4_E4M3 ? 64 : 32, kRowB = 32;           // bytes of 64 codes of a row
  static constexpr int kBytesA = kBM * kRowA * kKS, kBytesB = kBN * kRowB * kKS;
  static constexpr int kOffB = kBytesA, kOffS = kOffB + kBytesB, kOffSB = kOffS + kTilesA * 512;
  static constexpr int kStageBytes = kOffS + (kTilesA + kTilesB) * 512;
  // DMAs of a wave and stage: 1 KB slices of A and B, 256-byte pieces of the scale tiles (a wave past the last piece
  // repeats it), the same number for every wave, so that one vmcnt bounds a stage
  static constexpr int kSA = kBytesA / 1024 / kWaves, kSB = kBytesB / 1024 / kWaves;
  static constexpr int kPieces = (kTilesA + kTilesB) * 2, kSS = (kPieces + kWaves - 1) / kWaves;
  static constexpr int kDma = kSA + kSB + kSS;
  static constexpr int kRing = kStages * kStageBytes;
  static_assert(kSA * kWaves * 1024 == kBytesA && kSB * kWaves * 1024 == kBytesB && kRing <= 80 * 1024, "shape");
};

struct GemmArgs {
  const uint8_t* a;
  const uint8_t* sa;
  const uint8_t* b;
  const uint8_t* sb;
  int M, N, rows_b;  // rows_b: rows of B's operand (2 ceil(N / 32) 32 for the gated block)
  int kt;            // K tiles of 128
  int tm, tn, per;   // tiles along M and N; tiles an XCD
  void* c;           // C, or h of the gated block
  int64_t ldc;
  int type, b_pi, vec;
  const void* add;  // gated block: addend of [g | u], the saved [g | u]
  int64_t ld_add;
  void* gu;
  int fn, add_vec;
};

enum Epi { kPlain, kGated };

// The tile of this workgroup.  Workgroup i runs on XCD i % 8; each XCD takes a contiguous range of tiles in groups of 1024
// rows, M fastest, so that the tiles of an XCD share panels of A and B in its L2.
template <class S>
__device__ __forceinline__ bool tile_of(const GemmArgs& g, int& mt, int& nt) {
  const int j = blockIdx.x >> 3, t = (blockIdx.x & 7) * g.per + j;
  if (j >= g.per || t >= g.tm * g.tn) return false;
  const int grp = t / (S::kGroupM * g.tn), r = t - grp * (S::kGroupM * g.tn);
  const int rows = min(S::kGroupM, g.tm - grp * S::kGroupM);
  mt = grp * S::kGroupM + r % rows;
  nt = r / rows;
  return true;
}

template <int n>
__device__ __forceinline__ void read_words(const uint8_t* p, uint32_t* w) {
  if constexpr (n == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (n == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

__device__ __forceinline__ v8i frag4(const uint8_t* p) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  return v8i{(int)u.x, (int)u.y, (int)u.z, (int)u.w, 0, 0, 0, 0};
}
__device__ __forceinline__ v8i frag8(const uint8_t* lo, const uint8_t* hi) {
  const uint4 a = *reinterpret_cast<const uint4*>(lo), b = *reinterpret_cast<const uint4*>(hi);
  return v8i{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

// A bare barrier (a fence would wait for every DMA) that no LDS access is moved across
__device__ __forceinline__ void stage_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---- epilogues
template <class S, int kT>
__device__ __forceinline__ void store_plain(const GemmArgs& g, int m0, int n0, int lane, const v16f (*acc)[S::kMB]) {
  typedef typename Elem<kT>::T T;
#pragma unroll
  for (int nt = 0; nt < S::kNB; ++nt)
#pragma unroll
    for (int mt = 0; mt < S::kMB; ++mt) {
      const int m = m0 + mt * 32 + (lane & 31), nb = n0 + nt * 32;
      if (nb >= g.N) continue;
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = acc[nt][mt][i];
      if (g.b_pi) {
        store_block<kT>(reinterpret_cast<T*>(g.c), g.ldc, m0 + mt * 32, g.M, nb, g.N, g.vec, lane, v);
      } else if (m < g.M) {
        T* row = reinterpret_cast<T*>(g.c) + (int64_t)m * g.ldc;
#pragma unroll
        for (int q = 0; q < 4; ++q) store_run<kT, 4>(row, nb + q * 8 + (lane >> 5) * 4, g.N, g.vec, v + 4 * q);
      }
    }
}

template <int kT>
__device__ __forceinline__ void load_run16(const void* base, int64_t off, int64_t c, int64_t cols, bool vec, float* v) {
  const typename Elem<kT>::T* p = reinterpret_cast<const typename Elem<kT>::T*>(base) + off + c;
  if (vec && c + 16 <= cols) {
    load8<kT>(p, v);
    load8<kT>(p + 8, v + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = c + i < cols ? Elem<kT>::get(p[i]) : 0.f;
  }
}

template <int kT>
__device__ __forceinline__ void store_nt8(typename Elem<kT>::T* p, const float* f) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = f[i];
  store_codes<true>(reinterpret_cast<uint8_t*>(p), make_uint4(round2<kT>(v[0], v[1]), round2<kT>(v[2], v[3]),
                                                              round2<kT>(v[4], v[5]), round2<kT>(v[6], v[7])));
}

template <class S, int kT, int kFn>
__device__ __forceinline__ void store_gated(const GemmArgs& g, int m0, int n0, int lane, const v16f (*acc)[S::kMB]) {
  typedef typename Elem<kT>::T T;
  const int64_t nblk = (g.N + 31) / 32;
#pragma unroll
  for (int p = 0; p < S::kNB / 2; ++p)
#pragma unroll
    for (int mt = 0; mt < S::kMB; ++mt) {
      // rows past the last one compute the last one's and are not stored
      const int m = min(m0 + mt * 32 + (lane & 31), g.M - 1), c0 = (n0 >> 1) + p * 32;
      const int c = c0 + (lane >> 5) * 16;  // the lane's first gate and up column
      if (c0 >= g.N) continue;
      float gv[16], uv[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        gv[i] = acc[2 * p][mt][i];
        uv[i] = acc[2 * p + 1][mt][i];
      }
      if (g.add) {
        float t[16];
        load_run16<kT>(g.add, (int64_t)m * g.ld_add, c, g.N, g.add_vec, t);
#pragma unroll
        for (int i = 0; i < 16; ++i) gv[i] += t[i];
        load_run16<kT>(g.add, (int64_t)m * g.ld_add + g.N, c, g.N, g.add_vec, t);
#pragma unroll
        for (int i = 0; i < 16; ++i) uv[i] += t[i];
      }
      if (g.gu && m0 + mt * 32 + (lane & 31) < g.M) {
        T* s = reinterpret_cast<T*>(g.gu) + saved_offset(m, c, nblk);
        // read again by the backward pass alone: past the caches, which keep h
        store_nt8<kT>(s, gv);
        store_nt8<kT>(s + 512, gv + 8);
        store_nt8<kT>(s + 1024, uv);
        store_nt8<kT>(s + 1536, uv + 8);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) gv[i] = gate_fn<kFn>(gv[i]) * uv[i];
      store_block<kT>(reinterpret_cast<T*>(g.c), g.ldc, m0 + mt * 32, g.M, c0, g.N, g.vec, lane, gv);
    }
}

// ---- the kernel
template <class S, int kEpi>
__global__ __launch_bounds__(S::kThreads) __attribute__((amdgpu_waves_per_eu(2)))
void gemm_kernel(const GemmArgs g) {
  constexpr int kMB = S::kMB, kNB = S::kNB;
  __shared__ __attribute__((aligned(16))) uint8_t lds[S::kRing];
  int mt_, nt_;
  if (!tile_of<S>(g, mt_, nt_)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave / S::kWM, wm = wave % S::kWM;
  const int m0 = mt_ * S::kBM, n0 = nt_ * S::kBN, kt = g.kt;

  // this wave's slices of a stage.  E4M3: a slice is a block of 16 rows x 64 codes (two halves of a K tile: first all rows
  // of one, then of the other).  E2M1: a block of 16 rows x 128 codes, or with stages of 64 codes the halves of two blocks.
  const int last_a = ((g.M + 31) >> 5) * 2 - 1, last_b = ((g.rows_b + 31) >> 5) * 2 - 1;  // last row block of 16
  constexpr int kRowsA = S::kBM / 16;
  auto slice4 = [&](int r0, int sl, int last_rb) -> uint32_t {
    if constexpr (S::kKS == 2) return (uint32_t)((min((r0 >> 4) + sl, last_rb) - (r0 >> 4)) * kt * 1024) + lane * 16;
    return (uint32_t)((min((r0 >> 4) + 2 * sl + (lane >> 5), last_rb) - (r0 >> 4)) * kt * 1024) + (lane & 31) * 16;
  };
  constexpr int kBlkA = S::kAF == MXFP4_E4M3 ? 2048 : 1024;     // bytes of a 16-row K tile
  constexpr int kStepA = kBlkA * S::kKS / 2, kStepB = 512 * S::kKS;  // of a stage
  const uint8_t* ga = g.a + (int64_t)(m0 >> 4) * kt * kBlkA;
  const uint8_t* gb = g.b + (int64_t)(n0 >> 4) * kt * 1024;
  uint32_t oa[S::kSA], ob[S::kSB];
#pragma unroll
  for (int j = 0; j < S::kSA; ++j) {
    const int sl = wave * S::kSA + j;
    if constexpr (S::kAF == MXFP4_E4M3) {
      const int half = sl / kRowsA, rb = min((m0 >> 4) + sl % kRowsA, last_a) - (m0 >> 4);
      oa[j] = (uint32_t)(rb * kt * 2048 + half * 1024) + lane * 16;
    } else {
      oa[j] = slice4(m0, sl, last_a);
    }
  }
#pragma unroll
  for (int j = 0; j < S::kSB; ++j) ob[j] = slice4(n0, wave * S::kSB + j, last_b);
  const uint8_t* gsp[S::kSS];
  int so[S::kSS];
#pragma unroll
  for (int j = 0; j < S::kSS; ++j) {
    const int pc = min(wave * S::kSS + j, S::kPieces - 1), ti = pc >> 1;
    const bool is_a = ti < S::kTilesA;
    const int rt = is_a ? min((m0 >> 7) + ti, (g.M - 1) >> 7) : min((n0 >> 7) + ti - S::kTilesA, (g.rows_b - 1) >> 7);
    gsp[j] = (is_a ? g.sa : g.sb) + (int64_t)rt * kt * 512 + (pc & 1) * 256;
    so[j] = S::kOffS + pc * 256;
  }
  const uint32_t lds0 = lds_addr(lds);
  const int last = (S::kKS == 2 ? kt : 2 * kt) - 1;  // stage
  auto dma = [&](int s, int slot, int d) {  // DMA d of stage s into ring slot `slot`
    const uint32_t st = lds0 + slot * S::kStageBytes;
    if (d < S::kSA)
      dma16_at(ga + (int64_t)s * kStepA, oa[d], st + (wave * S::kSA + d) * 1024);
    else if (d < S::kSA + S::kSB)
      dma16_at(gb + (int64_t)s * kStepB, ob[d - S::kSA], st + S::kOffB + (wave * S::kSB + d - S::kSA) * 1024);
    else
      dma4_at(gsp[d - S::kSA - S::kSB] + (int64_t)(S::kKS == 2 ? s : s >> 1) * 512, lane * 4,
              st + so[d - S::kSA - S::kSB]);
  };

  v16f acc[kNB][kMB];
#pragma unroll
  for (int i = 0; i < kNB; ++i)
#pragma unroll
    for (int j = 0; j < kMB; ++j) acc[i][j] = v16f{};

  const int rl = lane & 31, hi = lane >> 5, sshift = hi * 8;
  const int rwa = (S::kBM < 128 ? m0 & 127 : 0) + wm * 32 * kMB, rwb = (S::kBN < 128 ? n0 & 127 : 0) + wn * 32 * kNB;
  const int sao = S::kOffS + (rwa >> 7) * 512 + rl * 16 + ((rwa >> 5) & 3) * 4;
  const int sbo = S::kOffSB + (rwb >> 7) * 512 + rl * 16 + ((rwb >> 5) & 3) * 4;
  struct Frags {
    v8i a[kMB], b[kNB];
  };
  uint32_t sca[kMB], scb[kNB], sna[kMB], snb[kNB];  // scale words of this K tile and the next
  constexpr int kReads = kMB + kNB, kMfma = kMB * kNB;
  auto read_scales = [&](int slot) {
    const uint8_t* st = lds + slot * S::kStageBytes;
    read_words<kMB>(st + sao, sna);
    read_words<kNB>(st + sbo, snb);
  };
  auto take_scales = [&] {
#pragma unroll
    for (int i = 0; i < kMB; ++i) sca[i] = sna[i] >> sshift;
#pragma unroll
    for (int i = 0; i < kNB; ++i) scb[i] = snb[i] >> sshift;
  };
  // E2M1: 16 bytes of a row, chunk hi at its place; E4M3: chunks hi and hi + 2 at theirs (tiled_offset in mx_device.h)
  const int c4 = (hi ^ ((rl >> 3) & 1)) << 4, c8 = (hi ^ ((rl >> 2) & 3)) << 4;
  auto row4 = [&](int row0, int half) {  // of row row0 + rl, row0 a multiple of 32
    return ((row0 + rl) >> 4) * (512 * S::kKS) + half * 512 + (rl & 15) * 32 + c4;
  };
  auto read_frag = [&](int slot, int half, Frags& f, int r) {
    const uint8_t* st = lds + slot * S::kStageBytes;
    if (r < kMB) {
      const int row0 = (wm * kMB + r) * 32;
      if constexpr (S::kAF == MXFP4_E4M3) {
        const uint8_t* p = st + half * (S::kBM * 64) + (row0 + rl) * 64;
        f.a[r] = frag8(p + c8, p + (c8 ^ 32));
      } else {
        f.a[r] = frag4(st + row4(row0, half));
      }
    } else {
      f.b[r - kMB] = frag4(st + S::kOffB + row4((wn * kNB + r - kMB) * 32, half));
    }
  };
  auto mma = [&](const Frags& f, int x, auto half) {  // serpentine: one operand stays from each product to the next
    const int j = x / kNB, i = (j & 1) ? kNB - 1 - x % kNB : x % kNB;
    constexpr int kA = S::kAF == MXFP4_E4M3 ? 0 : 4, kOp = 2 * decltype(half)::value;
    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(f.b[i], f.a[j], acc[i][j], 4, kA, kOp, (int)scb[i], kOp,
                                                                (int)sca[j]);
  };
  // One step: this step's products with, between them, the reads of the next step's fragments and this step's share of
  // the DMAs that refill the ring slot freed at the last barrier.
  constexpr int kD0 = (S::kDma + 1) / 2;  // DMAs of the second step of a K tile; the rest in the first of the next
  auto step = [&](const Frags& cur, Frags& nxt, int rslot, int rhalf, int ds, int dslot, int d0, int d1, auto half) {
#pragma unroll
    for (int x = 0; x < kMfma; ++x) {
      constexpr int kOver = kMfma > 1 ? kMfma - 1 : 1;
#pragma unroll
      for (int r = 0; r < kReads; ++r)
        if (r * kOver / kReads == x) read_frag(rslot, rhalf, nxt, r);
#pragma unroll
      for (int d = 0; d < S::kDma; ++d)
        if (d >= d0 && d < d1 && (d - d0) * kOver / (d1 - d0) == x) dma(ds, dslot, d);
      mma(cur, x, half);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using H0 = std::integral_constant<int, 0>;
  using H1 = std::integral_constant<int, 1>;

  int slot = 0;  // ring slot of the stage at hand
  if constexpr (S::kDeep) {
    // The fragments of a whole K tile are read while the products of the one before run, so the LDS's latency is paid beside
    // them.  At the barrier of tile s every wave has read tile s, whose slot takes tile s + kStages.
    struct Tile {
      Frags f[2];
      uint32_t sa[kMB], sb[kNB];
    };
    Tile t0, t1;
    auto read_tile = [&](int sl, Tile& t, int r) {
      if (r == 0) {
        read_words<kMB>(lds + sl * S::kStageBytes + sao, t.sa);
        read_words<kNB>(lds + sl * S::kStageBytes + sbo, t.sb);
      }
      read_frag(sl, r / kReads, t.f[r / kReads], r % kReads);
    };
#pragma unroll
    for (int q = 0; q < S::kStages; ++q)
#pragma unroll
      for (int d = 0; d < S::kDma; ++d) dma(min(q, last), q, d);
    wait_vmcnt<(S::kStages - 1) * S::kDma>();
    stage_barrier();
#pragma unroll
    for (int r = 0; r < 2 * kReads; ++r) read_tile(0, t0, r);
    auto one = [&](int s, Tile& cur, Tile& nxt) {
      wait_vmcnt<(S::kStages - 2) * S::kDma>();
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's reads of tile s are in registers
      stage_barrier();
      const int old = slot;
      slot = slot + 1 == S::kStages ? 0 : slot + 1;
#pragma unroll
      for (int i = 0; i < kMB; ++i) sca[i] = cur.sa[i] >> sshift;
#pragma unroll
      for (int i = 0; i < kNB; ++i) scb[i] = cur.sb[i] >> sshift;
      constexpr int kAll = 2 * kMfma, kOver = kAll - 1;
#pragma unroll
      for (int x = 0; x < kAll; ++x) {
        if (x < kMfma) mma(cur.f[0], x, H0{});
        else mma(cur.f[1], x - kMfma, H1{});
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 2 * kReads; ++r)
          if (r * kOver / (2 * kReads) == x) read_tile(slot, nxt, r);
#pragma unroll
        for (int d = 0; d < S::kDma; ++d)
          if (d * kOver / S::kDma == x) dma(min(s + S::kStages, last), old, d);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    int s = 0;
    for (; s < last; s += 2) {
      one(s, t0, t1);
      one(s + 1, t1, t0);
    }
    if (s == last) one(s, t0, t1);
  } else if constexpr (S::kKS == 2) {
    // K tile s frees its ring slot at the barrier in its second half; that half and the first half of tile s + 1 refill it
    // with tile s + kStages.  So the ring starts with the second part of its last stage still to come.  Tiles past the end
    // re-load the last one into slots that nothing reads any more: the number in flight is the same at every wait.
#pragma unroll
    for (int q = 0; q < S::kStages; ++q)
#pragma unroll
      for (int d = 0; d < (q + 1 < S::kStages ? S::kDma : kD0); ++d) dma(min(q, last), q, d);
    wait_vmcnt<(S::kStages - 2) * S::kDma + kD0>();
    stage_barrier();
    read_scales(0);
    Frags f0, f1;
#pragma unroll
    for (int r = 0; r < kReads; ++r) read_frag(0, 0, f0, r);
    int pslot = S::kStages - 1;  // of the tile before
    for (int s = 0; s <= last; ++s) {
      take_scales();
      step(f0, f1, slot, 1, min(s - 1 + S::kStages, last), pslot, kD0, S::kDma, H0{});
      wait_vmcnt<(S::kStages - 2) * S::kDma>();
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's reads of tile s are in registers
      stage_barrier();
      pslot = slot;
      slot = slot + 1 == S::kStages ? 0 : slot + 1;
      read_scales(slot);
      step(f1, f0, slot, 0, min(s + S::kStages, last), pslot, 0, kD0, H1{});
    }
  } else {
    // a barrier a step: its slot is refilled within the step
#pragma unroll
    for (int q = 0; q < S::kStages; ++q)
#pragma unroll
      for (int d = 0; d < S::kDma; ++d) dma(min(q, last), q, d);
    wait_vmcnt<(S::kStages - 1) * S::kDma>();
    stage_barrier();
    read_scales(0);
    Frags f0, f1;
#pragma unroll
    for (int r = 0; r < kReads; ++r) read_frag(0, 0, f0, r);
    auto one = [&](int s, Frags& cur, Frags& nxt, auto half) {
      wait_vmcnt<(S::kStages - 2) * S::kDma>();
      __builtin_amdgcn_s_waitcnt(0xc07f);
      stage_barrier();
      take_scales();
      const int old = slot;
      slot = slot + 1 == S::kStages ? 0 : slot + 1;
      read_scales(slot);
      step(cur, nxt, slot, 0, min(s + S::kStages, last), old, 0, S::kDma, half);
    };
    for (int s = 0; s <= last; s += 2) {
      one(s, f0, f1, H0{});
      one(s + 1, f1, f0, H1{});
    }
  }
  wait_vmcnt<0>();  // the redundant loads land before the workgroup's LDS is given away

  const int mw = m0 + wm * 32 * kMB, nw = n0 + wn * 32 * kNB;
  if constexpr (kEpi == kPlain) {
    if (g.type == MXFP4_BF16) store_plain<S, MXFP4_BF16>(g, mw, nw, lane, acc);
    else if (g.type == MXFP4_F16) store_plain<S, MXFP4_F16>(g, mw, nw, lane, acc);
    else store_plain<S, MXFP4_F32>(g, mw, nw, lane, acc);
  } else {
    if (g.type == MXFP4_BF16) {
      if (g.fn == MXFP4_SILU) store_gated<S, MXFP4_BF16, MXFP4_SILU>(g, mw, nw, lane, acc);
      else store_gated<S, MXFP4_BF16, MXFP4_GELU>(g, mw, nw, lane, acc);
    } else {
      if (g.fn == MXFP4_SILU) store_gated<S, MXFP4_F16, MXFP4_SILU>(g, mw, nw, lane, acc);
      else store_gated<S, MXFP4_F16, MXFP4_GELU>(g, mw, nw, lane, acc);
    }
  }
}

// Every ring leaves room for two workgroups a CU, so that one's pipeline fill, barriers and epilogue overlap the other's
// products: 256 x 256 tiles with one took 87 us (E2M1, 10752 x 6144 x 2048) and 148 (10752 x 2048 x 12288) where these take 78
// and 128, each product in a loop by itself.  In Tall the E4M3 stages are 64 codes wide, the E2M1 ones 128 (half the barriers).  The others hold a whole K
// tile's fragments ahead, for which Tall has no registers left: at 1000 x 1024 x 7168 in E4M3 that took Low from 16.3 to 14.2
// us, Mid from 22.0 to 20.4, and Mini (twice Low's workgroups where those leave CUs idle) from 14.6 to 13.6.
template <int kAF>
using Tall = Shape<kAF, 2, 4, 4, 1, kAF == MXFP4_E4M3 ? 1 : 2, 3>;  // 256 x 128, 65 or 76 KB
template <int kAF>
using Mid = Shape<kAF, 2, 2, 2, 2, 2, kAF == MXFP4_E4M3 ? 3 : 4>;  // 128 x 128, 75 or 68 KB
template <int kAF>
using Low = Shape<kAF, 1, 2, 2, 2, 2, 4>;  // 64 x 128, 68 or 52 KB
template <int kAF>
using Mini = Shape<kAF, 1, 1, 2, 2, 2, 4>;  // 64 x 64, 52 or 36 KB

template <class S, int kEpi>
int launch(GemmArgs& g, const char* what, hipStream_t st) {
  g.tm = (g.M + S::kBM - 1) / S::kBM;
  g.tn = (g.rows_b + S::kBN - 1) / S::kBN;
  MX_CHECK_ARG((int64_t)g.tm * g.tn < (1 << 30), "%s: too large", what);
  // a lane's offset from its tile's first row block is held in 32 bits
  MX_CHECK_ARG((int64_t)std::max(S::kBM, S::kBN) / 16 * g.kt * 2048 < (1LL << 31), "%s: K too large", what);
  g.per = (g.tm * g.tn + 7) / 8;
  gemm_kernel<S, kEpi><<<8 * g.per, S::kThreads, 0, st>>>(g);
  MX_CHECK_LAUNCH(what);
  return MXFP8_OK;
}

template <int kEpi, int kAF>
int dispatch(GemmArgs& g, const char* what, hipStream_t st) {
  switch (mx4_shape(g.M, g.rows_b, g.kt, kAF == MXFP4_E4M3, kEpi == kGated, g.b_pi && g.type != MXFP4_F32 && !g.gu, 256)) {
    case kMx4Thin:
      mx4_thin(kEpi == kGated, g.a, g.sa, kAF, g.b, g.sb, g.M, g.N, g.kt, g.add, g.ld_add, g.fn, g.c, g.ldc, g.type, st);
      MX_CHECK_LAUNCH(what);
      return MXFP8_OK;
    case kMx4Tall: return launch<Tall<kAF>, kEpi>(g, what, st);
    case kMx4Mid: return launch<Mid<kAF>, kEpi>(g, what, st);
    case kMx4Mini:
      if constexpr (kEpi == kPlain) return launch<Mini<kAF>, kEpi>(g, what, st);
    default: return launch<Low<kAF>, kEpi>(g, what, st);
  }
}
template <int kEpi>
int dispatch(GemmArgs& g, int64_t a_fmt, const char* what, hipStream_t st) {
  return a_fmt == MXFP4_E4M3 ? dispatch<kEpi, MXFP4_E4M3>(g, what, st) : dispatch<kEpi, MXFP4_E2M1>(g, what, st);
}

int check_operands(const char* what, const void* a, const void* sa, int64_t a_fmt, const void* b, const void* sb,
                   int64_t M, int64_t N, int64_t K) {
  MX_CHECK_ARG(a && sa && b && sb, "%s: null operand", what);
  MX_CHECK_ARG(a_fmt == MXFP4_E2M1 || a_fmt == MXFP4_E4M3, "%s: unknown format %lld", what, (long long)a_fmt);
  MX_CHECK_ARG(M < (1LL << 30) && N > 0 && N < (1LL << 29) && K > 0 && K % 128 == 0 && K < (1LL << 26),
               "%s: bad shape (M=%lld N=%lld K=%lld)", what, (long long)M, (long long)N, (long long)K);
  MX_CHECK_ARG(mx_aligned(a, 16) && mx_aligned(sa, 16) && mx_aligned(b, 16) && mx_aligned(sb, 16),
               "%s: misaligned operand", what);
  return MXFP8_OK;
}

}  // namespace

extern "C" int mxfp4_gemm(const void* a, const void* sa, int64_t a_fmt, const void* b, const void* sb, int64_t b_order,
                          int64_t M, int64_t N, int64_t K, void* c, int64_t ldc, int64_t type, void* stream) {
  MX_CHECK_ARG(M >= 0, "mxfp4_gemm: bad M");
  if (M == 0) return MXFP8_OK;
  if (int rc = check_operands("mxfp4_gemm", a, sa, a_fmt, b, sb, M, N, K)) return rc;
  MX_CHECK_ARG(type >= MXFP4_BF16 && type <= MXFP4_F32, "mxfp4_gemm: unknown element type %lld", (long long)type);
  MX_CHECK_ARG(b_order == MXFP4_ROWS_PLAIN || b_order == MXFP4_ROWS_PI, "mxfp4_gemm: B in an order of another call");
  const int es = type == MXFP4_F32 ? 4 : 2;
  MX_CHECK_ARG(c && ldc >= N && mx_aligned(c, es), "mxfp4_gemm: bad output");
  GemmArgs g{};
  g.a = (const uint8_t*)a; g.sa = (const uint8_t*)sa; g.b = (const uint8_t*)b; g.sb = (const uint8_t*)sb;
  g.M = (int)M; g.N = (int)N; g.rows_b = (int)N; g.kt = (int)(K / 128);
  g.c = c; g.ldc = ldc; g.type = (int)type; g.b_pi = b_order == MXFP4_ROWS_PI;
  g.vec = mx_aligned(c, 16) && ldc * es % 16 == 0;
  return dispatch<kPlain>(g, a_fmt, "mxfp4_gemm", (hipStream_t)stream);
}

extern "C" int64_t mxfp4_gated_saved_elems(int64_t M, int64_t N) {
  return M <= 0 || N <= 0 ? 0 : (M + 31) / 32 * ((N + 31) / 32) * 2048;
}

extern "C" int mxfp4_gated(const void* a, const void* sa, int64_t a_fmt, const void* b, const void* sb, int64_t M,
                           int64_t N, int64_t K, const void* add, int64_t ld_add, int64_t fn, void* h, int64_t ldh,
                           void* gu, int64_t type, void* stream) {
  MX_CHECK_ARG(M >= 0, "mxfp4_gated: bad M");
  if (M == 0) return MXFP8_OK;
  if (int rc = check_operands("mxfp4_gated", a, sa, a_fmt, b, sb, M, N, K)) return rc;
  MX_CHECK_ARG(type == MXFP4_BF16 || type == MXFP4_F16, "mxfp4_gated: bf16 or f16 (type %lld)", (long long)type);
  MX_CHECK_ARG(fn == MXFP4_SILU || fn == MXFP4_GELU, "mxfp4_gated: unknown gate function %lld", (long long)fn);
  MX_CHECK_ARG(h && ldh >= N && mx_aligned(h, 2) && mx_aligned(gu, 16), "mxfp4_gated: bad output");
  MX_CHECK_ARG(!add || ((ld_add == 0 || ld_add >= 2 * N) && mx_aligned(add, 2)), "mxfp4_gated: bad addend");
  GemmArgs g{};
  g.a = (const uint8_t*)a; g.sa = (const uint8_t*)sa; g.b = (const uint8_t*)b; g.sb = (const uint8_t*)sb;
  g.M = (int)M; g.N = (int)N; g.rows_b = (int)((N + 31) / 32 * 64); g.kt = (int)(K / 128);
  g.c = h; g.ldc = ldh; g.type = (int)type; g.b_pi = 1;
  g.vec = mx_aligned(h, 16) && ldh % 8 == 0;
  g.add = add; g.ld_add = ld_add; g.gu = gu; g.fn = (int)fn;
  g.add_vec = mx_aligned(add, 16) && ld_add % 8 == 0 && N % 8 == 0;
  return dispatch<kGated>(g, a_fmt, "mxfp4_gated", (hipStream_t)stream);
}
