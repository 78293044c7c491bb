// Backward of the gated block's gate: from the saved [g | u] and dh, du = dh fn(g) and dg = dh u fn'(g), quantized straight
// from fp32 into the operand of the product with [W_gate; W_up] (and, where an addend wants its gradient, rounded to the
// activations' type).
//
// What bounds it: memory, 6 bytes read and 2 (E4M3) or 1 (E2M1) written for each column of a row, and 4 more for the
// addend's gradient: 10752 x 6144 bf16 in E4M3 takes 98 us, 159 with the addend's gradient (5.4 and 5.0 TB/s; part of it
// comes from the last-level cache) in a training step, and 90 in a loop by itself; in pieces of 16 bytes of a row that
// gradient took 30 more.  The saved values lie in the order of the forward epilogue's lanes, which is this kernel's order
// too: lane l of a wave holds row l % 32 and 16 columns of a 32 x 32 block, a 32-column scale block is two lanes, and every
// load of the saved values is 1 KB in a row.  One block a wave: four in a row, each asked for while the one before was
// computed, took 98 us in that loop, and 11.7 where one takes 9.4 at 1000 x 3584, whose waves then waited four times for
// memory.
#include "abi_common.h"
#include "mx4_device.h"

using namespace mx4;

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint4 load_nt(const void* p) {
  const u32x4v v = __builtin_nontemporal_load(reinterpret_cast<const u32x4v*>(p));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

struct BwdArgs {
  const void* gu;
  const void* dh;
  int64_t ld_dh;
  int M, N;
  uint8_t* q;
  uint8_t* s;
  void* dgu;
  int vec_dh, vec_dgu;
};

// 16 codes of v (its other 16 in lane l ^ 32) at row m, column c of an operand with ct column tiles; returns the scale byte,
// 0 past the rows
template <int kFmt>
__device__ __forceinline__ uint32_t quant_store(const float* v, int64_t m, int64_t c, int64_t ct, bool live, uint8_t* q) {
  uint32_t a, b;
  pair32(max(absmax8(v), absmax8(v + 8)), a, b);
  const uint32_t e = block_exponent<kFmt>(max(a, b));
  uint32_t c0[2], c1[2];
  encode8<kFmt>(v, e, c0);
  encode8<kFmt>(v + 8, e, c1);
  if (live) {
    uint8_t* p = q + code_offset<kFmt>(m, c, ct);
    if constexpr (kFmt == MXFP4_E4M3) *reinterpret_cast<uint4*>(p) = make_uint4(c0[0], c0[1], c1[0], c1[1]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(c0[0], c1[0]);
  }
  return live ? e : 0u;
}

// A workgroup takes 32 rows and 128 columns, a wave a 32 x 32 block of them.  Rows up to the scale tiles' 128 take part, so that
// all scale bytes are written.
template <int kT, int kFn, int kFmt>
__global__ __launch_bounds__(kThreads) void gate_bwd_kernel(const BwdArgs a) {
  typedef typename Elem<kT>::T T;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hi = lane >> 5;
  const int64_t nblk = (a.N + 31) / 32;
  const uint32_t tiles = (uint32_t)(a.N + 127) / 128, rb = blockIdx.x / tiles, tile = blockIdx.x - rb * tiles;
  const int64_t m = (int64_t)rb * 32 + (lane & 31), mc = min(m, (int64_t)a.M - 1);
  const bool live = m < a.M;
  const int64_t cb = (int64_t)tile * 128 + w * 32, c = cb + hi * 16;
  float dg[16], du[16];
  if (cb < a.N) {
    Group<kT> gr[2], ur[2], dr[2];
    const T* s = reinterpret_cast<const T*>(a.gu) + saved_offset(mc, c, nblk);
    gr[0].w = load_nt(s);  // read once: past the caches
    gr[1].w = load_nt(s + 512);
    ur[0].w = load_nt(s + 1024);
    ur[1].w = load_nt(s + 1536);
    const T* p = reinterpret_cast<const T*>(a.dh) + mc * a.ld_dh;
    if (a.vec_dh && cb + 32 <= a.N) {
      dr[0] = load_group<kT>(p + c);
      dr[1] = load_group<kT>(p + c + 8);
    } else {
      dr[0] = load_group_edge<kT>(p, c, a.N);
      dr[1] = load_group_edge<kT>(p, c + 8, a.N);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float g[8], u[8], d[8];
      gr[h].values(g);
      ur[h].values(u);
      dr[h].values(d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float df;
        const float f = gate_fn<kFn>(g[i], df);
        dg[8 * h + i] = d[i] * u[i] * df;
        du[8 * h + i] = d[i] * f;
      }
    }
  }
  if (cb + 32 > a.N) {  // the saved values past the last column are undefined
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      dg[i] = c + i < a.N ? dg[i] : 0.f;
      du[i] = c + i < a.N ? du[i] : 0.f;
    }
  }
  const uint32_t sg = quant_store<kFmt>(dg, m, c, 2 * tiles, live, a.q);
  const uint32_t su = quant_store<kFmt>(du, m, (int64_t)tiles * 128 + c, 2 * tiles, live, a.q);
  const int64_t t = (int64_t)(rb >> 2) * 2 * tiles + tile + (hi ? tiles : 0);
  a.s[t * 512 + (lane & 31) * 16 + (rb & 3) * 4 + w] = (uint8_t)(hi ? su : sg);
  if (a.dgu) {
    T* o = reinterpret_cast<T*>(a.dgu);
    store_block<kT>(o, 2 * (int64_t)a.N, rb * 32, a.M, cb, a.N, a.vec_dgu, lane, dg);
    store_block<kT>(o + a.N, 2 * (int64_t)a.N, rb * 32, a.M, cb, a.N, a.vec_dgu, lane, du);
  }
}

template <int kT, int kFn>
void launch(const BwdArgs& a, int64_t fmt, unsigned grid, hipStream_t st) {
  if (fmt == MXFP4_E4M3) gate_bwd_kernel<kT, kFn, MXFP4_E4M3><<<grid, kThreads, 0, st>>>(a);
  else gate_bwd_kernel<kT, kFn, MXFP4_E2M1><<<grid, kThreads, 0, st>>>(a);
}

}  // namespace

extern "C" int mxfp4_gated_bwd(const void* gu, const void* dh, int64_t ld_dh, int64_t M, int64_t N, int64_t fn,
                               int64_t type, int64_t fmt, void* q, void* s, void* dgu, void* stream) {
  MX_CHECK_ARG(M >= 0 && N > 0 && M < (1LL << 30) && N < (1LL << 29), "mxfp4_gated_bwd: bad shape (M=%lld N=%lld)",
               (long long)M, (long long)N);
  MX_CHECK_ARG(type == MXFP4_BF16 || type == MXFP4_F16, "mxfp4_gated_bwd: bf16 or f16 (type %lld)", (long long)type);
  MX_CHECK_ARG(fn == MXFP4_SILU || fn == MXFP4_GELU, "mxfp4_gated_bwd: unknown gate function %lld", (long long)fn);
  MX_CHECK_ARG(fmt == MXFP4_E2M1 || fmt == MXFP4_E4M3, "mxfp4_gated_bwd: unknown format %lld", (long long)fmt);
  if (M == 0) return MXFP8_OK;
  MX_CHECK_ARG(gu && dh && q && s && ld_dh >= N, "mxfp4_gated_bwd: null pointer or bad stride");
  MX_CHECK_ARG(mx_aligned(gu, 16) && mx_aligned(dh, 2) && mx_aligned(q, 16) && mx_aligned(s, 16) && mx_aligned(dgu, 2),
               "mxfp4_gated_bwd: misaligned buffer");
  const int64_t wgs = (N + 127) / 128 * ((M + 127) / 128 * 4);
  MX_CHECK_ARG(wgs < (1 << 24), "mxfp4_gated_bwd: too large (M=%lld N=%lld)", (long long)M, (long long)N);
  const BwdArgs a{gu, dh, ld_dh, (int)M, (int)N, (uint8_t*)q, (uint8_t*)s, dgu, mx_aligned(dh, 16) && ld_dh % 8 == 0,
                  mx_aligned(dgu, 16) && N % 8 == 0};
  const unsigned grid = (unsigned)wgs;
  const hipStream_t st = (hipStream_t)stream;
  if (type == MXFP4_BF16)
    fn == MXFP4_SILU ? launch<MXFP4_BF16, MXFP4_SILU>(a, fmt, grid, st) : launch<MXFP4_BF16, MXFP4_GELU>(a, fmt, grid, st);
  else
    fn == MXFP4_SILU ? launch<MXFP4_F16, MXFP4_SILU>(a, fmt, grid, st) : launch<MXFP4_F16, MXFP4_GELU>(a, fmt, grid, st);
  MX_CHECK_LAUNCH("mxfp4_gated_bwd");
  return MXFP8_OK;
}
