// MX quantization to E2M1 (or E4M3) operands of the 4-bit products, along the rows and, from the same read, along the
// columns; and the values of an operand.
//
// What bounds it: memory.  A bf16 element is read once (2 bytes) and leaves as 17/32 byte an axis (E2M1).
// One 256-thread workgroup per 128 x 128 tile, which is one 512-byte scale tile of either axis: lane l of wave w (rg =
// l / 16, ch = l % 16) holds columns 8 ch .. + 7 of rows 32 w + 8 rg + 0..7, so a 32-column block of a row is four
// neighbouring lanes and a 32-row block of a column is one wave.
//   Row axis: the four lanes agree on their amax by two DPP moves; eight codes leave as one word (E2M1).
//   Column axis: the amax over the lane's eight rows and the lanes l, l ^ 16, l ^ 32, l ^ 48 (two lane swaps); the codes
//   are turned through LDS and leave in 16-byte chunks.
#include "abi_common.h"
#include "mx4_device.h"

using namespace mx4;

namespace {

constexpr int kTile = 128, kThreads = 256;

struct QuantArgs {
  const void* x;
  int64_t rows, cols, ld;
  uint8_t* q;
  uint8_t* s;
  int64_t q_tiles;
  int order;
  uint8_t* qt;
  uint8_t* st;
  int64_t t_tile0, t_tiles;
  int order_t;
  int vec;  // rows are aligned to 16 bytes
};

template <int kT, int kFmt, bool kRows, bool kCols>
__global__ __launch_bounds__(kThreads) void quant_kernel(const QuantArgs a) {
  constexpr int kB = kFmt == MXFP4_E4M3 ? 8 : 4;         // bytes of eight codes
  constexpr int kLd = 16 * kB + 16;                      // row stride of the turned codes (128 codes and a pad)
  __shared__ uint32_t stile[kTile], sttile[kCols ? kTile : 1];
  __shared__ __attribute__((aligned(16))) uint8_t qtt[kCols ? kTile * kLd : 16];
  typedef typename Elem<kT>::T T;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, rg = lane >> 4, ch = lane & 15;
  const int64_t ct = blockIdx.x, rt = blockIdx.y;
  const int64_t col = ct * kTile + ch * 8, row0 = rt * kTile + 32 * w + 8 * rg;
  const T* x = reinterpret_cast<const T*>(a.x);
  float v[8][8];
  if (a.vec && (ct + 1) * kTile <= a.cols) {
#pragma unroll
    for (int k = 0; k < 8; ++k) load8<kT>(x + min(row0 + k, a.rows - 1) * a.ld + col, v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const T t = x[min(row0 + k, a.rows - 1) * a.ld + min(col + i, a.cols - 1)];
        v[k][i] = col + i < a.cols ? Elem<kT>::get(t) : 0.f;
      }
  }
  if (kCols) {  // rows past the end are zeros of the column axis
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = row0 + k < a.rows ? v[k][i] : 0.f;
  }
  if (kRows) {
    uint8_t* sb = reinterpret_cast<uint8_t*>(stile);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t e = block_exponent<kFmt>(quad_umax(absmax8(v[k])));
      uint32_t c[2];
      encode8<kFmt>(v[k], e, c);
      const int64_t r = order_row(row0 + k, a.order);
      if (row0 + k < a.rows) {
        uint8_t* p = a.q + code_offset<kFmt>(r, col, a.q_tiles);
        if constexpr (kFmt == MXFP4_E4M3) store_codes<true>(p, make_uint2(c[0], c[1]));
        else store_codes<true>(p, c[0]);
      }
      // the gate and up orders spread a tile's rows over two scale tiles: their bytes go out one by one
      const uint8_t eb = row0 + k < a.rows ? (uint8_t)e : (uint8_t)0;
      if ((ch & 3) == 0) {
        if (a.order < MXFP4_ROWS_GATE) sb[(r & 31) * 16 + w * 4 + (ch >> 2)] = eb;
        else if (row0 + k < (a.rows + 31) / 32 * 32) a.s[blocked_offset(r, col >> 5, a.q_tiles)] = eb;
      }
    }
  }
  if constexpr (kCols) {
    uint8_t* stb = reinterpret_cast<uint8_t*>(sttile);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float t[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = v[k][i];
      uint32_t m = absmax8(t), pa, pb;
      pair16(m, pa, pb);
      pair32(max(pa, pb), pa, pb);
      const uint32_t e = block_exponent<kFmt>(max(pa, pb));
      uint32_t c[2];
      encode8<kFmt>(t, e, c);
      const int cl = ch * 8 + i;  // column in the tile; its codes of rows 32 w + 8 rg ..
      // slots of eight codes, turned by the lane's column group so that a write instruction spreads over the banks
      const int slot = (4 * w + rg) ^ (ch & 12);
      uint8_t* p = qtt + cl * kLd + slot * kB;
      if constexpr (kFmt == MXFP4_E4M3) *reinterpret_cast<uint2*>(p) = make_uint2(c[0], c[1]);
      else *reinterpret_cast<uint32_t*>(p) = c[0];
      if (rg == 0) {
        const int64_t r = order_row(ct * kTile + cl, a.order_t);
        stb[(r & 31) * 16 + (cl >> 5) * 4 + w] = ct * kTile + cl < a.cols ? (uint8_t)e : (uint8_t)0;
      }
    }
  }
  __syncthreads();
  if constexpr (kCols) {
    constexpr int kChunks = kB;  // 16-byte chunks of a row of 128 codes: 4 or 8
#pragma unroll
    for (int j = 0; j < kTile * kChunks / kThreads; ++j) {
      const int id = tid + j * kThreads, cl = id / kChunks, k = id % kChunks;
      if (ct * kTile + cl >= a.cols) continue;
      constexpr int kPer = 16 / kB;  // slots a chunk: 4 or 2
      const int slot = (k * kPer) ^ ((cl >> 3) & 12);
      const uint4 c = *reinterpret_cast<const uint4*>(qtt + cl * kLd + slot * kB);
      const int64_t r = order_row(ct * kTile + cl, a.order_t);
      store_codes<true>(a.qt + code_offset<kFmt>(r, (a.t_tile0 + rt) * kTile + k * (128 / kChunks), a.t_tiles), c);
    }
  }
  if (kRows && a.order < MXFP4_ROWS_GATE && tid < 32)
    store_codes<true>(a.s + (rt * a.q_tiles + ct) * 512 + tid * 16, reinterpret_cast<const uint4*>(stile)[tid]);
  if (kCols && tid >= 64 && tid < 96)
    store_codes<true>(a.st + (ct * a.t_tiles + a.t_tile0 + rt) * 512 + (tid - 64) * 16,
                      reinterpret_cast<const uint4*>(sttile)[tid - 64]);
}

// Eight values a thread; odd widths end in a shorter piece.
template <int kT, int kFmt>
__global__ __launch_bounds__(kThreads) void dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ s,
                                                           int64_t rows, int64_t cols, int64_t tiles, int64_t per_row,
                                                           void* out, int vec) {
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t r = id / per_row, c = (id - r * per_row) * 8;
  if (r >= rows) return;
  const uint32_t e = s[blocked_offset(r, c >> 5, tiles)];
  const uint8_t* p = q + code_offset<kFmt>(r, c, tiles);
  float v[8];
  if constexpr (kFmt == MXFP4_E4M3) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t code = ((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 0xffu;
      const uint32_t E = (code >> 3) & 15u, M = code & 7u;
      float f = E == 0 ? (float)M * 0x1p-9f : __builtin_ldexpf((float)(8u + M), (int)E - 10);
      f = (code & 0x80u) ? -f : f;
      v[i] = (code & 0x7fu) == 0x7fu ? __uint_as_float(0x7fc00000u) : __builtin_ldexpf(f, (int)e - 127);
    }
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t code = (w >> (4 * i)) & 15u, E = (code >> 1) & 3u, M = code & 1u;
      const float f = E == 0 ? 0.5f * M : __builtin_ldexpf((float)(2u + M), (int)E - 2);
      v[i] = __builtin_ldexpf((code & 8u) ? -f : f, (int)e - 127);
    }
  }
  if (e == 255u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(0x7fc00000u);
  }
  store_run<kT, 8>(reinterpret_cast<typename Elem<kT>::T*>(out) + r * cols, c, cols, vec, v);
}

template <int kT, int kFmt>
void launch_quant(const QuantArgs& a, dim3 grid, hipStream_t st) {
  if (a.q && a.qt) quant_kernel<kT, kFmt, true, true><<<grid, kThreads, 0, st>>>(a);
  else if (a.q) quant_kernel<kT, kFmt, true, false><<<grid, kThreads, 0, st>>>(a);
  else quant_kernel<kT, kFmt, false, true><<<grid, kThreads, 0, st>>>(a);
}

template <int kT>
void launch_dequant(const void* q, const void* s, int64_t rows, int64_t cols, int64_t fmt, void* out, int vec,
                    int64_t per_row, unsigned blocks, hipStream_t st) {
  const int64_t tiles = (cols + 127) / 128;
  if (fmt == MXFP4_E4M3)
    dequant_kernel<kT, MXFP4_E4M3><<<blocks, kThreads, 0, st>>>((const uint8_t*)q, (const uint8_t*)s, rows, cols, tiles,
                                                                per_row, out, vec);
  else
    dequant_kernel<kT, MXFP4_E2M1><<<blocks, kThreads, 0, st>>>((const uint8_t*)q, (const uint8_t*)s, rows, cols, tiles,
                                                                per_row, out, vec);
}

int elem_size(int64_t type) { return type == MXFP4_F32 ? 4 : 2; }

}  // namespace

extern "C" int mxfp4_abi_version(void) { return MXFP4_OPS_ABI_VERSION; }

extern "C" int mxfp4_quant(const void* x, int64_t type, int64_t rows, int64_t cols, int64_t ld_x, int64_t fmt, void* q,
                           void* s, int64_t order, void* qt, void* st, int64_t order_t, int64_t t_tile0,
                           int64_t t_tiles, void* stream) {
  MX_CHECK_ARG(type >= MXFP4_BF16 && type <= MXFP4_F32, "mxfp4_quant: unknown element type %lld", (long long)type);
  MX_CHECK_ARG(fmt == MXFP4_E2M1 || fmt == MXFP4_E4M3, "mxfp4_quant: unknown format %lld", (long long)fmt);
  MX_CHECK_ARG(order >= MXFP4_ROWS_PLAIN && order <= MXFP4_ROWS_UP &&
                   (order_t == MXFP4_ROWS_PLAIN || order_t == MXFP4_ROWS_PI),
               "mxfp4_quant: unknown row order");
  MX_CHECK_ARG(rows >= 0 && cols >= 0 && ld_x >= 0, "mxfp4_quant: bad shape (rows=%lld cols=%lld ld=%lld)",
               (long long)rows, (long long)cols, (long long)ld_x);
  if (rows == 0 || cols == 0) return MXFP8_OK;
  MX_CHECK_ARG(x && (q == nullptr) == (s == nullptr) && (qt == nullptr) == (st == nullptr) && (q || qt),
               "mxfp4_quant: null pointer (each axis needs codes and scales)");
  const int64_t rt = (rows + 127) / 128, ct = (cols + 127) / 128;
  MX_CHECK_ARG(!qt || (t_tile0 >= 0 && t_tile0 + rt <= t_tiles), "mxfp4_quant: column tiles out of range");
  MX_CHECK_ARG(mx_aligned(x, elem_size(type)) && mx_aligned(q, 16) && mx_aligned(s, 16) && mx_aligned(qt, 16) &&
                   mx_aligned(st, 16),
               "mxfp4_quant: misaligned buffer");
  MX_CHECK_ARG(rt <= 65535 && ct <= 0x7fffffff, "mxfp4_quant: too large");
  const int vec = mx_aligned(x, 16) && ld_x * elem_size(type) % 16 == 0;
  QuantArgs a{x, rows, cols, ld_x, (uint8_t*)q, (uint8_t*)s, ct, (int)order, (uint8_t*)qt, (uint8_t*)st, t_tile0, t_tiles,
              (int)order_t, vec};
  dim3 grid((unsigned)ct, (unsigned)rt);
  const hipStream_t hs = (hipStream_t)stream;
  const bool f8 = fmt == MXFP4_E4M3;
  if (type == MXFP4_BF16) f8 ? launch_quant<MXFP4_BF16, MXFP4_E4M3>(a, grid, hs) : launch_quant<MXFP4_BF16, MXFP4_E2M1>(a, grid, hs);
  else if (type == MXFP4_F16) f8 ? launch_quant<MXFP4_F16, MXFP4_E4M3>(a, grid, hs) : launch_quant<MXFP4_F16, MXFP4_E2M1>(a, grid, hs);
  else f8 ? launch_quant<MXFP4_F32, MXFP4_E4M3>(a, grid, hs) : launch_quant<MXFP4_F32, MXFP4_E2M1>(a, grid, hs);
  MX_CHECK_LAUNCH("mxfp4_quant");
  return MXFP8_OK;
}

extern "C" int mxfp4_dequant(const void* q, const void* s, int64_t rows, int64_t cols, int64_t fmt, void* out,
                             int64_t type, void* stream) {
  MX_CHECK_ARG(rows >= 0 && cols >= 0, "mxfp4_dequant: bad shape");
  MX_CHECK_ARG(type >= MXFP4_BF16 && type <= MXFP4_F32, "mxfp4_dequant: unknown element type %lld", (long long)type);
  MX_CHECK_ARG(fmt == MXFP4_E2M1 || fmt == MXFP4_E4M3, "mxfp4_dequant: unknown format %lld", (long long)fmt);
  if (rows == 0 || cols == 0) return MXFP8_OK;
  MX_CHECK_ARG(q && s && out, "mxfp4_dequant: null pointer");
  MX_CHECK_ARG(mx_aligned(q, 16) && mx_aligned(s, 16) && mx_aligned(out, elem_size(type)),
               "mxfp4_dequant: misaligned buffer");
  const int64_t per_row = (cols + 7) / 8, blocks = (rows * per_row + kThreads - 1) / kThreads;
  MX_CHECK_ARG(blocks <= 0x7fffffff, "mxfp4_dequant: too large");
  const int vec = mx_aligned(out, 16) && cols * elem_size(type) % 16 == 0;
  const hipStream_t hs = (hipStream_t)stream;
  if (type == MXFP4_BF16) launch_dequant<MXFP4_BF16>(q, s, rows, cols, fmt, out, vec, per_row, (unsigned)blocks, hs);
  else if (type == MXFP4_F16) launch_dequant<MXFP4_F16>(q, s, rows, cols, fmt, out, vec, per_row, (unsigned)blocks, hs);
  else launch_dequant<MXFP4_F32>(q, s, rows, cols, fmt, out, vec, per_row, (unsigned)blocks, hs);
  MX_CHECK_LAUNCH("mxfp4_dequant");
  return MXFP8_OK;
}
