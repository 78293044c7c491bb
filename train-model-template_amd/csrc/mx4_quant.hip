// MX quantization to E2M1 (or E4M3) operands of the 4-bit products, along the rows and, from the same read, along the
// columns; and the values of an operand.
//
// What bounds it: memory.  A bf16 element is read once (2 bytes) and leaves as 17/32 byte an axis (E2M1): in a training step
// [10752, 6144] takes 37 us (4.5 TB/s; 26 where the last-level cache holds the matrix), [10752, 2048] 16 (3.5 TB/s), 15 to 16 in
// E4M3 (12.9 at the rate of a large copy), both axes of [6144, 2048] 10.7; small matrices a launch and one round trip, 5 us.
// One 256-thread workgroup per 128 x 128 tile, which is one 512-byte scale tile of either axis: lane l of wave w (rg =
// l / 16, ch = l % 16) holds columns 8 ch .. + 7 of rows 32 w + 8 rg + 0..7, so a 32-column block of a row is four
// neighbouring lanes and a 32-row block of a column is one wave.
//   Row axis: the four lanes agree on their amax by two DPP moves.  A wave's 32 rows are two whole blocks of the operand's
//   layout, which pass through LDS (2 KB a wave in E2M1) and leave as 1 KB stores: stored from the lanes, as words of 32-byte
//   pieces, [10752, 2048] took 18 us and [10752, 6144] 41.
//   Column axis: the amax over the lane's eight rows and the lanes l, l ^ 16, l ^ 32, l ^ 48 (two lane swaps); the codes
//   are turned through LDS and leave in 16-byte chunks, 1 KB of whole 128-byte lines a wave.
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

__device__ __forceinline__ uint32_t word(const uint4& v, int p) { return p == 0 ? v.x : p == 1 ? v.y : p == 2 ? v.z : v.w; }

// Column i of eight rows' groups (i a constant once unrolled)
template <int kT>
__device__ __forceinline__ Group<kT> column(const Group<kT>* v, int i) {
  Group<kT> g;
  uint32_t u[8];
  if constexpr (kT == MXFP4_F32) {
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = i < 4 ? word(v[k].w, i) : word(v[k].x, i - 4);
    g.w = make_uint4(u[0], u[1], u[2], u[3]);
    g.x = make_uint4(u[4], u[5], u[6], u[7]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)  // the low or the high halves of two rows' words
      u[k] = __builtin_amdgcn_perm(word(v[2 * k + 1].w, i >> 1), word(v[2 * k].w, i >> 1), i & 1 ? 0x07060302u : 0x05040100u);
    g.w = make_uint4(u[0], u[1], u[2], u[3]);
  }
  return g;
}

template <int kT, int kFmt, bool kRows, bool kCols>
__global__ __launch_bounds__(kThreads) void quant_kernel(const QuantArgs a) {
  constexpr int kB = kFmt == MXFP4_E4M3 ? 8 : 4;         // bytes of eight codes
  constexpr int kLd = 16 * kB + 16;                      // row stride of the turned codes (128 codes and a pad)
  constexpr int kWaveBytes = 32 * 16 * kB;               // codes of a wave's 32 rows
  __shared__ uint32_t stile[kTile], sttile[kCols ? kTile : 1];
  __shared__ __attribute__((aligned(16))) uint8_t qtt[kCols ? kTile * kLd : 16];
  __shared__ __attribute__((aligned(16))) uint8_t qr[kRows ? 4 * kWaveBytes : 16];
  typedef typename Elem<kT>::T T;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, rg = lane >> 4, ch = lane & 15;
  const int64_t ct = blockIdx.x, rt = blockIdx.y;
  const int64_t col = ct * kTile + ch * 8, row32 = rt * kTile + 32 * w, row0 = row32 + 8 * rg;
  const T* x = reinterpret_cast<const T*>(a.x);
  Group<kT> v[8];
  if (a.vec && ((ct + 1) * kTile <= a.cols || a.cols % 8 == 0)) {
    // a row's last tile ends with a whole group: lanes past it read the group before and take zeros
    const int64_t cl = min(col, a.cols - 8);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = load_group<kT>(x + min(row0 + k, a.rows - 1) * a.ld + cl);
    if (cl != col) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = Group<kT>{};
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = load_group_edge<kT>(x + min(row0 + k, a.rows - 1) * a.ld, col, a.cols);
  }
  if (kCols) {  // rows past the end are zeros of the column axis
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t m = row0 + k < a.rows ? ~0u : 0u;
      v[k].w = make_uint4(v[k].w.x & m, v[k].w.y & m, v[k].w.z & m, v[k].w.w & m);
      if constexpr (kT == MXFP4_F32) v[k].x = make_uint4(v[k].x.x & m, v[k].x.y & m, v[k].x.z & m, v[k].x.w & m);
    }
  }
  if (kRows) {
    uint8_t* sb = reinterpret_cast<uint8_t*>(stile);
    uint8_t* mine = qr + w * kWaveBytes;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t e = block_exponent<kFmt>(quad_umax(v[k].absmax()));
      uint32_t c[2];
      encode_group<kT, kFmt>(v[k], e, c);
      // the row's place among the wave's 32, which stay together in every order
      const int rl = (int)order_row(8 * rg + k, a.order == MXFP4_ROWS_PLAIN ? MXFP4_ROWS_PLAIN : MXFP4_ROWS_PI);
      uint8_t* p = mine + code_offset<kFmt>(rl, ch * 8, 1);
      if constexpr (kFmt == MXFP4_E4M3) *reinterpret_cast<uint2*>(p) = make_uint2(c[0], c[1]);
      else *reinterpret_cast<uint32_t*>(p) = c[0];
      // the gate and up orders spread a tile's rows over two scale tiles: their bytes go out one by one
      const uint8_t eb = row0 + k < a.rows ? (uint8_t)e : (uint8_t)0;
      if ((ch & 3) == 0) {
        if (a.order < MXFP4_ROWS_GATE) sb[rl * 16 + w * 4 + (ch >> 2)] = eb;
        else if (row0 + k < (a.rows + 31) / 32 * 32) a.s[blocked_offset(order_row(row0 + k, a.order), col >> 5, a.q_tiles)] = eb;
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // a wave reads back what it wrote itself
    if (row32 < a.rows) {
      const int64_t r = order_row(row32, a.order);  // the first row of the 32 in every order
#pragma unroll
      for (int j = 0; j < kWaveBytes / 1024; ++j) {
        constexpr int kPer = kWaveBytes / 2048;  // KB of a 16-row block
        store_codes<true>(a.q + ((r >> 4) + j / kPer) * a.q_tiles * (1024 * kPer) + (ct * kPer + j % kPer) * 1024 + lane * 16,
                          *reinterpret_cast<const uint4*>(mine + j * 1024 + lane * 16));
      }
    }
  }
  if constexpr (kCols) {
    uint8_t* stb = reinterpret_cast<uint8_t*>(sttile);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const Group<kT> t = column<kT>(v, i);
      uint32_t pa, pb;
      pair16(t.absmax(), pa, pb);
      pair32(max(pa, pb), pa, pb);
      const uint32_t e = block_exponent<kFmt>(max(pa, pb));
      uint32_t c[2];
      encode_group<kT, kFmt>(t, e, c);
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

// A workgroup takes 16 rows of four column tiles; thread t row t / 16 and columns 8 (t % 16) .. of each.
template <int kT, int kFmt>
__global__ __launch_bounds__(kThreads) void dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ s,
                                                           int64_t rows, int64_t cols, int64_t tiles, void* out, int vec) {
  typedef typename Elem<kT>::T T;
  const int64_t r = (int64_t)blockIdx.y * 16 + (threadIdx.x >> 4);
  const int cl = (threadIdx.x & 15) * 8;
  uint2 code[4];
  uint32_t e[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // rows past the end lie in the operand's padding
    const int64_t t = min((int64_t)blockIdx.x * 4 + j, tiles - 1);
    const uint8_t* p = q + code_offset<kFmt>(r, t * 128 + cl, tiles);
    if constexpr (kFmt == MXFP4_E4M3) code[j] = *reinterpret_cast<const uint2*>(p);
    else code[j].x = *reinterpret_cast<const uint32_t*>(p);
    e[j] = s[blocked_offset(r, t * 4 + (cl >> 5), tiles)];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t c = ((int64_t)blockIdx.x * 4 + j) * 128 + cl;
    float v[8];
    const uint32_t w[2] = {code[j].x, code[j].y};
    // the hardware's conversion for scales whose products are normal numbers, else by hand (one branch a wave)
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(e[j] < 12u || e[j] > 245u) == 0, 1)) {
      const float sc = __uint_as_float(e[j] << 23);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v2f f;
        if constexpr (kFmt == MXFP4_E4M3) f = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i >> 1], sc, true)
                                                    : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i >> 1], sc, false);
        else f = i == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], sc, 0)
                 : i == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], sc, 1)
                 : i == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], sc, 2)
                          : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], sc, 3);
        v[2 * i] = f[0];
        v[2 * i + 1] = f[1];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float f;
        bool nan = e[j] == 255u;
        if constexpr (kFmt == MXFP4_E4M3) {
          const uint32_t b = (w[i >> 2] >> (8 * (i & 3))) & 0xffu, E = (b >> 3) & 15u, M = b & 7u;
          f = E == 0 ? (float)M * 0x1p-9f : __builtin_ldexpf((float)(8u + M), (int)E - 10);
          f = b & 0x80u ? -f : f;
          nan |= (b & 0x7fu) == 0x7fu;
        } else {
          const uint32_t b = (w[0] >> (4 * i)) & 15u, E = (b >> 1) & 3u, M = b & 1u;
          f = E == 0 ? 0.5f * M : __builtin_ldexpf((float)(2u + M), (int)E - 2);
          f = b & 8u ? -f : f;
        }
        v[i] = nan ? __uint_as_float(0x7fc00000u) : __builtin_ldexpf(f, (int)e[j] - 127);
      }
    }
    if (r < rows && c < cols) {
      T* row = reinterpret_cast<T*>(out) + r * cols;
      if (vec && c + 8 <= cols) {
        if constexpr (kT == MXFP4_F32) store_run<kT, 8>(row, c, cols, true, v);
        else
          store_codes<true>(reinterpret_cast<uint8_t*>(row + c),
                            make_uint4(round2<kT>(v[0], v[1]), round2<kT>(v[2], v[3]), round2<kT>(v[4], v[5]),
                                       round2<kT>(v[6], v[7])));
      } else {
        store_run<kT, 8>(row, c, cols, false, v);
      }
    }
  }
}

template <int kT, int kFmt>
void launch_quant(const QuantArgs& a, dim3 grid, hipStream_t st) {
  if (a.q && a.qt) quant_kernel<kT, kFmt, true, true><<<grid, kThreads, 0, st>>>(a);
  else if (a.q) quant_kernel<kT, kFmt, true, false><<<grid, kThreads, 0, st>>>(a);
  else quant_kernel<kT, kFmt, false, true><<<grid, kThreads, 0, st>>>(a);
}

// Rows past what a grid's second dimension counts take further launches, each from a scale tile's first row on (row blocks
// spread over a third dimension made every launch slower: both axes of 6144 x 2048, quantized and read back, 24.8 us in place of 22.2).
constexpr int64_t kDequantRows = 65528 * 16;
static_assert(kDequantRows % 128 == 0, "whole scale tiles");

template <int kT, int kFmt>
void launch_dequant(const void* q, const void* s, int64_t rows, int64_t cols, void* out, int vec, hipStream_t st) {
  const int64_t tiles = (cols + 127) / 128;
  for (int64_t r = 0; r < rows; r += kDequantRows) {
    const int64_t n = rows - r < kDequantRows ? rows - r : kDequantRows;
    const dim3 grid((unsigned)((tiles + 3) / 4), (unsigned)((n + 15) / 16));
    dequant_kernel<kT, kFmt><<<grid, kThreads, 0, st>>>(
        (const uint8_t*)q + r * tiles * 128 / (kFmt == MXFP4_E4M3 ? 1 : 2), (const uint8_t*)s + r / 128 * tiles * 512, n, cols,
        tiles, (typename Elem<kT>::T*)out + r * cols, vec);
  }
}
template <int kT>
void launch_dequant(const void* q, const void* s, int64_t rows, int64_t cols, int64_t fmt, void* out, int vec,
                    hipStream_t st) {
  if (fmt == MXFP4_E4M3) launch_dequant<kT, MXFP4_E4M3>(q, s, rows, cols, out, vec, st);
  else launch_dequant<kT, MXFP4_E2M1>(q, s, rows, cols, out, vec, st);
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
  MX_CHECK_ARG(rows < (1LL << 35) && cols < (1LL << 33), "mxfp4_dequant: too large");
  const int vec = mx_aligned(out, 16) && cols * elem_size(type) % 16 == 0;
  const hipStream_t hs = (hipStream_t)stream;
  if (type == MXFP4_BF16) launch_dequant<MXFP4_BF16>(q, s, rows, cols, fmt, out, vec, hs);
  else if (type == MXFP4_F16) launch_dequant<MXFP4_F16>(q, s, rows, cols, fmt, out, vec, hs);
  else launch_dequant<MXFP4_F32>(q, s, rows, cols, fmt, out, vec, hs);
  MX_CHECK_LAUNCH("mxfp4_dequant");
  return MXFP8_OK;
}
