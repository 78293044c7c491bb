// Distillation from a teacher's top logits: loss and gradient of a row of logits [V] against the teacher's k entries.
//
// Mathematics, with a = z / tau, q = softmax(a), S the row's entries and p the teacher's masses on them:
//   loss = tau^2 (sum_S p (log p - log q) + p_r (log p_r - log q_r)),   q_r = sum of q outside S
//   d loss / d z_j = tau (q_j P - p_j) on S, P = sum p + p_r;  tau q_j (P - p_r / q_r) elsewhere
// Without the rest bucket p_r = 0.  One pass over the row keeps a running maximum m and the sum s of exp((z - m) / tau) in
// fp32 over the columns outside S (a bit for every column in LDS says which), and S is added from its k values: q_r has its
// own maximum and sum and is no difference.  The factors exp((m - M) / tau) / sum and p_r / s that the gradient needs are at
// most 1 each.  z - m is taken before the division by tau: rows of the type's lowest value stay uniform.
// The loss sums logarithms and differences of logits apart, tau (tau l + d): a difference that reaches the type's end is not
// divided by tau.
//
// What bounds it: memory, the logits read once and the gradient written once.  A workgroup takes a row and holds it, or its
// first 128K (64K in fp32) columns, in registers between the two passes; what is left comes from the cache the second time.
// Few rows are split into pieces over two launches, joined by the second.  1000 rows of 65536 bf16 logits take 51 us (5.2
// TB/s), 2048 of 248001 478 (4.3 TB/s counted once; 32K columns in registers and two workgroups a CU take the same); vectors
// that begin 16-byte pieces but not lines took 3% more.  16 rows of 65536 fp32, the loss alone: 9.0 in the two launches.
#include <algorithm>

#include "abi_common.h"
#include "mx4_device.h"

using namespace mx4;

namespace {

constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kMaxPiece = 1 << 18;  // columns of a piece: its bits take 32 KB

struct Args {
  const void* z;
  int64_t ld, V;
  const void* idx;
  int idx8;
  int64_t ld_idx;
  const float* t;
  int64_t ld_t;
  int k;
  float tau;
  const float* lse;
  const float* weight;
  float* loss;
  void* grad;
  int64_t ld_grad;
  int parts;
  int wgs;         // workgroups of a row in this launch: parts, or 1 for the loss alone
  int64_t piece;   // vectors of a piece
  int bit_words;   // words of LDS for the bits
  float2* stats;   // [T][parts] running maximum and sum of the piece
  float2* entries; // [T][k] logit of the entry, and 1 if it is the first (of lowest index) of its column
};

struct Sum {
  float m, s;  // s = sum of exp((z - m) / tau)
};
__device__ __forceinline__ Sum join(Sum a, Sum b, float c) {
  const float m = fmaxf(a.m, b.m);
  return Sum{m, a.s * __builtin_amdgcn_exp2f((a.m - m) * c) + b.s * __builtin_amdgcn_exp2f((b.m - m) * c)};
}
// f over the 64 lanes, in every lane: lane swaps in the VALU (quad permutations, mirrors of 8 and of 16 lanes, swaps of 16 and
// of 32), where shuffles go through LDS
template <int kDpp>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kDpp, 0xF, 0xF, true));
}
__device__ __forceinline__ float first_lane(float v) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}
template <class F>
__device__ __forceinline__ float wave_reduce(float v, F f) {
  v = f(v, dpp<0xB1>(v));   // lane ^ 1
  v = f(v, dpp<0x4E>(v));   // lane ^ 2
  v = f(v, dpp<0x141>(v));  // 7 - lane of 8
  v = f(v, dpp<0x140>(v));  // 15 - lane of 16
  uint32_t a, b;
  pair16(__float_as_uint(v), a, b);
  v = f(__uint_as_float(a), __uint_as_float(b));
  pair32(__float_as_uint(v), a, b);
  return f(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_reduce(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v) {  // NaN stays
  return wave_reduce(v, [](float a, float b) { return a > b || a != a ? a : b; });
}
// The sum of all lanes: against the wave's maximum each lane is scaled once
__device__ __forceinline__ Sum wave_join(Sum a, float c) {
  const float m = wave_reduce(a.m, [](float x, float y) { return fmaxf(x, y); });
  return Sum{m, wave_sum(a.s * __builtin_amdgcn_exp2f((a.m - m) * c))};
}
template <int kWaves>
__device__ __forceinline__ Sum block_join(Sum a, float c, float* sh) {
  a = wave_join(a, c);
  const int lane = threadIdx.x & 63;
  if (lane == 0) {
    sh[threadIdx.x >> 6] = a.m;
    sh[kWaves + (threadIdx.x >> 6)] = a.s;
  }
  __syncthreads();
  const int w = lane & (kWaves - 1);  // kWaves is a power of two: every wave's sum 64 / kWaves times
  const Sum r = wave_join(Sum{sh[w], sh[kWaves + w]}, c);
  // one lane's: the others may have added with a product kept unrounded (a fused multiply-add), an ulp apart
  return Sum{first_lane(r.m), first_lane(r.s) * ((float)kWaves / 64.f)};
}

template <int kT>
struct Vec {
  static constexpr int n = kT == MXFP4_F32 ? 4 : 8;  // elements of 16 bytes
};
template <int kT>
__device__ __forceinline__ void unpack_vec(uint4 u, float* v) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kT == MXFP4_F32) {
      v[i] = __uint_as_float(w[i]);
    } else if constexpr (kT == MXFP4_BF16) {
      v[2 * i] = bf16_lo(w[i]);
      v[2 * i + 1] = bf16_hi(w[i]);
    } else {
      const f16x2 h = __builtin_bit_cast(f16x2, w[i]);
      v[2 * i] = (float)h[0];
      v[2 * i + 1] = (float)h[1];
    }
  }
}

template <int kT>
__device__ __forceinline__ uint4 pack_vec(float* v) {
  if constexpr (kT == MXFP4_F32)
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  else
    return make_uint4(round2<kT>(v[0], v[1]), round2<kT>(v[2], v[3]), round2<kT>(v[4], v[5]), round2<kT>(v[6], v[7]));
}

// What a row's entries give without the row's sums (one wave computes it while the others read the row)
struct Teacher {
  float live;    // a teacher entry of positive mass
  float psum;    // sum of p
  float rest;    // p_r
  float zm, own; // maximum and sum of exp((z - zm) / tau) over S
  float a;       // sum of p log p
  float b;       // sum of p (z - zm)
  float dup;     // a column comes twice
};

enum Mode { kWhole, kStats, kFinish };  // a whole row; a piece's sums; loss and gradient of a piece from all sums

template <int kT, int kMode, int kThreads, int kHold>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kHold > 8 ? 4 : 8)))
void distill_kernel(const Args a) {
  typedef typename Elem<kT>::T T;
  constexpr int n = Vec<kT>::n, kWaves = kThreads / 64;
  constexpr bool kStream = kHold == 0 || kHold == 16;  // columns past what the registers hold
  extern __shared__ uint32_t bits[];  // a bit for every column of the piece: S; then the entries
  __shared__ float sh[2 * kWaves];
  __shared__ Teacher teacher;
  __shared__ int twice;  // a column of the piece comes twice
  int* const s_idx = reinterpret_cast<int*>(bits + a.bit_words);  // column, < 0: padding
  int* const s_first = s_idx + a.k;
  float* const s_z = reinterpret_cast<float*>(s_first + a.k);
  float* const s_p = s_z + a.k;
  const int tid = threadIdx.x, k = a.k;
  const int64_t row = blockIdx.x / (uint32_t)a.wgs;
  const int part = (int)(blockIdx.x - row * a.wgs);
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ld;
  const float c = kLog2e / a.tau, itau = 1.f / a.tau;
  const float weight = a.weight ? a.weight[row] : 1.f;

  // the row's vectors: `head` elements before the first that begins a 128-byte line, this workgroup's vectors [v0, v1), a tail
  const int head = (int)min((int64_t)((128 - ((uintptr_t)z & 127)) & 127) / (int)sizeof(T), a.V);
  const int64_t nv = (a.V - head) / n;
  const int64_t v0 = min((int64_t)part * a.piece, nv), v1 = min(v0 + a.piece, nv);
  const bool first = part == 0, last = part == a.parts - 1;
  const int64_t tail0 = head + nv * n;
  const int64_t c0 = first ? 0 : head + v0 * n, c1 = last ? a.V : head + v1 * n;  // this workgroup's columns
  // the piece's vectors by a 32-bit index from a wave-uniform address
  const char* const zp = reinterpret_cast<const char*>(z + head + v0 * n);
  const int pv = (int)(v1 - v0);
  auto load = [&](int v) { return *reinterpret_cast<const uint4*>(zp + (uint32_t)v * 16u); };

  uint4 held[kHold > 0 ? kHold : 1];
  if constexpr (kHold > 0) {
#pragma unroll
    for (int u = 0; u < kHold; ++u)
      if (pv > 0) held[u] = load(min(tid + u * kThreads, pv - 1));
  }

  // ---- the teacher's entries
  if constexpr (kMode != kFinish)
    for (int i = tid; i < a.bit_words; i += kThreads) bits[i] = 0;
  if (tid == 0) twice = 0;
  for (int i = tid; i < k; i += kThreads) {
    const int64_t o = row * a.ld_idx + i;
    const int64_t j = a.idx8 ? reinterpret_cast<const int64_t*>(a.idx)[o] : (int64_t)reinterpret_cast<const int32_t*>(a.idx)[o];
    const float t = a.t[row * a.ld_t + i];
    const bool ok = j >= 0 && j < a.V && !(t == -__builtin_inff());
    s_idx[i] = ok ? (int)j : -1;
    s_p[i] = t;
    if constexpr (kMode == kFinish) {
      const float2 e = ok ? a.entries[row * k + i] : make_float2(0.f, 0.f);
      s_z[i] = e.x;
      s_first[i] = e.y != 0.f;
    }
  }
  __syncthreads();
  const int64_t b0 = head + v0 * n - 64;  // column of bit 0: a vector's bits lie in one byte, the head's before them
  if constexpr (kMode != kFinish) {
    for (int i = tid; i < k; i += kThreads) {
      const int j = s_idx[i];
      s_first[i] = 0;
      if (j < c0 || j >= c1) continue;
      const uint32_t bit = 1u << ((j - b0) & 31);
      s_first[i] = !(atomicOr(&bits[(j - b0) >> 5], bit) & bit);
      if (!s_first[i]) twice = 1;
      s_z[i] = Elem<kT>::get(z[j]);
    }
    __syncthreads();
    // Which of a column's entries came first is chance, and the order of S's sum with it: the first is that of lowest index.
    if (twice) {
      for (int i = tid; i < k; i += kThreads) {
        const int j = s_idx[i];
        if (j < c0 || j >= c1) continue;
        int o = 0;
        while (s_idx[o] != j) ++o;
        s_first[i] = o == i;
      }
      __syncthreads();
    }
    if constexpr (kMode == kStats) {
      for (int i = tid; i < k; i += kThreads)
        if (s_idx[i] >= c0 && s_idx[i] < c1) a.entries[row * k + i] = make_float2(s_z[i], (float)s_first[i]);
    }
  }
  if (kMode != kStats && tid < 64) {
    float tmax = kLowest, zm = kLowest, any = 0.f, dup = 0.f;
    for (int i = tid; i < k; i += 64)
      if (s_idx[i] >= 0) {
        const float t = s_p[i];
        any = 1.f;
        tmax = (t > tmax || t != t) ? t : tmax;
        zm = fmaxf(zm, s_z[i]);
        dup = s_first[i] ? dup : 1.f;
      }
    any = wave_max(any);
    tmax = wave_max(tmax);
    zm = wave_max(zm);
    dup = wave_max(dup);
    const float lse = a.lse ? a.lse[row] : 0.f;
    float psum = 0.f, own = 0.f, A = 0.f, B = 0.f;
    for (int i = tid; i < k; i += 64)
      if (s_idx[i] >= 0) {
        psum += a.lse ? expf(s_p[i] * itau - lse) : expf((s_p[i] - tmax) * itau);
        if (s_first[i]) own += __builtin_amdgcn_exp2f((s_z[i] - zm) * c);
      }
    psum = wave_sum(psum);
    own = wave_sum(own);
    const float norm = a.lse ? 0.f : logf(psum);
    for (int i = tid; i < k; i += 64)
      if (s_idx[i] >= 0) {
        const float logp = a.lse ? s_p[i] * itau - lse : (s_p[i] - tmax) * itau - norm;
        const float p = expf(logp);
        s_p[i] = p;
        if (p > 0.f || p != p) {
          A += p * logp;
          B += p * (s_z[i] - zm);
        }
      }
    A = wave_sum(A);
    B = wave_sum(B);
    if (tid == 0) teacher = Teacher{any, a.lse ? psum : 1.f, a.lse ? fmaxf(1.f - psum, 0.f) : 0.f, zm, own, A, B, dup};
  }

  // ---- the running maximum and sum outside S
  Sum tot{kLowest, 0.f};
  if constexpr (kMode != kFinish) {
    auto scalar = [&](int64_t j) {
      if (bits[(j - b0) >> 5] >> ((j - b0) & 31) & 1) return;
      tot = join(tot, Sum{Elem<kT>::get(z[j]), 1.f}, c);
    };
    auto vector = [&](int v, uint4 raw) {
      float x[n];
      unpack_vec<kT>(raw, x);
      const int b = v * n + 64;
      const uint32_t mask = (bits[b >> 5] >> (b & 31)) & ((1u << n) - 1);
      if (mask) {
#pragma unroll
        for (int i = 0; i < n; ++i) x[i] = (mask >> i & 1) ? -__builtin_inff() : x[i];
      }
      float m = tot.m;
#pragma unroll
      for (int i = 0; i < n; ++i) m = fmaxf(m, x[i]);
      float s = tot.s * __builtin_amdgcn_exp2f((tot.m - m) * c);
#pragma unroll
      for (int i = 0; i < n; ++i) s += __builtin_amdgcn_exp2f((x[i] - m) * c);
      tot = Sum{m, s};
    };
    if (first && tid < head) scalar(tid);
    if (last && tail0 + tid < a.V) scalar(tail0 + tid);
    if constexpr (kHold > 0) {
#pragma unroll
      for (int u = 0; u < kHold; ++u) {
        if (tid + u * kThreads < pv) vector(tid + u * kThreads, held[u]);
        // one vector unpacked at a time, and none of it kept for the second pass in place of the packed form
        asm("" : "+v"(held[u].x), "+v"(held[u].y), "+v"(held[u].z), "+v"(held[u].w));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (kStream) {
      int v = tid + kHold * kThreads;
      for (; v + 3 * kThreads < pv; v += 4 * kThreads) {
        uint4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = load(v + u * kThreads);
#pragma unroll
        for (int u = 0; u < 4; ++u) vector(v + u * kThreads, x[u]);
      }
      for (; v < pv; v += kThreads) vector(v, load(v));
    }
  } else {
    for (int i = tid; i < a.parts; i += kThreads) {
      const float2 st = a.stats[row * a.parts + i];
      tot = join(tot, Sum{st.x, st.y}, c);
    }
  }
  tot = block_join<kWaves>(tot, c, sh);
  if constexpr (kMode == kStats) {
    if (tid == 0) a.stats[row * a.parts + part] = make_float2(tot.m, tot.s);
    return;
  }

  // ---- loss and gradient
  if constexpr (kMode != kStats) {
    const Teacher tc = teacher;
    const bool live = tc.live > 0.f;
    const float big = fmaxf(tot.m, tc.zm);
    const float e_rest = __builtin_amdgcn_exp2f((tot.m - big) * c);
    const float total = tot.s * e_rest + tc.own * __builtin_amdgcn_exp2f((tc.zm - big) * c);
    // a rest that is the rounding of the sum is not held against a student with nothing outside S
    const float rest = tot.s == 0.f && tc.rest < 0x1p-16f ? 0.f : tc.rest;
    if (a.loss && first && tid == 0) {
      const float log_total = total == 0.f ? 0.f : logf(total);
      float l = tc.a + tc.psum * log_total, d = tc.psum * (big - tc.zm) - tc.b;
      if (rest > 0.f) {
        l += rest * (logf(rest) - logf(tot.s) + log_total);
        d += rest * (big - tot.m);
      }
      a.loss[row] = live ? a.tau * (a.tau * l + d) : 0.f;
    }
    if (!a.grad) return;
    const bool zero = !live || weight == 0.f || total == 0.f;
    const float P = a.lse ? tc.psum + rest : 1.f, scale = weight * a.tau;
    float f = 0.f;  // outside S: exp((z - m) / tau) f
    if (tot.s != 0.f) f = (P * e_rest / total - (rest > 0.f ? rest / tot.s : 0.f)) * scale;
    T* g = reinterpret_cast<T*>(a.grad) + row * a.ld_grad;
    const bool vec = (((uintptr_t)g ^ (uintptr_t)z) & 15) == 0;
    auto value = [&](float v) { return zero ? 0.f : __builtin_amdgcn_exp2f((v - tot.m) * c) * f; };
    if (!vec) {  // the gradient lies otherwise in its 16 bytes than the logits (so it is not in place)
      for (int64_t j = c0 + tid; j < c1; j += kThreads) g[j] = Elem<kT>::put(value(Elem<kT>::get(z[j])));
    } else {
      if (first && tid < head) g[tid] = Elem<kT>::put(value(Elem<kT>::get(z[tid])));
      if (last && tail0 + tid < a.V) g[tail0 + tid] = Elem<kT>::put(value(Elem<kT>::get(z[tail0 + tid])));
      char* const gp = reinterpret_cast<char*>(g + head + v0 * n);
      auto out = [&](int v, uint4 raw) {
        float x[n];
        unpack_vec<kT>(raw, x);
#pragma unroll
        for (int i = 0; i < n; ++i) x[i] = value(x[i]);
        store_codes<true>(reinterpret_cast<uint8_t*>(gp + (uint32_t)v * 16u), pack_vec<kT>(x));
      };
      if constexpr (kHold > 0) {
#pragma unroll
        for (int u = 0; u < kHold; ++u) {
          if (tid + u * kThreads < pv) out(tid + u * kThreads, held[u]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if constexpr (kStream) {
        int v = tid + kHold * kThreads;
        for (; v + 3 * kThreads < pv; v += 4 * kThreads) {
          uint4 x[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) x[u] = load(v + u * kThreads);
#pragma unroll
          for (int u = 0; u < 4; ++u) out(v + u * kThreads, x[u]);
        }
        for (; v < pv; v += kThreads) out(v, load(v));
      }
    }
    if (zero) return;
    __syncthreads();  // orders this workgroup's stores: S goes over them
    for (int i = tid; i < k; i += kThreads) {
      const int j = s_idx[i];
      if (j < c0 || j >= c1 || !s_first[i]) continue;
      float p = s_p[i];
      if (tc.dup != 0.f) {
        p = 0.f;
        for (int o = 0; o < k; ++o) p += s_idx[o] == j ? s_p[o] : 0.f;
      }
      g[j] = Elem<kT>::put((__builtin_amdgcn_exp2f((s_z[i] - big) * c) / total * P - p) * scale);
    }
  }
}

// Threads a workgroup: of a whole row of nv vectors, and of a piece
constexpr int64_t whole_threads(int64_t nv) { return nv <= 1024 ? 256 : nv <= 4096 ? 512 : 1024; }
constexpr int kSplitThreads = 512;

template <int kT>
void launch(const Args& a0, int64_t T, int stages, hipStream_t st) {
  Args a = a0;
  a.wgs = a.parts;
  const unsigned grid = (unsigned)(T * a.parts);
  const size_t entries = (size_t)a.k * 16;
  if (stages == (DISTILL_STATS | DISTILL_FINISH) && a.parts == 1) {
    const size_t lds = a.bit_words * 4 + entries;
    const int64_t nv = a.V / Vec<kT>::n, threads = whole_threads(nv);
    if (threads == 256) distill_kernel<kT, kWhole, 256, 4><<<grid, 256, lds, st>>>(a);
    else if (threads == 512) distill_kernel<kT, kWhole, 512, 8><<<grid, 512, lds, st>>>(a);
    else if (nv <= 8192) distill_kernel<kT, kWhole, 1024, 8><<<grid, 1024, lds, st>>>(a);
    else distill_kernel<kT, kWhole, 1024, 16><<<grid, 1024, lds, st>>>(a);
    return;
  }
  if (stages & DISTILL_STATS) distill_kernel<kT, kStats, kSplitThreads, 0><<<grid, kSplitThreads, a.bit_words * 4 + entries, st>>>(a);
  if (stages & DISTILL_FINISH) {
    a.wgs = a.grad ? a.parts : 1;
    a.bit_words = 0;
    distill_kernel<kT, kFinish, kSplitThreads, 0><<<(unsigned)(T * a.wgs), kSplitThreads, entries, st>>>(a);
  }
}

}  // namespace

// Splitting costs a launch and a second reading of the row, and pays where few long rows leave most CUs idle.  us with the
// gradient, whole / split: 16 rows of 128 KB 12.2 / 9.4 (16 pieces), of 496 KB 32 / 12.6; one row of 496 KB 31 / 10.2 (32);
// 64 rows of 128 KB 15.7 / 15.0, of 256 KB 20.0 / 13.4 (8), of 1 MB 46 / 37; 128 rows of 256 KB 24.3 / 22.2, of 1 MB 60 / 64;
// 16 rows of 32 KB 10.7 / 12.4.
extern "C" int64_t distill_parts(int64_t T, int64_t V, int64_t type) {
  if (T <= 0 || V <= 0) return 1;
  const int64_t bytes = V * (type == MXFP4_F32 ? 4 : 2);
  int64_t parts = 1;
  if (T <= 64 && bytes >= (T <= 16 ? 96 << 10 : 192 << 10))
    parts = std::min<int64_t>({32, std::max<int64_t>(256 / T, 8), bytes >> 13});  // pieces of 8 KB at least
  parts = std::max(parts, (V + kMaxPiece - 1) / kMaxPiece);
  return std::min<int64_t>(parts, DISTILL_MAX_PARTS);
}

extern "C" int64_t distill_workspace_size(int64_t T, int64_t k, int64_t parts) {
  return T <= 0 || k <= 0 || parts <= 0 ? 0 : T * parts * 8 + T * k * 8;
}

extern "C" int distill_topk_kl(const void* logits, int64_t type, int64_t ld, int64_t T, int64_t V, const void* idx,
                               int64_t idx_bytes, int64_t ld_idx, const float* t, int64_t ld_t, int64_t k, float tau,
                               const float* lse, const float* weight, float* loss, void* grad, int64_t ld_grad,
                               int64_t parts, int64_t stages, void* ws, void* stream) {
  MX_CHECK_ARG(T >= 0 && V > 0 && V < (1LL << 31) - 1 && ld >= 0, "distill_topk_kl: bad shape (T=%lld V=%lld ld=%lld)",
               (long long)T, (long long)V, (long long)ld);
  MX_CHECK_ARG(type >= MXFP4_BF16 && type <= MXFP4_F32, "distill_topk_kl: unknown element type %lld", (long long)type);
  MX_CHECK_ARG(k >= 1 && k <= DISTILL_MAX_K, "distill_topk_kl: 1 to %d teacher entries a row (k=%lld)", DISTILL_MAX_K,
               (long long)k);
  MX_CHECK_ARG(idx_bytes == 4 || idx_bytes == 8, "distill_topk_kl: 32- or 64-bit indices");
  MX_CHECK_ARG(tau > 0.f && tau < __builtin_inff(), "distill_topk_kl: the temperature has to be positive");
  MX_CHECK_ARG(parts >= 1 && parts <= DISTILL_MAX_PARTS && stages >= 1 && stages <= 3, "distill_topk_kl: bad plan");
  if (T == 0) return MXFP8_OK;
  const bool whole = stages == 3 && parts == 1;
  MX_CHECK_ARG(T < (1LL << 31) && T * parts * (whole ? whole_threads(V / (type == MXFP4_F32 ? 4 : 8)) : kSplitThreads) < (1LL << 32),
               "distill_topk_kl: more rows than one launch has threads for (T=%lld)", (long long)T);
  MX_CHECK_ARG(logits && idx && t && (whole || ws) && (loss || grad || stages == DISTILL_STATS),
               "distill_topk_kl: null pointer");
  MX_CHECK_ARG(!grad || ld_grad >= V, "distill_topk_kl: bad gradient stride");
  const int es = type == MXFP4_F32 ? 4 : 2;
  MX_CHECK_ARG(mx_aligned(logits, es) && mx_aligned(grad, es) && mx_aligned(idx, idx_bytes) && mx_aligned(ws, 8),
               "distill_topk_kl: misaligned buffer");
  const int64_t n = 16 / es, nv = V / n, piece = std::max<int64_t>((nv + parts - 1) / parts, 1);
  MX_CHECK_ARG(piece * n <= kMaxPiece + 8, "distill_topk_kl: too few parts");
  const Args a{logits, ld, V, idx, idx_bytes == 8, ld_idx, t, ld_t, (int)k, tau, lse, weight, loss, grad, ld_grad, (int)parts,
               0, piece, (int)((piece * n + 64 + 8) / 32 + 2),  // a piece's columns, 64 before it, the tail
               (float2*)ws, ws ? (float2*)((char*)ws + T * parts * 8) : nullptr};
  const hipStream_t st = (hipStream_t)stream;
  if (type == MXFP4_BF16) launch<MXFP4_BF16>(a, T, (int)stages, st);
  else if (type == MXFP4_F16) launch<MXFP4_F16>(a, T, (int)stages, st);
  else launch<MXFP4_F32>(a, T, (int)stages, st);
  MX_CHECK_LAUNCH("distill_topk_kl");
  return MXFP8_OK;
}
