// Distillation from a teacher's top logits: loss and gradient of a row of logits [V] against the teacher's k entries.
//
// Mathematics, with a = z / tau, q = softmax(a), S the row's entries and p the teacher's masses on them:
//   loss = tau^2 (sum_S p (log p - log q) + p_r (log p_r - log q_r)),   q_r = sum of q outside S
//   d loss / d z_j = tau (q_j P - p_j) on S, P = sum p + p_r;  tau q_j (P - p_r / q_r) elsewhere
// Without the rest bucket p_r = 0.  One pass over the row keeps a running maximum m and the sum s of exp((z - m) / tau) in
// fp32; with the bucket it leaves out S (a bit for every column in LDS), so that q_r comes from its own maximum and sum and
// not from a difference.  The factors exp((m - M) / tau) / sum and p_r / s that the gradient needs are at most 1 each.
// z - m is taken before the division by tau: rows of the type's lowest value stay uniform.
//
// What bounds it: memory, the logits read once and the gradient written once.  A workgroup takes a row (its second reading
// comes from the cache); few rows are split into pieces over two launches, joined by the second.
#include <algorithm>

#include "abi_common.h"
#include "mx4_device.h"

using namespace mx4;

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kMaxPiece = 1 << 18;  // columns of a piece with the rest bucket: its bits take 32 KB

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
  int wgs;        // workgroups of a row in this launch: parts, or 1 for the loss alone
  int64_t piece;  // vectors of a piece
  float2* stats;  // [T][parts]
  float* zs;      // [T][k] logits of the entries
};

struct Sum {
  float m, s;  // s = sum of exp((z - m) / tau)
};
__device__ __forceinline__ Sum join(Sum a, Sum b, float c) {
  const float m = fmaxf(a.m, b.m);
  return Sum{m, a.s * __builtin_amdgcn_exp2f((a.m - m) * c) + b.s * __builtin_amdgcn_exp2f((b.m - m) * c)};
}

template <class F>
__device__ __forceinline__ float wave_reduce(float v, F f) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = f(v, __shfl_xor(v, o));
  return v;
}
template <class F>
__device__ __forceinline__ float block_reduce(float v, F f, float* sh) {
  v = wave_reduce(v, f);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = sh[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) r = f(r, sh[w]);
  return r;
}
__device__ __forceinline__ Sum block_join(Sum a, float c, float* sh) {
#pragma unroll
  for (int o = 32; o; o >>= 1) a = join(a, Sum{__shfl_xor(a.m, o), __shfl_xor(a.s, o)}, c);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    sh[threadIdx.x >> 6] = a.m;
    sh[kWaves + (threadIdx.x >> 6)] = a.s;
  }
  __syncthreads();
  Sum r{sh[0], sh[kWaves]};
#pragma unroll
  for (int w = 1; w < kWaves; ++w) r = join(r, Sum{sh[w], sh[kWaves + w]}, c);
  return r;
}
__device__ __forceinline__ float fadd(float a, float b) { return a + b; }
__device__ __forceinline__ float fmax2(float a, float b) { return fmaxf(a, b); }

template <int kT>
struct Vec {
  static constexpr int n = kT == MXFP4_F32 ? 4 : 8;  // elements of 16 bytes
};
template <int kT>
__device__ __forceinline__ void load_vec(const typename Elem<kT>::T* p, float* v) {
  if constexpr (kT == MXFP4_F32) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i];
  } else {
    load8<kT>(p, v);
  }
}

// kStats: the running maximum and sum of this workgroup's piece.  kFinish: loss and gradient, from the sums of all pieces.
// Both: the piece is the whole row and nothing passes through memory.
template <int kT, bool kRest, bool kStats, bool kFinish>
__global__ __launch_bounds__(kThreads) void distill_kernel(const Args a) {
  typedef typename Elem<kT>::T T;
  constexpr int n = Vec<kT>::n;
  extern __shared__ uint32_t bits[];  // a bit for every column of the piece: S
  __shared__ int s_idx[DISTILL_MAX_K];
  __shared__ float s_z[DISTILL_MAX_K], s_p[DISTILL_MAX_K];
  __shared__ float sh[2 * kWaves];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / (uint32_t)a.wgs;
  const int part = (int)(blockIdx.x - row * a.wgs);
  const T* z = reinterpret_cast<const T*>(a.z) + row * a.ld;
  const float c = kLog2e / a.tau;
  const float weight = a.weight ? a.weight[row] : 1.f;

  // ---- the teacher's entries; s_idx < 0: padding
  float tmax = kLowest;
  for (int i = tid; i < a.k; i += kThreads) {
    const int64_t o = row * a.ld_idx + i;
    const int64_t j = a.idx8 ? reinterpret_cast<const int64_t*>(a.idx)[o] : (int64_t)reinterpret_cast<const int32_t*>(a.idx)[o];
    const float t = a.t[row * a.ld_t + i];
    const bool ok = j >= 0 && j < a.V && !(t == -__builtin_inff());
    s_idx[i] = ok ? (int)j : -1;
    s_p[i] = t;
    if (ok) {
      tmax = (t > tmax || t != t) ? t : tmax;
      s_z[i] = kStats ? Elem<kT>::get(z[j]) : a.zs[row * a.k + i];
    }
  }
  float any = 0.f;
  for (int i = tid; i < a.k; i += kThreads) any = s_idx[i] >= 0 ? 1.f : any;
  const bool live = block_reduce(any, fmax2, sh) > 0.f;  // block_reduce's barriers publish s_idx, s_z, s_p

  // the row's vectors: `head` elements before the first aligned one, this workgroup's vectors [v0, v1), a tail
  const int head = (int)min((int64_t)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(T), a.V);
  const int64_t nv = (a.V - head) / n;
  const int64_t v0 = min((int64_t)part * a.piece, nv), v1 = min(v0 + a.piece, nv);
  const bool first = part == 0, last = part == a.parts - 1;
  const int64_t tail0 = head + nv * n;
  // columns of this workgroup: [c0, c1)
  const int64_t c0 = first ? 0 : head + v0 * n, c1 = last ? a.V : head + v1 * n;

  Sum tot{kLowest, 0.f};
  if constexpr (kStats) {
    if (live) {
      // bit b of the piece: column head + v0 n - 8 + b, so that a vector's bits lie in one byte
      const int64_t b0 = head + v0 * n - 8;
      if constexpr (kRest) {
        const int words = (int)((c1 - b0 + 31) >> 5);
        for (int i = tid; i < words; i += kThreads) bits[i] = 0;
        __syncthreads();
        for (int i = tid; i < a.k; i += kThreads)
          if (s_idx[i] >= c0 && s_idx[i] < c1) atomicOr(&bits[(s_idx[i] - b0) >> 5], 1u << ((s_idx[i] - b0) & 31));
        __syncthreads();
      }
      auto take = [&](float v) {
        const float m = fmaxf(tot.m, v);
        tot.s = tot.s * __builtin_amdgcn_exp2f((tot.m - m) * c) + __builtin_amdgcn_exp2f((v - m) * c);
        tot.m = m;
      };
      auto scalar = [&](int64_t j) {
        if constexpr (kRest) {
          if (bits[(j - b0) >> 5] >> ((j - b0) & 31) & 1) return;
        }
        take(Elem<kT>::get(z[j]));
      };
      if (first && tid < head) scalar(tid);
      if (last && tail0 + tid < a.V) scalar(tail0 + tid);
      auto vector = [&](int64_t v, float* x) {
        if constexpr (kRest) {
          const int64_t b = (v - v0) * n + 8;
          const uint32_t mask = (bits[b >> 5] >> (b & 31)) & ((1u << n) - 1);
          if (mask) {
#pragma unroll
            for (int i = 0; i < n; ++i) x[i] = (mask >> i & 1) ? -__builtin_inff() : x[i];
          }
        }
        float m = tot.m;
#pragma unroll
        for (int i = 0; i < n; ++i) m = fmaxf(m, x[i]);
        float s = tot.s * __builtin_amdgcn_exp2f((tot.m - m) * c);
#pragma unroll
        for (int i = 0; i < n; ++i) s += __builtin_amdgcn_exp2f((x[i] - m) * c);
        tot = Sum{m, s};
      };
      int64_t v = v0 + tid;
      for (; v + 3 * kThreads < v1; v += 4 * kThreads) {
        float x[4][n];
#pragma unroll
        for (int u = 0; u < 4; ++u) load_vec<kT>(z + head + (v + u * kThreads) * n, x[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) vector(v + u * kThreads, x[u]);
      }
      for (; v < v1; v += kThreads) {
        float x[n];
        load_vec<kT>(z + head + v * n, x);
        vector(v, x);
      }
      tot = block_join(tot, c, sh);
    }
    if constexpr (!kFinish) {
      if (tid == 0) a.stats[row * a.parts + part] = make_float2(tot.m, tot.s);
      if (first)
        for (int i = tid; i < a.k; i += kThreads)
          if (s_idx[i] >= 0) a.zs[row * a.k + i] = s_z[i];
      return;
    }
  }
  if constexpr (kFinish) {
    const bool zero_grad = !live || weight == 0.f;
    float f = 0.f, big = 0.f, P = 1.f, log_sum = 0.f, scale = 0.f;
    if (live) {
      if constexpr (!kStats) {
        for (int i = tid; i < a.parts; i += kThreads) {
          const float2 st = a.stats[row * a.parts + i];
          tot = join(tot, Sum{st.x, st.y}, c);
        }
        tot = block_join(tot, c, sh);
      }
      // masses of the teacher; entries that repeat an earlier one's column count once in q
      tmax = block_reduce(tmax, [](float x, float y) { return (x > y || x != x) ? x : y; }, sh);
      const float lse = a.lse ? a.lse[row] : 0.f, itau = 1.f / a.tau;
      float psum = 0.f;
      for (int i = tid; i < a.k; i += kThreads)
        if (s_idx[i] >= 0)
          psum += kRest ? expf(s_p[i] * itau - lse) : __builtin_amdgcn_exp2f((s_p[i] - tmax) * c);
      psum = block_reduce(psum, fadd, sh);
      // a rest that is the rounding of the sum is not held against a student with nothing outside S
      float p_rest = kRest ? fmaxf(1.f - psum, 0.f) : 0.f;
      if (kRest && tot.s == 0.f && p_rest < 0x1p-16f) p_rest = 0.f;
      P = kRest ? psum + p_rest : 1.f;
      big = tot.m;
      float total = tot.s;
      if constexpr (kRest) {
        float zm = kLowest;
        for (int i = tid; i < a.k; i += kThreads)
          if (s_idx[i] >= 0) zm = fmaxf(zm, s_z[i]);
        big = fmaxf(big, block_reduce(zm, fmax2, sh));
        float own = 0.f;
        for (int i = tid; i < a.k; i += kThreads) {
          if (s_idx[i] < 0) continue;
          bool again = false;
          for (int o = 0; o < i; ++o) again |= s_idx[o] == s_idx[i];
          if (!again) own += __builtin_amdgcn_exp2f((s_z[i] - big) * c);
        }
        own = block_reduce(own, fadd, sh);
        total = own + tot.s * __builtin_amdgcn_exp2f((tot.m - big) * c);
      }
      log_sum = total == 0.f ? 0.f : logf(total);
      // loss
      float part_loss = 0.f;
      for (int i = tid; i < a.k; i += kThreads) {
        if (s_idx[i] < 0) continue;
        const float logp = kRest ? s_p[i] * itau - lse : (s_p[i] - tmax) * itau - logf(psum);
        const float logq = total == 0.f ? -__builtin_inff() : (s_z[i] - big) * itau - log_sum;
        const float p = expf(logp);
        if (p > 0.f || p != p) part_loss += p * (logp - logq);
      }
      part_loss = block_reduce(part_loss, fadd, sh);
      if (kRest && p_rest > 0.f)
        part_loss += p_rest * (logf(p_rest) - ((tot.m - big) * itau + logf(tot.s) - log_sum));
      if (a.loss && first && tid == 0) a.loss[row] = part_loss * a.tau * a.tau;
      // gradient outside S: exp((z - m) / tau) f
      scale = weight * a.tau;
      if (tot.s != 0.f) {
        f = P * __builtin_amdgcn_exp2f((tot.m - big) * c) / total;
        if (kRest) f -= p_rest / tot.s;
        f *= scale;
      }
      if (a.grad) {
        // s_p becomes the gradient on S, s_idx < 0 for the columns of other pieces and repeated entries
        __syncthreads();
        float gs[(DISTILL_MAX_K + kThreads - 1) / kThreads];
        int keep[(DISTILL_MAX_K + kThreads - 1) / kThreads];
#pragma unroll
        for (int r = 0; r < (DISTILL_MAX_K + kThreads - 1) / kThreads; ++r) {
          const int i = tid + r * kThreads;
          keep[r] = 0;
          if (i >= a.k || s_idx[i] < 0) continue;
          float p = 0.f;
          bool again = false;
          for (int o = 0; o < a.k; ++o)
            if (s_idx[o] == s_idx[i]) {
              again |= o < i;
              p += expf(kRest ? s_p[o] * itau - lse : (s_p[o] - tmax) * itau - logf(psum));
            }
          const float q = total == 0.f ? 0.f : __builtin_amdgcn_exp2f((s_z[i] - big) * c) / total;
          gs[r] = total == 0.f ? 0.f : (q * P - p) * scale;
          keep[r] = !again && s_idx[i] >= c0 && s_idx[i] < c1;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < (DISTILL_MAX_K + kThreads - 1) / kThreads; ++r) {
          const int i = tid + r * kThreads;
          if (i >= a.k) continue;
          if (!keep[r]) s_idx[i] = -1;
          s_p[i] = gs[r];
        }
      }
    } else if (a.loss && first && tid == 0) {
      a.loss[row] = 0.f;
    }
    if (!a.grad) return;
    T* g = reinterpret_cast<T*>(a.grad) + row * a.ld_grad;
    const bool vec = (((uintptr_t)g ^ (uintptr_t)z) & 15) == 0;
    auto value = [&](float v) { return zero_grad ? 0.f : __builtin_amdgcn_exp2f((v - tot.m) * c) * f; };
    if (first && tid < head) g[tid] = Elem<kT>::put(value(Elem<kT>::get(z[tid])));
    if (last && tail0 + tid < a.V) g[tail0 + tid] = Elem<kT>::put(value(Elem<kT>::get(z[tail0 + tid])));
    auto out = [&](int64_t v, float* x) {
#pragma unroll
      for (int i = 0; i < n; ++i) x[i] = value(x[i]);
      store_run<kT, n>(g, head + v * n, a.V, vec, x);
    };
    int64_t v = v0 + tid;
    for (; v + 3 * kThreads < v1; v += 4 * kThreads) {
      float x[4][n];
#pragma unroll
      for (int u = 0; u < 4; ++u) load_vec<kT>(z + head + (v + u * kThreads) * n, x[u]);
#pragma unroll
      for (int u = 0; u < 4; ++u) out(v + u * kThreads, x[u]);
    }
    for (; v < v1; v += kThreads) {
      float x[n];
      load_vec<kT>(z + head + v * n, x);
      out(v, x);
    }
    if (zero_grad) return;
    __syncthreads();  // this workgroup's stores have completed: S goes over them
    for (int i = tid; i < a.k; i += kThreads)
      if (s_idx[i] >= 0) g[s_idx[i]] = Elem<kT>::put(s_p[i]);
  }
}

template <int kT, bool kRest>
void launch(const Args& a, int64_t T, int stages, size_t lds, hipStream_t st) {
  Args b = a;
  b.wgs = a.parts;
  const unsigned grid = (unsigned)(T * a.parts);
  if (stages == (DISTILL_STATS | DISTILL_FINISH) && a.parts == 1) {
    distill_kernel<kT, kRest, true, true><<<grid, kThreads, lds, st>>>(b);
    return;
  }
  if (stages & DISTILL_STATS) distill_kernel<kT, kRest, true, false><<<grid, kThreads, lds, st>>>(b);
  if (stages & DISTILL_FINISH) {
    b.wgs = a.grad ? a.parts : 1;
    distill_kernel<kT, kRest, false, true><<<(unsigned)(T * b.wgs), kThreads, 0, st>>>(b);
  }
}

}  // namespace

extern "C" int64_t distill_parts(int64_t T, int64_t V, int64_t rest) {
  if (T <= 0 || V <= 0) return 1;
  int64_t parts = std::min((int64_t)1024 / T, V / 8192);
  if (rest) parts = std::max(parts, (V + kMaxPiece - 1) / kMaxPiece);
  return std::min<int64_t>(std::max<int64_t>(parts, 1), DISTILL_MAX_PARTS);
}

extern "C" int64_t distill_workspace_size(int64_t T, int64_t k, int64_t parts) {
  return T <= 0 || k <= 0 || parts <= 0 ? 0 : T * parts * 8 + T * k * 4;
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
  MX_CHECK_ARG(T * parts < (1LL << 31), "distill_topk_kl: too many rows");
  const bool whole = stages == 3 && parts == 1;
  MX_CHECK_ARG(logits && idx && t && (whole || ws) && (loss || grad || stages == DISTILL_STATS),
               "distill_topk_kl: null pointer");
  MX_CHECK_ARG(!grad || ld_grad >= V, "distill_topk_kl: bad gradient stride");
  const int es = type == MXFP4_F32 ? 4 : 2;
  MX_CHECK_ARG(mx_aligned(logits, es) && mx_aligned(grad, es) && mx_aligned(idx, idx_bytes) && mx_aligned(ws, 8),
               "distill_topk_kl: misaligned buffer");
  const int64_t n = 16 / es, nv = V / n;
  Args a{logits, ld, V, idx, idx_bytes == 8, ld_idx, t, ld_t, (int)k, tau, lse, weight, loss, grad, ld_grad, (int)parts, 0,
         std::max<int64_t>((nv + parts - 1) / parts, 1), (float2*)ws, ws ? (float*)((char*)ws + T * parts * 8) : nullptr};
  const bool rest = lse != nullptr;
  // a bit for every column of a piece, its head and tail
  const size_t lds = rest ? ((size_t)(a.piece * n + 8 + 64) / 32 + 2) * 4 : 0;
  MX_CHECK_ARG(!(rest && (stages & DISTILL_STATS)) || a.piece * n <= kMaxPiece + 8, "distill_topk_kl: too few parts");
  const hipStream_t st = (hipStream_t)stream;
#define RUN(T_) (rest ? launch<T_, true>(a, T, (int)stages, lds, st) : launch<T_, false>(a, T, (int)stages, lds, st))
  if (type == MXFP4_BF16) RUN(MXFP4_BF16);
  else if (type == MXFP4_F16) RUN(MXFP4_F16);
  else RUN(MXFP4_F32);
#undef RUN
  MX_CHECK_LAUNCH("distill_topk_kl");
  return MXFP8_OK;
}
