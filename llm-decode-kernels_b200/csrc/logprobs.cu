// Log probabilities of given tokens, the entropy of each row's distribution and its top alternatives, in one pass
// over the logits. With m = max x, y = (x - m) log2(e), s = sum 2^y and w = sum 2^y y:
//   log p(t) = (x_t - m) - ln s        entropy = ln 2 (log2 s - w / s)
// Neither subtracts two large numbers of the row's own size, so fp32 keeps both to a few units in the last place.
// The maximum, s and w run along (rescaled when the maximum grows), so the row is read once.
//
// The top alternatives (by value, ties to the lowest index) come from the same pass: an element is a candidate when
// it is not below a threshold that at least `top` elements of the row reach. The first tile gives one (the r-th
// largest of the lanes' maxima in each of A warps, r A >= top, and of those the smallest), so that a few dozen
// candidates of a long row go to a small list in shared memory. A full list is cut to its `top` best, which raises
// the threshold. The order in which candidates arrive changes nothing: selection ranks (value, index) pairs.
//
// Memory bound: one 16-byte load per 8 (fp32: 4) logits. Rows are split over a cluster of CTAs when there are few
// of them; the parts meet in the first CTA's shared memory.
#include <algorithm>

#include "paged.cuh"

namespace dk {
namespace {

using paged::Elem;
using paged::exp2_approx;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kVecs = 4;    // vectors a thread loads at once
constexpr int kCap = 1024;  // candidates the list holds
constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 8;

struct LogprobParams {
  const void* logits;
  int64_t ld;
  const int64_t* targets;
  float* logprob;
  float* entropy;
  float* top_logprob;
  int64_t* top_id;
  int64_t V;
  int M, top;
  int* err;
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Order of the values as unsigned numbers: NaN above everything (as in a descending sort), -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return __int_as_float(0x7fc00000);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t candidate(float x, int64_t index) {
  return (static_cast<uint64_t>(order_key(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(index));
}

template <typename T>
struct Vec {
  static constexpr int kN = 16 / sizeof(T);
  float x[kN];
  __device__ void set(uint4 v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Elem<T>::unpack(w[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      }
    }
  }
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

struct Stats {
  float m, s, w;
  // Adds (m2, s2, w2), whose sums are relative to its own maximum.
  __device__ void join(float m2, float s2, float w2) {
    const float n = fmaxf(m, m2);
    const float base = n == -INFINITY ? 0.f : n;
    move(base);
    const float d2 = fmaxf((m2 - base) * 1.44269504088896341f, -200.f), c2 = exp2_approx(d2);
    s = fmaf(s2, c2, s);
    w = fmaf(c2, fmaf(s2, d2, w2), w);
    m = n;
  }
  // Sums relative to `base` >= m. A maximum far below the new one (or none yet, -inf) leaves 0.
  __device__ void move(float base) {
    const float d = fmaxf((m - base) * 1.44269504088896341f, -200.f), c = exp2_approx(d);
    w = c * fmaf(s, d, w);
    s *= c;
  }
};

template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads, 2) logprob_kernel(const LogprobParams p) {
  constexpr int kN = Vec<T>::kN;
  __shared__ uint64_t list[kTop ? kCap : 1];
  __shared__ uint64_t best[kTop ? kMaxTop : 1];                // this CTA's selection, best first
  __shared__ uint64_t all_best[kTop ? kMaxCluster * kMaxTop : 1];
  __shared__ float stat[kWarps * 3], cta_stat[3];
  __shared__ float warp_thr[kWarps];
  __shared__ int count, n_best;
  __shared__ uint64_t thr_key;  // candidates have to be above this pair
  const uint32_t C = gridDim.y, rank = blockIdx.y;
  const int row = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_trigger();
  pdl_wait();
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  // Vectors of 16 aligned bytes that hold the row: the first and the last may be partly outside it.
  const uintptr_t a0 = reinterpret_cast<uintptr_t>(x) & ~uintptr_t(15);
  const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(x) - a0) / sizeof(T));
  const int64_t nvec = (skip + p.V + kN - 1) / kN;
  const int64_t share = (nvec + C - 1) / C;
  const int64_t v0 = min(rank * share, nvec), v1 = min(v0 + share, nvec);
  const uint4* base = reinterpret_cast<const uint4*>(a0);
  if (tid == 0) count = 0, thr_key = 0;

  auto fetch = [&](int64_t v, Vec<T>& out) {
    const int64_t e0 = v * kN - skip;  // row index of the vector's first element
    if (v < v1 && e0 >= 0 && e0 + kN <= p.V) {
      out.set(__ldcs(base + v));
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i)
        out.x[i] = v < v1 && e0 + i >= 0 && e0 + i < p.V ? to_float(x[e0 + i]) : -INFINITY;
    }
  };

  Stats st{-INFINITY, 0.f, 0.f};
  float thr = -INFINITY;
  for (int64_t t0 = v0; t0 < v1; t0 += kThreads * kVecs) {
    Vec<T> v[kVecs];
    float vmax[kVecs], top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) fetch(t0 + u * kThreads + tid, v[u]);
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      vmax[u] = v[u].x[0];
#pragma unroll
      for (int i = 1; i < kN; ++i) vmax[u] = max_nan(vmax[u], v[u].x[i]);
      top = max_nan(top, vmax[u]);
    }
    if (top > st.m) {
      st.move(top);
      st.m = top;
    }
    const float shift = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const float y = max_nan((v[u].x[i] - shift) * 1.44269504088896341f, -200.f);  // 2^-200 is 0 here
        const float e = exp2_approx(y);
        st.s += e;
        st.w = fmaf(e, y, st.w);
      }
    }
    if constexpr (kTop) {
      if (t0 == v0) {  // the first threshold
        const int64_t nv = min(v1 - v0, static_cast<int64_t>(kThreads * kVecs));
        const int A = max(1, min(kWarps, static_cast<int>(nv / 32)));
        const int r = (p.top + A - 1) / A;
        if (warp < A) {
          uint32_t key = order_key(top), kth = 0;
          for (int i = 0; i < min(r, 32); ++i) {
            kth = __reduce_max_sync(0xffffffffu, key);
            const unsigned who = __ballot_sync(0xffffffffu, key == kth);
            if (lane == __ffs(who) - 1) key = 0;
          }
          if (lane == 0) warp_thr[warp] = r > 32 ? -INFINITY : key_value(kth);
        }
        __syncthreads();
        thr = warp_thr[0];
        for (int i = 1; i < A; ++i) thr = fminf(thr, warp_thr[i]);
        if (thr != thr) thr = INFINITY;  // NaN rows: only NaN (and +inf) pass
      }
      unsigned pending = 0;  // a bit for each of this thread's vectors that may hold candidates
#pragma unroll
      for (int u = 0; u < kVecs; ++u)
        if (!(vmax[u] < thr)) pending |= 1u << u;
      unsigned done[kVecs] = {};
      for (;;) {
        const uint64_t floor_key = thr_key;
        bool left = false;
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
          if (!(pending >> u & 1)) continue;
          const int64_t e0 = (t0 + u * kThreads + tid) * kN - skip;
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            if (v[u].x[i] < thr || (done[u] >> i & 1) || e0 + i < 0 || e0 + i >= p.V || t0 + u * kThreads + tid >= v1)
              continue;
            const uint64_t c = candidate(v[u].x[i], e0 + i);
            if (c <= floor_key) continue;
            const int at = atomicAdd(&count, 1);
            if (at < kCap) {
              list[at] = c;
              done[u] |= 1u << i;
            } else {
              left = true;
            }
          }
        }
        if (!__syncthreads_or(left)) break;
        // the list is full: keep its `top` best
        uint64_t mine[kCap / kThreads];
        int place[kCap / kThreads];
#pragma unroll
        for (int j = 0; j < kCap / kThreads; ++j) {
          mine[j] = list[tid + j * kThreads];
          int better = 0;
          for (int i = 0; i < kCap; ++i) better += list[i] > mine[j];
          place[j] = better;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kCap / kThreads; ++j)
          if (place[j] < p.top) {
            list[place[j]] = mine[j];
            if (place[j] == p.top - 1) thr_key = mine[j];
          }
        if (tid == 0) count = p.top;
        __syncthreads();
        thr = key_value(static_cast<uint32_t>(thr_key >> 32));
        if (thr != thr) thr = INFINITY;
      }
    }
  }

  // ---------------------------------------------------------------- this CTA's sums and selection
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st.join(__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
            __shfl_xor_sync(0xffffffffu, st.w, o));
  if (lane == 0) stat[3 * warp] = st.m, stat[3 * warp + 1] = st.s, stat[3 * warp + 2] = st.w;
  __syncthreads();
  if constexpr (kTop) {
    const int n = count;
    for (int c = tid; c < n; c += kThreads) {
      const uint64_t mine = list[c];
      int better = 0;
      for (int i = 0; i < n; ++i) better += list[i] > mine;
      if (better < p.top) best[better] = mine;
    }
    if (tid == 0) n_best = min(n, p.top);
  }
  if (warp == 0) {
    Stats s{-INFINITY, 0.f, 0.f};
    if (lane < kWarps) s = Stats{stat[3 * lane], stat[3 * lane + 1], stat[3 * lane + 2]};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      s.join(__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.s, o),
             __shfl_xor_sync(0xffffffffu, s.w, o));
    if (lane == 0) cta_stat[0] = s.m, cta_stat[1] = s.s, cta_stat[2] = s.w;
  }
  if (C > 1)
    cluster_sync();
  else
    __syncthreads();
  if (rank == 0) {
    Stats s{cta_stat[0], cta_stat[1], cta_stat[2]};
    for (uint32_t q = 1; q < C; ++q)
      s.join(ld_shared_cluster_f32(map_shared_rank(&cta_stat[0], q)), ld_shared_cluster_f32(map_shared_rank(&cta_stat[1], q)),
             ld_shared_cluster_f32(map_shared_rank(&cta_stat[2], q)));
    const float ln_s = logf(s.s);
    if (tid == 0) {
      const int64_t t = p.targets[row];
      float lp = 0.f;
      if (t >= p.V) {
        record_device_error(p.err, DK_DEVERR_BAD_TOKEN);
        lp = __int_as_float(0x7fc00000);
      } else if (t >= 0) {
        lp = (to_float(x[t]) - s.m) - ln_s;
      }
      p.logprob[row] = lp;
      p.entropy[row] = 0.693147180559945309f * (log2f(s.s) - s.w / s.s);
    }
    if constexpr (kTop) {
      auto put = [&](int place, uint64_t c) {
        p.top_logprob[static_cast<int64_t>(row) * p.top + place] = (key_value(static_cast<uint32_t>(c >> 32)) - s.m) - ln_s;
        p.top_id[static_cast<int64_t>(row) * p.top + place] = 0xffffffffu - static_cast<uint32_t>(c);
      };
      if (C == 1) {
        if (tid < p.top) put(tid, best[tid]);
      } else {
        for (int e = tid; e < static_cast<int>(C) * kMaxTop; e += kThreads) {
          const uint32_t q = e / kMaxTop, i = e % kMaxTop;
          int nq;
          asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(nq) : "r"(map_shared_rank(&n_best, q)) : "memory");
          uint64_t c = 0;
          if (static_cast<int>(i) < nq)
            asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(c) : "r"(map_shared_rank(&best[i], q)) : "memory");
          all_best[e] = c;
        }
        __syncthreads();
        for (int e = tid; e < static_cast<int>(C) * kMaxTop; e += kThreads) {
          const uint64_t mine = all_best[e];
          if (mine == 0) continue;
          int better = 0;
          for (int i = 0; i < static_cast<int>(C) * kMaxTop; ++i) better += all_best[i] > mine;
          if (better < p.top) put(better, mine);
        }
      }
    }
  }
  if (C > 1) cluster_sync();  // the first CTA has read the others' shared memory
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" int dk_token_logprobs(const void* logits, int64_t ld, int32_t dtype, const int64_t* targets, int64_t M, int64_t V,
                                 int64_t top, float* logprob, float* entropy, float* top_logprob, int64_t* top_id,
                                 dk_stream_t stream) {
  if (M < 0 || V <= 0 || top < 0 || ld < V) return set_error(DK_ERR_INVALID, "token_logprobs: bad sizes");
  if (top > kMaxTop || top > V)
    return set_error(DK_ERR_UNSUPPORTED, "token_logprobs: %lld alternatives (at most %d and the vocabulary)", (long long)top,
                     kMaxTop);
  if (dtype != DK_F16 && dtype != DK_BF16 && dtype != DK_F32)
    return set_error(DK_ERR_UNSUPPORTED, "token_logprobs: dtype %d", dtype);
  if (M > INT32_MAX || V >= INT32_MAX) return set_error(DK_ERR_INVALID, "token_logprobs: sizes must fit 31 bits");
  if (M == 0) return DK_OK;
  if (!logits || !targets || !logprob || !entropy || (top > 0 && (!top_logprob || !top_id)))
    return set_error(DK_ERR_INVALID, "token_logprobs: NULL pointer");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == DK_F32 ? 4 : 2))
    return set_error(DK_ERR_ALIGN, "token_logprobs: logits are not aligned to their type");
  LogprobParams p{logits, ld, targets, logprob, entropy, top_logprob, top_id, V, static_cast<int>(M), static_cast<int>(top),
                  device_info().err_word};
  // CTAs per row: while the rows alone leave SMs without one, and a CTA still gets a tile's worth of vectors
  const int64_t tile = static_cast<int64_t>(kThreads) * kVecs * (dtype == DK_F32 ? 4 : 8);
  int C = 1;
  while (C < kMaxCluster && M * C * 2 <= device_info().num_sms && V >= C * tile / 2) C *= 2;
  const dim3 grid(static_cast<unsigned>(M), static_cast<unsigned>(C));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
#define DK_LOGPROB(TT)                                                                                                \
  e = top > 0 ? launch(logprob_kernel<TT, true>, grid, dim3(kThreads), 0, st, pdl_enabled(), dim3(1, C, 1), p)        \
              : launch(logprob_kernel<TT, false>, grid, dim3(kThreads), 0, st, pdl_enabled(), dim3(1, C, 1), p)
  if (dtype == DK_F16)
    DK_LOGPROB(__half);
  else if (dtype == DK_BF16)
    DK_LOGPROB(__nv_bfloat16);
  else
    DK_LOGPROB(float);
#undef DK_LOGPROB
  if (e != cudaSuccess) return set_error(DK_ERR_CUDA, "token_logprobs launch: %s", cudaGetErrorString(e));
  return DK_OK;
}
