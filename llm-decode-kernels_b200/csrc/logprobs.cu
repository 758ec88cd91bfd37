// Log probabilities of given tokens, the entropy of each row's distribution and its top alternatives, in one pass
// over the logits. With m = max x, y = (x - m) log2(e), s = sum 2^y and w = sum 2^y y:
//   log p(t) = (x_t - m) - ln s        entropy = ln 2 (log2 s - w / s)
// s lies between 1 and V and no term of w is positive, so fp32 keeps both to a few units in the last place of ln s, and neither
// a positive log probability nor a negative entropy comes out.
// The maximum, s and w run along (rescaled when the maximum grows), so the row is read once.
//
// A thread takes 2^y relative to its base, the largest of the logits that it and the CTA's first tile have had. Once that
// tile is known few threads meet a larger one (of random logits, one of 256 threads a tile), so the common path only
// compares. (A base that may stay up to 40 below the maximum: 138.5 against 138.7 us for 2048 rows, and log probabilities of
// sure tokens up to 2e-6 above zero.)
//
// The top alternatives (by value, ties to the lowest index) come from the same pass. The `top`-th largest of the maxima that
// 64 groups of threads have seen is a threshold that `top` elements reach; it is taken after the first tile, again a few
// tiles later, and at the end. Vectors that hold something not below it are listed (a few hundred of 19008), and at the
// end opened against the last threshold (a few dozen elements), which are ranked by (value, index): the order in which
// they arrive changes nothing. -inf is not listed. A list that runs over (many equal logits), or is too short (fewer
// tokens allowed than asked for), falls back to a search for the `top`-th key over the CTA's part of the row: 16 more reads
// of it, from L2, counting the keys above three pivots.
// Bound by HBM, closely followed by the 16 exponentials a cycle that an SM computes (152064 x 2048 bf16 logits: 95 us of
// bytes, 66 us of exponentials at 1.97 GHz; measured 130 us, 4.8 TB/s, with the exponentials' pipe 62% and the issue slots 67%
// busy; 141 us under the power cap). Rows are split over a cluster of CTAs when there are few of them; the parts meet in the first
// CTA's shared memory.
#include <algorithm>
#include <cfloat>
#include <mutex>

#include "paged.cuh"

namespace dk {
namespace {

using paged::Elem;
using paged::exp2_approx;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kResident = 5;  // CTAs an SM holds (2048 rows of 152064 fp16: 124 us; 130 with 4)
constexpr int kGroups = kThreads / 4;
static_assert(kGroups == 64, "two maxima a lane");
constexpr int kRaiseTile = 3;  // at this tile the threshold is taken again from all seen so far
constexpr int kVecs = 4;     // vectors a thread loads at once
constexpr int kCap = 1024;   // candidates the list holds
constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.44269504088896341f;
// Logits below it (the type's lowest value in masks) count as this: just below -1e30, a value of bf16, so that elements
// clamped in any type and the least base are the same number.
constexpr float kLow = -0x1.94p99f;

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

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// 16 bytes of logits of type T.
template <typename T>
struct Vec {
  static constexpr int kN = 16 / sizeof(T);
  static constexpr int kPairs = kN / 2;
  uint4 v;
  __device__ uint32_t word(int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
  __device__ float2 pair(int i) const {
    if constexpr (sizeof(T) == 4)
      return make_float2(__uint_as_float(word(2 * i)), __uint_as_float(word(2 * i + 1)));
    else
      return Elem<T>::unpack(word(i));
  }
  __device__ float at(int i) const { return i & 1 ? pair(i / 2).y : pair(i / 2).x; }
  __device__ float max() const {  // NaN if there is one
    if constexpr (sizeof(T) == 4) {
      return max_nan(max_nan(at(0), at(1)), max_nan(at(2), at(3)));
    } else {
      uint32_t m;
      if constexpr (std::is_same<T, __half>::value)
        asm("{.reg .b32 a, b;\nmax.NaN.f16x2 a, %1, %2;\nmax.NaN.f16x2 b, %3, %4;\nmax.NaN.f16x2 %0, a, b;}"
            : "=r"(m) : "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
      else
        asm("{.reg .b32 a, b;\nmax.NaN.bf16x2 a, %1, %2;\nmax.NaN.bf16x2 b, %3, %4;\nmax.NaN.bf16x2 %0, a, b;}"
            : "=r"(m) : "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
      const float2 f = Elem<T>::unpack(m);
      return max_nan(f.x, f.y);
    }
  }
  __device__ static T none() {  // -inf
    if constexpr (sizeof(T) == 4)
      return -INFINITY;
    else if constexpr (std::is_same<T, __half>::value)
      return __ushort_as_half(0xfc00);
    else
      return __ushort_as_bfloat16(0xff80);
  }
  __device__ static uint4 none4() {
    constexpr uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    return make_uint4(w, w, w, w);
  }
  // What stands for -inf in sums, so that 0 * y is 0 for it.
  __device__ static constexpr float lowest() { return std::is_same<T, __half>::value ? -65504.f : kLow; }
  __device__ float2 finite_pair(int i) const {
    if constexpr (sizeof(T) == 4) {
      const float2 f = pair(i);
      return make_float2(max_nan(f.x, kLow), max_nan(f.y, kLow));
    } else if constexpr (std::is_same<T, __half>::value) {
      uint32_t m;
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(m) : "r"(word(i)), "r"(0xfbfffbffu));  // -65504
      return Elem<T>::unpack(m);
    } else {
      uint32_t m;
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(word(i)), "r"(0xf14af14au));  // kLow twice
      return Elem<T>::unpack(m);
    }
  }
};

__device__ __forceinline__ uint64_t bits2(float2 v) {
  return static_cast<uint64_t>(__float_as_uint(v.x)) | (static_cast<uint64_t>(__float_as_uint(v.y)) << 32);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return make_float2(__uint_as_float(static_cast<uint32_t>(d)), __uint_as_float(static_cast<uint32_t>(d >> 32)));
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return make_float2(__uint_as_float(static_cast<uint32_t>(d)), __uint_as_float(static_cast<uint32_t>(d >> 32)));
}

struct Stats {
  float m, s, w;  // sums relative to m
  // Adds (m2, s2, w2), whose sums are relative to its own base.
  __device__ void join(float m2, float s2, float w2) {
    const float n = fmaxf(m, m2);
    const float base = n == -INFINITY ? 0.f : n;
    move(base);
    const float d2 = fmaxf((m2 - base) * kLog2e, -200.f), c2 = exp2_approx(d2);
    s = fmaf(s2, c2, s);
    w = fmaf(c2, fmaf(s2, d2, w2), w);
    m = n;
  }
  // Sums relative to `base` >= m. A base far below the new one (or none yet, -inf) leaves 0.
  __device__ void move(float base) {
    const float d = fmaxf((m - base) * kLog2e, -200.f), c = exp2_approx(d);
    w = c * fmaf(s, d, w);
    s *= c;
  }
};

template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads, kResident) logprob_kernel(const LogprobParams p) {
  constexpr int kN = Vec<T>::kN;
  __shared__ uint64_t list[kTop ? kCap : 1];
  __shared__ uint64_t best[kTop ? kMaxTop : 1];                // this CTA's selection, best first
  __shared__ uint64_t all_best[kTop ? kMaxCluster * kMaxTop : 1];
  __shared__ float first_max[kGroups];
  __shared__ float stat[kWarps * 3], cta_stat[3];
  __shared__ int tally[kWarps * 3];
  __shared__ int vec_list[kTop ? kCap : 1], vec_count;  // vectors that hold candidates
  __shared__ int count, n_best;
  __shared__ float thr_sh;
  const uint32_t C = gridDim.y, rank = blockIdx.y;
  const int row = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_trigger();
  pdl_wait();
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  // Vectors of 16 aligned bytes that hold the row: the first and the last may be partly outside it.
  const uintptr_t a0 = reinterpret_cast<uintptr_t>(x) & ~uintptr_t(15);
  const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(x) - a0) / sizeof(T));
  const int V = static_cast<int>(p.V), nvec = (skip + V + kN - 1) / kN;
  const int share = (nvec + C - 1) / C;
  const int v0 = min(static_cast<int>(rank) * share, nvec), v1 = min(v0 + share, nvec);
  const uint4* vecs = reinterpret_cast<const uint4*>(a0);
  // Vectors of this part that lie wholly in the row; its at most two others are taken element by element.
  const int f0 = v0 * kN < skip ? v0 + 1 : v0, f1 = min(v1, (skip + V) / kN);
  if (tid == 0) count = vec_count = 0, thr_sh = -INFINITY;
  __syncthreads();

  // element i of vector v: -inf where it is outside the row
  auto fetch = [&](int v) {
    Vec<T> out;
    const int e0 = v * kN - skip;
    if (v >= f0 && v < f1) {
      out.v = __ldg(vecs + v);
    } else {
      T e[kN];
#pragma unroll
      for (int i = 0; i < kN; ++i) e[i] = v < v1 && e0 + i >= 0 && e0 + i < V ? x[e0 + i] : Vec<T>::none();
      out.v = *reinterpret_cast<const uint4*>(e);
    }
    return out;
  };
  auto outside = [&](int v, int i) { return v >= v1 || v * kN - skip + i < 0 || v * kN - skip + i >= V; };
  auto push = [&](float value, int index) {
    const int place = atomicAdd(&count, 1);
    if (place < kCap) list[place] = candidate(value, index);
  };

  float base = kLow, thr = -FLT_MAX;
  float run = -INFINITY;  // the largest logit this thread has seen (NaN: the largest, as in order_key)
  // Raises the threshold to the top-th largest of the maxima that 64 groups of four threads have seen; all threads. Returns
  // this lane's part of the largest of them, read before the second barrier: after it a warp ahead of the others may
  // already write the next round's maxima.
  auto raise_threshold = [&] {
    float group = max_nan(run, __shfl_xor_sync(0xffffffffu, run, 1));
    group = max_nan(group, __shfl_xor_sync(0xffffffffu, group, 2));
    if ((lane & 3) == 0) first_max[tid >> 2] = group;
    __syncthreads();
    const float top_max = fmaxf(first_max[lane], first_max[lane + 32]);
    if (kTop && tid < kGroups) {
      const float me = first_max[tid];
      int above = 0, reach = 0;
      for (int i = 0; i < kGroups; ++i) {
        above += !(first_max[i] <= me);
        reach += !(first_max[i] < me);
      }
      if (above < p.top && reach >= p.top && me == me) thr_sh = me;  // (all such threads hold the same value)
    }
    __syncthreads();
    if (kTop) thr = fmaxf(thr_sh, -FLT_MAX);  // (-inf is below any threshold)
    return top_max;
  };

  float2 s2 = make_float2(0.f, 0.f), w2 = s2;
  bool low = true;  // nothing above what stands for -inf in sums has set the base yet: -inf is told apart one by one
  int tile = 0;
  for (int t0 = f0; t0 < f1; t0 += kThreads * kVecs, ++tile) {
    Vec<T> v[kVecs];
    float vmax[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int at = t0 + u * kThreads + tid;
      v[u].v = at < f1 ? __ldg(vecs + at) : Vec<T>::none4();
    }
#pragma unroll
    for (int u = 0; u < kVecs; ++u) vmax[u] = v[u].max();
    const float mine = max_nan(max_nan(vmax[0], vmax[1]), max_nan(vmax[2], vmax[3]));
    run = max_nan(run, mine);
    if (tile == 0) {
      float top_max = raise_threshold();
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top_max = fmaxf(top_max, __shfl_xor_sync(0xffffffffu, top_max, o));
      low = !(top_max > Vec<T>::lowest());
      base = fmaxf(top_max, kLow);
    } else if (kTop && tile == kRaiseTile) {
      raise_threshold();
    }
    // Rare: a logit above the base, candidates
    if (mine > base) {
      Stats a{base, s2.x, w2.x}, b{base, s2.y, w2.y};
      base = mine;
      a.move(base), b.move(base);
      s2 = make_float2(a.s, b.s), w2 = make_float2(a.w, b.w);
    }
    if constexpr (kTop) {
      if (!(mine < thr)) {
#pragma unroll
        for (int u = 0; u < kVecs; ++u)
          if (!(vmax[u] < thr)) {
            const int place = atomicAdd(&vec_count, 1);
            if (place < kCap) vec_list[place] = t0 + u * kThreads + tid;
          }
      }
    }
    const float2 scale = make_float2(kLog2e, kLog2e), off = make_float2(-base, -base), zero = make_float2(-0.f, -0.f);
    if (!low) {
#pragma unroll
      for (int u = 0; u < kVecs; ++u)
#pragma unroll
        for (int i = 0; i < Vec<T>::kPairs; ++i) {
          const float2 y = fma2(add2(v[u].finite_pair(i), off), scale, zero);
          const float2 e = make_float2(exp2_approx(y.x), exp2_approx(y.y));
          s2 = add2(s2, e);
          w2 = fma2(e, y, w2);
        }
    } else {
      for (int u = 0; u < kVecs; ++u) {
        const Vec<T> q = u == 0 ? v[0] : u == 1 ? v[1] : u == 2 ? v[2] : v[3];
#pragma unroll
        for (int i = 0; i < Vec<T>::kPairs; ++i) {
          const float2 y = fma2(add2(q.finite_pair(i), off), scale, zero), f = q.pair(i);
          const float2 e = make_float2(f.x == -INFINITY ? 0.f : exp2_approx(y.x), f.y == -INFINITY ? 0.f : exp2_approx(y.y));
          s2 = add2(s2, e);
          w2 = fma2(e, y, w2);
        }
      }
    }
  }

  // ---------------------------------------------------------------- this CTA's sums and selection
  Stats st{f0 < f1 ? base : -INFINITY, s2.x + s2.y, w2.x + w2.y};
  if (tid < 2 * kN) {  // the row's ends outside whole vectors: a thread per element
    const int v = tid < kN ? v0 : v1 - 1;
    if (v0 < v1 && (v < f0 || v >= f1) && (tid < kN || v > v0) && !outside(v, tid % kN)) {
      const float f = to_float(x[v * kN - skip + tid % kN]);
      if (f != -INFINITY) {
        st.join(max_nan(f, kLow), 1.f, 0.f);
        if (f != f) st.s = f;
        run = max_nan(run, f);
        if constexpr (kTop)
          if (!(f < thr)) push(f, v * kN - skip + tid % kN);  // (with the loop's threshold: only more)
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st.join(__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
            __shfl_xor_sync(0xffffffffu, st.w, o));
  if (lane == 0) stat[3 * warp] = st.m, stat[3 * warp + 1] = st.s, stat[3 * warp + 2] = st.w;
  if constexpr (kTop)
    raise_threshold();
  else
    __syncthreads();
  if constexpr (kTop) {
    // The listed vectors are opened: what is not below the last threshold.
    const int listed = vec_count;
    for (int c = tid; c < min(listed, kCap); c += kThreads) {
      const Vec<T> q = fetch(vec_list[c]);
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (!(q.at(i) < thr)) push(q.at(i), vec_list[c] * kN - skip + i);
    }
    __syncthreads();
    const int here = max(0, min(V, v1 * kN - skip) - max(0, v0 * kN - skip));  // elements of this CTA's part
    const int want = min(p.top, here);
    int n = count;
    if (listed > kCap || n > kCap || n < want) {
      __syncthreads();
      // The want-th largest key: two bits at a time, the number of keys at or above three pivots.
      uint32_t kth = 0;
      for (int bit = 30; bit >= 0; bit -= 2) {
        int c[3] = {0, 0, 0};
        for (int v = v0 + tid; v < v1; v += kThreads) {
          const Vec<T> q = fetch(v);
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            const uint32_t k = outside(v, i) ? 0u : order_key(q.at(i));
#pragma unroll
            for (int j = 0; j < 3; ++j) c[j] += k >= (kth | (j + 1u) << bit);
          }
        }
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          const int w = __reduce_add_sync(0xffffffffu, c[j]);
          if (lane == 0) tally[3 * warp + j] = w;
        }
        __syncthreads();
        uint32_t digit = 0;
        for (int j = 0; j < 3; ++j) {
          int sum = 0;
          for (int w = 0; w < kWarps; ++w) sum += tally[3 * w + j];
          if (sum >= want) digit = j + 1;
        }
        kth |= digit << bit;
        __syncthreads();
      }
      // All keys above it, then those equal to it in order of index until there are enough.
      if (tid == 0) count = 0;
      __syncthreads();
      for (int v = v0 + tid; v < v1; v += kThreads) {
        const Vec<T> q = fetch(v);
#pragma unroll
        for (int i = 0; i < kN; ++i)
          if (!outside(v, i) && order_key(q.at(i)) > kth) list[atomicAdd(&count, 1)] = candidate(q.at(i), v * kN - skip + i);
      }
      __syncthreads();
      n = count;  // < want
      for (int t0 = v0; t0 < v1 && n < want; t0 += kThreads) {
        const Vec<T> q = fetch(t0 + tid);
        int equal = 0;
#pragma unroll
        for (int i = 0; i < kN; ++i) equal += !outside(t0 + tid, i) && order_key(q.at(i)) == kth;
        int before = equal;  // inclusive scan over the warp, then over the warps
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += u;
        }
        if (lane == 31) tally[warp] = before;
        __syncthreads();
        int all = 0, place = n + before - equal;
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) place += tally[w];
          all += tally[w];
        }
#pragma unroll
        for (int i = 0; i < kN; ++i)
          if (!outside(t0 + tid, i) && order_key(q.at(i)) == kth) {
            if (place < want) list[place] = candidate(q.at(i), (t0 + tid) * kN - skip + i);
            ++place;
          }
        n += all;
        __syncthreads();
      }
      n = want;
      __syncthreads();
    }
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
    auto logprob = [&](float value) {
      if (s.s == 0.f) return __int_as_float(0x7fc00000);  // no logit above -inf
      if (value == -INFINITY) return s.s == s.s ? value : s.s;
      return ((s.m > kLow ? value : max_nan(value, kLow)) - s.m) - ln_s;
    };
    if (tid == 0) {
      const int64_t t = p.targets[row];
      float lp = 0.f;
      if (t >= p.V) {
        record_device_error(p.err, DK_DEVERR_BAD_TOKEN);
        lp = __int_as_float(0x7fc00000);
      } else if (t >= 0) {
        lp = logprob(to_float(x[t]));
      }
      p.logprob[row] = lp;
      p.entropy[row] = fmaf(-0.693147180559945309f, s.w / s.s, ln_s);
    }
    if constexpr (kTop) {
      auto put = [&](int place, uint64_t c) {
        p.top_logprob[static_cast<int64_t>(row) * p.top + place] = logprob(key_value(static_cast<uint32_t>(c >> 32)));
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

// `per_sm`: CTAs of the launch for each SM, or 0 where most SMs stay idle anyhow. Where less than kResident are needed on
// each, dynamic shared memory that nothing uses keeps more than that away, so that all SMs get the same (148 rows, us: 16.6,
// 24.7 without).
template <typename T, bool kTop>
cudaError_t launch_logprobs(dim3 grid, int64_t per_sm, cudaStream_t st, const LogprobParams& p) {
  static std::mutex mu;
  static int limits[64];  // by device; 0: not asked yet
  auto kernel = logprob_kernel<T, kTop>;
  const DeviceInfo& device = device_info();
  int dev = 0, limit;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    int& known = limits[dev & 63];
    if (known == 0) known = opt_in_dynamic_smem(kernel);
    limit = known;
  }
  int64_t bytes = 0;
  if (per_sm > 0 && per_sm < kResident) {  // per_sm + 1 shall not fit
    const int64_t own = device.max_smem_optin - limit + 1024;  // static, and what the system takes for each CTA
    bytes = std::max<int64_t>(0, std::min<int64_t>(limit, device.smem_per_sm / (per_sm + 1) + 128 - own));
  }
  return launch(kernel, grid, dim3(kThreads), static_cast<size_t>(bytes), st, pdl_enabled(), dim3(1, grid.y, 1), p);
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
  if (M > INT32_MAX || V > INT32_MAX - 16) return set_error(DK_ERR_INVALID, "token_logprobs: sizes must fit 31 bits");
  if (M == 0) return DK_OK;
  if (!logits || !targets || !logprob || !entropy || (top > 0 && (!top_logprob || !top_id)))
    return set_error(DK_ERR_INVALID, "token_logprobs: NULL pointer");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == DK_F32 ? 4 : 2))
    return set_error(DK_ERR_ALIGN, "token_logprobs: logits are not aligned to their type");
  LogprobParams p{logits, ld, targets, logprob, entropy, top_logprob, top_id, V, static_cast<int>(M), static_cast<int>(top),
                  device_info().err_word};
  // CTAs per row (152064 fp16 logits, us): a row is split over up to 8 CTAs while each gets an SM of its own and a tile or
  // more (1 row: 16.3 on one, 9.8 on eight; 32 rows: 17.2 on one, 13.7 on four, 15.1 on eight), and over two while the
  // SMs take all of them at once and each has 4 tiles or more (148 rows: 17.7 and 16.4; 592 rows: 42.8 and 52.3).
  const int64_t tile = static_cast<int64_t>(kThreads) * kVecs * (dtype == DK_F32 ? 4 : 8), sms = device_info().num_sms;
  int C = 1;
  while (C < kMaxCluster && M * C * 2 <= sms && V >= 2 * C * tile) C *= 2;
  if (C == 1 && M * 2 <= 4 * sms && V >= 8 * tile) C = 2;
  const dim3 grid(static_cast<unsigned>(M), static_cast<unsigned>(C));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t per_sm = M * C * 2 > sms ? (M * C + sms - 1) / sms : 0;
  cudaError_t e;
#define DK_LOGPROB(TT)                                                                                                  \
  e = top > 0 ? launch_logprobs<TT, true>(grid, per_sm, st, p)                                                          \
              : launch_logprobs<TT, false>(grid, per_sm, st, p)
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
