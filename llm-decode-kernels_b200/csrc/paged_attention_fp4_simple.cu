// Attention over a paged cache held in 4 bits, in its simplest form: a CTA for each row and kv head, whose warps take every
// fourth position and join at the end.
//   out[t] = sum_j p[t][j] v[j],  p[t] = softmax over the visible j of scale * q[t] . k[j]
// Row t at position p sees j <= p with (window <= 0 or j > p - window or j < sinks), and with a prefix all of it; a row that
// sees nothing is zero. Everything is fp32 but the inputs and the output.
#include <algorithm>
#include <climits>

#include "paged_fp4.cuh"

namespace dk {
namespace paged {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxGroup = 16;

struct Simple {
  const void* q;
  int64_t ldq;
  const uint8_t* pool[2];
  void* out;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lengths;
  const int32_t* starts;
  const int32_t* prefix_table;
  int prefix_len;
  int T, B, nkv, G, n_pages, page_size, page_shift, capacity;
  Mask mask;
  float scale2, v_power;
  int* err;
};

template <typename T, int kHd>
__global__ void __launch_bounds__(kWarps * 32) simple_kernel(const Simple p) {
  using F = Fp4<kHd>;
  constexpr int kDims = kHd / 32;  // of a lane
  __shared__ float q_sh[kMaxGroup][kHd];
  __shared__ float o_sh[kWarps][kMaxGroup][kHd];
  __shared__ float m_sh[kWarps][kMaxGroup], l_sh[kWarps][kMaxGroup];
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int b = t, pos;
  if (p.starts == nullptr) {
    pos = length_of(p.lengths, t) - 1;
  } else {
    b = find_tile_warp([&](int j) { return p.starts[j]; }, p.B, t, lane);
    const int end = p.starts[b + 1];
    pos = t >= p.starts[b] && t < end ? length_of(p.lengths, b) - (end - t) : -1;
  }
  for (int i = threadIdx.x; i < p.G * kHd; i += kWarps * 32)
    q_sh[i / kHd][i % kHd] = static_cast<float>(static_cast<const T*>(p.q)[t * p.ldq + (h * p.G + i / kHd) * kHd + i % kHd]) * p.scale2;
  if (pos >= p.capacity && threadIdx.x == 0) record_device_error(p.err, DK_DEVERR_BAD_POSITION);
  __syncthreads();
  float m[kMaxGroup], l[kMaxGroup], o[kMaxGroup][kDims];
#pragma unroll
  for (int g = 0; g < kMaxGroup; ++g) {
    m[g] = -INFINITY, l[g] = 0.f;
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[g][d] = 0.f;
  }
  // a lane's dims are kDims * lane on; values of a position, zeros without a page
  auto value = [&](int which, int page, int j, float (&x)[kDims]) {
    const uint8_t* block = p.pool[which] + (static_cast<int64_t>(page) * p.nkv + h) * p.page_size * F::kRow;
    const int slot = j & (p.page_size - 1);
    const float s = fp4_scale(block[p.page_size * F::kCodes + slot * F::kScales + kDims * lane / 16]);
    uint32_t w[4];  // of the aligned four bytes that hold the lane's
    fp4_codes(*reinterpret_cast<const uint32_t*>(block + slot * F::kCodes + (kDims * lane / 2 & ~3)), w);
    if constexpr (kDims == 4) {
      const float2 f = Elem<__half>::unpack(lane & 1 ? w[2] : w[0]), g = Elem<__half>::unpack(lane & 1 ? w[3] : w[1]);
      x[0] = f.x * s, x[1] = f.y * s, x[2] = g.x * s, x[3] = g.y * s;
    } else {
      const uint32_t u = lane & 2 ? (lane & 1 ? w[3] : w[2]) : (lane & 1 ? w[1] : w[0]);
      const float2 f = Elem<__half>::unpack(u);
      x[0] = f.x * s, x[1] = f.y * s;
    }
  };
  auto take = [&](const int32_t* table, int j) {
    const int page = table[j >> p.page_shift];
    const bool there = page >= 0 && page < p.n_pages;
    if (!there) record_device_error(p.err, DK_DEVERR_BAD_POSITION);
    float k[kDims] = {}, v[kDims] = {};
    if (there) {
      value(0, page, j, k);
      value(1, page, j, v);
    }
#pragma unroll
    for (int g = 0; g < kMaxGroup; ++g) {
      if (g >= p.G) break;
      float s = 0.f;
#pragma unroll
      for (int d = 0; d < kDims; ++d) s = fmaf(q_sh[g][kDims * lane + d], k[d], s);
#pragma unroll
      for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
      const float mx = fmaxf(m[g], s), keep = exp2f(m[g] - mx), w = exp2f(s - mx);
      m[g] = mx, l[g] = fmaf(l[g], keep, w);
#pragma unroll
      for (int d = 0; d < kDims; ++d) o[g][d] = fmaf(o[g][d], keep, w * v[d]);
    }
  };
  for (int j = warp; j < p.prefix_len; j += kWarps) take(p.prefix_table, j);
  const int end = min(pos + 1, p.capacity);
  const int lo = p.mask.window > 0 ? max(0, pos - p.mask.window + 1) : 0, sinks = min(p.mask.sinks, min(lo, end));
  for (int i = warp; i < sinks + max(end - lo, 0); i += kWarps) take(p.table + b * p.ld_table, i < sinks ? i : lo + i - sinks);
#pragma unroll
  for (int g = 0; g < kMaxGroup; ++g) {
    if (g >= p.G) break;
    if (lane == 0) m_sh[warp][g] = m[g], l_sh[warp][g] = l[g];
#pragma unroll
    for (int d = 0; d < kDims; ++d) o_sh[warp][g][kDims * lane + d] = o[g][d];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.G * kHd; i += kWarps * 32) {
    const int g = i / kHd, d = i % kHd;
    float mx = -INFINITY, sum = 0.f, acc = 0.f;
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, m_sh[w][g]);
    if (mx != -INFINITY)
      for (int w = 0; w < kWarps; ++w) {
        const float a = exp2f(m_sh[w][g] - mx);
        sum = fmaf(a, l_sh[w][g], sum), acc = fmaf(a, o_sh[w][g][d], acc);
      }
    static_cast<T*>(p.out)[(static_cast<int64_t>(t) * p.nkv * p.G + h * p.G + g) * kHd + d] =
        static_cast<T>(sum == 0.f ? 0.f : acc / sum * p.v_power);
  }
}

int attention_fp4(const char* what, const dk_paged_attention_fp4_args* args, bool prefix) {
  if (args == nullptr) return set_error(DK_ERR_INVALID, "%s: NULL arguments", what);
  const dk_paged_attention_args& a = args->attention;
  const int64_t T = a.T, B = a.B, nq = a.n_q, nkv = a.n_kv, hd = a.head_dim, prefix_len = prefix ? a.prefix_len : 0;
  const int64_t positions = a.table_width * a.page_size;
  if (T < 0 || B < 0 || (B == 0 && T > 0) || nq <= 0 || nkv <= 0 || prefix_len < 0)
    return set_error(DK_ERR_INVALID, "%s: bad sizes", what);
  if (hd != 64 && hd != 128) return set_error(DK_ERR_UNSUPPORTED, "%s: head_dim %lld (64 or 128)", what, (long long)hd);
  if (a.dtype != DK_F16 && a.dtype != DK_BF16) return set_error(DK_ERR_UNSUPPORTED, "%s: dtype %lld", what, (long long)a.dtype);
  if (nq % nkv != 0 || nq / nkv > kMaxGroup)
    return set_error(DK_ERR_UNSUPPORTED, "%s: %lld query heads over %lld kv heads (a multiple, at most 16 each)", what,
                     (long long)nq, (long long)nkv);
  if (a.starts == nullptr && T != B) return set_error(DK_ERR_INVALID, "%s: without starts there is one token per sequence", what);
  if (a.n_pages <= 0 || a.table_width <= 0 || a.window < 0 || a.sinks < 0) return set_error(DK_ERR_INVALID, "%s: bad sizes", what);
  if (a.page_size < 16 || a.page_size > 256 || (a.page_size & (a.page_size - 1)))
    return set_error(DK_ERR_UNSUPPORTED, "%s: page_size %lld (a power of two from 16 to 256)", what, (long long)a.page_size);
  if (a.n_pages > INT32_MAX || a.table_width > INT32_MAX || a.n_pages * nkv > INT32_MAX || a.n_pages * nkv * a.page_size > INT32_MAX ||
      positions + T > (int64_t(1) << 31) - 1024 || a.window > INT32_MAX || a.sinks > INT32_MAX || prefix_len > (1 << 30) || nkv > 65535)
    return set_error(DK_ERR_INVALID, "%s: sizes must stay below 2^31", what);
  if (!fp4_power(args->k_scale) || !fp4_power(args->v_scale))
    return set_error(DK_ERR_INVALID, "%s: k_scale and v_scale must be powers of two from 2^-64 to 2^64", what);
  if (T == 0) return DK_OK;
  const int64_t ldq = T > 1 ? a.ldq : nq * hd;
  if (ldq < nq * hd) return set_error(DK_ERR_INVALID, "%s: q's tokens overlap", what);
  if (!a.q || !a.k_pages || !a.v_pages || !a.page_table || !a.lengths || !a.out || (prefix_len > 0 && !a.prefix_table))
    return set_error(DK_ERR_INVALID, "%s: NULL pointer", what);
  if (!aligned16(a.q) || !aligned16(a.k_pages) || !aligned16(a.v_pages) || !aligned16(a.out) || (ldq & 7))
    return set_error(DK_ERR_ALIGN, "%s: q rows, pages and out need 16-byte alignment", what);
  Simple p;
  p.q = a.q, p.ldq = ldq, p.out = a.out;
  p.pool[0] = static_cast<const uint8_t*>(a.k_pages), p.pool[1] = static_cast<const uint8_t*>(a.v_pages);
  p.table = a.page_table, p.ld_table = a.ld_table, p.lengths = a.lengths, p.starts = a.starts;
  p.prefix_table = a.prefix_table, p.prefix_len = static_cast<int>(prefix_len);
  p.T = static_cast<int>(T), p.B = static_cast<int>(B), p.nkv = static_cast<int>(nkv), p.G = static_cast<int>(nq / nkv);
  p.n_pages = static_cast<int>(a.n_pages), p.page_size = static_cast<int>(a.page_size);
  p.page_shift = __builtin_ctzll(a.page_size), p.capacity = static_cast<int>(positions);
  const int64_t window = prefix ? 0 : std::min(a.window, positions), sinks = prefix ? 0 : std::min(a.sinks, positions);
  p.mask = Mask{static_cast<int>(window), window > 0 ? static_cast<int>(sinks) : 0};
  p.scale2 = static_cast<float>(a.scale * args->k_scale * 1.44269504088896341), p.v_power = static_cast<float>(args->v_scale);
  p.err = device_info().err_word;
  const dim3 grid(static_cast<unsigned>(T), static_cast<unsigned>(nkv));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a.stream);
  cudaError_t e;
#define DK_SIMPLE(TT) \
  e = launch(hd == 128 ? simple_kernel<TT, 128> : simple_kernel<TT, 64>, grid, dim3(kWarps * 32), 0, st, pdl_enabled(), dim3(1, 1, 1), p)
  if (a.dtype == DK_F16)
    DK_SIMPLE(__half);
  else
    DK_SIMPLE(__nv_bfloat16);
#undef DK_SIMPLE
  if (e != cudaSuccess) return set_error(DK_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return DK_OK;
}

}  // namespace

int simple_fp4(const char* what, const dk_paged_attention_fp4_args* args, bool prefix) { return attention_fp4(what, args, prefix); }

}  // namespace paged
}  // namespace dk

