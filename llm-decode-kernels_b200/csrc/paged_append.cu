// Append of keys and values to a paged cache with the rotary positions applied on the way:
// for every token row of qkv at position p of its sequence b (x: a head of q or k, half = head_dim / 2)
//   x'[d]        = x[d] * cos[p][d] - x[d + half] * sin[p][d]
//   x'[d + half] = x[d + half] * cos[p][d] + x[d] * sin[p][d]          (fp32, rounded once)
// q' goes to q_out, k' and v to row p % page_size of page table[b][p / page_size]. The sequence runner's
// counterpart for a contiguous cache is the head of csrc/attention.cu (kernels/e2e/model.py:236-241).
//
// Memory bound: every element is read once and written once. A warp takes up to kAhead groups of heads of one token at a
// time (a head's 8 dims and their 8 partners a lane, or 8 dims of v), loads them before it knows where they go - the
// token's sequence, position and page are a chain of small loads - and its angles once for all of them. With few tokens
// a token's heads are spread over several warps.
// Measured (36 heads of 128): 9000 tokens, 164 MB, 32 us, 78% of the copy rate (64 registers a thread, 4 CTAs an SM, 20 bytes of
// it spilled; with 5 or 6 CTAs 92 to 300 bytes spill, 42 and 53 us); one token 2.3 us without the host.
#include <algorithm>

#include "paged.cuh"

namespace dk {
namespace {

using namespace paged;

struct AppendParams {
  const void* qkv;
  int64_t ldqkv;
  void* k;
  void* v;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lengths;
  const int32_t* starts;
  const void* cos;
  const void* sin;
  int64_t ld_rope;
  int64_t rope_rows, rope_offset;
  void* q_out;
  int T, B, nq, nkv;
  int n_pages, page_size, page_shift, table_width;
  int* err;
};

template <typename T, typename R>
__device__ __forceinline__ void load8(const R* p, float (&v)[8]) {
  if constexpr (sizeof(R) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Elem<T>::unpack(w[i]);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]), Elem<T>::pack(v[4], v[5]),
                    Elem<T>::pack(v[6], v[7]));
}

constexpr int kAhead = 2;  // 4 with half the warps resident: 33.9 against 32.9 us for 164 MB
constexpr int kWarps = 8;

template <typename T, typename R, int kHd>
__global__ void __launch_bounds__(kWarps * 32, 4) paged_append_kernel(const AppendParams p, int segments, int per_warp) {
  constexpr int kRot = kHd / 16;         // lanes of a rotated head
  constexpr int kHeads = 32 / kRot;      // rotated heads of a segment
  constexpr int kCopy = kHd / 8;         // lanes of a head of v
  constexpr int kCopyHeads = 32 / kCopy;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int rot_heads = p.nq + p.nkv, rot_segments = (rot_heads + kHeads - 1) / kHeads;
  const int parts = (segments + per_warp - 1) / per_warp;
  const int64_t total = static_cast<int64_t>(p.T) * parts;
  for (int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); w < total; w += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int t = static_cast<int>(w / parts), s0 = static_cast<int>(w % parts) * per_warp, s1 = min(s0 + per_warp, segments);
    const T* row = static_cast<const T*>(p.qkv) + t * p.ldqkv;
    const int d = 8 * (lane % kRot), vd = 8 * (lane % kCopy);
    // the head of this lane in segment s, or -1
    auto rot_head = [&](int s) {
      const int h = s * kHeads + lane / kRot;
      return s < rot_segments && h < rot_heads ? h : -1;
    };
    auto copy_head = [&](int s) {
      const int h = (s - rot_segments) * kCopyHeads + lane / kCopy;
      return s >= rot_segments && s < s1 && h < p.nkv ? h : -1;
    };
    uint4 lo[kAhead], hi[kAhead];
    auto load = [&](int s) {
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int h = s + a < s1 ? rot_head(s + a) : -1, vh = copy_head(s + a);
        if (h >= 0) {
          lo[a] = *reinterpret_cast<const uint4*>(row + h * kHd + d);
          hi[a] = *reinterpret_cast<const uint4*>(row + h * kHd + d + kHd / 2);
        } else if (vh >= 0) {
          lo[a] = *reinterpret_cast<const uint4*>(row + static_cast<int64_t>(rot_heads + vh) * kHd + vd);
        }
      }
    };
    load(s0);
    int b = t, pos;
    if (p.starts == nullptr) {
      pos = length_of(p.lengths, t) - 1;
    } else {
      b = find_tile_warp([&](int j) { return p.starts[j]; }, p.B, t, lane);
      const int end = p.starts[b + 1];
      pos = t >= p.starts[b] && t < end ? length_of(p.lengths, b) - (end - t) : -1;
    }
    // A row of no sequence, or of one without positions (an unused slot of the batch), appends nothing; its q is zero.
    const int64_t angle = pos + p.rope_offset;
    const bool live = pos >= 0, turns = live && angle >= 0 && angle < p.rope_rows;
    const int at = pos >> p.page_shift;
    const int page = live && at < p.table_width ? p.table[b * p.ld_table + at] : -1;
    const bool lands = turns && page >= 0 && page < p.n_pages;
    if (live && !lands && lane == 0) record_device_error(p.err, DK_DEVERR_BAD_POSITION);
    float co[8], si[8];
    if (turns) {
      load8<T>(static_cast<const R*>(p.cos) + angle * p.ld_rope + d, co);
      load8<T>(static_cast<const R*>(p.sin) + angle * p.ld_rope + d, si);
    }
    const int64_t in_page = static_cast<int64_t>(pos & (p.page_size - 1)) * kHd;
    const int64_t page_heads = static_cast<int64_t>(page) * p.nkv;
    for (int s = s0; s < s1; s += kAhead) {
      if (s > s0) load(s);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int h = s + a < s1 ? rot_head(s + a) : -1, vh = copy_head(s + a);
        if (h >= 0) {
          const bool is_q = h < p.nq;
          if (!is_q && !lands) continue;
          uint4 u = make_uint4(0, 0, 0, 0), v = u;
          if (turns) {
            const uint32_t l[4] = {lo[a].x, lo[a].y, lo[a].z, lo[a].w}, r[4] = {hi[a].x, hi[a].y, hi[a].z, hi[a].w};
            float x[8], y[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = Elem<T>::unpack(l[j]), g = Elem<T>::unpack(r[j]);
              x[2 * j] = f.x * co[2 * j] - g.x * si[2 * j];
              x[2 * j + 1] = f.y * co[2 * j + 1] - g.y * si[2 * j + 1];
              y[2 * j] = g.x * co[2 * j] + f.x * si[2 * j];
              y[2 * j + 1] = g.y * co[2 * j + 1] + f.y * si[2 * j + 1];
            }
            u = pack8<T>(x), v = pack8<T>(y);
          }
          T* dst = is_q ? static_cast<T*>(p.q_out) + (static_cast<int64_t>(t) * p.nq + h) * kHd
                        : static_cast<T*>(p.k) + (page_heads + h - p.nq) * p.page_size * kHd + in_page;
          *reinterpret_cast<uint4*>(dst + d) = u;
          *reinterpret_cast<uint4*>(dst + d + kHd / 2) = v;
        } else if (vh >= 0 && lands) {
          *reinterpret_cast<uint4*>(static_cast<T*>(p.v) + (page_heads + vh) * p.page_size * kHd + in_page + vd) = lo[a];
        }
      }
    }
  }
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" int dk_paged_append(const dk_paged_append_args* args) {
  if (args == nullptr) return set_error(DK_ERR_INVALID, "paged_append: NULL arguments");
  const dk_paged_append_args& a = *args;
  const int64_t T = a.T, B = a.B, nq = a.n_q, nkv = a.n_kv, head_dim = a.head_dim, n_pages = a.n_pages,
                page_size = a.page_size, table_width = a.table_width;
  const int dtype = static_cast<int>(a.dtype);
  if (T < 0 || B < 0 || (B == 0 && T > 0) || nq <= 0 || nkv <= 0 || n_pages <= 0 || table_width <= 0)
    return set_error(DK_ERR_INVALID, "paged_append: bad sizes");
  if (head_dim != 64 && head_dim != 128)
    return set_error(DK_ERR_UNSUPPORTED, "paged_append: head_dim %lld (64 or 128)", (long long)head_dim);
  if (dtype != DK_F16 && dtype != DK_BF16) return set_error(DK_ERR_UNSUPPORTED, "paged_append: dtype %d", dtype);
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
    return set_error(DK_ERR_UNSUPPORTED, "paged_append: page_size %lld (a power of two from 16 to 256)",
                     (long long)page_size);
  if (T == 0) return DK_OK;
  if (a.starts == nullptr && T != B)
    return set_error(DK_ERR_INVALID, "paged_append: without starts there is one token per sequence");
  if (T > INT32_MAX || B > INT32_MAX || n_pages > INT32_MAX || table_width > INT32_MAX ||
      table_width * page_size > INT32_MAX)
    return set_error(DK_ERR_INVALID, "paged_append: sizes must fit 31 bits");
  if (!a.qkv || !a.k_pages || !a.v_pages || !a.page_table || !a.lengths || !a.cos || !a.sin || !a.q_out)
    return set_error(DK_ERR_INVALID, "paged_append: NULL pointer");
  if (!aligned16(a.qkv) || !aligned16(a.k_pages) || !aligned16(a.v_pages) || !aligned16(a.q_out) || !aligned16(a.cos) ||
      !aligned16(a.sin) || (T > 1 && (a.ldqkv & 7)) || (a.ld_rope & (a.rope_f32 ? 3 : 7)))
    return set_error(DK_ERR_ALIGN, "paged_append: rows of qkv, cos, sin, the pages and q_out need 16-byte alignment");
  AppendParams p;
  p.qkv = a.qkv, p.ldqkv = a.ldqkv, p.k = a.k_pages, p.v = a.v_pages;
  p.table = a.page_table, p.ld_table = a.ld_table, p.lengths = a.lengths, p.starts = a.starts;
  p.cos = a.cos, p.sin = a.sin, p.ld_rope = a.ld_rope, p.rope_rows = a.rope_rows, p.rope_offset = a.rope_offset;
  p.q_out = a.q_out;
  p.T = static_cast<int>(T), p.B = static_cast<int>(B), p.nq = static_cast<int>(nq), p.nkv = static_cast<int>(nkv);
  p.n_pages = static_cast<int>(n_pages), p.page_size = static_cast<int>(page_size);
  p.page_shift = __builtin_ctzll(page_size);
  p.table_width = static_cast<int>(table_width);
  p.err = device_info().err_word;
  const int heads = static_cast<int>(512 / head_dim), copies = static_cast<int>(256 / head_dim);
  const int segments = static_cast<int>((nq + nkv + heads - 1) / heads + (nkv + copies - 1) / copies);
  // Whole tokens a warp once there are 16 warps of them for every SM; fewer segments each with fewer tokens (36 heads of 128,
  // us: 64 tokens 2.5, 5.6 with whole tokens; 1024 tokens 5.3, 7.6 with whole tokens, 7.3 with single segments; 4096 tokens
  // 11.8, 21.7 with single segments).
  const int64_t want = 16ll * device_info().num_sms;
  const int per_warp = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(segments, T * segments / want)));
  const int64_t warps = T * ((segments + per_warp - 1) / per_warp);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((warps + kWarps - 1) / kWarps, 64ll * device_info().num_sms)));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a.stream);
  cudaError_t e;
#define DK_APPEND(TT, RR)                                                                                    \
  e = launch(head_dim == 128 ? paged_append_kernel<TT, RR, 128> : paged_append_kernel<TT, RR, 64>, grid, dim3(kWarps * 32), 0, \
             st, pdl_enabled(), dim3(1, 1, 1), p, segments, per_warp)
  if (dtype == DK_F16) {
    if (a.rope_f32)
      DK_APPEND(__half, float);
    else
      DK_APPEND(__half, __half);
  } else {
    if (a.rope_f32)
      DK_APPEND(__nv_bfloat16, float);
    else
      DK_APPEND(__nv_bfloat16, __nv_bfloat16);
  }
#undef DK_APPEND
  if (e != cudaSuccess) return set_error(DK_ERR_CUDA, "paged_append launch: %s", cudaGetErrorString(e));
  return DK_OK;
}
