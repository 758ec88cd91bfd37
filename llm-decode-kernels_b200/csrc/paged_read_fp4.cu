// Positions of a 4-bit paged cache read back as 16-bit values, k and v: row t of the call is a position of a sequence (the
// last ones of each, as in the other paged ops), value = code * scale * power, exact in T unless outside its range.
//
// Memory bound: 9 bytes are read for 32 written. A CTA takes up to 32 rows: its first threads look up where they lie, side by side (a
// chain of small loads each), then a warp takes a row's columns, 8 dims (4 bytes of codes, half a group) a lane, so that it
// stores 512 contiguous bytes, with the loads of several rows in flight.
// Measured (4 kv heads of 128, bf16): 16 sequences of up to 8192, 207 MB, 38.4 us, 5.4 TB/s, 82% of the copy rate; 525 positions of 2 kv
// heads 2.7 us without the host.
#include <algorithm>

#include "paged_fp4.cuh"

namespace dk {
namespace {

using namespace paged;

struct ReadParams {
  const uint8_t* pool[2];
  void* out[2];
  float power[2];
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lengths;
  const int32_t* starts;
  int T, B, nkv;
  int n_pages, page_size, page_shift, table_width;
  int* err;
};

constexpr int kWarps = 8;
constexpr int kMaxRows = 32;  // of a CTA
constexpr int kAhead = 8;     // items loaded at a time (16 sequences of up to 8192: 37.5 us, 41.5 with 4, 46.7 with 2)

// CTA x: rows per * x .. + per. A row has `columns` items of 32 pieces of 8 dims, of k, then of v.
template <typename T, int kHd>
__global__ void __launch_bounds__(kWarps * 32) paged_read_fp4_kernel(const ReadParams p, int columns, int per) {
  using F = Fp4<kHd>;
  __shared__ int2 place[kMaxRows];  // {page, row in it}; page -1: zeros
  pdl_trigger();
  pdl_wait();
  const int t0 = blockIdx.x * per, n = min(per, p.T - t0);
  if (static_cast<int>(threadIdx.x) < n) {
    // A row of no sequence, or before its sequence's first position, has no place; nor has a position without a page, which is
    // reported.
    const int t = t0 + threadIdx.x;
    int b = t, pos, page = -1;
    if (p.starts == nullptr) {
      pos = length_of(p.lengths, t) - 1;
    } else {
      b = find_tile([&](int j) { return p.starts[j]; }, p.B, t);
      const int end = p.starts[b + 1];
      pos = t >= p.starts[b] && t < end ? length_of(p.lengths, b) - (end - t) : -1;
    }
    if (pos >= 0) {
      const int at = pos >> p.page_shift;
      page = at < p.table_width ? p.table[b * p.ld_table + at] : -1;
      if (page < 0 || page >= p.n_pages) {
        page = -1;
        record_device_error(p.err, DK_DEVERR_BAD_POSITION);
      }
    }
    place[threadIdx.x] = make_int2(page, pos & (p.page_size - 1));
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pieces = p.nkv * (kHd / 8), half = columns / 2;
  const int64_t page_bytes = static_cast<int64_t>(p.nkv) * p.page_size * F::kRow;
  const int scales_at = p.page_size * F::kCodes;
  // A warp keeps its column where there are no more than warps (then they share it out by rows), so that little is computed for each item.
  const int step = columns <= kWarps ? kWarps / columns : 1;
  for (int column = warp % columns; column < columns; column += kWarps) {
    const int which = column >= half, piece = (column - which * half) * 32 + lane;
    if (columns <= kWarps && warp >= step * columns) break;
    const int h = piece / (kHd / 8), c = piece % (kHd / 8);
    const uint8_t* pool = (which ? p.pool[1] : p.pool[0]) + static_cast<int64_t>(h) * p.page_size * F::kRow;
    const uint8_t *codes = pool + 4 * c, *scales = pool + scales_at + c / 2;
    const float power = which ? p.power[1] : p.power[0];
    uint4* out = reinterpret_cast<uint4*>(which ? p.out[1] : p.out[0]) + static_cast<int64_t>(t0) * pieces + piece;
    if (piece >= pieces) continue;
    auto rows = [&](int i, auto count) {  // (loads under a row's own condition: 41 us instead of 37 for 16 sequences of up to 8192)
      constexpr int kRows = decltype(count)::value;
      uint32_t code[kRows];
      uint8_t scale[kRows];
#pragma unroll
      for (int a = 0; a < kRows; ++a) {
        const int2 at = place[i + a * step];
        code[a] = 0, scale[a] = 0;
        if (at.x >= 0) {
          code[a] = *reinterpret_cast<const uint32_t*>(codes + at.x * page_bytes + at.y * F::kCodes);
          scale[a] = scales[at.x * page_bytes + at.y * F::kScales];
        }
      }
#pragma unroll
      for (int a = 0; a < kRows; ++a) {
        const float s = fp4_scale(scale[a]) * power;
        uint32_t x[4], y[4];
        fp4_codes(code[a], x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = Elem<__half>::unpack(x[j]);
          y[j] = Elem<T>::pack(f.x * s, f.y * s);
        }
        out[static_cast<int64_t>(i + a * step) * pieces] = make_uint4(y[0], y[1], y[2], y[3]);
      }
    };
    int i = columns <= kWarps ? warp / columns : 0;
    for (; i + (kAhead - 1) * step < n; i += kAhead * step) rows(i, std::integral_constant<int, kAhead>());
    for (; i < n; i += step) rows(i, std::integral_constant<int, 1>());
  }
}

// Pages in 16 bits of what a call's rows see, for the 256-row tiles (paged_attention_tc.cu): a page of the copy for each entry of
// the page tables, and tables that list them. A warp takes 16 positions of a head's k or v; the powers are left out (the scores' scale
// and the output's have them). code * scale is exact in either type: k is of the call's, so that q is the other factor as it is, and
// v is fp16, so that p keeps 11 bits beside it as in the other kernels over such a cache (bf16 would leave it 8).
// Measured: 8192 positions of 2 kv heads of 128, 2.4 MB read and 8.4 written, 5.1 us with its launch (the plan, a launch before it,
// then added 4; now a CTA or two beside the copy make it).
struct CopyParams {
  const uint8_t* pool[2];
  void* out[2];  // [B * width, nkv, page_size, kHd]: k of type T, v fp16
  int32_t* table_out;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lengths;
  const int32_t* starts;
  int T, B, nkv, n_pages, page_size, page_shift, width;
  int above;  // sequences of more tokens are copied
  Mask mask;
  int* err;
};

// The first `plans` CTAs make the plans of the launches that follow: neither waits for the other.
template <typename T, int kHd>
__global__ void __launch_bounds__(kPlanThreads) fp4_copy_kernel(const CopyParams p, const Problem pa, const Problem pb, int plans) {
  using F = Fp4<kHd>;
  constexpr int kPieces = 16 * kHd / 8;  // of 8 dims of 16 positions of a head
  constexpr int kWarps = kPlanThreads / 32;
  pdl_trigger();
  pdl_wait();
  const int cta = static_cast<int>(blockIdx.x) - plans, ctas = static_cast<int>(gridDim.x) - plans;
  if (cta < 0) return make_plan(blockIdx.x == 0 ? pa : pb);
  const int lane = threadIdx.x & 31, per_seq = p.width << (p.page_shift - 4), heads = 2 * p.nkv;
  const int64_t units = static_cast<int64_t>(p.B) * per_seq * heads;
  for (int64_t u = static_cast<int64_t>(cta) * kWarps + (threadIdx.x >> 5); u < units; u += static_cast<int64_t>(ctas) * kWarps) {
    const int64_t group = u / heads;
    const int b = static_cast<int>(group / per_seq), j0 = static_cast<int>(group - static_cast<int64_t>(b) * per_seq) * 16;
    // seen: below the length, and from the first row's window on or below the sinks
    const int t0 = min(max(p.starts[b], 0), p.T), rows = min(max(p.starts[b + 1], t0), p.T) - t0;
    const int length = length_of(p.lengths, b);
    if (rows <= p.above || j0 >= length) continue;
    if (p.mask.window > 0 && j0 + 15 <= length - rows - p.mask.window && j0 >= p.mask.sinks) continue;
    const int at = j0 >> p.page_shift, page = p.table[b * p.ld_table + at];
    const int64_t to = static_cast<int64_t>(b) * p.width + at;
    const bool there = page >= 0 && page < p.n_pages;
    const int head = static_cast<int>(u - group * heads), which = head >= p.nkv, h = head - which * p.nkv;
    if (lane == 0 && head == 0) {
      p.table_out[to] = static_cast<int32_t>(to);
      if (!there) record_device_error(p.err, DK_DEVERR_BAD_POSITION);  // (zeros)
    }
    const int slot = j0 & (p.page_size - 1);
    const uint8_t* block = (which ? p.pool[1] : p.pool[0]) + (static_cast<int64_t>(there ? page : 0) * p.nkv + h) * p.page_size * F::kRow;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(block + slot * F::kCodes) + lane;
    const uint8_t* scales = block + p.page_size * F::kCodes + slot * F::kScales + lane / 2;
    uint32_t code[kPieces / 32];
    uint8_t scale[kPieces / 32];
#pragma unroll
    for (int i = 0; i < kPieces / 32; ++i) {
      code[i] = there ? codes[32 * i] : 0;
      scale[i] = there ? scales[16 * i] : 0;
    }
    uint4* out = static_cast<uint4*>(which ? p.out[1] : p.out[0]) + ((to * p.nkv + h) * p.page_size + slot) * (kHd / 8) + lane;
#pragma unroll
    for (int i = 0; i < kPieces / 32; ++i) {
      uint32_t x[4], one = fp4_scales(scale[i]);
      fp4_codes(code[i], x);
      one = prmt(one, one, 0x1010);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = hmul2_rn(x[k], one);
        if (!std::is_same<T, __half>::value && !which) {
          const float2 f = Elem<__half>::unpack(x[k]);
          x[k] = Elem<T>::pack(f.x, f.y);
        }
      }
      out[32 * i] = make_uint4(x[0], x[1], x[2], x[3]);
    }
  }
}

}  // namespace

namespace paged {

cudaError_t fp4_copy_launch(const Problem& p, const Problem& b, int plans, int64_t hd, int dtype, void* k, void* v, int32_t* table,
                            cudaStream_t st) {
  CopyParams c;
  c.pool[0] = p.pool[0], c.pool[1] = p.pool[1], c.out[0] = k, c.out[1] = v, c.table_out = table;
  c.table = p.table, c.ld_table = p.ld_table, c.lengths = p.lengths, c.starts = p.starts;
  c.T = p.T, c.B = p.B, c.nkv = p.nkv, c.n_pages = p.n_pages, c.page_size = p.page_size, c.page_shift = p.page_shift;
  c.above = p.above, c.width = p.capacity >> p.page_shift, c.mask = p.mask, c.err = p.err;
  const int64_t units = static_cast<int64_t>(p.B) * (p.capacity / 16) * 2 * p.nkv;
  constexpr int kCopyWarps = kPlanThreads / 32;
  const dim3 grid(static_cast<unsigned>(plans + std::min<int64_t>((units + kCopyWarps - 1) / kCopyWarps, 2ll * device_info().num_sms)));
#define DK_COPY(TT)                                                                                                              \
  launch(hd == 128 ? fp4_copy_kernel<TT, 128> : fp4_copy_kernel<TT, 64>, grid, dim3(kPlanThreads), 0, st, pdl_enabled(), dim3(1, 1, 1), \
         c, p, b, plans)
  return dtype == DK_F16 ? DK_COPY(__half) : DK_COPY(__nv_bfloat16);
#undef DK_COPY
}

}  // namespace paged
}  // namespace dk

using namespace dk;

extern "C" int dk_paged_read_fp4(const dk_paged_read_fp4_args* args) {
  if (args == nullptr) return set_error(DK_ERR_INVALID, "paged_read_fp4: NULL arguments");
  const dk_paged_read_fp4_args& a = *args;
  const int64_t T = a.T, B = a.B, nkv = a.n_kv, head_dim = a.head_dim, page_size = a.page_size, width = a.table_width;
  const int dtype = static_cast<int>(a.dtype);
  if (T < 0 || B < 0 || (B == 0 && T > 0) || nkv <= 0 || a.n_pages <= 0 || width <= 0)
    return set_error(DK_ERR_INVALID, "paged_read_fp4: bad sizes");
  if (head_dim != 64 && head_dim != 128)
    return set_error(DK_ERR_UNSUPPORTED, "paged_read_fp4: head_dim %lld (64 or 128)", (long long)head_dim);
  if (dtype != DK_F16 && dtype != DK_BF16) return set_error(DK_ERR_UNSUPPORTED, "paged_read_fp4: dtype %d", dtype);
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
    return set_error(DK_ERR_UNSUPPORTED, "paged_read_fp4: page_size %lld (a power of two from 16 to 256)", (long long)page_size);
  if (!fp4_power(a.k_scale) || !fp4_power(a.v_scale))
    return set_error(DK_ERR_INVALID, "paged_read_fp4: k_scale and v_scale must be powers of two from 2^-64 to 2^64");
  if (T == 0) return DK_OK;
  if (a.starts == nullptr && T != B)
    return set_error(DK_ERR_INVALID, "paged_read_fp4: without starts there is one row per sequence");
  if (T > INT32_MAX || B > INT32_MAX || a.n_pages > INT32_MAX || width > INT32_MAX || width * page_size > INT32_MAX || nkv > 65535)
    return set_error(DK_ERR_INVALID, "paged_read_fp4: sizes must fit 31 bits");
  if (!a.k_pages || !a.v_pages || !a.page_table || !a.lengths || !a.k_out || !a.v_out)
    return set_error(DK_ERR_INVALID, "paged_read_fp4: NULL pointer");
  if (!aligned16(a.k_pages) || !aligned16(a.v_pages) || !aligned16(a.k_out) || !aligned16(a.v_out))
    return set_error(DK_ERR_ALIGN, "paged_read_fp4: pages and outputs need 16-byte alignment");
  ReadParams p;
  p.pool[0] = static_cast<const uint8_t*>(a.k_pages), p.pool[1] = static_cast<const uint8_t*>(a.v_pages);
  p.out[0] = a.k_out, p.out[1] = a.v_out;
  p.power[0] = static_cast<float>(a.k_scale), p.power[1] = static_cast<float>(a.v_scale);
  p.table = a.page_table, p.ld_table = a.ld_table, p.lengths = a.lengths, p.starts = a.starts;
  p.T = static_cast<int>(T), p.B = static_cast<int>(B), p.nkv = static_cast<int>(nkv);
  p.n_pages = static_cast<int>(a.n_pages), p.page_size = static_cast<int>(page_size);
  p.page_shift = __builtin_ctzll(page_size);
  p.table_width = static_cast<int>(width);
  p.err = device_info().err_word;
  // Up to 32 rows a CTA (a power of two: whole batches of loads) as long as every SM has 4 CTAs.
  const int64_t columns = 2 * ((nkv * (head_dim / 8) + 31) / 32);
  int64_t per = kMaxRows;
  while (per > 1 && per * 4 * device_info().num_sms > T) per /= 2;
  const dim3 grid(static_cast<unsigned>((T + per - 1) / per));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a.stream);
  cudaError_t e;
#define DK_READ(TT) \
  e = launch(head_dim == 128 ? paged_read_fp4_kernel<TT, 128> : paged_read_fp4_kernel<TT, 64>, grid, dim3(kWarps * 32), 0, st, \
             pdl_enabled(), dim3(1, 1, 1), p, static_cast<int>(columns), static_cast<int>(per))
  if (dtype == DK_F16)
    DK_READ(__half);
  else
    DK_READ(__nv_bfloat16);
#undef DK_READ
  if (e != cudaSuccess) return set_error(DK_ERR_CUDA, "paged_read_fp4 launch: %s", cudaGetErrorString(e));
  return DK_OK;
}
