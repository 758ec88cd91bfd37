// What the paged-cache kernels share: 16-bit element types, the division of a batch's attention work
// into units and chunks, and the partial results of units that several CTAs work on.
//
// A cache is a pool of pages, k and v each [n_pages, n_kv, page_size, head_dim]; row b of the page
// table lists the pages of sequence b in order, so position j of kv head h is row
// (table[b][j / page_size] * n_kv + h) * page_size + j % page_size of the pool.
//
// The query rows of a launch are cut into tiles of consecutive tokens of one sequence, with the G =
// n_q / n_kv query heads of one kv head side by side (row r of a tile: token r / G, head r % G), so a
// tile reads each k and v row once for all of its rows. (kv head, tile) is a unit; its visible
// positions are cut into chunks of kChunk positions, at least one. All chunks of all units are laid
// on one line, kv head by kv head, and every CTA of the launch takes an equal contiguous piece of it:
// long and short sequences, many or few of them, fill the GPU alike. A unit cut by a piece's end
// leaves its partial results (row maximum, row sum, unnormalized output, fp32) in the workspace, and
// a second kernel joins them in order of position, so that results do not depend on timing.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace dk {
namespace paged {

// ---------------------------------------------------------------------------------- element types
template <typename T>
struct Elem;

template <>
struct Elem<__half> {
  static constexpr CUtensorMapDataType kMapType = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  __device__ static uint32_t pack(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
  }
  __device__ static float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  // D(16x8, f32) += A(16x16, row) * B(16x8, col)
  __device__ static void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                             uint32_t b1) {
    mma_16816(d, a0, a1, a2, a3, b0, b1);
  }
};

template <>
struct Elem<__nv_bfloat16> {
  static constexpr CUtensorMapDataType kMapType = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  __device__ static uint32_t pack(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
  }
  __device__ static float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  __device__ static void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bounded wait like mbar_wait, for waits on a loop's critical path: the timer, whose read takes longer than most of these
// waits, is looked at only once in 256 unsuccessful polls.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int* err, int code) {
  uint64_t t0 = 0;
  for (uint32_t i = 1; !mbar_try_wait(bar, parity); ++i) {
    if ((i & 255) != 0) continue;
    const uint64_t now = globaltimer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > kWaitLimitNs) {
      record_device_error(err, code);
      return false;
    }
  }
  return true;
}

// ------------------------------------------------------------------------------------ visible positions
// A row at position p sees position j when j <= p and (window <= 0 or j > p - window or j < sinks).
struct Mask {
  int window, sinks;
  __device__ bool sees(int p, int j) const { return j <= p && (window <= 0 || j > p - window || j < sinks); }
};

// What the rows at positions p0..p1 of one tile visit: the pages (or parts of kChunk positions of larger ones) with sinks and
// those from the window's first one on, without the positions between. Offsets count the visited positions, chunks of
// kChunk at a time: offset j is position j below `gap_at`, position j + shift from there on (both multiples of a page's
// part); a row's position minus shift takes the place of its position in offsets. At least one chunk, so that a tile that
// sees nothing is still visited once and gets its zeros.
template <int kChunk>
struct Span {
  int end;  // first offset after the last visible one
  int lo;   // first offset inside some row's window
  int gap_at, shift, n;
  Span() = default;
  __device__ Span(int p0, int p1, const Mask& m, int capacity, int page_size) {
    const int part = min(page_size, kChunk);
    end = min(max(p1 + 1, 0), capacity);
    lo = m.window > 0 ? max(0, p0 - m.window + 1) : 0;
    gap_at = m.window > 0 ? (min(m.sinks, lo) + part - 1) & -part : 0;
    shift = max(0, (lo & -part) - gap_at);
    lo -= shift;
    end = max(end - shift, min(end, gap_at));  // (a window wholly past the table leaves the sinks)
    n = max(1, (end + kChunk - 1) / kChunk);
  }
  __device__ int position(int j) const { return j < gap_at ? j : j + shift; }
  // Is some offset of [j, j + len) visible to some row of the tile?
  __device__ bool needs(int j, int len, const Mask& m) const {
    return j < end && (m.window <= 0 || j + len > lo || j < m.sinks);
  }
};

// ------------------------------------------------------------------------------------------ launches
enum Mode {
  kOneToken = 0,  // tile b is the one token of sequence b
  kRagged = 1,    // tiles from the plan kernel
  kPrefix = 2,    // tiles of consecutive tokens of the whole batch, all of the prefix visible to each
};

struct Problem {
  const void* q;  // [T, n_q, head_dim], tokens ldq elements apart
  int64_t ldq;
  void* out;  // [T, n_q, head_dim]
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lengths;
  const int32_t* starts;  // [B + 1] or null
  int T, B, nkv, G;
  int n_pages, page_size, page_shift, capacity;  // capacity: positions a table row can hold
  int prefix_len;
  Mask mask;
  float scale2;  // scale * log2(e); tiles_kernel: a positive one, with the sign in `signs`
  int signs;     // tiles_kernel: what Q is multiplied by in the products with K, -1, 0 or 1
  int mode;
  int tile_tokens;
  int half_tokens;  // tokens of 128 rows (tiles_kernel); 1 (rows_kernel)
  int early, lead;  // the launch's first `early` pieces are `lead` chunks longer than the others (their CTAs start while
                    // the kernel before still holds the other SMs)
  int unit_extra;   // chunks added to a unit's length on the line for what it costs besides its chunks
  int n_tiles;      // kOneToken, kPrefix; kRagged: the plan's
  // kRagged: plan[0] = tiles, plan[1] = length of one kv head's line, then cum[max_tiles + 1]; what tile_at needs of
  // each tile lies in tile_info
  const int32_t* plan;
  const int4* tile_info;  // {first token, tokens, position of the first one, sequence}
  int max_tiles;
  int32_t* cum_out;  // kOneToken: [B + 1], the chunks of one kv head before each sequence
  // Partial results: a CTA's first piece of a unit that began before it (slot 2 * CTA), its last piece of a unit that
  // goes on after it (slot 2 * CTA + 1), and with always_partial a slot for each uncut unit after those
  float* part_o;   // [slots][tile rows][head_dim], or with rows_inner [slots][head_dim / 4][tile rows][4]
  float* part_ml;  // [slots][tile rows][2]: row maximum (base 2), row sum
  int4* cut;           // [CTAs] the unit whose chunks a CTA begins but does not end: {first token, tokens, kv head, last CTA}
  int rows_inner;
  int always_partial;  // no unit writes its output itself
  int* err;
};

// Positions of sequence b; an unused slot has none, however negative its length (positions counted back from the lowest
// number would wrap).
__device__ __forceinline__ int length_of(const int32_t* lengths, int b) { return max(lengths[b], 0); }

struct Tile {
  int t0, ntok;  // tokens of q
  int p0;        // position of the first one
  const int32_t* table;
};

__device__ __forceinline__ Tile tile_at(const Problem& p, int i) {
  Tile t;
  if (p.mode == kOneToken) {
    t.t0 = i;
    t.ntok = 1;
    t.p0 = length_of(p.lengths, i) - 1;
    t.table = p.table + i * p.ld_table;
  } else if (p.mode == kPrefix) {
    t.t0 = i * p.tile_tokens;
    t.ntok = min(p.tile_tokens, p.T - t.t0);
    t.p0 = p.prefix_len - 1;
    t.table = p.table;
  } else {
    const int4 v = p.tile_info[i];
    t.t0 = v.x, t.ntok = v.y, t.p0 = v.z;
    t.table = p.table + v.w * p.ld_table;
  }
  return t;
}

// Last position of a tile's rows (the rows of a prefix launch all sit at its last position).
__device__ __forceinline__ int tile_last(const Problem& p, const Tile& t) {
  return p.mode == kPrefix ? t.p0 : t.p0 + t.ntok - 1;
}
__device__ __forceinline__ int row_position(const Problem& p, const Tile& t, int tok) {
  return p.mode == kPrefix ? t.p0 : t.p0 + tok;
}

__device__ __forceinline__ int64_t partial_slot(int ctas, int cta, bool from_start, bool whole, int unit) {
  return whole ? 2ll * ctas + unit : 2ll * cta + (from_start ? 1 : 0);
}

// Largest i with cum(i) <= x, for cum(0) = 0 <= x < cum(n); one thread.
template <typename Cum>
__device__ __forceinline__ int find_tile(const Cum& cum, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cum(mid) <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// The same by a whole warp: 32 probes a round instead of one (two dependent loads for 1024 tiles, not ten).
template <typename Cum>
__device__ __forceinline__ int find_tile_warp(const Cum& cum, int n, int x, int lane) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + step * (lane + 1);
    const int below = __popc(__ballot_sync(0xffffffffu, at < hi && cum(at) <= x));
    lo += step * below;
    hi = min(hi, lo + step);
  }
  return lo;
}

// The chunks of one kv head before tile i, for the three ways a launch is cut into tiles.
struct Line {
  const int* cum_in;  // kOneToken, kRagged
  int per_tile;       // kPrefix: length of each tile
  int tiles, chunks;  // of one kv head
  __device__ int cum(int i) const { return cum_in ? cum_in[i] : i * per_tile; }
};

// The line of a launch whose chunk sums lie in global memory (all but a kOneToken launch before its first CTA wrote them).
__device__ __forceinline__ Line line_of(const Problem& p, int chunk) {
  if (p.mode == kPrefix) {
    const int per_tile = (p.prefix_len + chunk - 1) / chunk + p.unit_extra;
    return {nullptr, per_tile, p.n_tiles, per_tile * p.n_tiles};
  }
  if (p.mode == kOneToken) return {p.cum_out, 0, p.n_tiles, p.cum_out[p.B]};
  return {p.plan + 2, 0, p.plan[0], p.plan[1]};
}

// How the line of a launch is cut into one piece for each CTA (or group of one).
// (A launch's line is shorter than 2^31: checked on the host. 64-bit divisions took a microsecond of these kernels' starts.)
struct Cuts {
  int long_end, per_long, per, early;
  __device__ Cuts(const Problem& p, const Line& line, int ctas) {
    const int all = line.chunks * p.nkv;
    early = p.early;
    const int ahead = early * p.lead;
    per = all > ahead ? (all - ahead + ctas - 1) / ctas : 0;
    per_long = early == 0 ? 0 : per > 0 ? per + p.lead : (all + early - 1) / early;
    long_end = early * per_long;
  }
  __device__ int begin(int cta) const { return cta < early ? cta * per_long : long_end + (cta - early) * per; }
  __device__ int owner(int x) const { return x < long_end ? x / per_long : early + (x - long_end) / per; }
};

// The pool's row of position j, whose page is `page`, for kv head h. A page outside the pool reads as zeros (a row past the
// maps' end) and is reported.
__device__ __forceinline__ int pool_row(const Problem& p, int page, int h, int j) {
  if (page >= 0 && page < p.n_pages) return (page * p.nkv + h) * p.page_size + (j & (p.page_size - 1));
  record_device_error(p.err, DK_DEVERR_BAD_POSITION);
  return p.n_pages * p.nkv * p.page_size;
}

// A CTA's piece of the line, unit by unit. Whole warps walk it.
template <int kChunk>
struct Walk {
  const Problem& p;
  const Line& line;
  int x, x1;
  int next_h, next_t, next_c;
  // the current part: chunks c0 .. c1 of the unit (h, ti)
  int h, ti, c0, c1;
  int u0;  // where the unit begins
  const Cuts cuts;
  Span<kChunk> span;  // the unit's chunks
  Tile t, next_tile;  // (the next tile's fields are loaded a part ahead)
  int last;           // the tile's last position
  __device__ Walk(const Problem& p_, const Line& line_, int cta, int ctas, int lane)
      : p(p_), line(line_), cuts(p_, line_, ctas) {
    const int all = line.chunks * p.nkv;
    x = min(cuts.begin(cta), all);
    x1 = min(cuts.begin(cta + 1), all);
    next_h = next_t = next_c = 0;
    if (x < x1) {
      next_h = x / line.chunks;
      const int r = x - next_h * line.chunks;
      next_t = find_tile_warp([&](int i) { return line.cum(i); }, line.tiles, r, lane);
      next_c = r - line.cum(next_t);
      next_tile = tile_at(p, next_t);
    }
  }
  __device__ bool more() const { return x < x1; }
  // Moves to the next part and returns the unit's chunks. A part may be empty (c1 <= c0): the end of a unit's stretch
  // of the line that stands for its fixed cost.
  __device__ Span<kChunk> step() {
    h = next_h, ti = next_t, c0 = next_c;
    u0 = x - c0;
    t = next_tile;
    last = tile_last(p, t);
    const Span<kChunk> span(t.p0, last, p.mask, p.capacity, p.page_size);
    const int to = min(span.n + p.unit_extra, c0 + (x1 - x));
    x += to - c0;
    c1 = min(to, span.n);
    next_c = 0;
    if (++next_t == line.tiles) next_t = 0, ++next_h;
    if (x < x1) next_tile = tile_at(p, next_t);
    return span;
  }
  // Moves to the next part that has chunks and whose tile has more than `tokens` tokens; false: there is none.
  __device__ bool next(int tokens) {
    while (more()) {
      span = step();
      if (c1 > c0 && t.ntok > tokens) return true;
    }
    return false;
  }
  // Does the unit begin in this part and go on in other CTAs' pieces? Then what the join needs of it.
  __device__ bool cut(const Span<kChunk>& span) const { return c0 == 0 && c1 < span.n; }
  __device__ int4 cut_record(const Span<kChunk>& span) const {
    return make_int4(t.t0, t.ntok, h, cuts.owner(u0 + span.n - 1));
  }
};

// Where the partial results of one unit lie: the CTAs first..last of the launch that took its chunks.
struct Pieces {
  int first, last;
  int64_t whole_slot;
};

// The unit's stretch of the line is u0 .. u1, `extra` of it at its end without chunks.
__device__ __forceinline__ Pieces pieces_of(const Cuts& cuts, int u0, int u1, int extra, int ctas, int64_t unit) {
  return {cuts.owner(u0), cuts.owner(u1 - extra - 1), 2ll * ctas + unit};
}

__device__ __forceinline__ int64_t piece_slot(const Pieces& w, int i) {
  return w.first == w.last ? w.whole_slot : 2ll * i + (i == w.first ? 1 : 0);
}

// Row of a tile's results that holds head g of its token `tok`: tiles of more than half_tokens tokens have a second
// half of 128 rows.
__device__ __forceinline__ int result_row(const Problem& p, int tok, int g) {
  return tok / p.half_tokens * 128 + tok % p.half_tokens * p.G + g;
}

// ------------------------------------------------------------------------------------------- host
// The launch of the 256-row tensor-core kernel (paged_attention_tc.cu): CTAs of one wave (0: it does not fit).
constexpr int kTcChunk = 128;
constexpr int kTcRows = 256;
constexpr int kTcUnitExtra = 3;  // a unit's fixed cost (its Q, first and last steps, output) in chunks (2, 4: up to 2 us more)
int tc_ctas(int64_t head_dim, int dtype);
// mk, mv: the pages as rows of head_dim, in boxes of 64 dims of min(page_size, kTcChunk) rows, 128-byte swizzle.
int tc_launch(const Problem& p, int64_t nq, int64_t head_dim, int dtype, int ctas, const CUtensorMap& mk,
              const CUtensorMap& mv, int wait_late, cudaStream_t st);

}  // namespace paged
}  // namespace dk
