// Attention over a paged cache: the plan of ragged launches, the kernel for few query rows per kv head
// (decode), the kernel that joins the partial results of split units, and the entry points.
//
//   out[t] = sum_j p[t][j] v[j],  p[t] = softmax over the visible j of scale * q[t] . k[j]
// Row t at position p sees j <= p with (window <= 0 or j > p - window or j < sinks); a row that sees
// nothing is zero. Scores, softmax statistics and sums are fp32; p is rounded to the cache's type for the
// tensor-core product with v, as its other operand is (the sum of p is not rounded).
//
// The decode kernel is bound by the bytes of k and v: each is read once for the G query heads that share
// it. A producer warp streams chunks of 64 positions, page by page, through a ring of TMA boxes (128-byte
// swizzle: the ldmatrix reads hit all banks); pages that no row sees are never read, and their table
// entries may be anything. Four consumer warps of a group take 16 positions each: q.k on the tensor cores with the
// query heads as the rows, online softmax in registers, p.v on the tensor cores with p taken from the
// score accumulators. A position that no row of the tile sees reads a zero row instead of v, so whatever
// the page holds there (infinities and NaN included) stays out; masked scores are replaced, not added to.
// Measured (28 heads over 4 kv heads of 128, bf16): 64 sequences of 8192, 1.07 GB, 174 us, 6.2 TB/s, 94% of the copy rate (168
// registers a thread, 20 to 28 bytes spilled); one of 640 (12 heads over 2) 7.8 us without the host, of 32768 16 us: a
// chain of launch, first copies and the join's launch.
#include <algorithm>
#include <climits>
#include <mutex>

#include "paged.cuh"

namespace dk {
namespace paged {
namespace {

constexpr int kChunk = 64;
constexpr int kGroups = 2;   // independent consumer groups of a CTA, each with a piece of the line of its own
constexpr int kCWarps = 4;   // warps of a group
constexpr int kThreads = kGroups * (kCWarps + 1) * 32;
constexpr int kMaxRing = 6;
constexpr int kPlanThreads = 1024;
constexpr int kRowsUnitExtra = 2;  // a unit's fixed cost (q, joining the warps, output) in chunks

// ------------------------------------------------------------------------------------ ragged plan
// One CTA cuts the sequences into tiles of tile_tokens tokens and sums up their chunks.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const Problem p, int32_t* plan, int4* info) {
  constexpr int kOwnTiles = 4;  // tiles of a sequence that its own thread writes
  __shared__ int warp_sum[kPlanThreads / 32];
  __shared__ int long_count;
  __shared__ int4 long_seq[kPlanThreads];  // {first tile, tiles, first token, end}
  __shared__ int2 long_len[kPlanThreads];  // {length, sequence}
  if (threadIdx.x == 0) long_count = 0;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // inclusive scan over the CTA; returns the exclusive prefix and the total
  auto scan = [&](int v, int& total) {
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    int w = warp_sum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, warp == 0 ? 0 : warp - 1);
    return (warp == 0 ? 0 : before) + s - v;
  };
  int32_t* cum = plan + 2;
  int tiles = 0, length = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    const int t0 = b < p.B ? min(max(p.starts[b], 0), p.T) : 0;
    const int t1 = b < p.B ? min(max(p.starts[b + 1], t0), p.T) : 0;
    const int mine = (t1 - t0 + p.tile_tokens - 1) / p.tile_tokens;
    int total;
    const int at = tiles + scan(mine, total);
    // sequence and first token of each tile; long sequences are filled in by the whole CTA below
    if (mine > 0 && at < p.max_tiles) info[at] = make_int4(t0, t1, length_of(p.lengths, b), b);
    for (int i = 1; i < min(mine, kOwnTiles) && at + i < p.max_tiles; ++i)
      info[at + i] = make_int4(t0 + i * p.tile_tokens, t1, length_of(p.lengths, b), b);
    __syncthreads();
    if (mine > kOwnTiles) {
      const int k = atomicAdd(&long_count, 1);
      long_seq[k] = make_int4(at, mine, t0, t1);
      long_len[k] = make_int2(length_of(p.lengths, b), b);
    }
    __syncthreads();
    for (int k = 0; k < long_count; ++k)
      for (int i = kOwnTiles + tid; i < long_seq[k].y && long_seq[k].x + i < p.max_tiles; i += kPlanThreads)
        info[long_seq[k].x + i] = make_int4(long_seq[k].z + i * p.tile_tokens, long_seq[k].w, long_len[k].x, long_len[k].y);
    __syncthreads();
    if (tid == 0) long_count = 0;
    tiles += total;
  }
  tiles = min(tiles, p.max_tiles);
  __syncthreads();  // the tiles written above are read by other threads below
  for (int i0 = 0; i0 < tiles; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int n = 0;
    if (i < tiles) {
      const int4 v = info[i];  // {first token, sequence's end, length, sequence}
      const int ntok = min(p.tile_tokens, v.y - v.x), p0 = v.z - (v.y - v.x);
      info[i] = make_int4(v.x, ntok, p0, v.w);
      n = Span<kTcChunk>(p0, p0 + ntok - 1, p.mask, p.capacity, p.page_size).n + p.unit_extra;
    }
    int total;
    const int at = length + scan(n, total);
    if (i < tiles) cum[i] = at;
    length += total;
  }
  if (tid == 0) {
    cum[tiles] = length;
    plan[0] = tiles;
    plan[1] = length;
  }
}

// ------------------------------------------------------------------------------------ decode kernel
template <int kHd>
struct Box {
  static constexpr int kSegs = kHd / 64;
  // A chunk of k or v: per 64-dim segment 64 rows of 128 bytes, 16-byte piece c of row r at c ^ (r % 8).
  static constexpr int kSegBytes = kChunk * 128;
  static constexpr int kTensorBytes = kSegs * kSegBytes;
  static constexpr int kSlotBytes = 2 * kTensorBytes;
  __device__ static const uint8_t* at(const uint8_t* t, int r, int d) {
    return t + (d >> 6) * kSegBytes + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4);
  }
};

__device__ __forceinline__ void group_sync(int group) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(kCWarps * 32) : "memory");
}

template <typename T, int kHd, int kRows>
__global__ void __launch_bounds__(kThreads)
    rows_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const Problem p,
                int ring, int wait_late) {
  using B = Box<kHd>;
  using E = Elem<T>;
  constexpr int kTiles = kHd / 8;
  constexpr bool kTwo = kRows == 16;  // rows 8..15 of the MMA in use
  constexpr int kR = kTwo ? 2 : 1;
  __shared__ __align__(16) uint4 vzero;
  __shared__ float pre_ml_sh[kGroups][kCWarps * kRows * 2];
  __shared__ float pre_w_sh[kGroups][kCWarps * kRows];
  __shared__ float fin_sh[kGroups][kRows * 2];
  __shared__ __align__(8) uint64_t full_sh[kGroups][kMaxRing], empty_sh[kGroups][kMaxRing];
  __shared__ int warp_sum[kThreads / 32 + 1];
  extern __shared__ __align__(128) uint8_t dsm_raw[];
  uint8_t* base = dsm_raw + ((1024u - (smem_addr(dsm_raw) & 1023u)) & 1023u);
  int* cum_sh = reinterpret_cast<int*>(base);  // [B + 1], before the first copies land there

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool producer = warp >= kGroups * kCWarps;
  const int group = producer ? warp - kGroups * kCWarps : warp / kCWarps;
  const int cta = blockIdx.x * kGroups + group, ctas = gridDim.x * kGroups;  // pieces of the line: one a group
  uint8_t* slots = base + group * ring * B::kSlotBytes;
  float* pre_o = reinterpret_cast<float*>(base + kGroups * ring * B::kSlotBytes) + group * kCWarps * kRows * kHd;
  float *pre_ml = pre_ml_sh[group], *pre_w = pre_w_sh[group], *fin = fin_sh[group];
  uint64_t *full = full_sh[group], *empty = empty_sh[group];
  if (tid == 0) {
    for (int i = 0; i < kGroups * kMaxRing; ++i) {
      mbar_init(&full_sh[0][i], 1);
      mbar_init(&empty_sh[0][i], kCWarps);
    }
    fence_mbar_init();
    vzero = make_uint4(0, 0, 0, 0);
    prefetch_tensormap(&mk);
    prefetch_tensormap(&mv);
  }
  if (!wait_late) pdl_wait();
  pdl_trigger();

  Line line{cum_sh, 0, p.n_tiles, 0};
  {  // every CTA sums up the sequences' chunks for itself
    int carry = 0;
    for (int b0 = 0; b0 < p.B; b0 += kThreads) {
      const int b = b0 + tid;
      int n = 0;
      if (b < p.B) {
        const int last = length_of(p.lengths, b) - 1;
        n = Span<kChunk>(last, last, p.mask, p.capacity, p.page_size).n + p.unit_extra;
      }
      int s = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
      }
      __syncthreads();
      if (lane == 31) warp_sum[warp] = s;
      __syncthreads();
      int before = carry;
      for (int w = 0; w < kThreads / 32; ++w) {
        const int ws = warp_sum[w];
        if (w < warp) before += ws;
        carry += ws;
      }
      if (b < p.B) cum_sh[b] = before + s - n;
    }
    if (tid == 0) cum_sh[p.B] = carry;
    line.chunks = carry;
    __syncthreads();
    if (blockIdx.x == 0)  // for the join kernel
      for (int i = tid; i <= p.B; i += kThreads) p.cum_out[i] = cum_sh[i];
  }
  __syncthreads();

  Walk<kChunk> walk(p, line, cta, ctas, lane);
  __syncthreads();  // the sums have been read: copies may land on them
  bool ok = true;
  int fill = 0;  // ring fills so far

  if (producer) {
    // ---------------------------------------------------------------- producer warps: one lane per box
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (the sums lay there)
    const int box = min(p.page_size, kChunk);  // rows of one box
    const int boxes = kChunk / box;
    const int kv = lane & 1, sg = (lane >> 1) % B::kSegs, pg = lane / (2 * B::kSegs);
    while (walk.more() && ok) {
      const Span<kChunk> span = walk.step();
      const int h = walk.h, c0 = walk.c0, c1 = walk.c1;
      const int32_t* table = walk.t.table;
      if (lane == 0 && walk.last >= p.capacity) record_device_error(p.err, DK_DEVERR_BAD_POSITION);  // cut to the table
      // this lane's page in chunk i of the unit; INT_MIN: none, or nothing that a row sees
      auto entry = [&](int i) {
        const int j = i * kChunk + pg * box;
        return i < c1 && pg < boxes && span.needs(j, box, p.mask) ? table[span.position(j) >> p.page_shift] : INT_MIN;
      };
      int next = entry(c0);
      for (int i = c0; i < c1; ++i, ++fill) {
        const int page = next;
        next = entry(i + 1);
        const int s = fill % ring;
        if (fill >= ring && !wait_for(&empty[s], ((fill / ring) - 1) & 1, p.err, DK_DEVERR_WAIT_EMPTY)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const bool mine = page != INT_MIN;
        const unsigned want = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) mbar_arrive_expect_tx(&full[s], __popc(want) * box * 128);
        __syncwarp();
        if (mine) {
          const int y = pool_row(p, page, h, span.position(i * kChunk + pg * box));
          uint8_t* dst = slots + s * B::kSlotBytes + kv * B::kTensorBytes + sg * B::kSegBytes + pg * box * 128;
          tma_load_2d(dst, kv ? &mv : &mk, sg * 64, y, &full[s]);
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- consumer warps
    const int g = lane >> 2, tq = lane & 3;
    const int mi = lane >> 3, rr = lane & 7;
    const int sub = warp % kCWarps, gtid = tid - group * kCWarps * 32;
    if (gtid == 0) p.cut[cta] = make_int4(0, 0, 0, 0);
    while (walk.more()) {
      const Span<kChunk> span = walk.step();
      const Tile t = walk.t;
      const int h = walk.h, c0 = walk.c0, c1 = walk.c1;
      if (c1 <= c0) continue;
      const int rows = p.G;  // one token's
      const int p0 = t.p0 - span.shift;
      // this lane's rows g and g + 8: positions, and q as the MMA's A operand
      int pos[kR];
      uint32_t qa[kHd / 16][2 * kR];
#pragma unroll
      for (int e = 0; e < kR; ++e) {
        const int row = g + 8 * e;
        pos[e] = row < rows ? p0 : -1;
        const T* qr = static_cast<const T*>(p.q) + t.t0 * p.ldq + (h * p.G + row) * kHd;
#pragma unroll
        for (int ks = 0; ks < kHd / 16; ++ks) {
          qa[ks][e] = row < rows ? *reinterpret_cast<const uint32_t*>(qr + 16 * ks + 2 * tq) : 0u;
          qa[ks][kR + e] = row < rows ? *reinterpret_cast<const uint32_t*>(qr + 16 * ks + 8 + 2 * tq) : 0u;
        }
      }
      float o[kTiles][4];
#pragma unroll
      for (int j = 0; j < kTiles; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      float m_run[kR], l_run[kR];
#pragma unroll
      for (int e = 0; e < kR; ++e) m_run[e] = -INFINITY, l_run[e] = 0.f;

      for (int i = c0; i < c1; ++i, ++fill) {
        const int s = fill % ring;
        if (ok && !wait_for(&full[s], (fill / ring) & 1, p.err, DK_DEVERR_WAIT_FULL)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        const int j0 = i * kChunk + 16 * sub;  // this warp's 16 positions
        if (ok && span.needs(j0, 16, p.mask)) {
          const uint8_t* kt = slots + s * B::kSlotBytes;
          const uint8_t* vt = kt + B::kTensorBytes;
          float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
          const int krow = 16 * sub + 8 * (mi >> 1) + rr;
#pragma unroll
          for (int ks = 0; ks < kHd / 16; ++ks) {
            uint32_t kb[4];
            ldmatrix_x4(kb, B::at(kt, krow, 16 * ks + 8 * (mi & 1)));
            const uint32_t a1 = kTwo ? qa[ks][kR - 1] : 0u, a3 = kTwo ? qa[ks][2 * kR - 1] : 0u;
            E::mma(sc[0], qa[ks][0], a1, qa[ks][kR], a3, kb[0], kb[1]);
            E::mma(sc[1], qa[ks][0], a1, qa[ks][kR], a3, kb[2], kb[3]);
          }
          // every row sees all 16 positions (nothing to mask)?
          const bool clear = j0 + 15 <= p0 && (p.mask.window <= 0 || j0 > p0 - p.mask.window || j0 + 15 < p.mask.sinks) &&
                             j0 + 15 < span.end;
          uint32_t pa[2][kR];  // p as the MMA's A operand
#pragma unroll
          for (int e = 0; e < kR; ++e) {
            float bm = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const int j = j0 + 8 * nt + 2 * tq + u;
                float v = sc[nt][2 * e + u] * p.scale2;
                if (!clear && !(j < span.end && p.mask.sees(pos[e], j))) v = -INFINITY;
                sc[nt][2 * e + u] = v;
                bm = fmaxf(bm, v);
              }
            bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 1));
            bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 2));
            const float m_new = fmaxf(m_run[e], bm);
            const float m_use = m_new == -INFINITY ? 0.f : m_new;  // a row that has seen nothing yet
            const float alpha = exp2_approx(m_run[e] - m_use);
            float pr[2][2], ls = 0.f;
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                pr[nt][u] = exp2_approx(sc[nt][2 * e + u] - m_use);
                ls += pr[nt][u];
              }
            l_run[e] = fmaf(l_run[e], alpha, ls);
            m_run[e] = m_new;
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
              o[j][2 * e] *= alpha;
              o[j][2 * e + 1] *= alpha;
            }
            pa[0][e] = E::pack(pr[0][0], pr[0][1]);
            pa[1][e] = E::pack(pr[1][0], pr[1][1]);
          }
          const int vrow = 16 * sub + (mi & 1) * 8 + rr;
          const bool zero = !clear && !span.needs(i * kChunk + vrow, 1, p.mask);
          const uint32_t a1 = kTwo ? pa[0][kR - 1] : 0u, a3 = kTwo ? pa[1][kR - 1] : 0u;
#pragma unroll
          for (int dp = 0; dp < kHd / 16; ++dp) {
            uint32_t vb[4];
            ldmatrix_x4_trans(vb, zero ? reinterpret_cast<const uint8_t*>(&vzero) : B::at(vt, vrow, 16 * dp + (mi >> 1) * 8));
            E::mma(o[2 * dp], pa[0][0], a1, pa[1][0], a3, vb[0], vb[1]);
            E::mma(o[2 * dp + 1], pa[0][0], a1, pa[1][0], a3, vb[2], vb[3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }
      // the warps' results of this part of the unit, joined
      if (gtid == 0 && walk.cut(span)) p.cut[cta] = walk.cut_record(span);
#pragma unroll
      for (int e = 0; e < kR; ++e) {
        l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 1);
        l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 2);
        const int row = g + 8 * e;
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
          *reinterpret_cast<float2*>(&pre_o[(sub * kRows + row) * kHd + 8 * j + 2 * tq]) =
              make_float2(o[j][2 * e], o[j][2 * e + 1]);
        if (tq == 0) {
          pre_ml[(sub * kRows + row) * 2] = m_run[e];
          pre_ml[(sub * kRows + row) * 2 + 1] = l_run[e];
        }
      }
      group_sync(group);
      const bool all_of_it = c0 == 0 && c1 == span.n, whole = all_of_it && !p.always_partial;
      if (gtid < kRows) {
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kCWarps; ++w) mx = fmaxf(mx, pre_ml[(w * kRows + gtid) * 2]);
        const float m_use = mx == -INFINITY ? 0.f : mx;
        float ls = 0.f;
#pragma unroll
        for (int w = 0; w < kCWarps; ++w) {
          const float wt = exp2_approx(pre_ml[(w * kRows + gtid) * 2] - m_use);
          pre_w[w * kRows + gtid] = wt;
          ls = fmaf(wt, pre_ml[(w * kRows + gtid) * 2 + 1], ls);
        }
        fin[2 * gtid] = mx;
        fin[2 * gtid + 1] = ls;
      }
      group_sync(group);
      const int64_t slot = partial_slot(ctas, cta, c0 == 0, all_of_it, h * line.tiles + walk.ti);
      if (ok) {
        for (int e = gtid; e < rows * (kHd / 4); e += kCWarps * 32) {
          const int row = e / (kHd / 4), d = 4 * (e % (kHd / 4));
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kCWarps; ++w) {
            const float wt = pre_w[w * kRows + row];
            const float4 v = *reinterpret_cast<const float4*>(&pre_o[(w * kRows + row) * kHd + d]);
            a.x = fmaf(wt, v.x, a.x), a.y = fmaf(wt, v.y, a.y), a.z = fmaf(wt, v.z, a.z), a.w = fmaf(wt, v.w, a.w);
          }
          if (whole) {
            const float l = fin[2 * row + 1];
            const float inv = l == 0.f ? 0.f : 1.f / l;
            T* dst = static_cast<T*>(p.out) + (static_cast<int64_t>(t.t0) * p.nkv * p.G + h * p.G + row) * kHd + d;
            *reinterpret_cast<uint2*>(dst) = make_uint2(E::pack(a.x * inv, a.y * inv), E::pack(a.z * inv, a.w * inv));
          } else {
            *reinterpret_cast<float4*>(&p.part_o[(slot * kRows + row) * kHd + d]) = a;
          }
        }
        if (!whole && gtid < rows)
          *reinterpret_cast<float2*>(&p.part_ml[(slot * kRows + gtid) * 2]) = make_float2(fin[2 * gtid], fin[2 * gtid + 1]);
      }
      group_sync(group);  // pre_o, pre_ml and fin are written again by the next piece
    }
  }
  if (__syncthreads_or(!ok) && producer && lane == 0) {
    // a wait gave up: let copies still in flight land before the shared memory goes away (bounded)
    const uint64_t t0 = globaltimer_ns();
    for (int f = max(0, fill - ring); f < fill; ++f)
      while (!mbar_try_wait(&full[f % ring], (f / ring) & 1) && globaltimer_ns() - t0 < 500000000ull) {
      }
  }
  if (wait_late) pdl_wait();
}

// ------------------------------------------------------------------------------------ join
// How a join's block takes results: kRows rows, kDims groups of four dims of each (the grid's z has the others), and kParts
// stretches of a unit's pieces, whose sums are joined in order at the end. A unit cut into many pieces (few sequences, long
// ones: up to one for every CTA) would otherwise be one long chain of loads on one SM.
template <int kR, int kD, int kP, int kA>
struct JoinShape {
  static constexpr int kRows = kR, kDims = kD, kParts = kP, kAhead = kA;  // kAhead: pieces loaded at a time
  static constexpr int kLanes = kR * kD, kThreads = kLanes * kP;
  int lane, part, row, d4;  // of this thread; row: in the whole grid's y (or x)
  __device__ explicit JoinShape(int y)
      : lane(threadIdx.x % kLanes), part(threadIdx.x / kLanes), row(y * kR + lane % kR), d4(blockIdx.z * kD + lane / kR) {}
};

template <typename T, int kHd>
struct Joined {
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ void add(float m2, float l2, const float4& o) {
    const float mx = fmaxf(m, m2), use = mx == -INFINITY ? 0.f : mx;
    const float keep = exp2_approx(m - use), take = exp2_approx(m2 - use);
    m = mx;
    l = fmaf(l, keep, l2 * take);
    acc.x = fmaf(acc.x, keep, o.x * take), acc.y = fmaf(acc.y, keep, o.y * take);
    acc.z = fmaf(acc.z, keep, o.z * take), acc.w = fmaf(acc.w, keep, o.w * take);
  }
  // Adds the pieces from..to of a unit's row in order, kAhead of them loaded at a time. d4: the lane's dims / 4.
  template <int kAhead>
  __device__ void add(const Problem& p, const Pieces& w, int from, int to, int tile_rows, int row, int d4) {
    const int64_t at = p.rows_inner ? static_cast<int64_t>(d4) * tile_rows + row : static_cast<int64_t>(row) * (kHd / 4) + d4;
    for (int i0 = from; i0 <= to; i0 += kAhead) {
      float2 ml[kAhead];
      float4 o[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (i0 + a > to) break;
        const int64_t slot = piece_slot(w, i0 + a);
        ml[a] = *reinterpret_cast<const float2*>(&p.part_ml[(slot * tile_rows + row) * 2]);
        o[a] = reinterpret_cast<const float4*>(p.part_o)[slot * tile_rows * (kHd / 4) + at];
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (i0 + a > to) break;
        add(ml[a].x, ml[a].y, o[a]);
      }
    }
  }
  // Part `part` of `parts` of a unit's pieces.
  template <int kAhead>
  __device__ void add_part(const Problem& p, const Pieces& w, int part, int parts, int tile_rows, int row, int d4) {
    const int n = w.last - w.first + 1;
    add<kAhead>(p, w, w.first + n * part / parts, w.first + n * (part + 1) / parts - 1, tile_rows, row, d4);
  }
  // Joins the parts of a block in order, called by all of its threads; the first has the result.
  template <typename Shape>
  __device__ void join_parts(const Shape& at) {
    if constexpr (Shape::kParts > 1) {
      __shared__ float2 part_ml[Shape::kParts - 1][Shape::kLanes];
      __shared__ float4 part_o[Shape::kParts - 1][Shape::kLanes];
      if (at.part > 0) {
        part_ml[at.part - 1][at.lane] = make_float2(m, l);
        part_o[at.part - 1][at.lane] = acc;
      }
      __syncthreads();
      if (at.part == 0)
        for (int i = 0; i < Shape::kParts - 1; ++i) add(part_ml[i][at.lane].x, part_ml[i][at.lane].y, part_o[i][at.lane]);
    }
  }
  __device__ void store(T* out, int d4) const {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(out + 4 * d4) = make_uint2(Elem<T>::pack(acc.x * inv, acc.y * inv), Elem<T>::pack(acc.z * inv, acc.w * inv));
  }
};

template <typename T, int kHd>
__device__ __forceinline__ T* out_row(const Problem& p, int t, int head) {
  return static_cast<T*>(p.out) + (static_cast<int64_t>(t) * p.nkv * p.G + head) * kHd;
}

// Joins the units that a piece's end cuts. Block (x, y): rows of the unit that CTA x began, if there is one, or with
// `by_unit` (launches of fewer units than CTAs) of unit x, if it is cut.
template <typename T, int kHd, typename Shape>
__global__ void __launch_bounds__(Shape::kThreads) join_split_kernel(const Problem p, int tile_rows, int ctas, int by_unit) {
  pdl_trigger();
  pdl_wait();
  int4 c;  // {first token, tokens, kv head, last CTA}
  Pieces w{static_cast<int>(blockIdx.x), 0, 0};
  if (by_unit) {
    const Line line = line_of(p, kTcChunk);
    const int x = blockIdx.x;
    if (x >= line.tiles * p.nkv) return;
    const int h = x / line.tiles, ti = x - h * line.tiles;
    const Tile t = tile_at(p, ti);
    w = pieces_of(Cuts(p, line, ctas), h * line.chunks + line.cum(ti), h * line.chunks + line.cum(ti + 1), p.unit_extra, ctas, 0);
    if (w.first == w.last) return;
    c = make_int4(t.t0, t.ntok, h, w.last);
  } else {
    c = p.cut[blockIdx.x];
    w.last = c.w;
  }
  const Shape at(blockIdx.y);
  const int rows = c.y * p.G, i = at.row;
  if (static_cast<int>(blockIdx.y) * Shape::kRows >= rows) return;
  Joined<T, kHd> sum;
  if (i < rows)
    sum.template add_part<Shape::kAhead>(p, w, at.part, Shape::kParts, tile_rows, result_row(p, i / p.G, i % p.G), at.d4);
  sum.join_parts(at);
  if (at.part == 0 && i < rows) sum.store(out_row<T, kHd>(p, c.x + i / p.G, c.z * p.G + i % p.G), at.d4);
}

// Joins the prefix's results (`a`) with those of the sequences' own positions (`b`). Block (x, h): rows (token, head of
// kv head h). The last part of a block takes the own positions, the others the prefix's pieces.
template <typename T, int kHd, typename Shape>
__global__ void __launch_bounds__(Shape::kThreads)
    join_prefix_kernel(const Problem a, int a_ctas, const Problem b, int b_ctas, int b_rows) {
  pdl_trigger();
  pdl_wait();
  const Shape at(blockIdx.x);
  const int h = blockIdx.y;
  const bool live = at.row < a.T * a.G;
  const int t = live ? at.row / a.G : 0, g = live ? at.row % a.G : 0;
  Joined<T, kHd> sum;
  if (live && at.part < Shape::kParts - 1) {
    const Line line = line_of(a, kTcChunk);
    const int unit = h * a.n_tiles + t / a.tile_tokens, a0 = unit * line.per_tile;
    const Pieces w = pieces_of(Cuts(a, line, a_ctas), a0, a0 + line.per_tile, a.unit_extra, a_ctas, unit);
    sum.template add_part<Shape::kAhead>(a, w, at.part, Shape::kParts - 1, kTcRows, result_row(a, t % a.tile_tokens, g), at.d4);
  } else if (live) {
    const Line own = line_of(b, 1);
    if (own.chunks > 0) {
      const int ti = b.mode == kRagged ? find_tile([&](int i) { return b.tile_info[i].x; }, own.tiles, t) : t;
      const Tile tile = tile_at(b, ti);
      const int tok = t - tile.t0;  // (a row that `starts` leaves out belongs to no tile)
      const int b0 = h * own.chunks + own.cum(ti), b1 = h * own.chunks + own.cum(ti + 1);
      const Pieces w = pieces_of(Cuts(b, own, b_ctas), b0, b1, b.unit_extra, b_ctas, h * own.tiles + ti);
      if (tok >= 0 && tok < tile.ntok) sum.template add<2>(b, w, w.first, w.last, b_rows, result_row(b, tok, g), at.d4);
    }
  }
  sum.join_parts(at);
  if (at.part == 0 && live) sum.store(out_row<T, kHd>(b, t, h * b.G + g), at.d4);
}

}  // namespace

// ------------------------------------------------------------------------------------ host
namespace {

// Tiles that are cut into more pieces than this, on average, are joined in parts (42 tokens after 32768 positions: 28 us, 46
// without; one short sequence 12.1, 12.2; 16 sequences of 8192 with 4 tokens each, 9 pieces a unit: 44, 40).
constexpr int kFewPieces = 8;
constexpr int kMaxBatch = 4096;  // kOneToken: the chunk sums of a batch lie in shared memory

// What a rows_kernel launch takes: slots of its ring, shared memory, and the CTAs of one wave (0: it does not fit).
struct RowsShape {
  int ring;
  size_t smem;
  int ctas;
};

template <typename T, int kHd, int kRows>
RowsShape rows_shape() {
  static std::mutex mu;
  static int per_sm[64];  // by device; 0: not asked yet
  RowsShape s;
  s.ring = kHd == 64 ? (kRows == 8 ? 6 : 5) : (kRows == 8 ? 3 : 2);
  s.smem = 1024 + static_cast<size_t>(kGroups) * (s.ring * Box<kHd>::kSlotBytes + kCWarps * kRows * kHd * 4);
  static_assert((kMaxBatch + 1) * 4 <= kGroups * 2 * Box<kHd>::kSlotBytes, "the chunk sums fit the ring");
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  int& n = per_sm[dev & 63];
  if (n == 0) {
    auto k = rows_kernel<T, kHd, kRows>;
    if (opt_in_dynamic_smem(k) < static_cast<int>(s.smem) ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, kThreads, s.smem) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
  }
  s.ctas = n * device_info().num_sms;
  return s;
}

struct Sizes {
  int64_t T, B, nq, nkv, hd, prefix_len;
  bool ragged;
  int dtype;
};

RowsShape rows_shape_of(const Sizes& z, int rows) {
#define DK_SHAPE(TT) \
  (z.hd == 128 ? (rows == 8 ? rows_shape<TT, 128, 8>() : rows_shape<TT, 128, 16>()) \
               : (rows == 8 ? rows_shape<TT, 64, 8>() : rows_shape<TT, 64, 16>()))
  return z.dtype == DK_F16 ? DK_SHAPE(__half) : DK_SHAPE(__nv_bfloat16);
#undef DK_SHAPE
}

cudaError_t launch_rows(const Sizes& z, int rows, const RowsShape& s, cudaStream_t st, const CUtensorMap& mk,
                        const CUtensorMap& mv, const Problem& p, int wait_late) {
#define DK_ROWS(TT, HH, RR) \
  launch(rows_kernel<TT, HH, RR>, dim3(s.ctas), dim3(kThreads), s.smem, st, pdl_enabled(), dim3(1, 1, 1), mk, mv, p, s.ring, wait_late)
#define DK_ROWS_T(TT) \
  (z.hd == 128 ? (rows == 8 ? DK_ROWS(TT, 128, 8) : DK_ROWS(TT, 128, 16)) : (rows == 8 ? DK_ROWS(TT, 64, 8) : DK_ROWS(TT, 64, 16)))
  return z.dtype == DK_F16 ? DK_ROWS_T(__half) : DK_ROWS_T(__nv_bfloat16);
#undef DK_ROWS_T
#undef DK_ROWS
}

// A workspace cut into aligned areas; with a null base it only counts.
struct Cutter {
  char* base;
  uint64_t used = 0;
  template <typename T>
  T* take(uint64_t count) {
    T* at = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += (count * sizeof(T) + 255) / 256 * 256;
    return at;
  }
};

// One launch over the chunks of one kind of tiles, with its areas of the workspace.
struct Pass {
  Problem p;
  bool tc;  // 256-row tiles on the tensor-core kernel
  RowsShape shape;
  int rows, ctas;
};

void cut_pass(const Sizes& z, Cutter& c, Pass& a, bool always_partial) {
  Problem& p = a.p;
  if (a.tc) {
    a.rows = kTcRows;
    p.unit_extra = kTcUnitExtra;
    p.rows_inner = 1;
    a.ctas = tc_ctas(z.hd, z.dtype);
  } else {
    a.rows = z.nq / z.nkv <= 8 ? 8 : 16;
    a.shape = rows_shape_of(z, a.rows);
    a.ctas = a.shape.ctas * kGroups;
    p.unit_extra = kRowsUnitExtra;
  }
  const int64_t tiles = p.mode == kRagged ? p.max_tiles : p.n_tiles;
  const int64_t slots = 2ll * a.ctas + (always_partial ? z.nkv * tiles : 0);
  p.always_partial = always_partial;
  p.part_o = c.take<float>(slots * a.rows * z.hd);
  p.part_ml = c.take<float>(slots * a.rows * 2);
  p.cut = c.take<int4>(a.ctas);
  p.cum_out = p.mode == kOneToken ? c.take<int32_t>(z.B + 1) : nullptr;
  p.plan = p.mode == kRagged ? c.take<int32_t>(3 + static_cast<int64_t>(p.max_tiles)) : nullptr;
  p.tile_info = p.mode == kRagged ? c.take<int4>(p.max_tiles) : nullptr;
}

// Tiles of one token, or of two halves of up to 128 rows each.
void set_tile(const Sizes& z, Pass& a, bool tc) {
  a.tc = tc;
  a.p.half_tokens = tc ? static_cast<int>(128 / (z.nq / z.nkv)) : 1;
  a.p.tile_tokens = tc ? 2 * a.p.half_tokens : 1;
}

// One token for each sequence goes to the rows kernel, several to the tiles (64 sequences of 8192, 12 heads over 2 kv heads,
// one token each, without the host: 91 us on the rows kernel, 111 as tiles; one of 640: 9.4 and 13.6; 4 tokens each as tiles:
// 109).
void shape_own(const Sizes& z, Pass& a) {
  set_tile(z, a, z.ragged);
  a.p.mode = z.ragged ? kRagged : kOneToken;
  a.p.max_tiles = z.ragged ? static_cast<int>(z.T / a.p.tile_tokens + z.B) : 0;
  a.p.n_tiles = static_cast<int>(z.B);
}

// A prefix is read by tiles however few the rows are (8192 positions for one token of 12 heads: 17 us, 29 on the rows
// kernel).
void shape_prefix(const Sizes& z, Pass& a) {
  set_tile(z, a, true);
  a.p.mode = kPrefix;
  a.p.n_tiles = static_cast<int>((z.T + a.p.tile_tokens - 1) / a.p.tile_tokens);
  a.p.prefix_len = static_cast<int>(z.prefix_len);
}

// The two launches of a call with a prefix run side by side: the prefix's takes most of the SMs, and the own positions'
// starts on the others right away, with longer pieces there. How long the prefix's takes is known here: about 6 us and 2 us
// for each chunk of a CTA's piece; a group of the other takes 1.1 us for a chunk.
void share_gpu(Pass& pre, Pass& own) {
  if (own.tc || !pdl_enabled()) return;
  const int sms = device_info().num_sms;
  const int64_t n = static_cast<int64_t>((pre.p.prefix_len + kTcChunk - 1) / kTcChunk + pre.p.unit_extra) * pre.p.n_tiles * pre.p.nkv;
  const int64_t most = sms * 7 / 8, per = (n + most - 1) / most;
  pre.ctas = static_cast<int>((n + per - 1) / per);
  own.p.early = kGroups * (sms - pre.ctas);
  own.p.lead = static_cast<int>((60 + 20 * per) / 11);
}

int check_sizes(const char* what, const Sizes& z) {
  if (z.T < 0 || z.B < 0 || (z.B == 0 && z.T > 0) || z.nq <= 0 || z.nkv <= 0 || z.prefix_len < 0)
    return set_error(DK_ERR_INVALID, "%s: bad sizes", what);
  if (z.hd != 64 && z.hd != 128) return set_error(DK_ERR_UNSUPPORTED, "%s: head_dim %lld (64 or 128)", what, (long long)z.hd);
  if (z.dtype != DK_F16 && z.dtype != DK_BF16) return set_error(DK_ERR_UNSUPPORTED, "%s: dtype %d", what, z.dtype);
  if (z.nq % z.nkv != 0 || z.nq / z.nkv > 16)
    return set_error(DK_ERR_UNSUPPORTED, "%s: %lld query heads over %lld kv heads (a multiple, at most 16 each)", what,
                     (long long)z.nq, (long long)z.nkv);
  if (!z.ragged && z.T != z.B) return set_error(DK_ERR_INVALID, "%s: without starts there is one token per sequence", what);
  if (!z.ragged && z.B > kMaxBatch)
    return set_error(DK_ERR_UNSUPPORTED, "%s: %lld sequences (at most %d without starts)", what, (long long)z.B, kMaxBatch);
  if (z.T * (z.nq / z.nkv) > (1 << 30) || z.T > (1 << 26) || z.B > (1 << 26) || z.nkv > 65535 || z.prefix_len > (1 << 30))
    return set_error(DK_ERR_INVALID, "%s: sizes out of range", what);
  return DK_OK;
}

template <typename Shape>
dim3 join_grid(int64_t x, int64_t y, int64_t hd) {
  return dim3(static_cast<unsigned>(x), static_cast<unsigned>(y), static_cast<unsigned>(hd / 4 / Shape::kDims));
}

template <typename T, int kHd>
cudaError_t launch_join(const Sizes& z, cudaStream_t st, const Pass* prefix, const Pass& own) {
  // Tiles are bound by the bytes of their pieces (for a prompt of 8192 about 40 MB in L2, 6 us) and by the number of blocks:
  // two or four rows a thread, or fewer blocks that loop, came out the same or slower.
  using Tiles = JoinShape<8, kHd / 4, 1, 2>;
  using Few = JoinShape<8, 8, 4, 4>;
  using OneToken = JoinShape<kHd == 128 ? 2 : 4, kHd / 4, 4, 4>;
  const dim3 one(1, 1, 1);
  if (prefix != nullptr) {
    const int64_t rows = z.T * (z.nq / z.nkv);
    return launch(join_prefix_kernel<T, kHd, Few>, join_grid<Few>((rows + Few::kRows - 1) / Few::kRows, z.nkv, kHd),
                  dim3(Few::kThreads), 0, st, pdl_enabled(), one, prefix->p, prefix->ctas, own.p, own.ctas, own.rows);
  }
  if (!own.tc)
    return launch(join_split_kernel<T, kHd, OneToken>, join_grid<OneToken>(own.ctas, own.rows / OneToken::kRows, kHd),
                  dim3(OneToken::kThreads), 0, st, pdl_enabled(), one, own.p, own.rows, own.ctas, 0);
  const int64_t units = static_cast<int64_t>(own.p.max_tiles) * z.nkv, x = std::min<int64_t>(units, own.ctas);
  const int64_t y = (std::min<int64_t>(z.T, own.p.tile_tokens) * (z.nq / z.nkv) + 7) / 8;
  const int by_unit = units < own.ctas;
  if (units * kFewPieces <= own.ctas)
    return launch(join_split_kernel<T, kHd, Few>, join_grid<Few>(x, y, kHd), dim3(Few::kThreads), 0, st, pdl_enabled(), one,
                  own.p, own.rows, own.ctas, by_unit);
  return launch(join_split_kernel<T, kHd, Tiles>, join_grid<Tiles>(x, y, kHd), dim3(Tiles::kThreads), 0, st, pdl_enabled(), one,
                own.p, own.rows, own.ctas, by_unit);
}

uint64_t workspace_of(const Sizes& z) {
  Cutter c{nullptr};
  Pass own = {}, pre = {};
  shape_own(z, own);
  cut_pass(z, c, own, z.prefix_len > 0);
  if (z.prefix_len > 0) {
    shape_prefix(z, pre);
    cut_pass(z, c, pre, true);
  }
  return c.used;
}

}  // namespace
}  // namespace paged
}  // namespace dk

using namespace dk;
using namespace dk::paged;

extern "C" int dk_paged_attention_workspace_bytes(int64_t T, int64_t B, int64_t nq, int64_t nkv, int64_t head_dim,
                                                  int32_t dtype, int32_t ragged, int64_t prefix_len, uint64_t* bytes) {
  const Sizes z{T, B, nq, nkv, head_dim, prefix_len, ragged != 0, dtype};
  if (const int rc = check_sizes("paged_attention_workspace_bytes", z)) return rc;
  if (!bytes) return set_error(DK_ERR_INVALID, "paged_attention_workspace_bytes: bytes is NULL");
  *bytes = workspace_of(z);
  return DK_OK;
}

namespace {

int attention(const char* what, const dk_paged_attention_args* args, bool prefix) {
  if (args == nullptr) return set_error(DK_ERR_INVALID, "%s: NULL arguments", what);
  const dk_paged_attention_args& a = *args;
  const Sizes z{a.T, a.B, a.n_q, a.n_kv, a.head_dim, prefix ? a.prefix_len : 0, a.starts != nullptr, static_cast<int>(a.dtype)};
  const int64_t n_pages = a.n_pages, page_size = a.page_size, table_width = a.table_width;
  int64_t window = prefix ? 0 : a.window;
  int64_t sinks = prefix ? 0 : a.sinks;
  if (const int rc = check_sizes(what, z)) return rc;
  if (n_pages <= 0 || table_width <= 0 || window < 0 || sinks < 0) return set_error(DK_ERR_INVALID, "%s: bad sizes", what);
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
    return set_error(DK_ERR_UNSUPPORTED, "%s: page_size %lld (a power of two from 16 to 256)", what, (long long)page_size);
  // Positions and offsets are 32-bit: the largest sums are a position rounded up to whole chunks with their boxes, and the
  // window before the position of a row that comes up to T rows before its sequence's first one.
  constexpr int64_t kMaxPositions = (int64_t(1) << 31) - 1024;
  if (n_pages > INT32_MAX || table_width > INT32_MAX || n_pages * z.nkv > INT32_MAX ||
      n_pages * z.nkv * page_size + kChunk > INT32_MAX || table_width * page_size + z.T > kMaxPositions ||
      window > INT32_MAX || sinks > INT32_MAX)
    return set_error(DK_ERR_INVALID,
                     "%s: pages x kv heads x page_size, window and sinks must stay below 2^31, a table row's positions with T 1024 below", what);
  // A window of all positions masks none, and sinks end with the positions: sums with them stay in range.
  window = std::min(window, table_width * page_size);
  sinks = std::min(sinks, table_width * page_size);
  const int64_t ldq = z.T > 1 ? a.ldq : z.nq * z.hd;
  if (z.T == 0) return DK_OK;
  if (ldq < z.nq * z.hd) return set_error(DK_ERR_INVALID, "%s: q's tokens overlap", what);
  if (!a.q || !a.k_pages || !a.v_pages || !a.page_table || !a.lengths || !a.out || !a.workspace ||
      (z.prefix_len > 0 && !a.prefix_table))
    return set_error(DK_ERR_INVALID, "%s: NULL pointer", what);
  if (!aligned16(a.q) || !aligned16(a.k_pages) || !aligned16(a.v_pages) || !aligned16(a.out) || (ldq & 7) ||
      (reinterpret_cast<uintptr_t>(a.workspace) & 255))
    return set_error(DK_ERR_ALIGN, "%s: q rows, pages and out need 16-byte alignment, the workspace 256", what);
  Pass own = {}, pre = {};
  Cutter c{static_cast<char*>(a.workspace)};
  shape_own(z, own);
  cut_pass(z, c, own, z.prefix_len > 0);
  if (z.prefix_len > 0) {
    shape_prefix(z, pre);
    cut_pass(z, c, pre, true);
  }
  for (const Pass* s : {&pre, &own}) {
    if (s == &pre && z.prefix_len == 0) continue;
    const int64_t chunk = s->tc ? kTcChunk : kChunk;
    const int64_t tiles = s->p.mode == kRagged ? s->p.max_tiles : s->p.n_tiles;
    const int64_t positions = s->p.mode == kPrefix ? z.prefix_len : table_width * page_size;
    if (tiles * ((positions + chunk - 1) / chunk + 1 + s->p.unit_extra) * z.nkv >= (int64_t(1) << 30))
      return set_error(DK_ERR_UNSUPPORTED, "%s: the call's work counts more than 2^30 chunks: fewer sequences or narrower page tables",
                       what);
  }
  if (c.used > a.workspace_bytes)
    return set_error(DK_ERR_INVALID, "%s: the workspace has %llu bytes, %llu are needed", what,
                     (unsigned long long)a.workspace_bytes, (unsigned long long)c.used);
  if (own.ctas == 0 || (z.prefix_len > 0 && pre.ctas == 0))
    return set_error(DK_ERR_UNSUPPORTED, "%s: the kernel's shared memory does not fit this device", what);
  const int beside = z.prefix_len > 0 && pdl_enabled() ? 1 : 0;
  for (Problem* p : {&own.p, &pre.p}) {
    p->q = a.q, p->ldq = ldq, p->out = a.out;
    p->table = a.page_table, p->ld_table = a.ld_table, p->lengths = a.lengths, p->starts = a.starts;
    p->T = static_cast<int>(z.T), p->B = static_cast<int>(z.B), p->nkv = static_cast<int>(z.nkv);
    p->G = static_cast<int>(z.nq / z.nkv);
    p->n_pages = static_cast<int>(n_pages), p->page_size = static_cast<int>(page_size);
    p->page_shift = __builtin_ctzll(page_size);
    p->capacity = static_cast<int>(table_width * page_size);
    p->mask = Mask{static_cast<int>(window), window > 0 ? static_cast<int>(sinks) : 0};
    p->scale2 = static_cast<float>(a.scale * 1.44269504088896341);
    p->err = device_info().err_word;
  }
  for (Pass* s : {&own, &pre}) {  // the tiles take the scale's sign apart from it
    if (!s->tc) continue;
    const float scale2 = s->p.scale2;
    s->p.signs = scale2 < 0.f ? -1 : scale2 == 0.f ? 0 : 1;
    s->p.scale2 = scale2 < 0.f ? -scale2 : scale2 == 0.f ? 1.f : scale2;
  }
  pre.p.table = a.prefix_table, pre.p.capacity = static_cast<int>(z.prefix_len), pre.p.mask = Mask{0, 0};
  if (z.prefix_len > 0) share_gpu(pre, own);

  cudaStream_t st = reinterpret_cast<cudaStream_t>(a.stream);
  const uint64_t rows = static_cast<uint64_t>(n_pages * z.nkv * page_size);
  const CUtensorMapDataType type = z.dtype == DK_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap mk, mv;
  uint32_t box = 0;
  auto page_maps = [&](int chunk) {  // in boxes of a page, or of a chunk's positions of one (0.3 us each, so not made twice)
    const uint32_t want = static_cast<uint32_t>(std::min<int64_t>(page_size, chunk));
    if (want == box) return true;
    box = want;
    return make_tensor_map_2d(&mk, a.k_pages, type, z.hd, rows, z.hd * 2, 64, box, CU_TENSOR_MAP_SWIZZLE_128B) &&
           make_tensor_map_2d(&mv, a.v_pages, type, z.hd, rows, z.hd * 2, 64, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  cudaError_t e = cudaSuccess;
  if (z.ragged)
    e = launch(plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, pdl_enabled(), dim3(1, 1, 1), own.p,
               const_cast<int32_t*>(own.p.plan), const_cast<int4*>(own.p.tile_info));
  for (const Pass* s : {&pre, &own}) {
    if (s->ctas == 0 || e != cudaSuccess) continue;
    if (!page_maps(s->tc ? kTcChunk : kChunk)) return DK_ERR_CUDA;
    if (s->tc) {
      if (const int rc = tc_launch(s->p, z.nq, z.hd, z.dtype, s->ctas, mk, mv, s == &own ? beside : 0, st)) return rc;
    } else {
      e = launch_rows(z, s->rows, s->shape, st, mk, mv, s->p, s == &own ? beside : 0);
    }
  }
  const Pass* with = z.prefix_len > 0 ? &pre : nullptr;
  if (e == cudaSuccess) {
    if (z.dtype == DK_F16)
      e = z.hd == 128 ? launch_join<__half, 128>(z, st, with, own) : launch_join<__half, 64>(z, st, with, own);
    else
      e = z.hd == 128 ? launch_join<__nv_bfloat16, 128>(z, st, with, own) : launch_join<__nv_bfloat16, 64>(z, st, with, own);
  }
  if (e != cudaSuccess) return set_error(DK_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return DK_OK;
}

}  // namespace

extern "C" int dk_paged_attention(const dk_paged_attention_args* args) { return attention("paged_attention", args, false); }

extern "C" int dk_shared_prefix_attention(const dk_paged_attention_args* args) {
  return attention("shared_prefix_attention", args, true);
}
