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

#include "paged_fp4.cuh"

namespace dk {
namespace paged {
namespace {

constexpr int kChunk = 64;
constexpr int kGroups = 2;   // independent consumer groups of a CTA, each with a piece of the line of its own
constexpr int kCWarps = 4;   // warps of a group
constexpr int kThreads = kGroups * (kCWarps + 1) * 32;
constexpr int kMaxRing = 6;
constexpr int kFp4UnitExtra = 1;   // the same over a 4-bit cache, whose chunks are longer
constexpr int kRowsUnitExtra = 2;  // a unit's fixed cost (q, joining the warps, output) in chunks

// ------------------------------------------------------------------------------------ ragged plan
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const Problem p) {
  pdl_trigger();
  pdl_wait();
  make_plan(p);
}

// The plans of a call's two launches, a CTA each. (As the only kernel it cost calls of one launch 0.2 us.)
__global__ void __launch_bounds__(kPlanThreads) plan_both_kernel(const Problem a, const Problem b) {
  pdl_trigger();
  pdl_wait();
  make_plan(blockIdx.x == 0 ? a : b);
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
  __device__ JoinShape(int y, int z)
      : lane(threadIdx.x % kLanes), part(threadIdx.x / kLanes), row(y * kR + lane % kR), d4(z * kD + lane / kR) {}
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
  __device__ void store(T* out, int d4, float scale) const {
    const float inv = l == 0.f ? 0.f : 1.f / l * scale;  // (a power of two: exact; a quotient takes longer)
    *reinterpret_cast<uint2*>(out + 4 * d4) = make_uint2(Elem<T>::pack(acc.x * inv, acc.y * inv), Elem<T>::pack(acc.z * inv, acc.w * inv));
  }
};

template <typename T, int kHd>
__device__ __forceinline__ T* out_row(const Problem& p, int t, int head) {
  return static_cast<T*>(p.out) + (static_cast<int64_t>(t) * p.nkv * p.G + head) * kHd;
}

// Joins the units that a piece's end cuts. Block (x, y, z): rows of the unit that CTA x began, if there is one, or with
// `by_unit` (launches of fewer units than CTAs) of unit x, if it is cut.
template <typename T, int kHd, typename Shape>
__device__ __forceinline__ void join_split(const Problem& p, int tile_rows, int ctas, int by_unit, int x, int y, int z) {
  int4 c;  // {first token, tokens, kv head, last CTA}
  Pieces w{x, 0, 0};
  if (by_unit) {
    const Line line = line_of(p, kTcChunk);
    if (x >= line.tiles * p.nkv) return;
    const int h = x / line.tiles, ti = x - h * line.tiles;
    const Tile t = tile_at(p, ti);
    w = pieces_of(Cuts(p, line, ctas), h * line.chunks + line.cum(ti), h * line.chunks + line.cum(ti + 1), p.unit_extra, ctas, 0);
    if (w.first == w.last) return;
    c = make_int4(t.t0, t.ntok, h, w.last);
  } else {
    c = p.cut[x];
    w.last = c.w;
  }
  const Shape at(y, z);
  const int rows = c.y * p.G, i = at.row;
  if (y * Shape::kRows >= rows) return;
  Joined<T, kHd> sum;
  if (i < rows)
    sum.template add_part<Shape::kAhead>(p, w, at.part, Shape::kParts, tile_rows, result_row(p, i / p.G, i % p.G), at.d4);
  sum.join_parts(at);
  if (at.part == 0 && i < rows) sum.store(out_row<T, kHd>(p, c.x + i / p.G, c.z * p.G + i % p.G), at.d4, p.out_scale);
}

template <typename T, int kHd, typename Shape>
__global__ void __launch_bounds__(Shape::kThreads) join_split_kernel(const Problem p, int tile_rows, int ctas, int by_unit) {
  pdl_trigger();
  pdl_wait();
  join_split<T, kHd, Shape>(p, tile_rows, ctas, by_unit, blockIdx.x, blockIdx.y, blockIdx.z);
}

// The same for the two launches of a call at once: the first `blocks` blocks are a's, (x, y) with y < ay, the others b's.
template <typename T, int kHd, typename ShapeA, typename ShapeB>
__global__ void __launch_bounds__(ShapeA::kThreads)
    join_both_kernel(const Problem a, int a_rows, int a_ctas, int blocks, int ay, const Problem b, int b_rows, int b_ctas, int by_unit, int by) {
  static_assert(ShapeA::kThreads == ShapeB::kThreads, "one block size");
  constexpr int kZ = kHd / 4 / ShapeB::kDims;
  pdl_trigger();
  pdl_wait();
  int x = blockIdx.x;
  if (x < blocks)
    return join_split<T, kHd, ShapeA>(a, a_rows, a_ctas, 0, x / ay, x % ay, 0);
  x -= blocks;
  join_split<T, kHd, ShapeB>(b, b_rows, b_ctas, by_unit, x / kZ / by, x / kZ % by, x % kZ);
}

// Joins the prefix's results (`a`) with those of the sequences' own positions (`b`). Block (x, h): rows (token, head of
// kv head h). The last part of a block takes the own positions, the others the prefix's pieces.
template <typename T, int kHd, typename Shape>
__global__ void __launch_bounds__(Shape::kThreads)
    join_prefix_kernel(const Problem a, int a_ctas, const Problem b, int b_ctas, int b_rows) {
  pdl_trigger();
  pdl_wait();
  const Shape at(blockIdx.x, blockIdx.z);
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
  if (at.part == 0 && live) sum.store(out_row<T, kHd>(b, t, h * b.G + g), at.d4, b.out_scale);
}

}  // namespace

// ------------------------------------------------------------------------------------ host
namespace {

// Tiles that are cut into more pieces than this, on average, are joined in parts (42 tokens after 32768 positions: 28 us, 46
// without; one short sequence 12.1, 12.2; 16 sequences of 8192 with 4 tokens each, 9 pieces a unit: 44, 40).
constexpr int kFewPieces = 8;

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
  bool fp4;           // the cache is held in 4 bits,
  int64_t positions;  // in a row of the page table
};

// A ragged call over a 4-bit cache: sequences of few tokens (drafted ones to check, decode steps beside prompts) go to the rows kernel,
// in tiles of up to 16 rows that each read the sequence again, up to kFewTiles of them; longer ones to the 256-row tiles (32 sequences
// of 4096, 28 heads over 4, tiles of 2 tokens, us on the rows kernel and as 256-row tiles: 2 tokens 31, 61; 4 39, 62; 6 53,
// 62; 8 62, 63; 12 93, 57. 16 of 4096, 8 over 8, tiles of 16: 32 44, 60; 64 69, 61). Which there are only the device
// knows, and a launch without any takes 3 to 5 us. A call whose sequences have kManyTokens on average is taken for
// prompts: then the tiles take all of them.
constexpr int kFewTiles = 3, kManyTokens = 256;
// Calls of little work, whatever their sequences have of it, all go to the rows kernel, which needs no second launch and mostly no join: up to
// kSmallFew chunks a group where the sequences have few tokens on average, kSmallMany else (up to that many tokens each, split by sequence
// or as tiles, and on the rows kernel, us; in brackets chunks a group). 28 heads over 4: 8 x 5: 250 17.4, 13.6; 4000 25.3, 23.0 (9). 64 x
// 2: 250 26.2, 13.3; 500 29.0, 16.4; 1000 32.6, 26.0 (12). 32 x 5: 500 27.2, 16.9. 16 x 20, 8 over 8: 2000 34.1, 29.2 (13). 12 over 2:
// 1 x 100: 500 19.6, 17.3 (1); 1000 20.3, 20.1 (3); 2000 21.6, 25.2 (6). 8 x 64: 500 27.9, 25.2 (5); 1000 28.9, 31.7 (10). 8 x 200, 8 over
// 8: 250 29.8, 22.4 (4); 500 33.6, 35.7 (8).
constexpr int64_t kSmallFew = 16, kSmallMany = 4;
struct Split {
  bool few, many;  // which kernels are launched
  int limit;       // the most tokens of a sequence of the first
};
Split split_of(const Sizes& z) {
  const int64_t limit = kFewTiles * (16 / (z.nq / z.nkv));
  if (!z.fp4 || !z.ragged || z.prefix_len > 0 || z.T >= kManyTokens * z.B) return {false, true, 0};
  const int64_t token = 16 / (z.nq / z.nkv), tiles = (z.T + token - 1) / token + z.B;
  const int64_t chunks = tiles * ((z.positions + kFp4Chunk - 1) / kFp4Chunk);  // of a kv head
  const int64_t small = (z.T <= limit * z.B ? kSmallFew : kSmallMany) * fp4_groups(16) * device_info().num_sms;
  if (z.T <= limit || chunks <= small / z.nkv) return {true, false, INT_MAX};
  return {z.B > 1, true, z.B > 1 ? static_cast<int>(limit) : 0};
}

// Prompts over a 4-bit cache first have the pages that they see copied in 16 bits, which the tiles then read, instead of converting
// each chunk for every tile anew: from kCopyTiles tiles a sequence on (positions, tokens each; us without and with a copy): 32
// sequences of 4096, 28 heads over 4, tiles of 36 tokens: 64 115, 126; 128 195, 175; 256 316, 252. 2 of 8192, 12 over 2, 42:
// 64 29, 30; 128 39, 38; 256 50, 44. 16 of 4096, 8 over 8, 256: 256 79, 103. The copy takes at most 1 GB of the workspace.
constexpr int64_t kCopyTiles = 3, kCopyBytes = int64_t(1) << 30;
bool copies(const Sizes& z) {
  const int64_t tile = 2 * (128 / (z.nq / z.nkv));
  return z.fp4 && z.ragged && z.prefix_len == 0 && split_of(z).many && z.T > 0 && z.T >= kCopyTiles * tile * z.B &&
         z.positions <= kCopyBytes / (4 * z.hd) / z.nkv / z.B;
}

Pages pages_of(const Sizes& z) { return !z.fp4 ? Pages::kPlain : copies(z) ? Pages::kCopy : Pages::kCodes; }

RowsShape rows_shape_of(const Sizes& z, int rows) {
  if (z.fp4) return fp4_rows_shape(z.hd, z.dtype, rows, z.ragged);
#define DK_SHAPE(TT) \
  (z.hd == 128 ? (rows == 8 ? rows_shape<TT, 128, 8>() : rows_shape<TT, 128, 16>()) \
               : (rows == 8 ? rows_shape<TT, 64, 8>() : rows_shape<TT, 64, 16>()))
  return z.dtype == DK_F16 ? DK_SHAPE(__half) : DK_SHAPE(__nv_bfloat16);
#undef DK_SHAPE
}

cudaError_t launch_rows(const Sizes& z, int rows, const RowsShape& s, cudaStream_t st, const CUtensorMap& mk,
                        const CUtensorMap& mv, const Problem& p, int wait_late) {
  if (z.fp4) return fp4_rows_launch(p, z.hd, z.dtype, rows, z.ragged, s, wait_late, st);
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
  int groups;  // of a CTA, each with a piece of the line (not tc)
};

void cut_pass(const Sizes& z, Cutter& c, Pass& a, bool always_partial) {
  Problem& p = a.p;
  if (a.tc) {
    a.rows = kTcRows;
    p.unit_extra = kTcUnitExtra;
    p.rows_inner = 1;
    a.ctas = tc_ctas(z.hd, z.dtype, pages_of(z));
  } else {
    a.rows = z.nq / z.nkv <= 8 && !z.ragged ? 8 : 16;
    a.shape = rows_shape_of(z, a.rows);
    a.groups = z.fp4 ? fp4_groups(a.rows) : kGroups;
    a.ctas = a.shape.ctas * a.groups;
    p.unit_extra = z.fp4 ? kFp4UnitExtra : kRowsUnitExtra;
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

// The copy of the pages and the tables that list them.
struct Copy {
  void *k, *v;
  int32_t* table;
};
Copy cut_copy(const Sizes& z, Cutter& c) {
  const uint64_t positions = static_cast<uint64_t>(z.B * z.positions), bytes = positions * z.nkv * z.hd * 2;
  return {c.take<char>(bytes), c.take<char>(bytes), c.take<int32_t>(positions / 16)};  // (a page has 16 positions at least)
}

// Tiles of one token (ragged: of up to 16 rows), or of two halves of up to 128 rows each.
void set_tile(const Sizes& z, Pass& a, bool tc) {
  const int group = static_cast<int>(z.nq / z.nkv);
  a.tc = tc;
  a.p.half_tokens = tc ? 128 / group : z.ragged ? 16 / group : 1;
  a.p.tile_tokens = tc ? 2 * a.p.half_tokens : a.p.half_tokens;
}

void set_ragged(const Sizes& z, Pass& a, int above, int most) {
  a.p.mode = kRagged;
  const int64_t of_one = (int64_t(most) + a.p.tile_tokens - 1) / a.p.tile_tokens;  // tiles of a sequence, at most
  a.p.max_tiles = static_cast<int>(std::min(z.T / a.p.tile_tokens + z.B, of_one * z.B));
  a.p.above = above, a.p.most = most;
}

// One token for each sequence goes to the rows kernel, several to the tiles (64 sequences of 8192, 12 heads over 2 kv heads,
// one token each, without the host: 91 us on the rows kernel, 111 as tiles; one of 640: 9.4 and 13.6; 4 tokens each as tiles:
// 109).
void shape_own(const Sizes& z, Pass& a) {
  const Split split = split_of(z);
  set_tile(z, a, z.ragged && split.many);
  a.p.n_tiles = static_cast<int>(z.B);
  if (z.ragged) set_ragged(z, a, split.many ? split.limit : 0, INT_MAX);
  a.p.zero_outside = z.ragged && z.prefix_len == 0;
}

// Over a 4-bit cache: the chunks of a rows pass's longest unit if the units are short, else 0. Short units are not cut, and no join follows:
// up to 3 chunks (short page tables or windows), and up to kShortUnit where the units keep two fifths of the groups busy in one
// round (one token each; us cut and joined, and whole, replayed from a graph; sequences, kv heads: positions): 1, 2: 60 8.4, 4.9;
// 380 9.8, 9.0; 500 9.7, 10.8. 16, 8: 380 10.9, 9.9; 500 10.9, 12.0. 48, 4: 380 12.7, 10.6; 640 15.1, 14.4; 760 15.3, 16.2.
// 64, 4: 500 15.0, 12.5; 640 15.4, 14.8. 112, 4 (a second round): 250 14.6, 13.8; 380 16.6, 17.1; 500 17.4, 20.2. 256, 4: 380 24.0, 23.1.
// Launched one by one, these calls of one launch take 12 us instead of 14.
constexpr int64_t kShortUnit = 5;
int short_unit(const Sizes& z, const Pass& a) {
  // A window takes its own positions, from the first token's to the last's, and parts of pages before them and at the sinks' end.
  const int64_t part = std::min(a.p.page_size, kFp4Chunk), all = a.p.capacity;
  const int64_t most = a.p.mask.window > 0
                           ? std::min<int64_t>(all, int64_t(a.p.mask.window) + a.p.mask.sinks + a.p.tile_tokens + 2 * part)
                           : all;
  const int64_t chunks = (most + kFp4Chunk - 1) / kFp4Chunk, units = z.B * z.nkv;
  const bool one_round = 5 * units >= 2 * a.ctas && units <= a.ctas;
  return chunks <= (one_round ? kShortUnit : 3) ? static_cast<int>(chunks) : 0;
}

// The sequences of few tokens of a ragged call that has others too.
void shape_few(const Sizes& z, Pass& a) {
  set_tile(z, a, false);
  set_ragged(z, a, 0, split_of(z).limit);
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
// for each chunk of a CTA's piece; a group of the other takes 1.1 us for a chunk. Over a 4-bit cache a chunk of the other takes twice that
// (prefix 64 x 8192: 37.1 us; a third more or less of that lead: 37.1, 37.6).
void share_gpu(const Sizes& z, Pass& pre, Pass& own) {
  if (own.tc || !pdl_enabled()) return;
  const int sms = device_info().num_sms;
  const int64_t n = static_cast<int64_t>((pre.p.prefix_len + kTcChunk - 1) / kTcChunk + pre.p.unit_extra) * pre.p.n_tiles * pre.p.nkv;
  const int64_t most = sms * 7 / 8, per = (n + most - 1) / most;
  pre.ctas = static_cast<int>((n + per - 1) / per);
  own.p.early = own.groups * (sms - pre.ctas);
  own.p.lead = static_cast<int>(z.fp4 ? (60 + 20 * per) / 22 : (60 + 20 * per) / 11);
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
cudaError_t launch_join(const Sizes& z, cudaStream_t st, const Pass* prefix, const Pass* few, const Pass& own) {
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
  if (few != nullptr) {
    using Wide = JoinShape<kHd == 128 ? 8 : 16, kHd / 4, 1, 2>;  // (Tiles in blocks of the other shapes' size)
    const int64_t ay = few->rows / OneToken::kRows, blocks = few->ctas * ay;
    const bool in_parts = units * kFewPieces <= own.ctas;
    const int64_t by = in_parts ? y : (y * 8 + Wide::kRows - 1) / Wide::kRows, bz = in_parts ? kHd / 4 / Few::kDims : 1;
    return launch(in_parts ? join_both_kernel<T, kHd, OneToken, Few> : join_both_kernel<T, kHd, OneToken, Wide>,
                  dim3(static_cast<unsigned>(blocks + x * by * bz)), dim3(Few::kThreads), 0, st, pdl_enabled(), one, few->p, few->rows,
                  few->ctas, static_cast<int>(blocks), static_cast<int>(ay), own.p, own.rows, own.ctas, by_unit, static_cast<int>(by));
  }
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
  if (split_of(z).few && split_of(z).many) {
    Pass few = {};
    shape_few(z, few);
    cut_pass(z, c, few, false);
  }
  if (copies(z)) cut_copy(z, c);
  return c.used;
}

}  // namespace
}  // namespace paged
}  // namespace dk

using namespace dk;
using namespace dk::paged;

namespace {

int workspace_bytes(const char* what, const Sizes& z, uint64_t* bytes) {
  if (const int rc = check_sizes(what, z)) return rc;
  if (!bytes) return set_error(DK_ERR_INVALID, "%s: bytes is NULL", what);
  *bytes = workspace_of(z);
  return DK_OK;
}

}  // namespace

extern "C" int dk_paged_attention_workspace_bytes(int64_t T, int64_t B, int64_t nq, int64_t nkv, int64_t head_dim,
                                                  int32_t dtype, int32_t ragged, int64_t prefix_len, uint64_t* bytes) {
  return workspace_bytes("paged_attention_workspace_bytes", Sizes{T, B, nq, nkv, head_dim, prefix_len, ragged != 0, dtype, false, 0}, bytes);
}

extern "C" int dk_paged_attention_fp4_workspace_bytes(int64_t T, int64_t B, int64_t nq, int64_t nkv, int64_t head_dim,
                                                      int32_t dtype, int32_t ragged, int64_t prefix_len, int64_t positions,
                                                      uint64_t* bytes) {
  if (positions <= 0 || positions > INT32_MAX) return set_error(DK_ERR_INVALID, "paged_attention_fp4_workspace_bytes: bad sizes");
  return workspace_bytes("paged_attention_fp4_workspace_bytes",
                         Sizes{T, B, nq, nkv, head_dim, prefix_len, ragged != 0, dtype, true, positions}, bytes);
}

namespace {

int attention(const char* what, const dk_paged_attention_args& a, bool prefix, bool fp4, double k_scale, double v_scale) {
  const Sizes z{a.T, a.B, a.n_q, a.n_kv, a.head_dim, prefix ? a.prefix_len : 0, a.starts != nullptr, static_cast<int>(a.dtype), fp4,
                a.table_width <= INT32_MAX ? a.table_width * a.page_size : 0};
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
  if (!fp4_power(k_scale) || !fp4_power(v_scale))
    return set_error(DK_ERR_INVALID, "%s: k_scale and v_scale must be powers of two from 2^-64 to 2^64", what);
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
  Pass own = {}, pre = {}, few = {};
  Cutter c{static_cast<char*>(a.workspace)};
  shape_own(z, own);
  cut_pass(z, c, own, z.prefix_len > 0);
  if (z.prefix_len > 0) {
    shape_prefix(z, pre);
    cut_pass(z, c, pre, true);
  }
  const bool has_few = split_of(z).few && split_of(z).many;
  if (has_few) {
    shape_few(z, few);
    cut_pass(z, c, few, false);
  }
  const bool copied = copies(z);
  const Copy copy = copied ? cut_copy(z, c) : Copy{};
  for (const Pass* s : {&pre, &few, &own}) {
    if ((s == &pre && z.prefix_len == 0) || (s == &few && !has_few)) continue;
    const int64_t chunk = s->tc ? kTcChunk : z.fp4 ? kFp4Chunk : kChunk;
    const int64_t tiles = s->p.mode == kRagged ? s->p.max_tiles : s->p.n_tiles;
    const int64_t positions = s->p.mode == kPrefix ? z.prefix_len : table_width * page_size;
    if (tiles * ((positions + chunk - 1) / chunk + 1 + s->p.unit_extra) > ((int64_t(1) << 30) - 1) / z.nkv)  // (the product may pass 2^63)
      return set_error(DK_ERR_UNSUPPORTED, "%s: the call's work counts more than 2^30 chunks: fewer sequences or narrower page tables",
                       what);
  }
  if (c.used > a.workspace_bytes)
    return set_error(DK_ERR_INVALID, "%s: the workspace has %llu bytes, %llu are needed", what,
                     (unsigned long long)a.workspace_bytes, (unsigned long long)c.used);
  if (own.ctas == 0 || (z.prefix_len > 0 && pre.ctas == 0) || (has_few && few.ctas == 0))
    return set_error(DK_ERR_UNSUPPORTED, "%s: the kernel's shared memory does not fit this device", what);
  const int beside = z.prefix_len > 0 && pdl_enabled() ? 1 : 0;
  for (Problem* p : {&own.p, &pre.p, &few.p}) {
    p->q = a.q, p->ldq = ldq, p->out = a.out;
    p->table = a.page_table, p->ld_table = a.ld_table, p->lengths = a.lengths, p->starts = a.starts;
    p->T = static_cast<int>(z.T), p->B = static_cast<int>(z.B), p->nkv = static_cast<int>(z.nkv);
    p->G = static_cast<int>(z.nq / z.nkv);
    p->n_pages = static_cast<int>(n_pages), p->page_size = static_cast<int>(page_size);
    p->page_shift = __builtin_ctzll(page_size);
    p->capacity = static_cast<int>(table_width * page_size);
    p->mask = Mask{static_cast<int>(window), window > 0 ? static_cast<int>(sinks) : 0};
    p->scale2 = static_cast<float>(a.scale * k_scale * 1.44269504088896341);
    p->pool[0] = static_cast<const uint8_t*>(a.k_pages), p->pool[1] = static_cast<const uint8_t*>(a.v_pages);
    p->out_scale = static_cast<float>(v_scale);
    p->err = device_info().err_word;
  }
  for (Pass* s : {&own, &pre}) {  // the tiles take the scale's sign apart from it
    if (!s->tc) continue;
    const float scale2 = s->p.scale2;
    s->p.signs = scale2 < 0.f ? -1 : scale2 == 0.f ? 0 : 1;
    s->p.scale2 = scale2 < 0.f ? -scale2 : scale2 == 0.f ? 1.f : scale2;
  }
  pre.p.table = a.prefix_table, pre.p.capacity = static_cast<int>(z.prefix_len), pre.p.mask = Mask{0, 0};
  if (z.prefix_len > 0) share_gpu(z, pre, own);
  else if (z.fp4 && !own.tc) own.p.unit_len = short_unit(z, own);

  cudaStream_t st = reinterpret_cast<cudaStream_t>(a.stream);
  cudaError_t e = cudaSuccess;
  if (z.ragged && !copied)
    e = has_few ? launch(plan_both_kernel, dim3(2), dim3(kPlanThreads), 0, st, pdl_enabled(), dim3(1, 1, 1), own.p, few.p)
                : launch(plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, pdl_enabled(), dim3(1, 1, 1), own.p);
  if (copied) {
    e = fp4_copy_launch(own.p, few.p, has_few ? 2 : 1, z.hd, z.dtype, copy.k, copy.v, copy.table, st);
    own.p.table = copy.table, own.p.ld_table = table_width;
    own.p.n_pages = static_cast<int>(z.B * table_width);
  }
  const void *k_pages = copied ? copy.k : a.k_pages, *v_pages = copied ? copy.v : a.v_pages;
  const uint64_t rows = static_cast<uint64_t>(own.p.n_pages * z.nkv * page_size);
  const CUtensorMapDataType k_type = z.dtype == DK_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapDataType v_type = copied ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : k_type;
  CUtensorMap mk, mv;
  uint32_t box = 0;
  auto page_maps = [&](int chunk) {  // in boxes of a page, or of a chunk's positions of one (0.3 us each, so not made twice)
    const uint32_t want = static_cast<uint32_t>(std::min<int64_t>(page_size, chunk));
    if (want == box) return true;
    box = want;
    return make_tensor_map_2d(&mk, k_pages, k_type, z.hd, rows, z.hd * 2, 64, box, CU_TENSOR_MAP_SWIZZLE_128B) &&
           make_tensor_map_2d(&mv, v_pages, v_type, z.hd, rows, z.hd * 2, 64, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  for (const Pass* s : {&pre, &few, &own}) {
    if (s->ctas == 0 || e != cudaSuccess) continue;
    if ((!z.fp4 || (copied && s->tc)) && !page_maps(s->tc ? kTcChunk : kChunk)) return DK_ERR_CUDA;
    if (s->tc) {
      if (const int rc = tc_launch(s->p, z.nq, z.hd, z.dtype, pages_of(z), s->ctas, mk, mv, s == &own ? beside : 0, st)) return rc;
    } else {
      e = launch_rows(z, s->rows, s->shape, st, mk, mv, s->p, s == &own ? beside : 0);
    }
  }
  if (e == cudaSuccess && own.p.unit_len == 0) {
    const Pass *with = z.prefix_len > 0 ? &pre : nullptr, *beside_it = has_few ? &few : nullptr;
    if (z.dtype == DK_F16)
      e = z.hd == 128 ? launch_join<__half, 128>(z, st, with, beside_it, own) : launch_join<__half, 64>(z, st, with, beside_it, own);
    else
      e = z.hd == 128 ? launch_join<__nv_bfloat16, 128>(z, st, with, beside_it, own)
                      : launch_join<__nv_bfloat16, 64>(z, st, with, beside_it, own);
  }
  if (e != cudaSuccess) return set_error(DK_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return DK_OK;
}

}  // namespace

extern "C" int dk_paged_attention(const dk_paged_attention_args* args) {
  if (args == nullptr) return set_error(DK_ERR_INVALID, "paged_attention: NULL arguments");
  return attention("paged_attention", *args, false, false, 1., 1.);
}

extern "C" int dk_shared_prefix_attention(const dk_paged_attention_args* args) {
  if (args == nullptr) return set_error(DK_ERR_INVALID, "shared_prefix_attention: NULL arguments");
  return attention("shared_prefix_attention", *args, true, false, 1., 1.);
}

extern "C" int dk_paged_attention_fp4(const dk_paged_attention_fp4_args* args) {
  if (args == nullptr) return set_error(DK_ERR_INVALID, "paged_attention_fp4: NULL arguments");
  return attention("paged_attention_fp4", args->attention, false, true, args->k_scale, args->v_scale);
}

extern "C" int dk_shared_prefix_attention_fp4(const dk_paged_attention_fp4_args* args) {
  if (args == nullptr) return set_error(DK_ERR_INVALID, "shared_prefix_attention_fp4: NULL arguments");
  return attention("shared_prefix_attention_fp4", args->attention, true, true, args->k_scale, args->v_scale);
}
