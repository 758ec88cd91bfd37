// Attention over a paged cache held in 4 bits for few query rows per kv head: decode steps, and sequences with a few tokens each
// (tiles of up to 16 rows: floor(16 / G) tokens).
//
//   out[t] = sum_j p[t][j] v[j],  p[t] = softmax over the visible j of scale * q[t] . k[j]
// with the masks, units, pieces and joins of paged_attention.cu; here is the kernel between them.
//
// The bytes of k and v are 9/32 of a 16-bit cache's, so the conversion of codes competes with them: at the copy rate an SM gets
// 41 values a cycle, and one costs at least a conversion and a product with its scale for each pair. So every value is converted
// once, in registers, right in the place where the tensor-core product takes it from:
// * the cache's values are the 16 rows of the product (m16n8k16), the query heads its 8 columns: S^T = K Q^T, O^T = V^T P^T.
//   The other way round the 16 rows would be half empty for groups of up to 8 heads and each value would cost twice the products;
// * a lane takes the codes of one position as 16 contiguous bytes (k: a quarter of the dims, in the order they lie in; the product's
//   inner index runs over the dims in that order, and q is loaded to match) or 8 (v: 16 dims, one scale's). In v's product
//   the inner index runs over positions, so the pairs that a register holds are of two positions: the halves of the bytes are
//   exchanged between two positions' words first (four operations for eight registers);
// * p in fp16 goes from the accumulators' layout to the operand's by transposing 8 x 8 blocks between lanes (movmatrix). The 16
//   positions of a product are dealt to its rows such that each load of v reads 4 neighbouring positions: no bank conflicts.
// code * scale is exact in fp16, and so is q once its row is scaled by a power of two (bf16 rows; their largest value comes to 2^14,
// and what falls below 2^-24 there counts for nothing beside it): the products are those of the cache's values. p is rounded to
// fp16 for the product with v; its reference is 2^6 below the maximum seen when it was set, and it is set anew when a score
// passes it by 2^14, so that the largest p lies 30 to 38 binades above fp16's smallest step.
// A producer warp a group streams chunks of 128 positions through a ring of bulk copies, as in the 16-bit kernel; a consumer warp
// takes 32 of them, so that the operands of two tiles are on their way at a time. A position that no row of the tile
// sees gets a scale of zero in place of v's, whatever its page holds; a page outside the pool gets scales of zero in
// shared memory. Codes are finite whatever they are.
// What bounds it: no unit is full. Measured (28 heads over 4 kv heads of 128, bf16, 64 sequences of up to 8192, 212 MB): 52 us with the
// join, 4.1 TB/s, 62% of the copy rate; over the launch 59% of issue, 51% of the ALU, 51% of DRAM's nominal peak. Start, join and tail take
// 12 us of it, without any arithmetic the same loads take 40, and 12 consumer warps an SM do not cover one another's waits and conversions:
// a tile of 16 positions takes a warp about 260 instructions (64 conversions, 64 products with scales, 16 tensor-core products, 16
// exchanges of halves) besides 80 for the chunk, the part and the kernel's start, all of them 26 us of issue. 16-bit pages take 116 us.
// Chunks of 64 (a tile a warp): 61 us, but one sequence of 640 8.5 us instead of 9.4. 4 groups an SM, 96 registers a thread: 59.
// 32 sequences of 4096 with 2 to 5 tokens each: 41 us for three tiles a sequence.
#include <algorithm>
#include <climits>
#include <mutex>

#include "paged_fp4.cuh"

namespace dk {
namespace paged {
namespace {

constexpr int kCWarps = 4;  // warps of a group
constexpr int kSub = 2;     // 16-position tiles of a warp in a chunk
constexpr int kChunk = kFp4Chunk;
static_assert(kChunk == kCWarps * kSub * 16, "a chunk is one round of the warps");
// Groups of a CTA, one CTA an SM, each with a piece of the line and a producer warp of its own. What counts is the registers of a
// thread: with 8 rows 3 groups have 128 and keep a chunk's operands in them; 4 groups have 96 (64 x 8192: 59 us against 52).
template <int kBlocks>
constexpr int kGroups = fp4_groups(8 * kBlocks);
template <int kBlocks>
constexpr int kThreads = kGroups<kBlocks> * (kCWarps + 1) * 32;
// Slots of a group's ring: what fits beside the warps' results.
template <int kHd, int kBlocks>
constexpr int kRing = (kHd == 64 ? 2 : 1) * 3;
constexpr float kRefBelow = 6.f, kRefReach = 14.f;

// A chunk in shared memory: for k and v each the codes of kChunk positions, then their scales.
template <int kHd>
struct Slot {
  static constexpr int kScalesAt = kChunk * Fp4<kHd>::kCodes;
  static constexpr int kTensor = kChunk * Fp4<kHd>::kRow;
  static constexpr int kBytes = 2 * kTensor;
};

__device__ __forceinline__ void group_sync(int group) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(kCWarps * 32) : "memory");
}

// An 8 x 8 block of 16-bit values, a row's pair a lane, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

// Bits of a where m has ones, of b elsewhere.
__device__ __forceinline__ uint32_t choose(uint32_t a, uint32_t b, uint32_t m) { return (a & m) | (b & ~m); }

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }

// kRaggedTiles: tiles of the plan, a few tokens each; otherwise tile b is the one token of sequence b.
template <typename T, int kHd, int kBlocks, bool kRaggedTiles>
__global__ void __launch_bounds__(kThreads<kBlocks>, 1) fp4_rows_kernel(const Problem p, int wait_late) {
  constexpr int ring = kRing<kHd, kBlocks>;
  using F = Fp4<kHd>;
  using S = Slot<kHd>;
  constexpr int kG = kGroups<kBlocks>, kT = kThreads<kBlocks>;
  constexpr int kRows = 8 * kBlocks;      // query rows: the product's columns
  constexpr int kSteps = kHd / 16;        // products of a tile of k, and tiles of v's product
  constexpr int kWords = kHd / 32;        // words of a lane's codes of k; v's has kHd / 64
  constexpr uint32_t kLow = 0x0f0f0f0fu;
  __shared__ float2 pre_ml_sh[kG][kRows * kCWarps];
  __shared__ __align__(8) uint64_t full_sh[kG][ring], empty_sh[kG][ring];
  __shared__ int warp_sum[kT / 32 + 1];
  extern __shared__ __align__(128) uint8_t dsm[];
  int* cum_sh = reinterpret_cast<int*>(dsm);  // [B + 1], before the first copies land there

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool producer = warp >= kG * kCWarps;
  const int group = producer ? warp - kG * kCWarps : warp / kCWarps;
  const int cta = blockIdx.x * kG + group, ctas = gridDim.x * kG;  // pieces of the line: one a group
  uint8_t* slots = dsm + group * ring * S::kBytes;
  float* pre_o = reinterpret_cast<float*>(dsm + kG * ring * S::kBytes) + group * kCWarps * kRows * kHd;
  float2* pre_ml = pre_ml_sh[group];
  uint64_t *full = full_sh[group], *empty = empty_sh[group];
  if (tid == 0) {
    for (int i = 0; i < kG * ring; ++i) {
      mbar_init(&full_sh[0][i], 1);
      mbar_init(&empty_sh[0][i], kCWarps);
    }
    fence_mbar_init();
  }
  if (!wait_late) pdl_wait();
  pdl_trigger();

  Line line{cum_sh, 0, p.n_tiles, 0};
  if (p.unit_len > 0) {
    const int tiles = kRaggedTiles ? p.plan[0] : p.n_tiles;
    line = {nullptr, p.unit_len, tiles, tiles * p.unit_len};
  } else if constexpr (kRaggedTiles) {
    line = line_of(p, kChunk);
  } else {  // every CTA sums up the sequences' chunks for itself
    int carry = 0;
    for (int b0 = 0; b0 < p.B; b0 += kT) {
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
      for (int w = 0; w < kT / 32; ++w) {
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
      for (int i = tid; i <= p.B; i += kT) p.cum_out[i] = cum_sh[i];
  }
  __syncthreads();

  Walk<kChunk, true> walk(p, line, cta, ctas, lane);
  __syncthreads();  // the sums have been read: copies may land on them
  bool ok = true;
  int fill = 0;          // ring fills so far,
  int s = 0, round = 0;  // fill % ring and fill / ring
  auto filled = [&] {
    ++fill;
    if (++s == ring) s = 0, ++round;
  };

  if (producer) {
    // ---------------------------------------------------------------- producer warps: one lane per copy
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (the sums lay there)
    const int box = min(p.page_size, kChunk);  // positions of one copy
    const int boxes = kChunk / box;
    const int kv = lane & 1, scales = (lane >> 1) & 1, pg = lane >> 2;
    const int row_bytes = scales ? F::kScales : F::kCodes;
    const uint32_t bytes = box * row_bytes;
    const uint8_t* pool = (kv ? p.pool[1] : p.pool[0]) + (scales ? p.page_size * F::kCodes : 0);
    uint8_t* dst = slots + kv * S::kTensor + (scales ? S::kScalesAt : 0) + pg * bytes;
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
      for (int i = c0; i < c1; ++i, filled()) {
        const int page = next;
        next = entry(i + 1);
        if (round > 0 && !wait_for(&empty[s], (round - 1) & 1, p.err, DK_DEVERR_WAIT_EMPTY)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint8_t* at = dst + s * S::kBytes;
        const bool wanted = page != INT_MIN, mine = wanted && page >= 0 && page < p.n_pages;
        if (wanted && !mine) {  // no page of the pool: scales of zero
          record_device_error(p.err, DK_DEVERR_BAD_POSITION);
          if (scales)
            for (uint32_t b = 0; b < bytes; b += 16) *reinterpret_cast<uint4*>(at + b) = make_uint4(0, 0, 0, 0);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        const unsigned codes = __popc(__ballot_sync(0xffffffffu, mine && !scales)), grids = __popc(__ballot_sync(0xffffffffu, mine && scales));
        if (lane == 0) mbar_arrive_expect_tx(&full[s], box * (codes * F::kCodes + grids * F::kScales));
        __syncwarp();
        if (mine) {
          const int in_page = span.position(i * kChunk + pg * box) & (p.page_size - 1);
          bulk_g2s(at, pool + (static_cast<int64_t>(page) * p.nkv + h) * (p.page_size * F::kRow) + in_page * row_bytes, bytes, &full[s]);
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- consumer warps
    const int g = lane >> 2, tq = lane & 3;
    const int sub = warp % kCWarps, gtid = tid - group * kCWarps * 32;
    const int row_a = (g >> 1) + 4 * (g & 1);  // the position of a tile in the products' row g; row g + 8 has the one 8 on
    if (gtid == 0) p.cut[cta] = make_int4(0, 0, 0, 0);
    bool joined = false;
    while (walk.more()) {
      const Span<kChunk> span = walk.step();
      const Tile t = walk.t;
      const int h = walk.h, c0 = walk.c0, c1 = walk.c1;
      if (c1 <= c0) continue;
      const int rows = t.ntok * p.G, p0 = t.p0 - span.shift, p1 = p0 + t.ntok - 1;  // (positions in the span's offsets)
      // the chunks that every row sees all of (nothing to mask)
      const int clear_from = p.mask.window > 0 ? (max(0, p1 - p.mask.window + 1) + kChunk - 1) / kChunk : 0;
      const int clear_to = max(min(p0 + 1, span.end), 0) / kChunk;
      int pos[kBlocks][2];  // of the rows in columns 2 tq and 2 tq + 1
      // q as the products' column operand: column g has query row 8 * block + g, the lane its dims from tq * kHd / 4 on
      uint32_t qb[kBlocks][kSteps][2];
      float scale2[kBlocks][2];  // of columns 2 tq and 2 tq + 1
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb) {
        const int row = 8 * nb + g;
        const int tok = kRaggedTiles ? row / p.G : 0;
        const T* qr = static_cast<const T*>(p.q) + (t.t0 + tok) * p.ldq + (h * p.G + row - tok * p.G) * kHd + tq * (kHd / 4);
        uint4 raw[kSteps / 2];
#pragma unroll
        for (int i = 0; i < kSteps / 2; ++i)
          raw[i] = row < rows ? *reinterpret_cast<const uint4*>(qr + 8 * i) : make_uint4(0, 0, 0, 0);
        int e = 0;  // q is taken times 2^e
        if constexpr (!std::is_same<T, __half>::value) {
          float most = 0.f;
#pragma unroll
          for (int i = 0; i < kSteps / 2; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = Elem<T>::unpack(w[k]);
              most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          }
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
          e = most == 0.f ? 0 : min(100, 14 + 127 - static_cast<int>(__float_as_uint(most) >> 23));
        }
#pragma unroll
        for (int i = 0; i < kSteps / 2; ++i) {
          const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t v = w[k];
            if constexpr (!std::is_same<T, __half>::value) {
              const float2 f = Elem<T>::unpack(v);
              const float by = power_of_two(e);
              v = Elem<__half>::pack(f.x * by, f.y * by);
            }
            qb[nb][2 * i + (k >> 1)][k & 1] = v;
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) pos[nb][u] = p0 + (kRaggedTiles ? (8 * nb + 2 * tq + u) / p.G : 0);
#pragma unroll
        for (int u = 0; u < 2; ++u) scale2[nb][u] = p.scale2 * power_of_two(-__shfl_sync(0xffffffffu, e, 4 * (2 * tq + u)));
      }
      float o[kBlocks][kSteps][4];
      float base[kBlocks][2], reach[kBlocks][2], l[kBlocks][2];  // p = 2^(score - base); a score past base + reach sets it anew
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) o[nb][i][0] = o[nb][i][1] = o[nb][i][2] = o[nb][i][3] = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) base[nb][u] = 0.f, reach[nb][u] = -INFINITY, l[nb][u] = 0.f;
      }

      // The warp's kSub tiles of chunk i, in slot s. clear: every row sees all of the positions.
      auto tiles = [&](int i, bool clear) {
        const int r0 = 16 * kSub * sub;
        const uint8_t* kt = slots + s * S::kBytes;
        const uint8_t* vt = kt + S::kTensor;
        // S^T: rows are positions, columns query rows
        float sc[kSub][kBlocks][4];
        uint32_t ks[kSub][2][2];  // scales of rows g and g + 8, of both halves of a lane's dims
#pragma unroll
        for (int tile = 0; tile < kSub; ++tile) {
#pragma unroll
          for (int nb = 0; nb < kBlocks; ++nb) sc[tile][nb][0] = sc[tile][nb][1] = sc[tile][nb][2] = sc[tile][nb][3] = 0.f;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = r0 + 16 * tile + row_a + 8 * e;
            if constexpr (kHd == 128) {
              const uint32_t two = fp4_scales(*reinterpret_cast<const uint16_t*>(kt + S::kScalesAt + r * F::kScales + 2 * tq));
              ks[tile][e][0] = prmt(two, two, 0x1010), ks[tile][e][1] = prmt(two, two, 0x3232);
            } else {
              const uint32_t one = fp4_scales(kt[S::kScalesAt + r * F::kScales + tq]);
              ks[tile][e][0] = ks[tile][e][1] = prmt(one, one, 0x1010);
            }
          }
        }
        uint32_t kw[kSub][2][kWords];
#pragma unroll
        for (int tile = 0; tile < kSub; ++tile)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint8_t* at = kt + (r0 + 16 * tile + row_a + 8 * e) * F::kCodes + (kHd / 8) * tq;
            if constexpr (kHd == 128) {
              const uint4 w = *reinterpret_cast<const uint4*>(at);
              kw[tile][e][0] = w.x, kw[tile][e][1] = w.y, kw[tile][e][2] = w.z, kw[tile][e][3] = w.w;
            } else {
              const uint2 w = *reinterpret_cast<const uint2*>(at);
              kw[tile][e][0] = w.x, kw[tile][e][1] = w.y;
            }
          }
#pragma unroll
        for (int w = 0; w < kWords; ++w)
#pragma unroll
          for (int tile = 0; tile < kSub; ++tile) {
            uint32_t a[2][4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              fp4_codes(kw[tile][e][w], a[e]);
#pragma unroll
              for (int k = 0; k < 4; ++k) a[e][k] = hmul2_rn(a[e][k], ks[tile][e][2 * w / kWords]);
            }
#pragma unroll
            for (int nb = 0; nb < kBlocks; ++nb) {
              mma_16816(sc[tile][nb], a[0][0], a[1][0], a[0][1], a[1][1], qb[nb][2 * w][0], qb[nb][2 * w][1]);
              mma_16816(sc[tile][nb], a[0][2], a[1][2], a[0][3], a[1][3], qb[nb][2 * w + 1][0], qb[nb][2 * w + 1][1]);
            }
          }
        uint32_t pb[kSub][kBlocks][2];  // p as the products' column operand
#pragma unroll
        for (int nb = 0; nb < kBlocks; ++nb) {
          float y[kSub][4], top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int tile = 0; tile < kSub; ++tile)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[tile][e] = fmaf(sc[tile][nb][e], scale2[nb][e & 1], -base[nb][e & 1]);
            }
          if (!clear) {
#pragma unroll
            for (int tile = 0; tile < kSub; ++tile)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int j = i * kChunk + r0 + 16 * tile + row_a + 8 * (e >> 1);
                if (!(j < span.end && p.mask.sees(pos[nb][e & 1], j))) y[tile][e] = -INFINITY;
              }
          }
#pragma unroll
          for (int tile = 0; tile < kSub; ++tile)
#pragma unroll
            for (int e = 0; e < 4; ++e) top[e & 1] = fmaxf(top[e & 1], y[tile][e]);
          if (__any_sync(0xffffffffu, top[0] > reach[nb][0] || top[1] > reach[nb][1])) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float most = top[u];
              most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
              most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
              most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
              if (most > reach[nb][u]) {
                const float to = base[nb][u] + (most - kRefBelow), up = to - base[nb][u];
                const float keep = reach[nb][u] == -INFINITY ? 0.f : exp2_approx(-up);
                base[nb][u] = to;
                reach[nb][u] = kRefReach;
                l[nb][u] *= keep;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                  o[nb][k][u] *= keep;
                  o[nb][k][u + 2] *= keep;
                }
#pragma unroll
                for (int tile = 0; tile < kSub; ++tile) y[tile][u] -= up, y[tile][u + 2] -= up;
              }
            }
          }
#pragma unroll
          for (int tile = 0; tile < kSub; ++tile) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[e] = exp2_approx(y[tile][e]);
              l[nb][e & 1] += w[e];
            }
            pb[tile][nb][0] = transpose8(Elem<__half>::pack(w[0], w[1]));
            pb[tile][nb][1] = transpose8(Elem<__half>::pack(w[2], w[3]));
          }
        }
        // O^T: rows are dims (row g of tile k: the lane's dim 2 k, row g + 8: 2 k + 1), the inner index runs over positions:
        // the lane's four are tq, tq + 4, tq + 8, tq + 12
#pragma unroll
        for (int tile = 0; tile < kSub; ++tile) {
          uint32_t vw[4][kHd / 64], vs[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = r0 + 16 * tile + tq + 4 * e;
            if constexpr (kHd == 128) {
              const uint2 w = *reinterpret_cast<const uint2*>(vt + r * F::kCodes + 8 * g);
              vw[e][0] = w.x, vw[e][1] = w.y;
              vs[e] = vt[S::kScalesAt + r * F::kScales + g];
            } else {
              vw[e][0] = *reinterpret_cast<const uint32_t*>(vt + r * F::kCodes + 4 * g);
              vs[e] = vt[S::kScalesAt + r * F::kScales + (g >> 1)];
            }
          }
          if (!clear) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!span.needs(i * kChunk + r0 + 16 * tile + tq + 4 * e, 1, p.mask)) vs[e] = 0;
          }
          const uint32_t s01 = fp4_scales(vs[0] | vs[1] << 8), s23 = fp4_scales(vs[2] | vs[3] << 8);
#pragma unroll
          for (int w = 0; w < kHd / 64; ++w) {
            uint32_t a[4][4];
            fp4_codes(choose(vw[0][w], vw[1][w] << 4, kLow), a[0]);
            fp4_codes(choose(vw[0][w] >> 4, vw[1][w], kLow), a[1]);
            fp4_codes(choose(vw[2][w], vw[3][w] << 4, kLow), a[2]);
            fp4_codes(choose(vw[2][w] >> 4, vw[3][w], kLow), a[3]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t a0 = hmul2_rn(a[0][k], s01), a1 = hmul2_rn(a[1][k], s01), a2 = hmul2_rn(a[2][k], s23), a3 = hmul2_rn(a[3][k], s23);
#pragma unroll
              for (int nb = 0; nb < kBlocks; ++nb) mma_16816(o[nb][4 * w + k], a0, a1, a2, a3, pb[tile][nb][0], pb[tile][nb][1]);
            }
          }
        }
      };
      for (int i = c0; i < c1; ++i, filled()) {
        if (ok && !wait_for(&full[s], round & 1, p.err, DK_DEVERR_WAIT_FULL)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          const bool clear = i >= clear_from && i < clear_to;
          if (clear || span.needs(i * kChunk + 16 * kSub * sub, 16 * kSub, p.mask)) tiles(i, clear);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }
      // the warps' results of this part of the unit, joined
      if (gtid == 0 && walk.cut(span)) p.cut[cta] = walk.cut_record(span);
      if (joined) group_sync(group);  // (the last part's results have been read)
      joined = true;
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float sum = l[nb][u];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int row = 8 * nb + 2 * tq + u;
          float* to = &pre_o[(sub * kRows + row) * kHd + g * (kHd / 8)];
#pragma unroll
          for (int k = 0; k < kSteps; k += 2)
            *reinterpret_cast<float4*>(to + 2 * k) = make_float4(o[nb][k][u], o[nb][k][u + 2], o[nb][k + 1][u], o[nb][k + 1][u + 2]);
          if (g == 0) pre_ml[row * kCWarps + sub] = make_float2(reach[nb][u] == -INFINITY ? -INFINITY : base[nb][u], sum);
        }
      group_sync(group);
      const bool all_of_it = c0 == 0 && c1 == span.n, whole = all_of_it && !p.always_partial;
      const int64_t slot = partial_slot(ctas, cta, c0 == 0, all_of_it, h * line.tiles + walk.ti);
      for (int e = gtid; e < rows * (kHd / 4) && ok; e += kCWarps * 32) {
        const int row = e / (kHd / 4), d = 4 * (e % (kHd / 4));
        float2 ml[kCWarps];
        float m = -INFINITY, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kCWarps; ++w) {
          ml[w] = pre_ml[row * kCWarps + w];
          m = fmaxf(m, ml[w].x);
        }
        const float use = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int w = 0; w < kCWarps; ++w) {
          const float wt = exp2_approx(ml[w].x - use);
          const float4 v = *reinterpret_cast<const float4*>(&pre_o[(w * kRows + row) * kHd + d]);
          sum = fmaf(wt, ml[w].y, sum);
          acc.x = fmaf(wt, v.x, acc.x), acc.y = fmaf(wt, v.y, acc.y), acc.z = fmaf(wt, v.z, acc.z), acc.w = fmaf(wt, v.w, acc.w);
        }
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum * p.out_scale;
          const int tok = kRaggedTiles ? row / p.G : 0;
          T* dst = static_cast<T*>(p.out) + ((static_cast<int64_t>(t.t0 + tok) * p.nkv + h) * p.G + row - tok * p.G) * kHd + d;
          *reinterpret_cast<uint2*>(dst) = make_uint2(Elem<T>::pack(acc.x * inv, acc.y * inv), Elem<T>::pack(acc.z * inv, acc.w * inv));
        } else {
          *reinterpret_cast<float4*>(&p.part_o[(slot * kRows + row) * kHd + d]) = acc;
          if (d == 0) *reinterpret_cast<float2*>(&p.part_ml[(slot * kRows + row) * 2]) = make_float2(m, sum);
        }
      }
    }
  }
  if (kRaggedTiles && p.zero_outside && producer) zero_outside_rows<kHd>(p, cta, ctas, lane);
  if (__syncthreads_or(!ok) && producer && lane == 0) {
    // a wait gave up: let copies still in flight land before the shared memory goes away (bounded)
    const uint64_t t0 = globaltimer_ns();
    for (int f = max(0, fill - ring); f < fill; ++f)
      while (!mbar_try_wait(&full[f % ring], (f / ring) & 1) && globaltimer_ns() - t0 < 500000000ull) {
      }
  }
  if (wait_late) pdl_wait();
}

template <typename T, int kHd, int kBlocks, bool kRaggedTiles>
RowsShape shape() {
  static std::mutex mu;
  static int per_sm[64];  // by device; 0: not asked yet
  RowsShape s;
  s.ring = kRing<kHd, kBlocks>;
  s.smem = static_cast<size_t>(kGroups<kBlocks>) * (s.ring * Slot<kHd>::kBytes + kCWarps * 8 * kBlocks * kHd * 4);
  static_assert((kMaxBatch + 1) * 4 <= kGroups<kBlocks> * kRing<kHd, kBlocks> * Slot<kHd>::kBytes,
                "the chunk sums fit the ring");
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  int& n = per_sm[dev & 63];
  if (n == 0) {
    auto k = fp4_rows_kernel<T, kHd, kBlocks, kRaggedTiles>;
    if (opt_in_dynamic_smem(k) < static_cast<int>(s.smem) ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, kThreads<kBlocks>, s.smem) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
  }
  s.ctas = n * device_info().num_sms;
  return s;
}

}  // namespace

// One token each: tiles of 8 or 16 rows; ragged: of 16.
#define DK_BY_KIND(CALL, TT, HH) (ragged ? CALL(TT, HH, 2, true) : rows == 8 ? CALL(TT, HH, 1, false) : CALL(TT, HH, 2, false))
#define DK_BY_TYPE(CALL)                                                                                  \
  (dtype == DK_F16 ? (hd == 128 ? DK_BY_KIND(CALL, __half, 128) : DK_BY_KIND(CALL, __half, 64))           \
                   : (hd == 128 ? DK_BY_KIND(CALL, __nv_bfloat16, 128) : DK_BY_KIND(CALL, __nv_bfloat16, 64)))

RowsShape fp4_rows_shape(int64_t hd, int dtype, int rows, bool ragged) {
#define DK_SHAPE(TT, HH, NB, RR) shape<TT, HH, NB, RR>()
  return DK_BY_TYPE(DK_SHAPE);
#undef DK_SHAPE
}

cudaError_t fp4_rows_launch(const Problem& p, int64_t hd, int dtype, int rows, bool ragged, const RowsShape& s, int wait_late,
                            cudaStream_t st) {
#define DK_ROWS(TT, HH, NB, RR) \
  launch(fp4_rows_kernel<TT, HH, NB, RR>, dim3(s.ctas), dim3(kThreads<NB>), s.smem, st, pdl_enabled(), dim3(1, 1, 1), p, wait_late)
  return DK_BY_TYPE(DK_ROWS);
#undef DK_ROWS
}

}  // namespace paged
}  // namespace dk
