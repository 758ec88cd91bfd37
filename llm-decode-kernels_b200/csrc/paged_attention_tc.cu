// Attention over a paged cache for many query rows per kv head (prompts, and the prefix a batch shares) on the
// 5th-generation tensor cores.
//
// A CTA works on units of 256 query rows (two halves A and B of up to 128 rows: the G heads of 128 / G tokens each) and
// walks its chunks of 128 positions. Per chunk and half, S = Q K^T and O += P V are 128 x 128 x head_dim products,
// 4 * 128^2 * head_dim flops, whose operands Q, K and V lie in shared memory and whose accumulators and P lie in tensor
// memory:
// * warp 9 streams Q (a box of the half's heads and tokens) and, page by page, K and V (64-dim columns of 128 rows) with
//   TMA into the 128-byte-swizzled layout that tcgen05.mma reads; K's rows are contiguous along the product's inner
//   dimension (K-major), V's along its outer one (N-major), so neither is transposed in memory;
// * warp 8 issues the products, in the order PV_A(i), QK_A(i+1), PV_B(i), QK_B(i+1): while one half's softmax runs, the
//   other half's products do. Products of one thread run in order, so P(i) may lie where S(i+1) will;
// * warps 0-3 and 4-7 are the softmax of A and B, a thread per row: S from tensor memory, the row maximum, P = 2^(S - m) in
//   16 bits back to tensor memory. The maximum that P refers to is raised only when a row's grows by 2^8 or more; then
//   the row of O is rescaled in tensor memory (P stays below 2^8, far inside fp16; sums are fp32).
// The maximum and -inf for a masked score come before the scale, so it has to be positive there: of a negative one the products
// negate Q, and of zero they get a Q of zeros.
// V rows that no row of the unit sees (past the end, between sinks and window, pages that were not read) are zeroed in
// shared memory before the product, so that P = 0 does not meet a NaN; masked scores are replaced before the maximum.
// Every wait is bounded.
// kFp4: the pages are held in 4 bits. Chunks come as they lie in the pages (bulk copies of codes and scales) into a ring of their own, and
// four more warps convert them to fp16 into the slots that the products read, zeroing the V rows that no row sees on the way;
// all operands are fp16 (code * scale is exact there), so bf16 Q is turned into fp16 by its rows' softmax threads first, times a
// power of two that the row's scale takes back. For prompts the conversion of every chunk for every tile costs more than it
// saves: MMAs read shared memory at nearly its full rate, and the converted tiles are stored beside that (a prompt of 8192, 12 heads
// over 2: 271 us, 280 with two converting warps of twice the registers; copied to 16-bit pages first 193). It is used for prefixes
// and for ragged calls of fewer tokens.
// What bounds it: a chunk's four products take 4 x 8 x 65 = 2080 cycles at head_dim 128, its 32768 exponentials 2048 (16 a
// cycle), and they run beside each other; a pair of half chunks takes about 1.65 us (1.15 at least), a unit's start, masks
// and output about 5 us more. Measured: a prompt of 8192, 12 heads over 2 of 128, 197 us in short bursts, 1.05 PFLOP/s, 64%
// of the cuBLAS rate; under the power cap (1.69 GHz) 228 us, 65% of cuBLAS's there. 220 to 228 bytes of a thread's registers are
// spilled, 428 to 520 with kFp4 (128 registers at launch). 16 softmax warps, two a row: 362 us. Exponentials
// on the FMA units for an eighth of the positions: 206 us. Steps of 64 positions: their products take nearly as long (58 cycles).
#include <climits>
#include <mutex>

#include "paged_fp4.cuh"
#include "tcgen05.cuh"

namespace dk {
namespace paged {
namespace {

constexpr int kMmaWarp = 8, kLoadWarp = 9, kZeroWarp = 10;
constexpr int kConvertWarp = 10, kConvertWarps = 4;  // kFp4: of warps 10..15; without it warps 10 and 11 only give their registers away
// The softmax warpgroups take what the others give up of the registers that the launch holds:
// 256 * 208 + 128 * 88 = 384 * 168, and with two warpgroups more 256 * 208 + 256 * 48 = 512 * 128.
template <bool kFp4>
constexpr int kThreads = kFp4 ? 512 : 384;
template <bool kFp4>
constexpr int kRegsLaunch = kFp4 ? 128 : 168;
template <bool kFp4>
constexpr int kRegsOther = kFp4 ? 48 : 88;
constexpr int kRegsSoftmax = 208;
static_assert(256 * kRegsSoftmax + 128 * kRegsOther<false> <= kThreads<false> * kRegsLaunch<false> &&
                  256 * kRegsSoftmax + 256 * kRegsOther<true> <= kThreads<true> * kRegsLaunch<true>,
              "register split");
constexpr int kC = kTcChunk;
constexpr float kLazy = 8.f;  // growth (base 2) of a row's maximum that P takes without rescaling O
// P is handed over in two parts, positions 0..95 and 96..127: the products of the first run while the exponentials of the
// second are computed, so that only a quarter of P V is left after the softmax (a prompt of 8192: 196 us; 198 us with
// parts of 64 and 64, 202 us in one piece).
constexpr int kPartChunks = 3;  // 32-position chunks of the first part
constexpr int kPartSteps = 2 * kPartChunks;  // its products of 16 positions each

template <int kHd, bool kFp4>
struct Smem {
  static constexpr int kSegs = kHd / 64;
  static constexpr int kSegBytes = 128 * 128;            // 128 rows of 64 dims
  static constexpr int kTileBytes = kSegs * kSegBytes;   // Q half, K chunk or V chunk
  static constexpr int kSlots = (kHd == 128 ? 5 : 10) - (kFp4 ? (kHd == 128 ? 1 : 2) : 0);
  // kFp4: a K or V chunk as it lies in the pages, its codes before its scales
  static constexpr int kRawScalesAt = kC * Fp4<kHd>::kCodes;
  static constexpr int kRawBytes = kC * Fp4<kHd>::kRow;
  static constexpr int kRaw = kFp4 ? (kHd == 128 ? 3 : 6) : 0;
  static constexpr int kBytes = 1024 + (2 + kSlots) * kTileBytes + kRaw * kRawBytes;
};

struct Barriers {
  uint64_t kv_full[10], kv_empty[10];
  uint64_t q_full[2], q_empty;  // kFp4: a half's own; otherwise the first of both
  uint64_t q_ready[2];          // kFp4, bf16: the half's Q is in fp16
  uint64_t raw_full[6], raw_empty[6];  // kFp4
  uint64_t s_full[2], p_full[2][2], o_full[2];  // p_full: [half][the two parts of P]
  uint64_t drain;
};

// Shared-memory matrix descriptor of an N-major operand in the 128-byte-swizzled layout: rows of 128 bytes (64 values along
// N), one row per value along K; 8-row atoms follow each other along K (stride byte offset 1024), blocks of 64 along N
// lie kSegBytes apart (leading byte offset). The start moves along K by whole atoms.
__device__ __forceinline__ uint64_t sdesc_n_sw128(uint32_t smem_byte_addr, uint32_t block_bytes) {
  return static_cast<uint64_t>((smem_byte_addr >> 4) & 0x3FFF) | (static_cast<uint64_t>(block_bytes >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor: fp32 accumulator, A and B both of type T, A K-major, B K-major or N-major.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int M, int N, bool b_n_major) {
  const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (b_n_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

constexpr uint32_t kNegateA = 1u << 13;

// The products are issued by whole warps with one lane elected inside the instruction sequence: the operands stay
// warp-uniform values, where a branch on the lane would make each of them a value of one thread (and a product took
// about 130 cycles to issue, twice its execution).
// D[tmem] (+)= A[smem] * B[smem]^T for one K = 16 slice.
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, q;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem] for one K = 16 slice: A is 128 rows (lanes) of 8 columns of 16-bit pairs.
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p, q;\nelect.sync _|q, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on `bar` when all products issued so far have completed (the same elected lane).
__device__ __forceinline__ void commit_elected(uint64_t* bar) {
  asm volatile(
      "{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\n"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 64 columns of one lane per thread. The wait is part of the statement: until it, the registers must not even be moved.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
      "%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,"
      "%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];\ntcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
        "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
        "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
        "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
        "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
      : "r"(taddr)
      : "memory");
}

// The lowest n bits, for any n.
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t bits2(float2 v) {
  return static_cast<uint64_t>(__float_as_uint(v.x)) | (static_cast<uint64_t>(__float_as_uint(v.y)) << 32);
}
__device__ __forceinline__ float2 from_bits2(uint64_t v) {
  return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return from_bits2(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return from_bits2(d);
}

// Of four lanes' four 16-byte pieces each: lane l of the four gets piece l of all of them.
__device__ __forceinline__ void exchange(uint4& a, uint4& b, bool upper, int with) {
  const uint4 send = upper ? a : b;
  uint4 got;
  got.x = __shfl_xor_sync(0xffffffffu, send.x, with);
  got.y = __shfl_xor_sync(0xffffffffu, send.y, with);
  got.z = __shfl_xor_sync(0xffffffffu, send.z, with);
  got.w = __shfl_xor_sync(0xffffffffu, send.w, with);
  if (upper)
    a = got;
  else
    b = got;
}
__device__ __forceinline__ void transpose4(uint4 (&w)[4], int lane) {
  exchange(w[0], w[1], lane & 1, 1);
  exchange(w[2], w[3], lane & 1, 1);
  exchange(w[0], w[2], lane & 2, 2);
  exchange(w[1], w[3], lane & 2, 2);
}

__device__ __forceinline__ float row_max(const float (&s)[kC]) {
  float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int c = 4; c < kC; ++c) m4[c & 3] = fmaxf(m4[c & 3], s[c]);
  return fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
}

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(smem_addr(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}

// kFp4. A row of Q in shared memory from bf16 to fp16, times the power of two that brings its largest value to 2^14: what falls
// below fp16's smallest step then is 2^-38 of that. Returns the power's exponent. One thread per row; swizzled 16-byte pieces are
// taken in an order that spreads a warp's rows over the banks.
template <int kHd, bool kFp4>
__device__ __forceinline__ int q_to_fp16(uint8_t* row, int r) {
  using L = Smem<kHd, kFp4>;
  uint4 w[kHd / 8];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kHd / 8; ++i) {
    w[i] = *reinterpret_cast<const uint4*>(row + (i >> 3) * L::kSegBytes + (((i & 7) ^ (r & 7)) << 4));
    const uint32_t m = 0x7fff7fffu;
    most = __vmaxu2(most, __vmaxu2(__vmaxu2(w[i].x & m, w[i].y & m), __vmaxu2(w[i].z & m, w[i].w & m)));
  }
  most = max(most >> 16, most & 0xffffu);
  const int e = most == 0 ? 0 : min(100, 14 + 127 - static_cast<int>(most >> 7));
  const float by = __int_as_float((127 + e) << 23);
  auto turn = [&](uint32_t v) {
    const float2 f = Elem<__nv_bfloat16>::unpack(v);
    return Elem<__half>::pack(f.x * by, f.y * by);
  };
#pragma unroll
  for (int i = 0; i < kHd / 8; ++i)
    *reinterpret_cast<uint4*>(row + (i >> 3) * L::kSegBytes + (((i & 7) ^ (r & 7)) << 4)) =
        make_uint4(turn(w[i].x), turn(w[i].y), turn(w[i].z), turn(w[i].w));
  return e;
}

// P: the type of P and V in their product. K and Q are of type T, with kFp4 fp16.
template <typename T, int kHd, bool kFp4, typename P>
__global__ void __launch_bounds__(kThreads<kFp4>, 1)
    tiles_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                 const __grid_constant__ CUtensorMap mv, const Problem p, int wait_late) {
  using L = Smem<kHd, kFp4>;
  using K = typename std::conditional<kFp4, __half, T>::type;
  constexpr bool kTurnQ = !std::is_same<T, K>::value;
  constexpr uint32_t kS[2] = {0, 128}, kO[2] = {256, 256 + kHd};  // tensor-memory columns; P(X) lies over S(X)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* q_sm = smem;
  uint8_t* slots = smem + 2 * L::kTileBytes;
  uint8_t* raw = slots + L::kSlots * L::kTileBytes;
  __shared__ __align__(8) Barriers bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (kFp4 && p.above > 0) {  // beside a launch for the sequences of few tokens: there may be no others
    pdl_wait();
    if (p.plan[0] == 0) {
      pdl_trigger();
      if (tid == 0) p.cut[blockIdx.x] = make_int4(0, 0, 0, 0);  // (the join reads every CTA's)
      if (warp == kZeroWarp && p.zero_outside) zero_outside_rows<kHd>(p, blockIdx.x, gridDim.x, lane);
      return;
    }
  }
  if (tid == 0) {
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(&bar.kv_full[i], kFp4 ? kConvertWarps : 1);
      mbar_init(&bar.kv_empty[i], 1);
    }
    for (int i = 0; i < L::kRaw; ++i) {
      mbar_init(&bar.raw_full[i], 1);
      mbar_init(&bar.raw_empty[i], kConvertWarps);
    }
    mbar_init(&bar.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.q_full[i], 1);
      mbar_init(&bar.q_ready[i], 4);
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.p_full[i][0], 4);
      mbar_init(&bar.p_full[i][1], 4);
      mbar_init(&bar.o_full[i], 1);
    }
    mbar_init(&bar.drain, 1);
    failed = 0;
    fence_mbar_init();
    prefetch_tensormap(&mq);
    if constexpr (!kFp4) {
      prefetch_tensormap(&mk);
      prefetch_tensormap(&mv);
    }
  }
  if (warp == kMmaWarp) {
    tc::tmem_alloc(&tmem_slot, 512);
    tc::tmem_relinquish();
    tc::fence_before_sync();
  }
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_slot;
  if (!wait_late) pdl_wait();
  pdl_trigger();

  const Line line = line_of(p, kC);
  Walk<kC> walk(p, line, blockIdx.x, gridDim.x, lane);
  bool ok = true;

  if (warp >= kMmaWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther<kFp4>));
  if (warp == kLoadWarp) {
    // ---------------------------------------------------------------- loads
    const int box = min(p.page_size, kC), boxes = kC / box;
    const int sg = lane % L::kSegs, pg = kFp4 ? lane >> 1 : lane / L::kSegs;
    int fill = 0;
    // kFp4: a lane copies the codes or the scales of its page
    const int row_bytes = lane & 1 ? Fp4<kHd>::kScales : Fp4<kHd>::kCodes;
    for (int part = 0; walk.more() && ok; ++part) {
      const Span<kC> span = walk.step();
      if (walk.c1 <= walk.c0) {
        --part;
        continue;
      }
      const int h = walk.h, c0 = walk.c0, c1 = walk.c1;
      const int32_t* table = walk.t.table;
      if (lane == 0 && walk.last >= p.capacity) record_device_error(p.err, DK_DEVERR_BAD_POSITION);  // cut to the table
      const bool two = walk.t.ntok > p.half_tokens;
      auto entry = [&](int i) {  // this lane's page in chunk i of the unit; INT_MIN: none, or nothing that a row sees
        const int j = i * kC + pg * box;
        return i < c1 && pg < boxes && span.needs(j, box, p.mask) ? table[span.position(j) >> p.page_shift] : INT_MIN;
      };
      auto put = [&](const CUtensorMap* map, int i, int page) {
        const int s = fill % L::kSlots;
        if (fill >= L::kSlots && !wait_for(&bar.kv_empty[s], ((fill / L::kSlots) - 1) & 1, p.err, DK_DEVERR_WAIT_EMPTY))
          ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        const bool mine = page != INT_MIN;
        const unsigned want = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) mbar_arrive_expect_tx(&bar.kv_full[s], __popc(want) * box * 128);
        __syncwarp();
        if (mine) {
          const int y = pool_row(p, page, h, span.position(i * kC + pg * box));
          tma_load_2d(slots + s * L::kTileBytes + sg * L::kSegBytes + pg * box * 128, map, sg * 64, y, &bar.kv_full[s]);
        }
        ++fill;
      };
      auto put_raw = [&](int kv, int i, int page) {
        const int s = fill % max(L::kRaw, 1);
        if (fill >= L::kRaw && !wait_for(&bar.raw_empty[s], ((fill / max(L::kRaw, 1)) - 1) & 1, p.err, DK_DEVERR_WAIT_EMPTY)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        const uint32_t bytes = box * row_bytes;
        uint8_t* at = raw + s * L::kRawBytes + (lane & 1 ? L::kRawScalesAt : 0) + pg * bytes;
        const bool wanted = page != INT_MIN, mine = wanted && page >= 0 && page < p.n_pages;
        if (wanted && !mine) {  // no page of the pool: scales of zero
          record_device_error(p.err, DK_DEVERR_BAD_POSITION);
          if (lane & 1)
            for (uint32_t b = 0; b < bytes; b += 16) *reinterpret_cast<uint4*>(at + b) = make_uint4(0, 0, 0, 0);
          tc::fence_proxy_async_smem();
        }
        __syncwarp();
        const unsigned pages = __popc(__ballot_sync(0xffffffffu, mine)) / 2;
        if (lane == 0) mbar_arrive_expect_tx(&bar.raw_full[s], pages * box * Fp4<kHd>::kRow);
        __syncwarp();
        if (mine) {
          const int in_page = span.position(i * kC + pg * box) & (p.page_size - 1);
          bulk_g2s(at, p.pool[kv] + (static_cast<int64_t>(page) * p.nkv + h) * (p.page_size * Fp4<kHd>::kRow) +
                           (lane & 1 ? p.page_size * Fp4<kHd>::kCodes : 0) + in_page * row_bytes,
                   bytes, &bar.raw_full[s]);
        }
        ++fill;
      };
      auto put_chunk = [&](int kv, int i, int page) {
        if constexpr (kFp4)
          put_raw(kv, i, page);
        else
          put(kv ? &mv : &mk, i, page);
      };
      int page = entry(c0);
      // Q, once the last part's products with it have completed
      if (part > 0 && !wait_for(&bar.q_empty, (part - 1) & 1, p.err, DK_DEVERR_WAIT_EMPTY)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) {
        if constexpr (!kFp4) mbar_arrive_expect_tx(&bar.q_full[0], (two ? 2 : 1) * L::kSegs * p.half_tokens * p.G * 128);
        for (int x = 0; x < (two ? 2 : 1); ++x) {
          if constexpr (kFp4) mbar_arrive_expect_tx(&bar.q_full[x], L::kSegs * p.half_tokens * p.G * 128);
          for (int s = 0; s < L::kSegs; ++s)
            tma_load_3d(q_sm + x * L::kTileBytes + s * L::kSegBytes, &mq, s * 64, h * p.G,
                        p.signs == 0 ? p.T : walk.t.t0 + x * p.half_tokens, &bar.q_full[kFp4 ? x : 0]);  // (past the end: zeros)
        }
      }
      __syncwarp();
      put_chunk(0, c0, page);
      for (int i = c0; i < c1 && ok; ++i) {
        const int next = entry(i + 1);
        put_chunk(1, i, page);
        if (i + 1 < c1 && ok) put_chunk(0, i + 1, next);
        page = next;
      }
    }
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- products
    int fill = 0;         // ring slots consumed
    unsigned p_seen[2] = {0, 0}, q_seen[2] = {0, 0};
    auto q_wait = [&](int x) {
      if (!wait_for(kTurnQ ? &bar.q_ready[x] : &bar.q_full[x], q_seen[x]++ & 1, p.err, DK_DEVERR_WAIT_FULL)) ok = false;
    };
    auto slot_wait = [&](int f) {
      if (ok && !wait_for(&bar.kv_full[f % L::kSlots], (f / L::kSlots) & 1, p.err, DK_DEVERR_WAIT_FULL)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
    };
    auto slot_at = [&](int f) { return smem_addr(slots + (f % L::kSlots) * L::kTileBytes); };
    auto qk = [&](int x, int f) {
      const uint64_t a = tc::sdesc_k_sw128(smem_addr(q_sm + x * L::kTileBytes)), b = tc::sdesc_k_sw128(slot_at(f));
#pragma unroll
      for (int k = 0; k < kHd / 16; ++k) {
        const uint32_t off = ((k / 4) * L::kSegBytes + (k % 4) * 32) >> 4;  // (descriptors count 16 bytes)
        mma_ss(tmem + kS[x], a + off, b + off, idesc<K>(128, kC, false) | (p.signs < 0 ? kNegateA : 0u), k > 0);
      }
      commit_elected(&bar.s_full[x]);
    };
    auto pv = [&](int x, int f, bool first) {
      const uint64_t b = sdesc_n_sw128(slot_at(f), L::kSegBytes);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (ok && !wait_for(&bar.p_full[x][half], p_seen[x] & 1, p.err, DK_DEVERR_WAIT_FULL)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        tc::fence_after_sync();
#pragma unroll
        for (int k = half * kPartSteps; k < (half ? kC / 16 : kPartSteps); ++k)
          mma_ts(tmem + kO[x], tmem + kS[x] + 8 * k, b + ((k * 2048) >> 4), idesc<P>(128, kHd, true), !first || k > 0);
      }
      ++p_seen[x];
    };
    while (walk.more() && ok) {
      const Span<kC> span = walk.step();
      const int n = walk.c1 - walk.c0;
      if (n <= 0) continue;
      const bool two = walk.t.ntok > p.half_tokens;
      q_wait(0);
      if (kFp4 && two) q_wait(1);
      slot_wait(fill);
      if (!ok) break;
      tc::fence_after_sync();
      qk(0, fill);
      if (two) qk(1, fill);
      commit_elected(&bar.kv_empty[fill % L::kSlots]);
      if (n == 1) commit_elected(&bar.q_empty);
      for (int i = 0; i < n && ok; ++i) {
        const int fv = fill + 2 * i + 1, fk = fv + 1;
        slot_wait(fv);
        if (!ok) break;
        const int j0 = (walk.c0 + i) * kC;
        // does every row of v belong to a position that some row of the unit sees?
        const bool clear = j0 + kC <= span.end && (p.mask.window <= 0 || j0 >= span.lo || j0 + kC <= p.mask.sinks);
        if (!kFp4 && !clear) {
          uint8_t* v = slots + (fv % L::kSlots) * L::kTileBytes + (lane & 7) * 16;
          auto zero = [&](int from, int to) {  // 8 lanes a row of 64 dims
            for (int r = min(max(from, 0), kC) + (lane >> 3); r < min(to, kC); r += 4)
#pragma unroll
              for (int c = 0; c < L::kSegs; ++c)
                *reinterpret_cast<uint4*>(v + c * L::kSegBytes + r * 128) = make_uint4(0, 0, 0, 0);
          };
          zero(p.mask.sinks - j0, min(span.lo, span.end) - j0);
          zero(span.end - j0, kC);
          tc::fence_proxy_async_smem();
          __syncwarp();
        }
        const bool more = i + 1 < n;
        pv(0, fv, i == 0);
        if (!ok) break;
        if (more) {
          slot_wait(fk);
          if (!ok) break;
          qk(0, fk);
        } else {
          commit_elected(&bar.o_full[0]);
        }
        if (two) {
          pv(1, fv, i == 0);
          if (!ok) break;
          if (more)
            qk(1, fk);
          else
            commit_elected(&bar.o_full[1]);
        }
        commit_elected(&bar.kv_empty[fv % L::kSlots]);
        if (more) commit_elected(&bar.kv_empty[fk % L::kSlots]);
        if (i + 2 == n) commit_elected(&bar.q_empty);
      }
      fill += 2 * n;
    }
  } else if (warp < kMmaWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ---------------------------------------------------------------- softmax: a thread per row
    const int x = warp >> 2, r = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lanes + kS[x], o_col = tmem + lanes + kO[x];
    unsigned s_seen = 0, o_seen = 0;
    if (tid == 0) p.cut[blockIdx.x] = make_int4(0, 0, 0, 0);
    const int first = x * p.half_tokens;  // this half's first token
    const int tok = first + r / p.G, g = r % p.G;
    bool more_parts = walk.next(first);
    while (more_parts && ok) {
      const Span<kC> span = walk.span;
      const Tile t = walk.t;
      const int c0 = walk.c0, c1 = walk.c1, head = walk.h * p.G + g;
      const bool live = r < p.half_tokens * p.G && tok < t.ntok;
      const int pos = live ? row_position(p, t, tok) - span.shift : -1;  // (in the span's offsets)
      const int p_lo = row_position(p, t, first) - span.shift;
      const int p_hi = row_position(p, t, min(t.ntok, first + p.half_tokens) - 1) - span.shift;
      float scale2 = p.scale2;
      if constexpr (kTurnQ) {
        if (!wait_for(&bar.q_full[x], o_seen & 1, p.err, DK_DEVERR_WAIT_FULL)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        scale2 *= __int_as_float((127 - q_to_fp16<kHd, kFp4>(q_sm + x * L::kTileBytes + r * 128, r)) << 23);
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.q_ready[x]);
      }
      float m = -INFINITY, l = 0.f;  // of scale2 * score
      for (int i = c0; i < c1; ++i) {
        if (!wait_for(&bar.s_full[x], s_seen & 1, p.err, DK_DEVERR_WAIT_FULL)) ok = false;
        ++s_seen;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::fence_after_sync();
        float s[kC];
#pragma unroll
        for (int c = 0; c < kC; c += 64) tmem_ld64(s_col + c, *reinterpret_cast<float(*)[64]>(&s[c]));
        const int j0 = i * kC;
        const bool clear = j0 + kC - 1 <= p_lo && j0 + kC <= span.end &&
                           (p.mask.window <= 0 || j0 > p_hi - p.mask.window || j0 + kC <= p.mask.sinks);
        if (!clear) {
          // the row's visible positions of this chunk, a bit each: [lo, end) and those below the sinks' end
          const int end = min(span.end, pos + 1) - j0, sinks = min(p.mask.sinks - j0, end);
          const int lo = p.mask.window > 0 ? pos - p.mask.window + 1 - j0 : INT_MIN;
#pragma unroll
          for (int c = 0; c < kC / 32; ++c) {
            const uint32_t see = (low_bits(end - 32 * c) & ~low_bits(lo - 32 * c)) | low_bits(sinks - 32 * c);
            if (__all_sync(0xffffffffu, see == 0xffffffffu)) continue;  // (a warp's rows are few tokens: true for most c)
#pragma unroll
            for (int d = 0; d < 32; ++d) s[32 * c + d] = see & (1u << d) ? s[32 * c + d] : -INFINITY;
          }
        }
        // P refers to a maximum that is only raised when a row's grows by 2^kLazy or more.
        const float mx = row_max(s) * scale2;
        const bool raise = mx > m + kLazy || (m == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xffffffffu, raise)) {
          const float keep = raise ? exp2_approx(m - mx) : 1.f;
          if (raise) {
            m = mx;
            l *= keep;
          }
          if (i > c0) {  // O's products up to the last chunk are done: S came after them
#pragma unroll
            for (int c = 0; c < kHd / 16; ++c) {
              float o[16];
              uint32_t w[16];
              tc::tmem_ld16(o_col + 16 * c, o);
#pragma unroll
              for (int d = 0; d < 16; ++d) w[d] = __float_as_uint(o[d] * keep);
              tmem_st16(o_col + 16 * c, w);
            }
          }
        }
        const float base = m == -INFINITY ? 0.f : m;
        const float2 scale = make_float2(scale2, scale2), off = make_float2(-base, -base);
        float2 sum[4] = {};
#pragma unroll
        for (int c = 0; c < kC / 32; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int d = 0; d < 16; ++d) {
            float2 y = fma2(make_float2(s[32 * c + 2 * d], s[32 * c + 2 * d + 1]), scale, off);
            y = make_float2(exp2_approx(y.x), exp2_approx(y.y));
            sum[d & 3] = add2(sum[d & 3], y);
            w[d] = Elem<P>::pack(y.x, y.y);
          }
          tmem_st16(s_col + 16 * c, w);
          if (c == kPartChunks - 1 || c == kC / 32 - 1) {  // a part of P is complete
            tmem_wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.p_full[x][c / kPartChunks]);
          }
        }
        const float2 sums = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
        l += sums.x + sums.y;
      }
      // The next part is looked up while the last products run.
      const bool all_of_it = c0 == 0 && c1 == span.n, whole = all_of_it && !p.always_partial;
      const int64_t slot = partial_slot(gridDim.x, blockIdx.x, c0 == 0, all_of_it, walk.h * line.tiles + walk.ti);
      if (ok && tid == 0 && walk.cut(span)) p.cut[blockIdx.x] = walk.cut_record(span);
      more_parts = walk.next(first);
      if (ok && !wait_for(&bar.o_full[x], o_seen & 1, p.err, DK_DEVERR_WAIT_FULL)) ok = false;
      ++o_seen;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc::fence_after_sync();
      const int row = x * 128 + r;
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l * p.out_scale;
        // Four lanes exchange 16-byte pieces so that together they store 64 bytes of one row at a time: a lane storing its
        // own row would touch 32 lines with every instruction.
        T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(t.t0 + tok) * p.nkv * p.G + head) * kHd;
        T* row_out[4];
        bool row_live[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          row_out[k] = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), (lane & ~3) + k));
          row_live[k] = __shfl_sync(0xffffffffu, static_cast<int>(live), (lane & ~3) + k) != 0;
        }
#pragma unroll
        for (int c = 0; c < kHd; c += 64) {
          float o[64];
          tmem_ld64(o_col + c, o);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint4 w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float* v = &o[32 * half + 8 * k];
              w[k] = make_uint4(Elem<T>::pack(v[0] * inv, v[1] * inv), Elem<T>::pack(v[2] * inv, v[3] * inv),
                                Elem<T>::pack(v[4] * inv, v[5] * inv), Elem<T>::pack(v[6] * inv, v[7] * inv));
            }
            transpose4(w, lane);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (row_live[k]) *reinterpret_cast<uint4*>(row_out[k] + c + 32 * half + 8 * (lane & 3)) = w[k];
          }
        }
      } else {
        // Partial results lie with the rows innermost, [dims / 4][256 rows][4]: a warp stores 512 contiguous bytes.
        float* part = p.part_o + slot * kTcRows * kHd + row * 4;
#pragma unroll
        for (int c = 0; c < kHd; c += 64) {
          float o[64];
          tmem_ld64(o_col + c, o);
#pragma unroll
          for (int d = 0; d < 64; d += 4)
            if (live) *reinterpret_cast<float4*>(part + static_cast<int64_t>(c + d) * kTcRows) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
          __syncwarp();
        }
      }
      if (!whole && live) *reinterpret_cast<float2*>(&p.part_ml[(slot * kTcRows + row) * 2]) = make_float2(m, l);
      tc::fence_before_sync();
    }
  }

  if (kFp4 && warp >= kConvertWarp && warp < kConvertWarp + kConvertWarps) {
    // ---------------------------------------------------------------- conversion: a quarter of a chunk's rows each, K and V in turn
    // A lane takes 16 bytes of codes, 32 dims of a row, to four 16-byte pieces. The second segment's lanes (head_dim 128) take their
    // pieces in another order, so that 8 lanes' stores hit all banks.
    constexpr int kRowLanes = kHd / 32, kRowsAtOnce = 32 / kRowLanes, kSteps = kC / kConvertWarps / kRowsAtOnce;
    constexpr int kAhead = 2;  // steps whose codes are loaded at a time
    const int q = lane % kRowLanes, flip = q & 2;
    const int first = (warp - kConvertWarp) * (kC / kConvertWarps) + lane / kRowLanes;  // this lane's rows: first + i * kRowsAtOnce
    int fill = 0;
    while (walk.more() && ok) {
      const Span<kC> span = walk.step();
      for (int i = 2 * walk.c0; i < 2 * walk.c1; ++i, ++fill) {
        const int from = fill % max(L::kRaw, 1), s = fill % L::kSlots;
        if (!wait_for(&bar.raw_full[from], (fill / max(L::kRaw, 1)) & 1, p.err, DK_DEVERR_WAIT_FULL)) ok = false;
        if (ok && fill >= L::kSlots && !wait_for(&bar.kv_empty[s], ((fill / L::kSlots) - 1) & 1, p.err, DK_DEVERR_WAIT_EMPTY)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint8_t* codes_in = raw + from * L::kRawBytes + first * Fp4<kHd>::kCodes + 16 * q;
        const uint8_t* scales_in = raw + from * L::kRawBytes + L::kRawScalesAt + first * Fp4<kHd>::kScales + 2 * q;
        uint8_t* out = slots + s * L::kTileBytes + (q >> 1) * L::kSegBytes + first * 128;
        uint8_t* piece[4];  // (the rows of a lane are alike modulo 8, and so is their swizzle)
#pragma unroll
        for (int k = 0; k < 4; ++k) piece[k] = out + ((((q & 1) * 4 + (k ^ flip)) ^ (first & 7)) << 4);
        const int j0 = (i >> 1) * kC;
        // V rows of positions that no row of the unit sees become zeros (codes are finite whatever they are)
        const bool clear = (i & 1) == 0 || (j0 + kC <= span.end && (p.mask.window <= 0 || j0 >= span.lo || j0 + kC <= p.mask.sinks));
#pragma unroll
        for (int r0 = 0; r0 < kSteps; r0 += kAhead) {
          uint4 codes[kAhead];
          uint32_t scales[kAhead];
#pragma unroll
          for (int a = 0; a < kAhead; ++a) {
            codes[a] = *reinterpret_cast<const uint4*>(codes_in + (r0 + a) * kRowsAtOnce * Fp4<kHd>::kCodes);
            scales[a] = *reinterpret_cast<const uint16_t*>(scales_in + (r0 + a) * kRowsAtOnce * Fp4<kHd>::kScales);
          }
          if (!clear) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
              if (!span.needs(j0 + first + (r0 + a) * kRowsAtOnce, 1, p.mask)) scales[a] = 0;
          }
#pragma unroll
          for (int a = 0; a < kAhead; ++a) {
            const uint32_t two = fp4_scales(scales[a]);
            const uint32_t lo = prmt(two, two, flip ? 0x3232 : 0x1010), hi = prmt(two, two, flip ? 0x1010 : 0x3232);
            const uint4 c = codes[a];
            const uint32_t w[4] = {flip ? c.z : c.x, flip ? c.w : c.y, flip ? c.x : c.z, flip ? c.y : c.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t scale = k < 2 ? lo : hi;
              uint32_t v[4];
              fp4_codes(w[k], v);
              *reinterpret_cast<uint4*>(piece[k] + (r0 + a) * kRowsAtOnce * 128) =
                  make_uint4(hmul2_rn(v[0], scale), hmul2_rn(v[1], scale), hmul2_rn(v[2], scale), hmul2_rn(v[3], scale));
            }
          }
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar.kv_full[s]);
          mbar_arrive(&bar.raw_empty[from]);
        }
      }
    }
  }
  if (warp == kZeroWarp && p.zero_outside) zero_outside_rows<kHd>(p, blockIdx.x, gridDim.x, lane);

  __syncwarp();
  if (!ok && lane == 0) failed = 1;
  tc::fence_before_sync();
  __syncthreads();
  if (failed && warp == kMmaWarp) {
    // a wait gave up: let products and copies still in flight finish before their memory goes away (bounded)
    commit_elected(&bar.drain);
    if (lane == 0) {
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(&bar.drain, 0) && globaltimer_ns() - t0 < 500000000ull) {
      }
      const uint64_t t1 = globaltimer_ns();
      while (globaltimer_ns() - t1 < 20000000ull) {  // 20 ms: far more than any copy takes
      }
    }
    __syncwarp();
  }
  tc::fence_after_sync();
  if (warp == kMmaWarp) tc::tmem_dealloc(tmem, 512);
  if (wait_late) pdl_wait();
}

bool make_q_map(CUtensorMap* map, const Problem& p, int64_t nq, int64_t hd, CUtensorMapDataType type) {
  const uint64_t dims[3] = {static_cast<uint64_t>(hd), static_cast<uint64_t>(nq), static_cast<uint64_t>(p.T)};
  const uint64_t strides[2] = {static_cast<uint64_t>(hd) * 2, static_cast<uint64_t>(p.ldq) * 2};
  const uint32_t box[3] = {64, static_cast<uint32_t>(p.G), static_cast<uint32_t>(p.half_tokens)};
  return make_tensor_map(map, p.q, type, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T, int kHd, bool kFp4, typename P>
int ctas_of() {
  static std::mutex mu;
  static int known[64];  // by device; 0: not asked yet, -1: does not fit
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  int& n = known[dev & 63];
  if (n == 0) {
    cudaFuncAttributes a;  // the register split needs the launch to hold exactly what it divides
    const bool split = cudaFuncGetAttributes(&a, tiles_kernel<T, kHd, kFp4, P>) == cudaSuccess && a.numRegs == kRegsLaunch<kFp4>;
    n = split && opt_in_dynamic_smem(tiles_kernel<T, kHd, kFp4, P>) >= Smem<kHd, kFp4>::kBytes ? device_info().num_sms : -1;
  }
  return n < 0 ? 0 : n;
}

}  // namespace

#define DK_BY_PAGES(CALL, TT, HH)                       \
  (pages == Pages::kCodes  ? CALL(TT, HH, true, __half) \
   : pages == Pages::kCopy ? CALL(TT, HH, false, __half) : CALL(TT, HH, false, TT))
#define DK_BY_KIND(CALL)                                                                          \
  (dtype == DK_F16 ? (hd == 128 ? DK_BY_PAGES(CALL, __half, 128) : DK_BY_PAGES(CALL, __half, 64)) \
                   : (hd == 128 ? DK_BY_PAGES(CALL, __nv_bfloat16, 128) : DK_BY_PAGES(CALL, __nv_bfloat16, 64)))

int tc_ctas(int64_t hd, int dtype, Pages pages) {
#define DK_CTAS(TT, HH, FF, PP) ctas_of<TT, HH, FF, PP>()
  return DK_BY_KIND(DK_CTAS);
#undef DK_CTAS
}

int tc_launch(const Problem& p, int64_t nq, int64_t hd, int dtype, Pages pages, int ctas, const CUtensorMap& mk, const CUtensorMap& mv,
              int wait_late, cudaStream_t st) {
  const CUtensorMapDataType type = dtype == DK_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap mq;
  if (!make_q_map(&mq, p, nq, hd, type)) return DK_ERR_CUDA;
#define DK_TILES(TT, HH, FF, PP)                                                                                                    \
  launch(tiles_kernel<TT, HH, FF, PP>, dim3(ctas), dim3(kThreads<FF>), Smem<HH, FF>::kBytes, st, pdl_enabled(), dim3(1, 1, 1), mq, mk, \
         mv, p, wait_late)
  const cudaError_t e = DK_BY_KIND(DK_TILES);
#undef DK_TILES
  if (e != cudaSuccess) return set_error(DK_ERR_CUDA, "paged attention (256-row tiles) launch: %s", cudaGetErrorString(e));
  return DK_OK;
}

}  // namespace paged
}  // namespace dk
