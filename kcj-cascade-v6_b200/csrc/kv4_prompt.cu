// Attention of prompt chunks over a paged KV cache held in 4 bits: requests with
// more query rows than the few-row kernel takes (kv4_attend.cu).
//
// Bound by the tensor cores (4 D operations for each of 128 x 128 scores, 16 bits in)
// and, as much, by the exponentials: 16 a cycle against 4096 multiply-adds, so that
// at D = 128 a tile of scores takes 1024 cycles of either. One block an SM works on
// two tiles of 128 query rows against the same 128 tokens:
//   * 4 dequantising warps bring cache tiles in by bulk copies, turn the codes into
//     fp16 values and lay K and V^T out as the products' operands in shared memory;
//     both row tiles use them, which halves this work for each score;
//   * one thread issues the products (tcgen05, sums in tensor memory): S = Q K^T,
//     then O += P V with P from tensor memory, where it has taken S's place;
//   * 2 x 4 softmax warps, a thread to a query row: maximum, exponentials, P back as
//     fp16. While one row tile is in its softmax, the other one's products run.
// A running maximum is raised only when a score passes it by 2^8, which seldom
// happens after a row's first tokens, so that O is seldom rescaled.
//
// Measured: chunks of 900 to 1,537 tokens behind 5,200 to 9,100 cached ones, 64 / 8
// heads of 128, bf16: 639 us replayed in a CUDA graph, 761 TFLOP/s. The tensor cores are busy a third of the
// time, and what stands in their way is shared memory: for two row tiles the products
// read 192 KB of operands a tile of tokens and the dequantising warps store 64 KB, 2,000
// cycles of its bandwidth at best; of the 5,000 that a tile takes, a dequantising
// warp spends 4,000 in its stores' queue (with that work left out, a tile takes
// 4,000, with the softmax left out too, 3,600). Pairs of SMs that share a product
// would halve the reads of K and V and their stores. Tried without gain: 8
// dequantising warps, half of the exponentials as polynomials, the weights handed
// over in two halves, no pass for the maximum.
//
// Roundings to 16 bits: K and V as dequantised (2^-11 of a value; the price of one
// product for a score, where exact codes would need one for every group and two
// multiplications for every score), P, and the output; q is exact, as in
// kv4_attend.cu. A group of V that is not finite is zero as an operand, or rows that
// do not see its token would be hurt; in rows that do, its dims become NaN (the
// whole row and its log-sum-exp for such a K), whatever the token's weight.
#include "kv4_attend.cuh"

namespace cb {

namespace {

constexpr int kTok = 128;         // tokens of a tile
constexpr int kTileRows = 128;    // rows of a product
constexpr int kSoftWarps = 8, kDeqWarps = 4, kMmaWarp = kSoftWarps + kDeqWarps;
constexpr int kPromptWarps = 16, kPromptThreads = kPromptWarps * 32;  // the last three only make up a warpgroup
// Registers of a thread: 512 * 128 at launch, then for a softmax thread as many as
// hold a row of scores.
constexpr int kSoftRegs = 184, kDeqRegs = 88, kMmaRegs = 56;
static_assert(256 * kSoftRegs + 128 * kDeqRegs + 128 * kMmaRegs <= kPromptThreads * 128, "registers");
constexpr int kRaw = 3;           // cache tiles in a dequantising warp's ring
constexpr int kTmemCols = 512;

struct PromptLine {
  static constexpr int kRows = 2 * kTileRows, kTokens = kTok, kCost = 2, kWarps = kPromptWarps;
  static constexpr bool kBlock = true;
};

// What the dequantising warps say of 128 tokens, a byte each: a bit for each of the
// warp's two cache tiles that is there, and one if a token's K or V is not finite.
constexpr uint32_t kAllThere = 0x03030303u, kOdd = 0x04040404u;

template <int D, int NG>
struct PromptForm {
  static constexpr int kTile = 16 * D + 128 * NG;
  static constexpr int kOperand = 128 * D * 2;  // bytes of Q, K or V^T
  static constexpr int kQ = 0, kK = 2 * kOperand, kV = 4 * kOperand, kRing = 6 * kOperand;
  static constexpr int kFlags = kRing + kDeqWarps * kRaw * kTile;
  static constexpr int kBars = kFlags + 16;  // of four tiles
  static constexpr int kSmemUsed = kBars + 256;
  // one block an SM: each takes all of the tensor memory
  static constexpr int kSmem = kSmemUsed > 120 * 1024 ? kSmemUsed : 120 * 1024;
  static constexpr int kPart = PromptLine::kRows * (D + 2);
};

// ---- tcgen05

CB_D void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
CB_D void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
CB_D void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
CB_D void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
CB_D void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// Operands in shared memory: rows of 64 fp16 (128 bytes) along the axis that is
// summed over, 16-byte chunks exchanged within 8 rows by their number. A
// descriptor's low word holds the address, its high word is the same for all.
constexpr uint32_t kOperandHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
CB_D uint32_t operand_low(uint32_t addr) { return ((addr & 0x3ffff) >> 4) | (1u << 16); }

__host__ __device__ constexpr uint32_t product_shape(int n) {
  return (1u << 4) | (uint32_t)(n / 8) << 17 | (uint32_t)(kTileRows / 16) << 24;
}

// d (+)= a b. What the one thread issues has to be in uniform registers: with all
// operands known to be the same for the warp, a product of 16 steps' worth is
// issued in a few cycles, from ordinary registers in about 100 (measured), more
// than it takes to compute.
template <bool ADD>
CB_D void product_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t shape) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 da, db;\nmov.b64 da, {%1, %4};\nmov.b64 db, {%2, %4};\nsetp.ne.u32 p, %5, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}" ::"r"(d), "r"(a), "r"(b), "r"(shape),
      "n"(kOperandHigh), "n"((int)ADD)
      : "memory");
}
CB_D void product_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, uint32_t add) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 db;\nmov.b64 db, {%2, %4};\nsetp.ne.u32 p, %5, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}" ::"r"(d), "r"(a), "r"(b), "r"(shape),
      "n"(kOperandHigh), "r"(add)
      : "memory");
}
CB_D bool elected() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one;
}
// The same value, known to be so for the whole warp.
CB_D uint32_t uniform(uint32_t x) { return __reduce_or_sync(0xffffffffu, x); }

CB_D void tmem_load32(uint32_t addr, float *v) {
  uint32_t *r = reinterpret_cast<uint32_t *>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
CB_D void tmem_store32(uint32_t addr, const float *v) {
  const uint32_t *r = reinterpret_cast<const uint32_t *>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
CB_D void tmem_store16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

CB_D void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
CB_D void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(bar) : "memory"); }

// A warp's arrival, after what all its lanes have done.
CB_D void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) arrive(bar);
}

// A wait of a whole warp, which goes one way for all of it.
CB_D bool warp_wait(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, bar_wait(bar, parity)); }

// Two fp32 values in one 64-bit register.
CB_D uint64_t pair(float x, float y) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
CB_D float2 unpair(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
CB_D uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
CB_D uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}

CB_D float max3(float x, float y, float z) {
  float v;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(x), "f"(y), "f"(z));
  return v;
}

CB_D __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2 *>(&x); }
CB_D uint32_t as_u32(__half2 x) { return *reinterpret_cast<const uint32_t *>(&x); }

// Nibbles k of both halves of a word as code - 8: 0x6400 | c is 1024 + c, and
// 0x6400 | c << 4 is 1024 + 16 c.
CB_D __half2 code_low(uint32_t w) {
  return __hadd2(as_half2((w & 0x000f000fu) | 0x64006400u), __half2half2(__ushort_as_half(0xe408)));  // - 1032
}
CB_D __half2 code_high(uint32_t w) {
  return __hfma2(as_half2((w & 0x00f000f0u) | 0x64006400u), __half2half2(__ushort_as_half(0x2c00)),  // 1/16
                 __half2half2(__ushort_as_half(0xd480)));                                             // - 72
}

// An exponent of all ones in a scale or an offset.
CB_D bool not_finite(uint32_t par) { return (par & 0x7c00) == 0x7c00 || (par >> 16 & 0x7c00) == 0x7c00; }

// The first tokens of [from, to) that have a V which is not finite, for each group, and a K
// (first[NG]): a row sees the tokens below its limit, so that the first decides. It reads the
// pages again, on the way out of an item: with flags of single tokens in the loop over the
// tiles the prompt chunks named above took 674 us instead of 639. A whole warp calls.
template <int D, int NG>
CB_D void first_odd(const Kv4View &c, const AttendArgs &a, const Item &it, int from, int to, int *first) {
#pragma unroll
  for (int gi = 0; gi <= NG; ++gi) first[gi] = 0x7fffffff;
  for (int t = from + (threadIdx.x & 31); t < to; t += 32) {
    const int page = __ldg(a.block_table + it.b * a.table_stride + (t >> c.page_log2));
    if (page < 0 || page >= c.num_pages) continue;
    const uint32_t *p =
        reinterpret_cast<const uint32_t *>(c.base + (uint64_t)page * c.page_stride + (uint64_t)it.h * c.head_bytes +
                                           (t & (c.page_size - 1)) / kKv4Tile * (16 * D + 128 * NG) + 16 * D) +
        t % kKv4Tile * NG;
#pragma unroll
    for (int gi = 0; gi < NG; ++gi) {
      if (not_finite(p[gi])) first[NG] = min(first[NG], t);
      if (not_finite(p[16 * NG + gi])) first[gi] = min(first[gi], t);
    }
  }
#pragma unroll
  for (int gi = 0; gi <= NG; ++gi) first[gi] = __reduce_min_sync(0xffffffffu, first[gi]);
}

// Barriers, 8 bytes each.
enum {
  kFullK = 0,
  kFullV = 2,
  kEmptyK = 4,
  kEmptyV = 6,
  kScores = 8,
  kWeights = 10,
  kQuery = 12,
  kRawBars = 14,
  kBarCount = kRawBars + kDeqWarps * kRaw
};

template <int D, int NG>
__global__ void __launch_bounds__(kPromptThreads, 1) attend_prompt_kernel(const Kv4View c, const AttendArgs a) {
  using F = PromptForm<D, NG>;
  using L = PromptLine;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint32_t tmem_s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t base = smem_addr(smem), bars = base + F::kBars;
  uint32_t *flags = reinterpret_cast<uint32_t *>(smem + F::kFlags);
  const int most = a.columns * c.page_size, piece = blockIdx.x;

  asm volatile("griddepcontrol.launch_dependents;");
  long long share, f0, f1, first;
  Walk w;
  long long *room = reinterpret_cast<long long *>(smem);
  if (!find_piece<L>(a, c, most, room, room + 2 * kPromptWarps, share, f0, f1, first, w.it)) {
    if (threadIdx.x == 0) a.join_how[piece] = kJoinNone;
    return;
  }
  if (warp == kMmaWarp) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        bar_init(bars + 8 * (kFullK + i), kDeqWarps);
        bar_init(bars + 8 * (kFullV + i), kDeqWarps);
        bar_init(bars + 8 * (kEmptyK + i), 1);
        bar_init(bars + 8 * (kEmptyV + i), 1);
        bar_init(bars + 8 * (kScores + i), 1);
        bar_init(bars + 8 * (kWeights + i), kTileRows / 32);
        bar_init(bars + 8 * (kQuery + i), kTileRows / 32);
      }
      for (int i = 0; i < kDeqWarps * kRaw; ++i) bar_init(bars + 8 * (kRawBars + i), 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_s)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  const int units = (int)(f1 - f0);
  w.at = (int)(first - f0) + L::kCost;
  w.cut(units);
  bool more = w.t1 > w.t0 || next_in_piece<L>(a, c.kv_heads, most, units, w);
  bool fine = true;  // no wait ran out
  int how = kJoinNone;

  if (warp < kSoftWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    // -------------------------------------------------------------- softmax
    const int x = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's lanes of tensor memory
    const uint32_t s_at = tmem + lanes + x * kTok, o_at = tmem + lanes + 2 * kTok + x * D;
    uint32_t scores_parity = 0;
    int tile_no = 0;
    bool first_segment = true;
    for (; more && fine; more = next_in_piece<L>(a, c.kv_heads, most, units, w)) {
      const Item &it = w.it;
      const int n = w.t1 - w.t0, total = it.qn * a.ratio, row = it.rt * L::kRows + x * kTileRows + r;
      const bool two = total - it.rt * L::kRows > kTileRows;
      const bool whole = w.t0 == 0 && w.t1 == it.tiles;
      if (x == 0 || two) {
        // ---- this row of Q: fp16 times 2^(14 - e), e the exponent of its largest
        const int64_t at = (int64_t)(it.q0 + min(row, total - 1) / a.ratio) * a.q_token_stride +
                           (int64_t)(it.h * a.ratio + min(row, total - 1) % a.ratio) * a.q_head_stride;
        const uint16_t *src = static_cast<const uint16_t *>(a.q) + at;
        auto load8 = [&](int i) {
          if (a.q_vec) return __ldg(reinterpret_cast<const uint4 *>(src) + i);
          uint32_t y[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = __ldg(src + 8 * i + 2 * k) | (uint32_t)__ldg(src + 8 * i + 2 * k + 1) << 16;
          return make_uint4(y[0], y[1], y[2], y[3]);
        };
        auto two_of = [&](uint32_t v) {
          if (a.bf16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
          return __half22float2(as_half2(v));
        };
        float top = 0.0f;
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
          const uint4 v = load8(i);
          const uint32_t y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = two_of(y[k]);
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 110);
        const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23) * (a.scale < 0.0f ? -1.0f : 1.0f);
        // (never 0: times minus infinity it has to hide)
        const float to_log2 = fmaxf(__uint_as_float((uint32_t)(e - 14 + 127) << 23) * fabsf(a.scale) * kLog2e, 1e-37f);
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
          const uint4 v = load8(i);
          const uint32_t y[4] = {v.x, v.y, v.z, v.w};
          uint32_t z[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = two_of(y[k]);
            z[k] = as_u32(__floats2half2_rn(f.x * up, f.y * up));
          }
          *reinterpret_cast<uint4 *>(smem + F::kQ + x * F::kOperand + (i / 8) * 16384 + r * 128 +
                                     (((i & 7) ^ (r & 7)) << 4)) = make_uint4(z[0], z[1], z[2], z[3]);
        }
        fence_async();
        warp_arrive(bars + 8 * (kQuery + x));

        const int limit = row_limit(a, it, min(row, total - 1));
        float l = 0.0f, over = -INFINITY, sub = 0.0f;
        uint32_t odd = 0;
        for (int j = 0; j < n && fine; ++j) {
          fine = warp_wait(bars + 8 * (kScores + x), scores_parity);
          scores_parity ^= 1;
          tc_fence_after();
          const uint32_t there = flags[(tile_no + j) & 3];
          odd |= there;
          const int visible = limit - (w.t0 + j) * kTok;  // columns below it are seen
          const bool masked = __any_sync(0xffffffffu, visible < kTok) || (there & kAllThere) != kAllThere;
          float v[kTok];
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) tmem_load32(s_at + 32 * ch, v + 32 * ch);
          tc_wait_ld();
          if (masked) {
#pragma unroll
            for (int k = 0; k < kTok; ++k)
              if (k >= visible || !(there >> (8 * (k / 32) + k / 16 % 2) & 1)) v[k] = -INFINITY;
          }
          // ---- the row's largest score
          float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int k = 0; k < kTok; k += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i) tops[i] = max3(tops[i], v[k + 2 * i], v[k + 2 * i + 1]);
          const float top2 = fmaxf(tops[0], tops[1]), top3 = fmaxf(tops[2], tops[3]);
          const float m = fmaxf(top2, top3) * to_log2;
          float f = 1.0f;
          if (m > over) {
            if (over != -INFINITY) f = ex2(sub - m);
            sub = m;
            over = m + kSlack;
          }
          if (j > 0 && __any_sync(0xffffffffu, f != 1.0f)) {
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
              float y[32];
              tmem_load32(o_at + d, y);
              tc_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k) y[k] *= f;
              tmem_store32(o_at + d, y);
            }
          }
          l *= f;
          // ---- weights, P over the columns of S
          const uint64_t by = pair(to_log2, to_log2), minus = pair(-sub, -sub);
          uint64_t sums[2] = {0, 0};
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) {
            uint32_t p[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float2 y = unpair(fma2(pair(v[32 * ch + 2 * k], v[32 * ch + 2 * k + 1]), by, minus));
              const float p0 = ex2(y.x), p1 = ex2(y.y);
              sums[k & 1] = add2(sums[k & 1], pair(p0, p1));
              p[k] = as_u32(__floats2half2_rn(p0, p1));
            }
            tmem_store16(s_at + 16 * ch, p);
          }
          const float2 sum = unpair(add2(sums[0], sums[1]));
          l += sum.x + sum.y;
          tc_wait_st();
          tc_fence_before();
          warp_arrive(bars + 8 * (kWeights + x));
        }
        // ---- out, or a part of it
        if (fine) {
          fine = warp_wait(bars + 8 * (kScores + x), scores_parity);
          scores_parity ^= 1;
          tc_fence_after();
          uint32_t nan_v = 0;  // a bit for each group of which the row sees a V that is not finite
          if (odd & kOdd) {
            int first[NG + 1];
            first_odd<D, NG>(c, a, it, w.t0 * kTok, min(w.t1 * kTok, it.len), first);
            if (first[NG] < limit) l = NAN;
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) nan_v |= (first[gi] < limit ? 1u : 0u) << gi;
          }
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          const int at_row = x * kTileRows + r;
          float *part = a.parts + ((long long)piece * 2 + (first_segment ? 0 : 1)) * F::kPart;
          const int64_t to_row = out_row(a, it, min(row, total - 1));
#pragma unroll 1
          for (int d = 0; d < D; d += 32) {
            float v[32];
            tmem_load32(o_at + d, v);
            tc_wait_ld();
            if (nan_v >> (d / (D / NG)) & 1) {
#pragma unroll
              for (int k = 0; k < 32; ++k) v[k] = NAN;
            }
            if (!whole) {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                reinterpret_cast<float4 *>(part)[(d / 4 + k) * L::kRows + at_row] =
                    make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
            } else if (row < total) {
              uint4 *to = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + to_row * D + d);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                to[k] = make_uint4(pack2(a.bf16, v[8 * k] * inv, v[8 * k + 1] * inv),
                                   pack2(a.bf16, v[8 * k + 2] * inv, v[8 * k + 3] * inv),
                                   pack2(a.bf16, v[8 * k + 4] * inv, v[8 * k + 5] * inv),
                                   pack2(a.bf16, v[8 * k + 6] * inv, v[8 * k + 7] * inv));
            }
          }
          if (!whole) {
            reinterpret_cast<float2 *>(part + L::kRows * D)[at_row] =
                make_float2(over == -INFINITY && l == 0.0f ? -INFINITY : sub, l);
          } else if (row < total && a.lse) {
            a.lse[to_row] = l == 0.0f ? -INFINITY : (sub + log2f(l)) * kLn2;
          }
          tc_fence_before();
        }
      }
      if (w.t0 == 0 && w.t1 < it.tiles) {  // begun here, ended elsewhere
        how = kJoinFew;
        if (threadIdx.x == 0) {
          const int parts = (int)((f0 + w.at + it.tiles - 1) / share) - piece + 1;
          a.joins[piece] = make_int4(it.q0, it.rt, it.h, total);
          a.join_n[piece] = parts * 2 + (first_segment ? 0 : 1);
        }
      }
      first_segment = false;
      tile_no += n;
    }
    if (threadIdx.x == 0) a.join_how[piece] = (uint8_t)how;
  } else if (warp < kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kDeqRegs));
    // --------------------------------------------------------- dequantising
    const int dw = warp - kSoftWarps, g = lane >> 2, t = lane & 3;
    constexpr int kWords = D / 32, kGroupWords = kWords / NG;
    const uint8_t *ring = smem + F::kRing + dw * kRaw * F::kTile;
    const uint32_t ring_at = smem_addr(ring), raw_bars = bars + 8 * (kRawBars + dw * kRaw);
    const int per_page = c.page_log2 - 4;
    // The warp's cache tiles are tokens 32 dw and 32 dw + 16 of every tile. `ahead`
    // fetches them kRaw in advance; the lanes hold the pages of the next 32.
    Walk ahead = w;
    bool a_more = more;
    int a_no = 0, a_i = 0, a_page = -1;  // a_no: in the item's part, two for each tile
    uint32_t a_ok = 0, ok = 0;
    auto ahead_pages = [&]() {
      const int no = a_no + lane, tile = (ahead.t0 + no / 2) * (kTok / kKv4Tile) + dw * 2 + (no & 1);
      a_i = 0;
      a_page = -1;
      if (no < 2 * (ahead.t1 - ahead.t0) && tile * kKv4Tile < ahead.it.len) {
        a_page = __ldg(a.block_table + ahead.it.b * a.table_stride + (tile >> per_page));
        if (a_page < 0 || a_page >= c.num_pages) {
          kv4_error(c.errors, kErrBounds);
          a_page = -1;
        }
      }
      a_ok = __ballot_sync(0xffffffffu, a_page >= 0);
    };
    auto ahead_issue = [&](int stage) {
      if (!a_more) return;
      ok = (ok & ~(1u << stage)) | (a_ok >> a_i & 1u) << stage;
      if (lane == a_i) {
        const int tile = (ahead.t0 + a_no / 2) * (kTok / kKv4Tile) + dw * 2 + (a_no & 1);
        if (a_page >= 0) {
          asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"(raw_bars + 8 * stage), "r"(F::kTile)
                       : "memory");
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                           ring_at + stage * F::kTile),
                       "l"(c.base + (uint64_t)a_page * c.page_stride + (uint64_t)ahead.it.h * c.head_bytes +
                           (uint32_t)((tile & ((1 << per_page) - 1)) * F::kTile)),
                       "r"(F::kTile), "r"(raw_bars + 8 * stage)
                       : "memory");
        } else {
          arrive(raw_bars + 8 * stage);
        }
      }
      ++a_no;
      ++a_i;
      if (a_no == 2 * (ahead.t1 - ahead.t0)) {
        a_more = next_in_piece<L>(a, c.kv_heads, most, units, ahead);
        a_no = 0;
        if (a_more) ahead_pages();
      } else if (a_i == 32) {
        ahead_pages();
      }
    };
    if (a_more) ahead_pages();
    for (int i = 0; i < kRaw; ++i) ahead_issue(i);
    int stage = 0, no = 0;
    uint32_t raw_parity = 0;
    for (; more && fine; more = next_in_piece<L>(a, c.kv_heads, most, units, w)) {
      const Item &it = w.it;
      const int last = min((it.rt + 1) * L::kRows, it.qn * a.ratio) - 1, sees_most = row_limit(a, it, last);
      for (int tl = w.t0; tl < w.t1 && fine; ++tl, ++no) {
        // K of both cache tiles, then V: a buffer of K is free again after the
        // scores, one of V only after the second row tile's values.
        const int half = no & 1, next = stage + 1 == kRaw ? 0 : stage + 1;
        fine = warp_wait(bars + 8 * (kEmptyK + half), (no >> 1 & 1) ^ 1);
        fine = fine && warp_wait(raw_bars + 8 * stage, raw_parity >> stage & 1);
        fine = fine && warp_wait(raw_bars + 8 * next, raw_parity >> next & 1);
        if (!fine) break;
        raw_parity ^= 1u << stage | 1u << next;
        const uint32_t there = (ok >> stage & 1) | (ok >> next & 1) << 1;
        uint8_t *k_to = smem + F::kK + half * F::kOperand, *v_to = smem + F::kV + half * F::kOperand;
        const int tok0 = tl * kTok + dw * 32;
        {  // lane: a token
          const uint32_t *kp = reinterpret_cast<const uint32_t *>(ring + (lane < 16 ? stage : next) * F::kTile + 16 * D) +
                               (lane & 15) * NG;
          bool bad = false;
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) bad |= not_finite(kp[gi]) || not_finite(kp[16 * NG + gi]);
          bad = bad && tok0 + lane < sees_most && (there >> (lane >> 4) & 1);
          const bool any = __any_sync(0xffffffffu, bad);
          if (lane == 0)
            reinterpret_cast<uint8_t *>(flags + (no & 3))[dw] = (uint8_t)(there | (any ? kOdd & 0xffu : 0u));
        }
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
          const uint8_t *buf = ring + (ct ? next : stage) * F::kTile;
          // rows g and g + 8, 8 dims of 32 a word
          uint32_t kw[2][kWords], kp[2][NG];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            load_words<kWords>(buf + (g + 8 * h) * 16 * kWords + t * 4 * kWords, kw[h]);
            load_words<NG>(buf + 16 * D + (g + 8 * h) * NG * 4, kp[h]);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = dw * 32 + ct * 16 + 8 * h + g;
#pragma unroll
            for (int s = 0; s < kWords; ++s) {
              // odd rows take the words of a pair the other way round: no two lanes
              // that store together then meet in a bank
              const bool odd = g & 1;
              const uint32_t wd = odd ? kw[h][s ^ 1] : kw[h][s];
              const int i = odd ? s ^ 1 : s;
              const uint32_t par = NG == kWords && odd ? kp[h][(s ^ 1) / kGroupWords] : kp[h][s / kGroupWords];
              const __half2 sc = __half2half2(__ushort_as_half((unsigned short)(par & 0xffff)));
              const __half2 of = __half2half2(__ushort_as_half((unsigned short)(par >> 16)));
              uint4 y;
              y.x = as_u32(__hfma2(code_low(wd), sc, of));
              y.y = as_u32(__hfma2(code_high(wd), sc, of));
              y.z = as_u32(__hfma2(code_low(wd >> 8), sc, of));
              y.w = as_u32(__hfma2(code_high(wd >> 8), sc, of));
              *reinterpret_cast<uint4 *>(k_to + (i >> 1) * 16384 + row * 128 + ((((i & 1) * 4 + t) ^ (row & 7)) << 4)) = y;
            }
          }
        }
        fence_async();
        warp_arrive(bars + 8 * (kFullK + half));
        fine = warp_wait(bars + 8 * (kEmptyV + half), (no >> 1 & 1) ^ 1);
        if (!fine) break;
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
          const uint8_t *buf = ring + (ct ? next : stage) * F::kTile;
          // token pairs 8 h + 2t, 4 dims a word
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t vw[kWords], vp[2 * NG];
            load_words<kWords>(buf + 8 * D + (h * 32 + lane) * 4 * kWords, vw);
            load_words<2 * NG>(buf + 16 * D + 64 * NG + (8 * h + 2 * t) * NG * 4, vp);
            const int tok = tok0 + ct * 16 + 8 * h + 2 * t;
            const bool on0 = (there >> ct & 1) && tok < sees_most, on1 = (there >> ct & 1) && tok + 1 < sees_most;
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
              uint32_t p0 = vp[gi], p1 = vp[NG + gi];
              if (!on0 || not_finite(p0)) p0 = 0;
              if (!on1 || not_finite(p1)) p1 = 0;
              const __half2 sc = as_half2(__byte_perm(p0, p1, 0x5410)), of = as_half2(__byte_perm(p0, p1, 0x7632));
#pragma unroll
              for (int j = gi * kGroupWords; j < (gi + 1) * kGroupWords; ++j) {
                uint32_t y[4];
                y[0] = as_u32(__hfma2(code_low(vw[j]), sc, of));
                y[1] = as_u32(__hfma2(code_high(vw[j]), sc, of));
                y[2] = as_u32(__hfma2(code_low(vw[j] >> 8), sc, of));
                y[3] = as_u32(__hfma2(code_high(vw[j] >> 8), sc, of));
                const int chunk = (dw & 1) * 4 + ct * 2 + h;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  *reinterpret_cast<uint32_t *>(v_to + (dw >> 1) * (D * 128) + (32 * j + 8 * k + g) * 128 +
                                                ((chunk ^ g) << 4) + 4 * t) = y[k];
              }
            }
          }
          __syncwarp();
          ahead_issue(ct ? next : stage);
        }
        fence_async();
        warp_arrive(bars + 8 * (kFullV + half));
        stage = next + 1 == kRaw ? 0 : next + 1;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs));
    // --------------------------------------------------------- the products
    more = more && warp == kMmaWarp;
    constexpr uint32_t kShapeS = product_shape(kTok), kShapeO = product_shape(D);
    const uint32_t tm = uniform(tmem), at = uniform(base);
    uint32_t weights_parity[2] = {0, 0}, query_parity[2] = {0, 0};
    int no = 0;  // tile of the piece
    auto scores = [&](int x, int half, bool release) {
      tc_fence_after();
      if (elected()) {
        const uint32_t qa = operand_low(at + F::kQ + x * F::kOperand), kb = operand_low(at + F::kK + half * F::kOperand);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k / 4) * 16384 + (k % 4) * 32) >> 4;
          if (k == 0) product_ss<false>(tm + x * kTok, qa, kb, kShapeS);
          else product_ss<true>(tm + x * kTok, qa + off, kb + off, kShapeS);
        }
        tc_commit(bars + 8 * (kScores + x));
        if (release) tc_commit(bars + 8 * (kEmptyK + half));
      }
      __syncwarp();
    };
    auto values = [&](int x, int half, bool add, bool release) {
      tc_fence_after();
      if (elected()) {
        const uint32_t vb = operand_low(at + F::kV + half * F::kOperand);
#pragma unroll
        for (int k = 0; k < kTok / 16; ++k)
          product_ts(tm + 2 * kTok + x * D, tm + x * kTok + 8 * k, vb + (((k / 4) * (D * 128) + (k % 4) * 32) >> 4),
                     kShapeO, k > 0 ? 1u : (uint32_t)add);
        if (release) tc_commit(bars + 8 * (kEmptyV + half));
      }
      __syncwarp();
    };
    for (; more && fine; more = next_in_piece<L>(a, c.kv_heads, most, units, w)) {
      const int n = (int)uniform(w.t1 - w.t0);
      const int tiles = uniform(w.it.qn * a.ratio - w.it.rt * L::kRows > kTileRows) ? 2 : 1;  // of rows
      fine = fine && warp_wait(bars + 8 * (kFullK + (no & 1)), no >> 1 & 1);
      for (int x = 0; x < tiles && fine; ++x) {
        fine = warp_wait(bars + 8 * (kQuery + x), query_parity[x]);
        query_parity[x] ^= 1;
        if (fine) scores(x, no & 1, x == tiles - 1);
      }
      for (int j = 0; j < n && fine; ++j, ++no) {
        const int half = no & 1, next = (no + 1) & 1;
        for (int x = 0; x < tiles && fine; ++x) {
          fine = warp_wait(bars + 8 * (kWeights + x), weights_parity[x]);
          weights_parity[x] ^= 1;
          if (x == 0) fine = fine && warp_wait(bars + 8 * (kFullV + half), no >> 1 & 1);
          if (!fine) break;
          values(x, half, j > 0, x == tiles - 1);
          if (j + 1 < n) {
            if (x == 0) fine = warp_wait(bars + 8 * (kFullK + next), (no + 1) >> 1 & 1);
            if (fine) scores(x, next, x == tiles - 1);
          } else {
            if (elected()) tc_commit(bars + 8 * (kScores + x));  // O is complete
            __syncwarp();
          }
        }
      }
    }
  }
  if (!fine) {
    kv4_error(c.errors, kErrTimeout);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // what was issued comes to its end
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

// Joins the parts of items that a block began and did not end: block (piece, i) does
// rows 32 i .. 32 i + 31 of them, a lane to a row, parts in order.
template <int D>
__global__ void __launch_bounds__(256) prompt_join_kernel(const AttendArgs a) {
  using L = PromptLine;
  constexpr int kPart = L::kRows * (D + 2), kMine = D / 32;  // 4-dim pieces of a thread
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, piece = blockIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (a.join_how[piece] == kJoinNone) return;
  const int4 join = a.joins[piece];
  Item it;
  it.q0 = join.x, it.rt = join.y, it.h = join.z;
  const int r = blockIdx.y * 32 + lane, row = it.rt * L::kRows + r;
  if (it.rt * L::kRows + (int)blockIdx.y * 32 >= join.w) return;
  const int places = a.join_n[piece], parts = places >> 1;
  const float *base = a.parts + (long long)piece * 2 * kPart;
  float m = -INFINITY, l = 0.0f;
  float4 x[kMine];
#pragma unroll
  for (int k = 0; k < kMine; ++k) x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i = 0; i < parts; ++i) {
    const float *from = base + (long long)i * 2 * kPart + (i ? 0 : (places & 1) * kPart);
    const float2 ml = reinterpret_cast<const float2 *>(from + L::kRows * D)[r];
    const float top = fmaxf(m, ml.x), at = top == -INFINITY ? 0.0f : top;
    const float f = ex2(m - at), fi = ex2(ml.x - at);
    m = top;
    l = l * f + ml.y * fi;
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const float4 v = reinterpret_cast<const float4 *>(from)[(warp * kMine + k) * L::kRows + r];
      x[k].x = x[k].x * f + v.x * fi, x[k].y = x[k].y * f + v.y * fi;
      x[k].z = x[k].z * f + v.z * fi, x[k].w = x[k].w * f + v.w * fi;
    }
  }
  if (row >= join.w) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t to = out_row(a, it, row);
  uint2 *out = reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + to * D + warp * kMine * 4);
#pragma unroll
  for (int k = 0; k < kMine; ++k)
    out[k] = make_uint2(pack2(a.bf16, x[k].x * inv, x[k].y * inv), pack2(a.bf16, x[k].z * inv, x[k].w * inv));
  if (a.lse && warp == 0) a.lse[to] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <int D, int NG>
cudaError_t launch(const Kv4View &c, const AttendArgs &a, const Launch &l, cudaStream_t stream) {
  using F = PromptForm<D, NG>;
  static_assert(F::kSmem <= 227 * 1024 && kBarCount * 8 <= 256, "shared memory");
  static std::atomic<uint64_t> ready{0};  // a bit for each device
  cudaError_t e = allow_shared(attend_prompt_kernel<D, NG>, F::kSmem, ready);
  if (e != cudaSuccess) return e;
  e = kv4_launch(attend_prompt_kernel<D, NG>, dim3(l.pieces), kPromptThreads, F::kSmem, stream, false, c, a);
  if (e != cudaSuccess) return e;
  return kv4_launch(prompt_join_kernel<D>, dim3(l.pieces, PromptLine::kRows / 32), 256, 0, stream, true, a);
}

}  // namespace

Launch prompt_launch(int head_dim, int sms) {
  Launch l;
  l.sms = l.pieces = sms;
  l.rows = PromptLine::kRows;
  l.part = l.rows * (head_dim + 2);
  return l;
}

cudaError_t run_prompt(const Kv4View &c, const AttendArgs &a, int head_dim, int group, const Launch &l,
                       cudaStream_t stream) {
  const int ng = head_dim / group;
  if (head_dim == 64) return ng == 1 ? launch<64, 1>(c, a, l, stream) : launch<64, 2>(c, a, l, stream);
  if (ng == 1) return launch<128, 1>(c, a, l, stream);
  return ng == 2 ? launch<128, 2>(c, a, l, stream) : launch<128, 4>(c, a, l, stream);
}

}  // namespace cb
