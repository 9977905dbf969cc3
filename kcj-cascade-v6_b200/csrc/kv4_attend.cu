// Attention over a paged KV cache held in 4 bits (cb_kv4_attend). Format:
// kv4.cuh.
//
//   out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q.k_t - max)
//
// in one pass over a row's tokens with the running maximum and sum.
#include "kv4_attend.cuh"

namespace cb {

namespace {

// Row tiles of 8*NT rows (query row x query head of one KV head), tokens in
// tiles of 16, a piece of the line (kv4_attend.cuh) for every WARP: warps share
// nothing and never wait for one another. (With a piece for every block, whose
// warps met at each item's end, 61 ragged requests took 53 us instead of 49.) An
// item that ends up in several warps leaves partial sums in the workspace, joined
// by a second kernel in a fixed order.
//
// Tensor-core form (16x8x16, fp16 in, fp32 sums): the cache is the 16-row
// operand of both products and the 8*NT query rows the 8-wide one, so that the
// at most 8 or 16 query heads of a KV head do not leave half of a product
// empty:
//   S[token][row]  = K[token][dim] . Q[dim][row]
//   O[dim][row]   += V[dim][token] . P[token][row]
// Both operands of the cache are raw codes: a nibble under a mask is the fp16
// subnormal code * 2^-24 (second nibble: * 2^-20, undone in Q, or in O's rows),
// exact, with no conversion. Scales and offsets act on 16x8 scores instead of
// 16xD values: s = scale_k (q.c) + (offset_k - 8 scale_k) sum(q), and V's scale
// goes into P, p' = p * scale_v, its offset into a sum of p * offset_v - 8 p'.
// So the only roundings to 16 bits are p' (relative 2^-11, and 2^-25 of the largest for
// what is far below it; its rounded value is the one that the centring by 8
// uses) and the output. For an fp16 output that is an error of 2.4 to 3.1e-4 where
// the output's rounding alone makes 2.1e-4; the rest of p' as a second operand would
// take it away for 10 % of the time, and 4-bit values are off by hundreds of
// times as much. q is brought to fp16 by a power of two per row: exact for fp16 and,
// above 2^-28 of the row's largest, for bf16 (from 2^111 on it counts as infinite).
//
// Bound by HBM where the tokens are many: 1 + 8/group bytes for a cached value pair
// of K and V. Measured (replayed in a CUDA graph): 48 requests of 9,000 to 32,000
// tokens, 64 / 8 heads of 128, group 128: 216 us, 5.0 TB/s; the rest of the way is instructions (266 for a tile
// of 16 tokens, 16 of them products and 80 the unpacking, at 0.6 an SM quarter and
// cycle). A single short request is bound by latency: 10.9 us for 1,100 tokens.
// mma.sync and not tcgen05: its operands come from registers, where the codes become
// them with one instruction for two values, and 8 rows leave 15/16 of a 128-row
// product empty; kv4_prompt.cu has the rows for that.
constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kRecentre = 4;      // pairs of tiles between centrings of the sums
constexpr int kManyParts = 24;    // parts of an item that a warp joins alone
// What an item costs a warp beside its tiles (query rows in, results out), in
// tiles: it takes this much of the line too.
// (130 requests of up to 3,000 tokens, 64 dims: 66 us with 3, 59 with 5 or 8.)
constexpr int kItemCost = 8;
constexpr int kJoinWarps = 8, kJoinThreads = kJoinWarps * 32;

template <int D, int NG, int NT>
struct Form {
  static constexpr int kRows = 8 * NT;
  static constexpr int kTile = 16 * D + 128 * NG;   // bytes
  static constexpr int kSlabs = D > 128 ? 2 : 1;
  static constexpr int kWpr = D / kSlabs / 32;      // words a lane reads of a row and slab
  static constexpr int kWords = D / 32;
  static constexpr int kGroupWords = kWords / NG;
  // A warp's ring is two pairs of tiles. Bytes in flight: 8 or 16 warps with 2 to 4
  // tiles of 1.2 - 5.1 KB are 35 KB and more on an SM; HBM needs about
  // 6.5 TB/s * 0.8 us / 148 = 35 KB. Products of two tiles side by side (kJoint)
  // hide each other's latency where registers allow: 275 us without, 220 with, on
  // the 48 long requests.
  static constexpr int kJoint = NT == 1 ? 2 : 1;  // tiles whose products run side by side
  static constexpr int kCtasPerSm = NT == 1 && D <= 128 ? 2 : 1;
  static constexpr int kRing = 4 * kTile;           // of a warp, as are the next two
  static constexpr int kQ = NT * (D / 16) * 32 * 8;
  static constexpr int kConst = kRows * (2 + NG) * 4;
  static constexpr int kWarp = (kRing + kQ + kConst + 16 + 127) / 128 * 128;
  static constexpr int kSmem = kWarps * kWarp;
  static constexpr int kStatic = (2 * kWarps + kThreads) * (int)sizeof(long long);  // of find_piece
  static constexpr int kPart = kRows * (D + 2);     // floats of a partial result
  struct Line {
    static constexpr int kRows = 8 * NT, kTokens = kKv4Tile, kCost = kItemCost, kWarps = cb::kWarps;
    static constexpr bool kBlock = false;
  };
};

CB_D void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

CB_D void mma(float *c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

CB_D uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// A load that stays where it is written, before what waits for it.
CB_D float4 load_now(const float *p) {
  float4 v;
  asm volatile("ld.global.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
  return v;
}

template <int D, int NG, int NT>
__global__ void __launch_bounds__(kThreads, Form<D, NG, NT>::kCtasPerSm)
    attend_few_kernel(const Kv4View c, const AttendArgs a) {
  using F = Form<D, NG, NT>;
  using L = typename F::Line;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint8_t *ring = smem + warp * F::kWarp;
  uint2 *qs = reinterpret_cast<uint2 *>(smem + warp * F::kWarp + F::kRing);
  float *q_scale = reinterpret_cast<float *>(smem + warp * F::kWarp + F::kRing + F::kQ);
  int *limits = reinterpret_cast<int *>(q_scale + F::kRows);
  float *q_sum = reinterpret_cast<float *>(limits + F::kRows);  // [NG][rows]
  const uint32_t ring_at = smem_addr(ring);
  const uint32_t bars = ring_at + F::kRing + F::kQ + F::kConst;
  const int most = a.columns * c.page_size;
  const int per_page = c.page_log2 - 4;
  const int piece = warp * gridDim.x + blockIdx.x;

  asm volatile("griddepcontrol.launch_dependents;");
  if (lane == 0) {
    bar_init(bars, 2);  // two lanes arrive, one for each tile
    bar_init(bars + 8, 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  long long share, f0, f1, first;
  Walk w;
  __shared__ long long sums[2 * kWarps], ends[kThreads];
  if (!find_piece<L>(a, c, most, sums, ends, share, f0, f1, first, w.it)) {
    if (lane == 0) a.join_how[piece] = kJoinNone;
    return;
  }
  const int units = (int)(f1 - f0);
  w.at = (int)(first - f0) + L::kCost;
  w.cut(units);
  bool more = w.t1 > w.t0 || next_in_piece<L>(a, c.kv_heads, most, units, w);

  // `ahead` runs two pairs of tiles before the products; the lanes hold the pages of
  // the next 16 pairs of the item, and a pair's two lanes fetch its tiles, whose
  // presence is in `ok`.
  Walk ahead = w;
  int a_tile = w.t0, a_i = 0, a_page = -1;
  uint32_t a_ok = 0, ok = 0;                // ok: two bits for each half of the ring
  bool a_more = more;
  auto ahead_pages = [&]() {
    const int tile = a_tile + lane;
    a_i = 0;
    a_page = -1;
    if (tile < ahead.t1 && tile * kKv4Tile < ahead.it.len) {  // else none, or a row tile that sees nothing
      a_page = __ldg(a.block_table + ahead.it.b * a.table_stride + (tile >> per_page));
      if (a_page < 0 || a_page >= c.num_pages) {
        kv4_error(c.errors, kErrBounds);
        a_page = -1;
      }
    }
    a_ok = __ballot_sync(0xffffffffu, a_page >= 0);
  };
  auto ahead_issue = [&](int half) {
    if (!a_more) return;
    ok = half ? (ok & 3u) | (a_ok >> a_i & 3u) << 2 : (ok & 12u) | (a_ok >> a_i & 3u);
    const int j = lane - a_i;
    if (j == 0 || j == 1) {
      const uint32_t bar = bars + 8 * half;
      if (a_page >= 0) {
        bulk_load(ring_at + (2 * half + j) * F::kTile,
                  c.base + (uint64_t)a_page * c.page_stride + (uint64_t)ahead.it.h * c.head_bytes +
                      (uint32_t)(((a_tile + j) & ((1 << per_page) - 1)) * F::kTile),
                  F::kTile, bar);
      } else {
        asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(bar) : "memory");
      }
    }
    a_tile += 2;
    a_i += 2;
    if (a_tile >= ahead.t1) {
      a_more = next_in_piece<L>(a, c.kv_heads, most, units, ahead);
      a_tile = ahead.t0;
      if (a_more) ahead_pages();
    } else if (a_i == 32) {
      ahead_pages();
    }
  };
  if (a_more) ahead_pages();
  ahead_issue(0);
  ahead_issue(1);

  int half = 0;
  uint32_t parity = 0;
  int how = kJoinNone;
  bool first_segment = true;
  for (; more; more = next_in_piece<L>(a, c.kv_heads, most, units, w)) {
    const Item &it = w.it;
    const int rows = min(F::kRows, it.qn * a.ratio - it.rt * F::kRows);
    // ---- the query rows as operands: fp16, their scale, their sums by group.
    // A lane holds 8 dims of 32 of row g of each n-tile.
    __syncwarp();
#pragma unroll 1
    for (int n = 0; n < NT; ++n) {
      const int row = it.rt * F::kRows + n * 8 + g;
      uint32_t x[F::kWords][4];
      if (n * 8 + g < rows) {
        const uint16_t *src = static_cast<const uint16_t *>(a.q) + (int64_t)(it.q0 + row / a.ratio) * a.q_token_stride +
                              (int64_t)(it.h * a.ratio + row % a.ratio) * a.q_head_stride + 8 * t;
        if (a.q_vec) {
#pragma unroll
          for (int i = 0; i < F::kWords; ++i) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(src + 32 * i));
            x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < F::kWords; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              x[i][k] = __ldg(src + 32 * i + 2 * k) | (uint32_t)__ldg(src + 32 * i + 2 * k + 1) << 16;
        }
      } else {
#pragma unroll
        for (int i = 0; i < F::kWords; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) x[i][k] = 0;
      }
      auto two = [&](uint32_t v) {
        if (a.bf16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
        return __half22float2(*reinterpret_cast<const __half2 *>(&v));
      };
      float top = 0.0f, sum[NG];
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) sum[gi] = 0.0f;
#pragma unroll
      for (int i = 0; i < F::kWords; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 v = two(x[i][k]);
          top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          sum[i / F::kGroupWords] += v.x + v.y;
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^(14 - e) with e the exponent of the largest; powers of two are exact
      const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 110);
      const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
      const float down = __uint_as_float((uint32_t)(14 - 24 - e + 127) << 23);
#pragma unroll
      for (int i = 0; i < F::kWords; ++i) {
        uint32_t y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 v = two(x[i][k]);
          const float f = k & 1 ? up * 0.0625f : up;
          const __half2 hv = __floats2half2_rn(v.x * f, v.y * f);
          y[k] = *reinterpret_cast<const uint32_t *>(&hv);
        }
        qs[(n * (D / 16) + 2 * i) * 32 + lane] = make_uint2(y[0], y[1]);
        qs[(n * (D / 16) + 2 * i + 1) * 32 + lane] = make_uint2(y[2], y[3]);
      }
#pragma unroll
      for (int gi = 0; gi < NG; ++gi) {
        sum[gi] += __shfl_xor_sync(0xffffffffu, sum[gi], 1);
        sum[gi] += __shfl_xor_sync(0xffffffffu, sum[gi], 2);
        if (t == 0) q_sum[gi * F::kRows + n * 8 + g] = sum[gi] * down;
      }
      if (t == 0) {
        q_scale[n * 8 + g] = __uint_as_float((uint32_t)(24 - 14 + e + 127) << 23) * a.scale * kLog2e;
        limits[n * 8 + g] = row_limit(a, it, min(row, it.qn * a.ratio - 1));
      }
    }
    __syncwarp();
    // The tile loop asks shared memory for these only where registers are short.
    constexpr bool kCache = NT * NG <= 2;
    float2 qa_[kCache ? NT : 1], qb_[kCache ? NT : 1][NG];
    auto q_scales = [&](int n) { return *reinterpret_cast<const float2 *>(q_scale + n * 8 + 2 * t); };
    auto q_sums = [&](int n, int gi) { return *reinterpret_cast<const float2 *>(q_sum + gi * F::kRows + n * 8 + 2 * t); };
    if constexpr (kCache) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        qa_[n] = q_scales(n);
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) qb_[n][gi] = q_sums(n, gi);
      }
    }
    const int sees_least = limits[0], sees_most = limits[F::kRows - 1];

    // z: sum of p * offset_v - 8 p', p' as rounded
    float o[D / 16][NT][4], z[NT][2][NG], l[NT][2], over[NT][2], sub[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][n][e] = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[n][h] = 0.0f;
        over[n][h] = -INFINITY;  // the running maximum plus kSlack
        sub[n][h] = 0.0f;        // the running maximum, 0 before there is one
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) z[n][h][gi] = 0.0f;
      }
    }
    auto recentre = [&]() {  // o += z, summed over the lanes that share a row
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            float x = z[n][h][gi];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            z[n][h][gi] = 0.0f;
#pragma unroll
            for (int i = gi * F::kGroupWords * 2; i < (gi + 1) * F::kGroupWords * 2; ++i) {
              o[i][n][h] = fmaf(x, 0x1p-24f, o[i][n][h]);
              o[i][n][2 + h] = fmaf(x, 0x1p-20f, o[i][n][2 + h]);
            }
          }
    };

    int since = 0;
#pragma unroll 1
    for (int tile0 = w.t0; tile0 < w.t1; tile0 += 2) {
      if (!__all_sync(0xffffffffu, bar_wait(bars + 8 * half, parity >> half & 1))) {
        // The results are void. The other half's copies are given their time to end.
        kv4_error(c.errors, kErrTimeout);
        bar_wait(bars + 8 * (half ^ 1), parity >> (half ^ 1) & 1);
        if (lane == 0) a.join_how[piece] = kJoinNone;
        return;
      }
      parity ^= 1u << half;
      const uint32_t there = ok >> (2 * half) & 3u;
      constexpr int J = F::kJoint;
#pragma unroll 1
      for (int j0 = 0; j0 < 2; j0 += J) {
        const uint8_t *buf = ring + (2 * half + j0) * F::kTile;
        // ---- scores
        float s[J][NT][4];
        uint32_t par[J][2][NG];
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
          for (int h = 0; h < 2; ++h) load_words<NG>(buf + j * F::kTile + 16 * D + (g + 8 * h) * NG * 4, par[j][h]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][n][e] = 0.0f;
        }
        uint32_t w0[J][F::kWpr], w1[J][F::kWpr];
        float acc[J][NT][4];
#pragma unroll
        for (int i = 0; i < F::kWords; ++i) {
          if (i % F::kWpr == 0) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
              const uint8_t *p =
                  buf + j * F::kTile + (i / F::kWpr) * 16 * 16 * F::kWpr + g * 16 * F::kWpr + t * 4 * F::kWpr;
              load_words<F::kWpr>(p, w0[j]);
              load_words<F::kWpr>(p + 8 * 16 * F::kWpr, w1[j]);
            }
          }
          if (i % F::kGroupWords == 0) {
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[j][n][e] = 0.0f;
          }
#pragma unroll
          for (int hw = 0; hw < 2; ++hw) {
            uint2 b[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              b[n] = qs[(n * (D / 16) + 2 * i + hw) * 32 + lane];
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
              const uint32_t x = w0[j][i % F::kWpr] >> (8 * hw), y = w1[j][i % F::kWpr] >> (8 * hw);
              const uint32_t a0 = x & 0x000f000fu, a1 = y & 0x000f000fu, a2 = x & 0x00f000f0u, a3 = y & 0x00f000f0u;
#pragma unroll
              for (int n = 0; n < NT; ++n) mma(acc[j][n], a0, a1, a2, a3, b[n].x, b[n].y);
            }
          }
          if (i % F::kGroupWords == F::kGroupWords - 1) {
            const int gi = i / F::kGroupWords;
#pragma unroll
            for (int j = 0; j < J; ++j) {
              const float s0 = kv4_scale(par[j][0][gi]), s1 = kv4_scale(par[j][1][gi]);
              const float b0 = fmaf(-8.0f, s0, kv4_offset(par[j][0][gi]));
              const float b1 = fmaf(-8.0f, s1, kv4_offset(par[j][1][gi]));
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float2 qb;
                if constexpr (kCache) qb = qb_[n][gi];
                else qb = q_sums(n, gi);
                s[j][n][0] = fmaf(s0, acc[j][n][0], fmaf(b0, qb.x, s[j][n][0]));
                s[j][n][1] = fmaf(s0, acc[j][n][1], fmaf(b0, qb.y, s[j][n][1]));
                s[j][n][2] = fmaf(s1, acc[j][n][2], fmaf(b1, qb.x, s[j][n][2]));
                s[j][n][3] = fmaf(s1, acc[j][n][3], fmaf(b1, qb.y, s[j][n][3]));
              }
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float2 qa;
          if constexpr (kCache) qa = qa_[n];
          else qa = q_scales(n);
#pragma unroll
          for (int j = 0; j < J; ++j)
            s[j][n][0] *= qa.x, s[j][n][1] *= qa.y, s[j][n][2] *= qa.x, s[j][n][3] *= qa.y;
        }
        // ---- V: everything leaves the ring here, so that the next pair may come in
        uint32_t vpar[J][2][NG], vw[J][2][F::kWords];
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint8_t *p = buf + j * F::kTile;
            load_words<NG>(p + 16 * D + 64 * NG + (g + 8 * h) * NG * 4, vpar[j][h]);
#pragma unroll
            for (int sl = 0; sl < F::kSlabs; ++sl)
              load_words<F::kWpr>(p + 8 * D + ((sl * 2 + h) * 32 + lane) * 4 * F::kWpr, vw[j][h] + sl * F::kWpr);
          }
        const int tile = tile0 + j0;
        if (j0 + J == 2) {
          __syncwarp();
          ahead_issue(half);
        }

        // ---- weights. Rows of tokens t0 + g and t0 + g + 8 of each tile.
        const bool partial = (tile + J) * kKv4Tile > sees_least || (there >> j0) != (J == 2 ? 3u : 3u >> j0);
        if (partial) {
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const int tok = (there >> (j0 + j) & 1) ? (tile + j) * kKv4Tile + g : 0x7fffff00;  // a tile not there
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int2 lim = *reinterpret_cast<const int2 *>(limits + n * 8 + 2 * t);
              s[j][n][0] = tok < lim.x ? s[j][n][0] : -INFINITY;
              s[j][n][1] = tok < lim.y ? s[j][n][1] : -INFINITY;
              s[j][n][2] = tok + 8 < lim.x ? s[j][n][2] : -INFINITY;
              s[j][n][3] = tok + 8 < lim.y ? s[j][n][3] : -INFINITY;
            }
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) {
              if (tok >= sees_most) vpar[j][0][gi] = 0;
              if (tok + 8 >= sees_most) vpar[j][1][gi] = 0;
            }
          }
        }
        // p' = p * scale_v stays near 1 if the maximum is taken over s + log2
        // scale_v (its exponent; a subnormal scale counts as 2^-15). One that is not
        // finite wraps to 0, or it would cost the other groups' weights their bits.
        float ev[J][2];
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t top = 0;
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) top = max(top, (vpar[j][h][gi] << 17) + (1u << 27));
            ev[j][h] = (float)((int)(top >> 27) - 16);
          }
        float high[NT][2];
        bool raise = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            high[n][h] = fmaxf(s[0][n][h] + ev[0][0], s[0][n][2 + h] + ev[0][1]);
            if (J == 2)
              high[n][h] = fmaxf(high[n][h], fmaxf(s[J - 1][n][h] + ev[J - 1][0], s[J - 1][n][2 + h] + ev[J - 1][1]));
            raise |= high[n][h] > over[n][h];
          }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float m = high[n][h];
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
              const bool fresh = over[n][h] == -INFINITY;
              if (!(m > over[n][h])) continue;  // a row goes by its own scores; a NaN is no maximum
              const float f = fresh ? 1.0f : ex2(sub[n][h] - m);
              sub[n][h] = m;
              over[n][h] = m + kSlack;
              l[n][h] *= f;
#pragma unroll
              for (int gi = 0; gi < NG; ++gi) z[n][h][gi] *= f;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) {
                o[i][n][h] *= f;
                o[i][n][2 + h] *= f;
              }
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[j][n][e] = ex2(s[j][n][e] - sub[n][e & 1]);
              l[n][e & 1] += s[j][n][e];
            }
        // ---- O += V P'
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            const float s0 = kv4_scale(vpar[j][0][gi]), s1 = kv4_scale(vpar[j][1][gi]);
            const float y0 = kv4_offset(vpar[j][0][gi]), y1 = kv4_offset(vpar[j][1][gi]);
            uint32_t b[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float *p = s[j][n];
              float p0 = p[0] * s0, p1 = p[1] * s0, p2 = p[2] * s1, p3 = p[3] * s1;
              if (partial) {  // a hidden token's parameters are nothing; a weight of 0 beside a NaN is NaN
                const int2 lim = *reinterpret_cast<const int2 *>(limits + n * 8 + 2 * t);
                const int tok = (tile + j) * kKv4Tile + g;
                if (tok < lim.x) z[n][0][gi] = fmaf(p[0], y0, z[n][0][gi]);
                else p0 = 0.0f;
                if (tok < lim.y) z[n][1][gi] = fmaf(p[1], y0, z[n][1][gi]);
                else p1 = 0.0f;
                if (tok + 8 < lim.x) z[n][0][gi] = fmaf(p[2], y1, z[n][0][gi]);
                else p2 = 0.0f;
                if (tok + 8 < lim.y) z[n][1][gi] = fmaf(p[3], y1, z[n][1][gi]);
                else p3 = 0.0f;
              } else {
                z[n][0][gi] = fmaf(p[0], y0, fmaf(p[2], y1, z[n][0][gi]));
                z[n][1][gi] = fmaf(p[1], y0, fmaf(p[3], y1, z[n][1][gi]));
              }
              const __half2 h0 = __floats2half2_rn(p0, p1), h1 = __floats2half2_rn(p2, p3);
              b[n][0] = transpose8(*reinterpret_cast<const uint32_t *>(&h0));
              b[n][1] = transpose8(*reinterpret_cast<const uint32_t *>(&h1));
              const float2 r0 = __half22float2(h0), r1 = __half22float2(h1);
              z[n][0][gi] = fmaf(-8.0f, r0.x + r1.x, z[n][0][gi]);
              z[n][1][gi] = fmaf(-8.0f, r0.y + r1.y, z[n][1][gi]);
            }
#pragma unroll
            for (int i = gi * F::kGroupWords; i < (gi + 1) * F::kGroupWords; ++i)
#pragma unroll
              for (int hw = 0; hw < 2; ++hw) {
                const uint32_t x = vw[j][0][i] >> (8 * hw), y = vw[j][1][i] >> (8 * hw);
                const uint32_t a0 = x & 0x000f000fu, a1 = x & 0x00f000f0u, a2 = y & 0x000f000fu, a3 = y & 0x00f000f0u;
#pragma unroll
                for (int n = 0; n < NT; ++n) mma(o[2 * i + hw][n], a0, a1, a2, a3, b[n][0], b[n][1]);
              }
          }
      }
      // Codes are sums around 7.5 scale until they are centred; the tensor cores
      // cut low bits off a sum, which would add up over a long row.
      if (++since == kRecentre) {
        recentre();
        since = 0;
      }
      half ^= 1;
    }
    recentre();

    // ---- out: the result of an item that is all here, else a part of it
    const bool whole = w.t0 == 0 && w.t1 == it.tiles;
    float *part = a.parts + ((long long)piece * 2 + (first_segment ? 0 : 1)) * F::kPart;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float inv[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = l[n][h];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        inv[h] = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int r = n * 8 + 2 * t + h;
        if (g == 0 && whole) {
          if (a.lse && r < rows)
            a.lse[out_row(a, it, it.rt * F::kRows + r)] = sum == 0.0f ? -INFINITY : (sub[n][h] + log2f(sum)) * kLn2;
        } else if (g == 0) {
          reinterpret_cast<float2 *>(part + F::kRows * D)[r] =
              make_float2(over[n][h] == -INFINITY && sum == 0.0f ? -INFINITY : sub[n][h], sum);
        }
      }
      if (!whole) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          reinterpret_cast<float4 *>(part)[(n * (D / 16) + i) * 32 + lane] =
              make_float4(o[i][n][0], o[i][n][1], o[i][n][2], o[i][n][3]);
      } else {
        // lanes g and g ^ 1 exchange, so that each stores two adjacent dims of one row
        const int r = n * 8 + 2 * t + (g & 1);
        uint32_t *to = static_cast<uint32_t *>(a.out) +
                       (out_row(a, it, it.rt * F::kRows + min(r, rows - 1)) * D + (g & 6)) / 2;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f = e ? 0x1p20f : 0x1p24f;
            const float x = o[i][n][2 * e] * f * inv[0], y = o[i][n][2 * e + 1] * f * inv[1];
            const float got = __shfl_xor_sync(0xffffffffu, g & 1 ? x : y, 4);
            if (r < rows) to[(16 * i + 8 * e) / 2] = g & 1 ? pack2(a.bf16, got, y) : pack2(a.bf16, x, got);
          }
      }
    }
    if (w.t0 == 0 && w.t1 < it.tiles) {  // begun here, ended elsewhere
      const int parts = (int)((f0 + w.at + it.tiles - 1) / share) - piece + 1;
      how = parts > kManyParts ? kJoinMany : kJoinFew;
      if (lane == 0) {
        a.joins[piece] = make_int4(it.q0, it.rt, it.h, it.qn * a.ratio);
        a.join_n[piece] = parts * 2 + (first_segment ? 0 : 1);
      }
    }
    first_segment = false;
  }
  if (lane == 0) a.join_how[piece] = (uint8_t)how;
}

// Rows of no request: zeros, and a log-sum-exp of -inf. They are before the first request's
// rows or behind the last one's.
template <int D>
CB_D void fill_rows(const AttendArgs &a) {
  const int begin = min(max(__ldg(a.q_start), 0), a.total_q);
  const int end = min(max(__ldg(a.q_start + a.requests), begin), a.total_q);
  const int64_t rest = (int64_t)(begin + a.total_q - end) * a.q_heads, skip = (int64_t)(end - begin) * a.q_heads;
  const int64_t from = (int64_t)begin * a.q_heads, step = (int64_t)gridDim.x * kJoinThreads;
  if (a.fill & CB_KV4_FILL_OUT)
    for (int64_t i = (int64_t)blockIdx.x * kJoinThreads + threadIdx.x; i < rest * (D / 8); i += step)
      static_cast<uint4 *>(a.out)[i < from * (D / 8) ? i : i + skip * (D / 8)] = make_uint4(0, 0, 0, 0);
  if (a.fill & CB_KV4_FILL_LSE)
    for (int64_t i = (int64_t)blockIdx.x * kJoinThreads + threadIdx.x; i < rest; i += step)
      a.lse[i < from ? i : i + skip] = -INFINITY;
}

// Joins the parts of the items that a piece began and did not end, 16 dims of 8
// rows (a chunk) at a time. A block does eight chunks of an item, a warp each, or
// one chunk with all its warps where the item has many parts (a long request that
// is alone). The order of the sums depends on the number of parts alone.
template <int D>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(const AttendArgs a, const int pieces, const int nt) {
  __shared__ int counts[kJoinWarps], task_s[3];
  __shared__ float4 sums[kJoinWarps][32];
  __shared__ float4 tops[kJoinWarps][4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int chunks = nt * (D / 16), groups = (chunks + kJoinWarps - 1) / kJoinWarps;
  // The kernel in front began after everything before it had ended, and leaves these rows alone.
  if (a.fill) fill_rows<D>(a);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // the blocks' tasks, in the order of the pieces; a thread counts 16 pieces
  uint4 how = make_uint4(0, 0, 0, 0);
  if (threadIdx.x * 16 < pieces) how = reinterpret_cast<const uint4 *>(a.join_how)[threadIdx.x];
  const uint32_t words[4] = {how.x, how.y, how.z, how.w};
  int mine = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    mine += __popc(words[k] & 0x01010101u * kJoinFew) * groups + __popc(words[k] & 0x01010101u * kJoinMany) * chunks;
  int v = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) counts[warp] = v;
  __syncthreads();
  int tasks = 0, begin = v - mine;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    if (w < warp) begin += counts[w];
    tasks += counts[w];
  }
  const int part = nt * 8 * (D + 2);
  for (int task = blockIdx.x; task < tasks; task += gridDim.x) {
    __syncthreads();
    if (task >= begin && task < begin + mine) {
      int at = task - begin;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int h = words[k / 4] >> (8 * (k % 4)) & 0xff, n = h == kJoinFew ? groups : h == kJoinMany ? chunks : 0;
        if (at >= 0 && at < n) task_s[0] = threadIdx.x * 16 + k, task_s[1] = at, task_s[2] = h;
        at -= n;
      }
    }
    __syncthreads();
    const int p = task_s[0], team = task_s[2] == kJoinMany ? kJoinWarps : 1;
    const int chunk = team > 1 ? task_s[1] : task_s[1] * kJoinWarps + warp, n = chunk / (D / 16), i = chunk % (D / 16);
    const int4 join = a.joins[p];
    const int places = a.join_n[p], parts = places >> 1;
    Item it;
    it.q0 = join.x, it.rt = join.y, it.h = join.z;
    const int rows = join.w - (it.rt * nt + n) * 8;
    const bool here = chunk < chunks && rows > 0;
    float4 m = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);  // maximum and sum of rows 2t, 2t + 1
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [](float &m, float &l, float &x, float &y, float mk, float lk, float xk, float yk) {
      const float top = fmaxf(m, mk), at = top == -INFINITY ? 0.0f : top;  // parts may hold nothing
      const float f = ex2(m - at), fk = ex2(mk - at);
      m = top;
      l = l * f + lk * fk;
      x = x * f + xk * fk;
      y = y * f + yk * fk;
    };
    if (here) {
      const float *base = a.parts + (long long)p * 2 * part;
      constexpr int kBatch = 4;
      for (int k0 = team > 1 ? warp : 0; k0 < parts; k0 += kBatch * team) {
        float4 vs[kBatch], ms[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int at = min(k0 + k * team, parts - 1);
          const float *from = base + (long long)at * 2 * part + (at ? 0 : (places & 1) * part);
          vs[k] = load_now(from + (chunk * 32 + lane) * 4);
          ms[k] = load_now(from + nt * 8 * D + (n * 4 + t) * 4);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (k0 + k * team >= parts) ms[k].x = ms[k].z = -INFINITY, ms[k].y = ms[k].w = 0.0f;
          add(m.x, m.y, x.x, x.z, ms[k].x, ms[k].y, vs[k].x, vs[k].z);
          add(m.z, m.w, x.y, x.w, ms[k].z, ms[k].w, vs[k].y, vs[k].w);
        }
      }
    }
    if (team > 1) {
      sums[warp][lane] = x;
      if (g == 0) tops[warp][t] = m;
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int w = 1; w < kJoinWarps; ++w) {
          const float4 mw = tops[w][t], vw = sums[w][lane];
          add(m.x, m.y, x.x, x.z, mw.x, mw.y, vw.x, vw.z);
          add(m.z, m.w, x.y, x.w, mw.z, mw.w, vw.y, vw.w);
        }
      }
    }
    if (here && (team == 1 || warp == 0)) {
      const int row = (it.rt * nt + n) * 8;
      const float i0 = m.y == 0.0f ? 0.0f : 1.0f / m.y, i1 = m.w == 0.0f ? 0.0f : 1.0f / m.w;
      if (i == 0 && g == 0 && a.lse) {
        if (2 * t < rows) a.lse[out_row(a, it, row + 2 * t)] = m.y == 0.0f ? -INFINITY : (m.x + log2f(m.y)) * kLn2;
        if (2 * t + 1 < rows)
          a.lse[out_row(a, it, row + 2 * t + 1)] = m.w == 0.0f ? -INFINITY : (m.z + log2f(m.w)) * kLn2;
      }
      const int r = 2 * t + (g & 1);
      uint32_t *to =
          static_cast<uint32_t *>(a.out) + (out_row(a, it, row + min(r, rows - 1)) * D + 16 * i + (g & 6)) / 2;
      const float x0 = x.x * 0x1p24f * i0, y0 = x.y * 0x1p24f * i1, x1 = x.z * 0x1p20f * i0, y1 = x.w * 0x1p20f * i1;
      const float got0 = __shfl_xor_sync(0xffffffffu, g & 1 ? x0 : y0, 4);
      const float got1 = __shfl_xor_sync(0xffffffffu, g & 1 ? x1 : y1, 4);
      if (r < rows) {
        to[0] = g & 1 ? pack2(a.bf16, got0, y0) : pack2(a.bf16, x0, got0);
        to[4] = g & 1 ? pack2(a.bf16, got1, y1) : pack2(a.bf16, x1, got1);
      }
    }
  }
}

// ------------------------------------------------------------------- the host

constexpr int kMaxDevices = 64;

int sm_count(int device) {
  static std::atomic<int> known[kMaxDevices];  // calls may come from several threads
  if (device < 0 || device >= kMaxDevices) return 148;
  int n = known[device].load(std::memory_order_relaxed);
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = 148;
    }
    known[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int D, int NG, int NT>
cudaError_t run_few(const Kv4View &c, const AttendArgs &a, const Launch &l, cudaStream_t stream) {
  using F = Form<D, NG, NT>;
  static std::atomic<uint64_t> ready{0};  // a bit for each device
  static_assert(F::kCtasPerSm * (F::kSmem + F::kStatic + 1024) <= 228 * 1024, "shared memory of an SM");
  cudaError_t e = allow_shared(attend_few_kernel<D, NG, NT>, F::kSmem, ready);
  if (e != cudaSuccess) return e;
  e = kv4_launch(attend_few_kernel<D, NG, NT>, dim3(l.pieces / kWarps), kThreads, F::kSmem, stream, false, c, a);
  if (e != cudaSuccess) return e;
  return kv4_launch(attend_join_kernel<D>, dim3(8 * l.sms), kJoinThreads, 0, stream, true, a, l.pieces, NT);
}

// n-tiles of a row tile at most: O is head_dim * rows / 32 registers of a lane, and 8
// warps' rings and query rows have to fit an SM (256 dims in 8 groups, 16 rows: 230 KB).
constexpr int most_tiles(int d, int ng) { return d <= 128 ? 4 : ng <= 4 ? 2 : 1; }

// f(integral constants D, NG, NT) for a cache and a number of n-tiles.
template <typename F>
auto by_form(int d, int ng, int nt, F f) {
  auto with_nt = [&](auto dd, auto gg) {
    constexpr int kMost = most_tiles(decltype(dd)::value, decltype(gg)::value);
    if (nt == 1) return f(dd, gg, std::integral_constant<int, 1>{});
    if (nt == 2) return f(dd, gg, std::integral_constant<int, (kMost < 2 ? kMost : 2)>{});
    return f(dd, gg, std::integral_constant<int, kMost>{});
  };
  auto with_ng = [&](auto dd) {
    constexpr int kD = decltype(dd)::value;
    if (ng == 1) return with_nt(dd, std::integral_constant<int, 1>{});
    if (ng == 2 || kD < 128) return with_nt(dd, std::integral_constant<int, 2>{});
    if (ng == 4 || kD < 256) return with_nt(dd, std::integral_constant<int, (kD < 128 ? 2 : 4)>{});
    return with_nt(dd, std::integral_constant<int, (kD < 256 ? kD / 32 : 8)>{});
  };
  if (d == 64) return with_ng(std::integral_constant<int, 64>{});
  if (d == 128) return with_ng(std::integral_constant<int, 128>{});
  return with_ng(std::integral_constant<int, 256>{});
}

// n-tiles of a row tile (8, 16 or 32 rows) for requests of `rows` rows. A tile of 32
// rows has room for 8 warps on an SM (O is head_dim * rows / 32 registers in a lane),
// one of 8 rows for 16, and costs 3.5 times as much; what several tiles read again is
// in L2. 24 requests of up to 7,000 tokens, 8 KV heads of 128, us with tiles of 8,
// 16, 32 rows: 16 rows 54, 52, -; 24 rows 74, 87, 79; 32 rows 91, 89, 84; 40
// rows 111, 126, 133; 64 rows 166, 163, 139. (In one group; other forms go by the same
// rule.) 256 dims in 8 groups take 69 us for 24 such requests of 16 rows, in 4 groups, with
// tiles of 16 rows, 57.
int few_tiles(int head_dim, int group, int64_t rows) {
  const int most = most_tiles(head_dim, head_dim / group);
  if (rows <= 8 || most == 1) return 1;
  if (rows <= 16 || most == 2) return 2;
  return 2 * ((rows + 7) / 8) > 7 * ((rows + 31) / 32) ? 4 : 1;
}

// Above this many rows of a request the prompt kernel takes it (where it is
// offered: head_dim 64 and 128). It works on 128 rows whether there are or not, the
// few-row kernel reads the cache again for every 8 or 32. 24 requests of up to 7,000
// tokens, 8 KV heads of 128, few-row against prompt kernel: 64 rows 139 against 180
// us, 96 rows 197 against 186, 128 rows 252 against 186.
constexpr int kFewRows = 64;

struct Launches {
  Launch few, prompt;
  bool prompts;  // whether a request may have more than kFewRows rows
};

Launches plan_launches(const cb_kv4_cache *cache, const cb_kv4_attend_args *a) {
  const int64_t ratio = a->q_heads / cache->kv_heads, rows = ratio * (a->max_q > 1 ? a->max_q : 1);
  const int d = cache->head_dim;
  Launches l = {};
  l.prompts = d <= 128 && rows > kFewRows;
  // beside prompt chunks the others are single tokens in the main
  const int nt = few_tiles(d, cache->group, l.prompts ? ratio : rows);
  l.few.sms = min(sm_count(cache->device) & ~1, kJoinThreads);  // a thread of the join counts 16 pieces
  l.few.rows = 8 * nt;
  l.few.part = l.few.rows * (d + 2);
  l.few.pieces = l.few.sms * (nt == 1 && d <= 128 ? 2 : 1) * kWarps;
  if (l.prompts) l.prompt = prompt_launch(d, l.few.sms);
  return l;
}

int check(const cb_kv4_cache *cache, const cb_kv4_attend_args *a, Kv4View *c) {
  if (!a) return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: no arguments");
  if (int rc = kv4_check_cache(cache, a->layer, "cb_kv4_attend: no cache", c)) return rc;
  if (a->dtype != CB_KV4_F16 && a->dtype != CB_KV4_BF16)
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: q must be fp16 or bf16");
  if (a->requests < 0 || a->columns <= 0 || a->total_q < 0 || a->q_heads <= 0 || a->table_stride < 0)
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: bad sizes");
  if (a->q_heads % cache->kv_heads) return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: q_heads is not a multiple of kv_heads");
  if ((long long)a->total_q * a->q_heads > 0x3fffffffll) return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: too many rows");
  if (!a->q_start && a->total_q != a->requests)
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: without q_start there is one row for each request");
  if ((long long)a->columns * cache->page_size > kKv4MostTokens)
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: a row may not hold more than 2^30 tokens");
  if (a->requests > 0 && a->total_q > 0 && (!a->q || !a->out || !a->block_table || !a->kv_lens))
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: missing array");
  if (reinterpret_cast<uintptr_t>(a->out) & 15)
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: out must be 16-byte aligned");
  if (a->total_q > 0 && (((a->fill & CB_KV4_FILL_OUT) && !a->out) || ((a->fill & CB_KV4_FILL_LSE) && !a->lse)))
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: nothing to fill");
  return CB_OK;
}

}  // namespace

}  // namespace cb

extern "C" uint64_t cb_kv4_attend_workspace(const cb_kv4_cache *cache, const cb_kv4_attend_args *a) {
  using namespace cb;
  Kv4View c;
  if (check(cache, a, &c) != CB_OK) return 0;
  const Launches l = plan_launches(cache, a);
  return launch_bytes(l.few) + (l.prompts ? launch_bytes(l.prompt) : 0);
}

extern "C" int cb_kv4_attend(const cb_kv4_cache *cache, const cb_kv4_attend_args *args, void *stream) {
  using namespace cb;
  Kv4View c;
  if (int rc = check(cache, args, &c)) return rc;
  if (args->total_q == 0 || (args->requests == 0 && !args->fill)) return CB_OK;
  const Launches l = plan_launches(cache, args);
  const uint64_t need = launch_bytes(l.few) + (l.prompts ? launch_bytes(l.prompt) : 0);
  if (args->requests > 0 &&
      (!args->workspace || args->workspace_bytes < need || (reinterpret_cast<uintptr_t>(args->workspace) & 15)))
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: workspace too small or not 16-byte aligned");
  Kv4Device dev(cache->device);
  if (dev.err != cudaSuccess) return kv4_fail(CB_ERR_CUDA, "cb_kv4_attend: device", dev.err);
  AttendArgs a = {};
  a.q = args->q;
  a.out = args->out;
  a.lse = args->lse;
  a.block_table = args->block_table;
  a.kv_lens = args->kv_lens;
  a.q_start = args->q_start;
  a.table_stride = args->table_stride;
  a.q_token_stride = args->q_token_stride;
  a.q_head_stride = args->q_head_stride;
  a.scale = args->scale;
  a.requests = args->requests;
  a.columns = args->columns;
  a.total_q = args->total_q;
  a.q_heads = args->q_heads;
  a.ratio = args->q_heads / cache->kv_heads;
  a.causal = args->causal;
  a.bf16 = args->dtype == CB_KV4_BF16;
  a.q_vec = ((reinterpret_cast<uintptr_t>(a.q) | (a.q_token_stride | a.q_head_stride) * 2) & 15) == 0;
  a.fill = args->q_start ? args->fill : 0;  // without q_start every row is a request's
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (args->requests == 0) {
    const auto join = cache->head_dim == 64    ? attend_join_kernel<64>
                      : cache->head_dim == 128 ? attend_join_kernel<128>
                                               : attend_join_kernel<256>;
    e = kv4_launch(join, dim3(8 * l.few.sms), kJoinThreads, 0, st, false, a, 0, 1);
    return e == cudaSuccess ? CB_OK : kv4_fail(CB_ERR_CUDA, "cb_kv4_attend: launch", e);
  }
  if (l.prompts) {
    launch_arrays(l.prompt, static_cast<char *>(args->workspace) + launch_bytes(l.few), a);
    a.rows_above = kFewRows;
    a.rows_most = 0x7fffffff;
    a.min_share = 1;
    e = run_prompt(c, a, cache->head_dim, cache->group, l.prompt, st);
  }
  if (e == cudaSuccess) {
    launch_arrays(l.few, args->workspace, a);
    a.rows_above = 0;
    a.rows_most = l.prompts ? kFewRows : 0x7fffffff;
    a.min_share = 2;
    e = by_form(cache->head_dim, cache->head_dim / cache->group, l.few.rows / 8, [&](auto d, auto ng, auto nt) {
      return run_few<decltype(d)::value, decltype(ng)::value, decltype(nt)::value>(c, a, l.few, st);
    });
  }
  return e == cudaSuccess ? CB_OK : kv4_fail(CB_ERR_CUDA, "cb_kv4_attend: launch", e);
}
