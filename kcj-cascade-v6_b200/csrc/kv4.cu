// Paged KV cache held in 4 bits: the page table (cb_kv4_plan), and the
// quantising write and the dequantising read of tokens (cb_kv4_append,
// cb_kv4_read). Format: kv4.cuh.
#include <cooperative_groups.h>

#include <string>
#include <type_traits>

#include "kv4.cuh"

namespace cg = cooperative_groups;

namespace cb {

extern thread_local std::string g_create_error;  // store.cu: message of store-less calls

int kv4_fail(int code, const char *msg, cudaError_t e) {
  if (e != cudaSuccess) (void)cudaGetLastError();  // reported here, and not again by the next launch
  try {
    g_create_error = msg;
    if (e != cudaSuccess) {
      g_create_error += ": ";
      g_create_error += cudaGetErrorString(e);
    }
  } catch (...) {  // no memory for the message: the code alone
  }
  return code;
}

namespace {

bool form_offered(int layers, int kv_heads, int d, int page_size, int group) {
  if (layers <= 0 || kv_heads <= 0 || layers > (1 << 16) || kv_heads > (1 << 16)) return false;
  if (d != 64 && d != 128 && d != 256) return false;
  if (group != 32 && group != 64 && group != 128 && group != 256) return false;
  if (group > d) return false;
  return page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128 || page_size == 256;
}

}  // namespace

int kv4_check_cache(const cb_kv4_cache *c, int32_t layer, const char *who, Kv4View *out) {
  if (!c || !c->pages) return kv4_fail(CB_ERR_ARG, who);
  const uint64_t bytes = cb_kv4_page_bytes(c->layers, c->kv_heads, c->head_dim, c->page_size, c->group);
  if (!bytes) return kv4_fail(CB_ERR_ARG, "cb_kv4: head_dim, page_size or group not offered");
  if (layer < 0 || layer >= c->layers) return kv4_fail(CB_ERR_ARG, "cb_kv4: layer out of range");
  if (c->num_pages <= 0) return kv4_fail(CB_ERR_ARG, "cb_kv4: the cache has no pages");
  if (c->page_stride < bytes || (c->page_stride & 15) || (reinterpret_cast<uintptr_t>(c->pages) & 15))
    return kv4_fail(CB_ERR_ARG, "cb_kv4: pages must be 16-byte aligned and not overlap");
  out->head_bytes = kv4_head_bytes(c->head_dim, c->group, c->page_size);
  out->base = static_cast<uint8_t *>(c->pages) + (uint64_t)layer * c->kv_heads * out->head_bytes;
  out->page_stride = c->page_stride;
  out->errors = c->errors;
  out->num_pages = c->num_pages;
  out->kv_heads = c->kv_heads;
  out->page_size = c->page_size;
  out->page_log2 = 31 - __builtin_clz((unsigned)c->page_size);
  return CB_OK;
}

namespace {

// ------------------------------------------------------------------ the plan
//
// One cluster does a step: every CTA runs the same scans over the rows (chunks
// of kPlanThreads rows, two prefix sums: new tokens, then pages needed) and takes
// its share of the tokens; the cluster's barrier stands between reading the old
// state and writing the new one, so the state may be updated in place with one
// launch and no counters in memory.
//
// A warp takes 8 x 32 tokens at a time (32 where there are few): each lane's eight
// rows are found first, then its eight page numbers are under way together; one at a
// time, every token would wait for a search and a load.
constexpr int kPlanThreads = 512;
constexpr int kPlanCtas = 16;  // the largest cluster
constexpr int kPlanRun = 8;

// Exclusive prefix sum over the block; `total` is the block's sum.
CB_D long long block_scan(long long x, long long *warp_sums, long long &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    const long long s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  __syncthreads();
  total = all;
  return before + v - x;
}

// Last index i in [0, n) with start[i] <= e (start ascending, start[0] <= e).
template <typename I>
CB_D int find_row(const I *start, int n, I e) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= e) lo = mid;
    else hi = mid;
  }
  return lo;
}

CB_D void plan_barrier(int ctas) {
  if (ctas > 1) cg::this_cluster().sync();
  else __syncthreads();
}

template <int RUN>
__global__ void __launch_bounds__(kPlanThreads) kv4_plan_kernel(const cb_kv4_plan_args a, const int ctas) {
  __shared__ long long start[kPlanThreads], warp_sums[kPlanThreads / 32];
  __shared__ int begin_s[kPlanThreads], base_s[kPlanThreads];
  __shared__ int len_s[kPlanThreads], held_s[kPlanThreads];  // held_s: -1 for a refused row
  const int tid = threadIdx.x, lane = tid & 31;
  const long long stride = (long long)ctas * kPlanThreads * RUN;  // of the cluster
  const int rank = ctas > 1 ? (int)cg::this_cluster().block_rank() : 0;
  const long long mine = ((long long)rank * kPlanThreads + (tid & ~31)) * RUN + lane;
  const int ps = a.page_size, log2 = (ps & (ps - 1)) == 0 ? 31 - __clz(ps) : -1;
  const long long most = (long long)a.columns * ps;
  long long count = min(max(*a.free_count, 0), a.num_pages);

  if (a.done) {  // finished rows give their pages back
    long long back = 0;
    for (int r0 = 0; r0 < a.requests; r0 += kPlanThreads) {
      const int r = r0 + tid;
      long long rel = 0;
      int bor = 0;
      if (r < a.requests && a.done[r]) {
        long long len = max(a.kv_lens[r], 0);
        if (len > most) {
          len = most;
          if (rank == 0) kv4_error(a.errors, kErrBounds);
        }
        const int held = (int)((len + ps - 1) / ps);
        bor = min(max(a.borrowed[r], 0), held);
        rel = held - bor;
      }
      long long total;
      const long long at = block_scan(rel, warp_sums, total);
      start[tid] = at;
      held_s[tid] = bor;
      __syncthreads();
      for (long long e0 = mine; e0 - lane < total; e0 += stride) {
        int page[RUN];
        int i = e0 < total ? find_row(start, kPlanThreads, e0) : 0;
#pragma unroll
        for (int u = 0; u < RUN; ++u) {
          const long long e = e0 + 32 * u;
          while (e < total && i + 1 < kPlanThreads && start[i + 1] <= e) ++i;
          if (e < total) page[u] = a.block_table[(r0 + i) * a.table_stride + held_s[i] + (e - start[i])];
        }
#pragma unroll
        for (int u = 0; u < RUN; ++u) {
          const long long e = e0 + 32 * u, to = count + back + e;
          if (e < total && to < a.num_pages) a.free[to] = page[u];
          else if (e < total) kv4_error(a.errors, kErrBounds);  // more pages came back than there are
        }
      }
      back += total;
      __syncthreads();
    }
    count = min(count + back, (long long)a.num_pages);
    plan_barrier(ctas);  // the pages are on the stack
  }

  long long tokens = 0, needed = 0, used = 0;
  for (int r0 = 0; r0 < a.requests; r0 += kPlanThreads) {
    const int r = r0 + tid;
    long long len = 0, q = 0;
    bool known = false;
    if (r < a.requests) {
      q = max(a.q_lens[r], 0);
      len = a.done && a.done[r] ? 0 : a.kv_lens[r];
      known = len >= 0 && len <= most;
      if (!known) {
        if (rank == 0) kv4_error(a.errors, kErrBounds);
        len = len < 0 ? 0 : most;
      }
    }
    long long total;
    const long long at = tokens + block_scan(q, warp_sums, total);
    const int held = (int)((len + ps - 1) / ps);
    const bool fits = known && at + q <= a.tokens && len + q <= most;
    const long long need = fits ? (len + q + ps - 1) / ps - held : 0;
    long long need_total;
    const long long first = needed + block_scan(need, warp_sums, need_total);
    const bool ok = fits && (need == 0 || first + need <= count);
    long long used_total;
    block_scan(ok ? need : 0, warp_sums, used_total);
    begin_s[tid] = (int)min(at, 0x7fffffffll);
    base_s[tid] = (int)min(first, 0x7fffffffll);
    len_s[tid] = (int)len;
    held_s[tid] = ok ? held : -1;
    if (rank == 0 && r < a.requests) {
      a.q_start[r] = (int)min(at, 0x7fffffffll);
      a.status[r] = ok ? CB_PUT_STORED : CB_PUT_FAILED;
    }
    __syncthreads();
    const int end = (int)min(tokens + total, (long long)a.tokens);
    for (long long n0_ = tokens + mine; n0_ - lane < end; n0_ += stride) {
      const int n0 = (int)min(n0_, 0x7fffffffll);
      int page[RUN], pos[RUN], row[RUN];
      int i = n0 < end ? find_row(begin_s, kPlanThreads, n0) : 0;
      int next = i + 1 < kPlanThreads ? begin_s[i + 1] : 0x7fffffff;
#pragma unroll
      for (int u = 0; u < RUN; ++u) {
        const int n = n0 + 32 * u;
        page[u] = -1, pos[u] = 0, row[u] = -1;
        if (n0 < end && 32 * u < end - n0) {
          while (next <= n) {
            ++i;
            next = i + 1 < kPlanThreads ? begin_s[i + 1] : 0x7fffffff;
          }
          pos[u] = (int)min((uint32_t)len_s[i] + (uint32_t)(n - begin_s[i]), 0x7fffffffu);
          const int held = held_s[i];
          if (held >= 0) {
            const int col = log2 >= 0 ? pos[u] >> log2 : pos[u] / ps;
            row[u] = i;
            page[u] = col < held ? a.block_table[(r0 + i) * a.table_stride + col]
                                 : a.free[(int)count - 1 - (base_s[i] + col - held)];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < RUN; ++u) {
        if (n0 >= end || 32 * u >= end - n0) break;
        long long slot = -1;
        if (row[u] >= 0) {
          const int col = log2 >= 0 ? pos[u] >> log2 : pos[u] / ps, in_page = pos[u] - col * ps;
          if (in_page == 0 && col >= held_s[row[u]])  // the first token of a new page
            a.block_table[(r0 + row[u]) * a.table_stride + col] = page[u];
          if (page[u] >= 0 && page[u] < a.num_pages) slot = (long long)page[u] * ps + in_page;
          else kv4_error(a.errors, kErrBounds);
        }
        a.slots[n0 + 32 * u] = slot;
        a.positions[n0 + 32 * u] = pos[u];
      }
    }
    tokens += total;
    needed += need_total;
    used += used_total;
    __syncthreads();
  }
  for (long long n = tokens + (long long)rank * kPlanThreads + tid; n < a.tokens;
       n += (long long)ctas * kPlanThreads) {
    a.slots[n] = -1;
    a.positions[n] = 0;
  }
  plan_barrier(ctas);  // everyone has read the old state
  if (rank != 0) return;
  for (int r = tid; r < a.requests; r += kPlanThreads) {
    // status was written by this thread
    const bool done = a.done && a.done[r];
    const int len = done ? 0 : a.kv_lens[r];
    a.kv_lens_out[r] = a.status[r] == CB_PUT_STORED ? len + max(a.q_lens[r], 0) : len;
    if (done) a.borrowed[r] = 0;
  }
  if (tid == 0) {
    a.q_start[a.requests] = (int)min(tokens, 0x7fffffffll);
    *a.free_count_out = (int)(count - used);
  }
}

// ---------------------------------------------------------- append and read
//
// A warp takes 8 tokens of the call, wherever their slots are, and K or V of one
// head. In registers a lane (g, t) has the dims 32 i + 8 t .. + 7 of token g: 64
// contiguous bytes of a 16-bit row for every four lanes and i. For K that
// is the order of the words in a page: a token's minimum and maximum are shuffles
// among four lanes, and its row of codes is 16 bytes a lane. For V the lanes
// exchange: four lanes collect the nibbles of dims 8 apart, then two rows their
// halves of a word. Bound by HBM: 4 D bytes of values and 1 - 1.25 D of codes for
// a token and head.
constexpr int kTokenThreads = 128, kTokensWarp = 8;

// 8 values; `vec`: on a 16-byte boundary.
template <typename T>
CB_D void load8(const T *p, bool vec, float *x) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p));
      const T *t = reinterpret_cast<const T *>(&a);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)t[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = kv4_load1(p + i);
  }
}

template <typename T>
CB_D void store8(T *p, bool vec, const float *x) {
  alignas(16) T y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = kv4_round<T>(x[i]);
  if (vec) {
#pragma unroll
    for (int w = 0; w < (int)sizeof(T) / 2; ++w)
      reinterpret_cast<uint4 *>(p)[w] = reinterpret_cast<const uint4 *>(y)[w];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = y[i];
  }
}

CB_D float max_nan(float x, float y) {
  float v;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(x), "f"(y));
  return v;
}

// x / 15, correctly rounded: a product with the rounded reciprocal, corrected once by
// its exact remainder (Markstein). x is 0 or far above the smallest normal number.
CB_D float fifteenth(float x) {
  constexpr float r = 1.0f / 15.0f;
  const float q = __fmul_rn(x, r);
  return __fmaf_rn(__fmaf_rn(-15.0f, q, x), r, q);
}

struct TokenStrides {
  int64_t k_token, k_head, v_token, v_head;
};

// Where a token of the call lives: its tile (of the head) and place, or no tile.
struct Spot {
  uint8_t *tile;
  int tok;
};

// The spots of the warp's 8 tokens, one in each of lanes 0 .. 7.
CB_D Spot load_spot(const Kv4View &c, const int64_t *slots, int64_t n, int64_t first, int head, int tile_bytes) {
  const int lane = threadIdx.x & 31;
  Spot s = {nullptr, 0};
  if (lane < kTokensWarp && first + lane < n) {
    const int64_t slot = __ldg(slots + first + lane);
    const int64_t page = slot >> c.page_log2;
    if (slot >= 0 && page < c.num_pages) {
      const int in_page = (int)(slot & (c.page_size - 1));
      s.tok = in_page % kKv4Tile;
      s.tile = c.base + page * c.page_stride + head * c.head_bytes + (uint64_t)(in_page / kKv4Tile) * tile_bytes;
    } else if (slot >= 0) {
      kv4_error(c.errors, kErrBounds);
    }
  }
  return s;
}

CB_D Spot spot_of(const Spot &s, int token) {
  Spot r;
  r.tile = reinterpret_cast<uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(s.tile), token));
  r.tok = __shfl_sync(0xffffffffu, s.tok, token);
  return r;
}

template <int N>
CB_D void load_words4(const void *p, uint32_t *w) {
  if constexpr (N == 2) {
    const uint2 v = *static_cast<const uint2 *>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    const uint4 v = *static_cast<const uint4 *>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
}
template <int N>
CB_D void store_words4(void *p, const uint32_t *w) {
  if constexpr (N == 2) *static_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
  else *static_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int D>
__global__ void __launch_bounds__(kTokenThreads)
    kv4_append_kernel(const Kv4View c, const int group_log2, const T *__restrict__ k, const T *__restrict__ v,
                      const TokenStrides st, const bool vec, const int64_t *__restrict__ slots, const int n) {
  constexpr int kSlabs = D > 128 ? 2 : 1, kWpr = D / kSlabs / 32, kWords = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = 1 << group_log2, ng = D >> group_log2;
  const uint32_t id = blockIdx.x * (kTokenThreads / 32) + (threadIdx.x >> 5), part = id / (uint32_t)c.kv_heads;
  const int head = (int)(id - part * c.kv_heads);
  const bool is_v = part & 1;
  const int64_t first = (int64_t)(part >> 1) * kTokensWarp;
  if (first >= n) return;
  const Spot mine = load_spot(c, slots, n, first, head, 16 * D + 128 * ng);
  uint32_t words[kWords];  // codes of token g: dims 8 t + e of block i in nibble e
  {
    const Spot to = spot_of(mine, g);
    const int64_t row = first + (first + g < n ? g : 0);
    const T *src = (is_v ? v + row * st.v_token + head * st.v_head : k + row * st.k_token + head * st.k_head) + 8 * t;
    float x[kWords][8], lo[kWords], hi[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) load8(src + 32 * i, vec, x[i]);
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      lo[i] = INFINITY, hi[i] = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[i] = fminf(lo[i], x[i][e]);
        hi[i] = max_nan(hi[i], x[i][e]);  // a NaN stays, and makes the scale NaN
        x[i][e] = fminf(fmaxf(x[i][e], -kKv4Most), kKv4Most);
      }
    }
#pragma unroll
    for (int span = 1; span < kWords; span *= 2) {
      if (group <= 32 * span) break;
#pragma unroll
      for (int i = 0; i < kWords; i += 2 * span) lo[i] = fminf(lo[i], lo[i + span]), hi[i] = max_nan(hi[i], hi[i + span]);
    }
    const int step_log2 = group_log2 - 5;
    float off = 0.0f, inv = 0.0f;
    bool any = false;
    __half scale_h = __float2half_rn(0.0f), offset_h = scale_h;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if ((i & ((1 << step_log2) - 1)) == 0) {  // a group begins: its parameters
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          lo[i] = fminf(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
          hi[i] = max_nan(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
        }
        const float low = fminf(fmaxf(lo[i], -kKv4Most), kKv4Most);
        const float high = hi[i] != hi[i] ? hi[i] : fminf(fmaxf(hi[i], -kKv4Most), kKv4Most);
        scale_h = __float2half_rn(fifteenth(__fsub_rn(high, low)));
        const float s = __half2float(scale_h);
        offset_h = __float2half_rn(__fadd_rn(low, __fmul_rn(8.0f, s)));
        off = __half2float(offset_h);
        any = s > 0.0f;
        inv = any ? __frcp_rn(s) : 0.0f;
        if (t == 0 && to.tile)
          reinterpret_cast<uint32_t *>(to.tile + 16 * D + (is_v ? 64 * ng : 0))[to.tok * ng + (i >> step_log2)] =
              (uint32_t)__half_as_ushort(scale_h) | (uint32_t)__half_as_ushort(offset_h) << 16;
      }
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // to the nearest integer, ties to even, by adding 1.5 * 2^23 (and the 8): it is then
        // in the low bits; conversions would go through the unit with 16 results a cycle
        const float y = any ? fminf(fmaxf(__fmul_rn(__fsub_rn(x[i][e], off), inv), -8.0f), 7.0f) : 0.0f;
        const uint32_t code = __float_as_uint(__fadd_rn(y, 12582920.0f)) & 15u;
        w |= code << (4 * (is_v ? e : (e & 1) * 4 + e / 2));
      }
      words[i] = w;
    }
    if (!is_v && to.tile) {
#pragma unroll
      for (int sl = 0; sl < kSlabs; ++sl)
        store_words4<kWpr>(to.tile + ((sl * 16 + to.tok) * 4 + t) * kWpr * 4, words + sl * kWpr);
    }
  }
  if (!is_v) return;
  // V. Lane (e, p) is to have dims e + 8 {0, 1, 2, 3} of tokens 2 p and 2 p + 1.
  uint32_t out[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    uint32_t w = 0;  // nibbles 2 t (low half) and 2 t + 1 of the four lanes' words
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t b = __shfl_sync(0xffffffffu, words[i], (lane & 28) + q) >> (8 * t);
      w |= (b & 15u) << (4 * q) | (b >> 4 & 15u) << (16 + 4 * q);
    }
    const uint32_t a = __shfl_sync(0xffffffffu, w, (2 * t) * 4 + g / 2);
    const uint32_t b = __shfl_sync(0xffffffffu, w, (2 * t + 1) * 4 + g / 2);
    out[i] = __byte_perm(a, b, g & 1 ? 0x7632 : 0x5410);
  }
  const Spot s0 = spot_of(mine, 2 * t), s1 = spot_of(mine, 2 * t + 1);
  if (s0.tile && s0.tile == s1.tile && s1.tok == s0.tok + 1 && !(s0.tok & 1)) {  // a pair of the page
#pragma unroll
    for (int sl = 0; sl < kSlabs; ++sl)
      store_words4<kWpr>(s0.tile + 8 * D + (((sl * 2 + s0.tok / 8) * 8 + g) * 4 + s0.tok % 8 / 2) * kWpr * 4,
                         out + sl * kWpr);
  } else {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const Spot &s = b ? s1 : s0;
      if (!s.tile) continue;
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        reinterpret_cast<uint16_t *>(s.tile + 8 * D)[((((i / kWpr * 2 + s.tok / 8) * 8 + g) * 4 + s.tok % 8 / 2) * kWpr +
                                                      i % kWpr) * 2 + s.tok % 2] = (uint16_t)(out[i] >> (16 * b));
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kTokenThreads)
    kv4_read_kernel(const Kv4View c, const int group_log2, T *__restrict__ k, T *__restrict__ v, const bool vec,
                    const int64_t *__restrict__ slots, const int n) {
  constexpr int kSlabs = D > 128 ? 2 : 1, kWpr = D / kSlabs / 32, kWords = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int ng = D >> group_log2;
  const uint32_t id = blockIdx.x * (kTokenThreads / 32) + (threadIdx.x >> 5), part = id / (uint32_t)c.kv_heads;
  const int head = (int)(id - part * c.kv_heads);
  const bool is_v = part & 1;
  const int64_t first = (int64_t)(part >> 1) * kTokensWarp;
  if (first >= n) return;
  const Spot mine = load_spot(c, slots, n, first, head, 16 * D + 128 * ng);
  {
    const Spot at = spot_of(mine, g);
    uint32_t w[kWords], par[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = par[i] = 0;
    if (at.tile) {
      const uint32_t *params = reinterpret_cast<const uint32_t *>(at.tile + 16 * D + (is_v ? 64 * ng : 0)) + at.tok * ng;
#pragma unroll
      for (int i = 0; i < kWords; ++i) par[i] = params[i >> (group_log2 - 5)];
    }
    if (!is_v) {
      if (at.tile) {
#pragma unroll
        for (int sl = 0; sl < kSlabs; ++sl)
          load_words4<kWpr>(at.tile + ((sl * 16 + at.tok) * 4 + t) * kWpr * 4, w + sl * kWpr);
      }
    } else {
      // a lane fetches words of tokens 2 t and 2 t + 1 (dims g + 8 {0 .. 3}), as they lie
      const Spot s0 = spot_of(mine, 2 * t), s1 = spot_of(mine, 2 * t + 1);
      uint32_t a[kWords], b[kWords];
#pragma unroll
      for (int i = 0; i < kWords; ++i) a[i] = b[i] = 0;
#pragma unroll
      for (int sl = 0; sl < kSlabs; ++sl) {
        if (s0.tile)
          load_words4<kWpr>(s0.tile + 8 * D + (((sl * 2 + s0.tok / 8) * 8 + g) * 4 + s0.tok % 8 / 2) * kWpr * 4, a + sl * kWpr);
        if (s1.tile)
          load_words4<kWpr>(s1.tile + 8 * D + (((sl * 2 + s1.tok / 8) * 8 + g) * 4 + s1.tok % 8 / 2) * kWpr * 4, b + sl * kWpr);
      }
      const uint32_t pick = (s0.tok & 1 ? 0x32u : 0x10u) | (s1.tok & 1 ? 0x7600u : 0x5400u);
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        // 4 nibbles (dims 8 apart) of each token: as 16-bit elements an 8 x 8 matrix, dims by
        // tokens. Transposed, a lane has dims 2 t and 2 t + 1 of its own token, and wants
        // nibble t of all eight, which are with the four lanes of the token.
        uint32_t both = __byte_perm(a[i], b[i], pick), y = 0;
        asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(both));
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t x = __shfl_sync(0xffffffffu, both, (lane & 28) + q) >> (4 * t);
          y |= ((x & 15u) | (x >> 12 & 0xf0u)) << (8 * q);
        }
        w[i] = y;
      }
    }
    if (first + g < n) {
      T *dst = (is_v ? v : k) + ((first + g) * c.kv_heads + head) * D + 8 * t;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const float s = kv4_scale(par[i]), o = kv4_offset(par[i]);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int nib = is_v ? e : (e & 1) * 4 + e / 2;
          x[e] = kv4_value(w[i] >> (4 * nib) & 15u, s, o);
        }
        store8(dst + 32 * i, vec, x);
      }
    }
  }
}

// A warp for 8 tokens, K or V, and head.
inline uint64_t token_blocks(const Kv4View &c, int n) {
  const uint64_t warps = ((uint64_t)n + kTokensWarp - 1) / kTokensWarp * 2 * c.kv_heads;
  return (warps + kTokenThreads / 32 - 1) / (kTokenThreads / 32);
}

template <typename T, int D>
cudaError_t launch_append(const Kv4View &c, int group, const void *k, const void *v, const TokenStrides &st,
                          const int64_t *slots, int n, cudaStream_t stream) {
  const uint64_t unit = 16 / sizeof(T);
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 &&
                   ((st.k_token | st.k_head | st.v_token | st.v_head) & (int64_t)(unit - 1)) == 0;
  return kv4_launch(kv4_append_kernel<T, D>, dim3((unsigned)token_blocks(c, n)), kTokenThreads, 0, stream, false, c,
                    31 - __builtin_clz((unsigned)group), static_cast<const T *>(k), static_cast<const T *>(v), st, vec,
                    slots, n);
}

template <typename T, int D>
cudaError_t launch_read(const Kv4View &c, int group, void *k, void *v, const int64_t *slots, int n,
                        cudaStream_t stream) {
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  return kv4_launch(kv4_read_kernel<T, D>, dim3((unsigned)token_blocks(c, n)), kTokenThreads, 0, stream, false, c,
                    31 - __builtin_clz((unsigned)group), static_cast<T *>(k), static_cast<T *>(v), vec, slots, n);
}

// f(T{}, std::integral_constant<int, D>{}) for the cache's type and head size.
template <typename F>
cudaError_t by_form(int dtype, int d, F f) {
  auto with = [&](auto t) {
    if (d == 64) return f(t, std::integral_constant<int, 64>{});
    if (d == 128) return f(t, std::integral_constant<int, 128>{});
    return f(t, std::integral_constant<int, 256>{});
  };
  if (dtype == CB_KV4_F16) return with(__half{});
  if (dtype == CB_KV4_BF16) return with(__nv_bfloat16{});
  return with(float{});
}

// The warps of a launch over n tokens are counted in 31 bits.
bool tokens_fit(const Kv4View &c, int32_t n) { return token_blocks(c, n) * (kTokenThreads / 32) < 0x7fffffffull; }

}  // namespace

}  // namespace cb

extern "C" uint64_t cb_kv4_page_bytes(int32_t layers, int32_t kv_heads, int32_t head_dim, int32_t page_size,
                                      int32_t group) {
  if (!cb::form_offered(layers, kv_heads, head_dim, page_size, group)) return 0;
  return (uint64_t)layers * kv_heads * cb::kv4_head_bytes(head_dim, group, page_size);
}

extern "C" int cb_kv4_plan(const cb_kv4_plan_args *a, void *stream) {
  using namespace cb;
  if (!a || a->requests < 0 || a->tokens < 0 || a->columns <= 0 || a->num_pages <= 0 || a->page_size <= 0 ||
      a->table_stride < a->columns)
    return kv4_fail(CB_ERR_ARG, "cb_kv4_plan: bad sizes");
  if ((long long)a->columns * a->page_size > kKv4MostTokens)
    return kv4_fail(CB_ERR_ARG, "cb_kv4_plan: a row may not hold more than 2^30 tokens");
  if (!a->free || !a->free_count || !a->free_count_out || !a->q_start || (a->tokens > 0 && (!a->slots || !a->positions)) ||
      (a->requests > 0 && (!a->q_lens || !a->kv_lens || !a->kv_lens_out || !a->block_table || !a->status)) ||
      (a->done && !a->borrowed))
    return kv4_fail(CB_ERR_ARG, "cb_kv4_plan: missing array");
  Kv4Device dev(a->device);
  if (dev.err != cudaSuccess) return kv4_fail(CB_ERR_CUDA, "cb_kv4_plan: device", dev.err);
  int ctas = 1;
  // 16,384 tokens: one run of 32 for every warp of the largest cluster
  const bool many = a->tokens > 2 * kPlanCtas * kPlanThreads;
  while (ctas < kPlanCtas && a->tokens > ctas * 2 * kPlanThreads) ctas *= 2;
  const auto kernel = many ? kv4_plan_kernel<kPlanRun> : kv4_plan_kernel<1>;
  if (ctas > 8) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return kv4_fail(CB_ERR_CUDA, "cb_kv4_plan: cluster size", e);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, *a, ctas);
  return e == cudaSuccess ? CB_OK : kv4_fail(CB_ERR_CUDA, "cb_kv4_plan: launch", e);
}

extern "C" int cb_kv4_append(const cb_kv4_cache *cache, int32_t layer, int32_t dtype, const void *k, const void *v,
                             int32_t n, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                             int64_t v_head_stride, const int64_t *slots, void *stream) {
  using namespace cb;
  Kv4View c;
  if (int rc = kv4_check_cache(cache, layer, "cb_kv4_append: no cache", &c)) return rc;
  if (dtype < CB_KV4_F16 || dtype > CB_KV4_F32) return kv4_fail(CB_ERR_ARG, "cb_kv4_append: unknown dtype");
  if (n < 0 || (n > 0 && (!k || !v || !slots))) return kv4_fail(CB_ERR_ARG, "cb_kv4_append: bad arguments");
  if (!tokens_fit(c, n)) return kv4_fail(CB_ERR_ARG, "cb_kv4_append: too many tokens in one call");
  if (n == 0) return CB_OK;
  Kv4Device dev(cache->device);
  if (dev.err != cudaSuccess) return kv4_fail(CB_ERR_CUDA, "cb_kv4_append: device", dev.err);
  const TokenStrides st = {k_token_stride, k_head_stride, v_token_stride, v_head_stride};
  const cudaError_t e = by_form(dtype, cache->head_dim, [&](auto t, auto d) {
    return launch_append<decltype(t), decltype(d)::value>(c, cache->group, k, v, st, slots, n,
                                                          static_cast<cudaStream_t>(stream));
  });
  return e == cudaSuccess ? CB_OK : kv4_fail(CB_ERR_CUDA, "cb_kv4_append: launch", e);
}

extern "C" int cb_kv4_read(const cb_kv4_cache *cache, int32_t layer, int32_t dtype, void *k_out, void *v_out,
                           int32_t n, const int64_t *slots, void *stream) {
  using namespace cb;
  Kv4View c;
  if (int rc = kv4_check_cache(cache, layer, "cb_kv4_read: no cache", &c)) return rc;
  if (dtype < CB_KV4_F16 || dtype > CB_KV4_F32) return kv4_fail(CB_ERR_ARG, "cb_kv4_read: unknown dtype");
  if (n < 0 || (n > 0 && (!k_out || !v_out || !slots))) return kv4_fail(CB_ERR_ARG, "cb_kv4_read: bad arguments");
  if (!tokens_fit(c, n)) return kv4_fail(CB_ERR_ARG, "cb_kv4_read: too many tokens in one call");
  if (n == 0) return CB_OK;
  Kv4Device dev(cache->device);
  if (dev.err != cudaSuccess) return kv4_fail(CB_ERR_CUDA, "cb_kv4_read: device", dev.err);
  const cudaError_t e = by_form(dtype, cache->head_dim, [&](auto t, auto d) {
    return launch_read<decltype(t), decltype(d)::value>(c, cache->group, k_out, v_out, slots, n,
                                                        static_cast<cudaStream_t>(stream));
  });
  return e == cudaSuccess ? CB_OK : kv4_fail(CB_ERR_CUDA, "cb_kv4_read: launch", e);
}
