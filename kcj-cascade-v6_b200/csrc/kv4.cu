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
constexpr int kPlanThreads = 512;
constexpr int kPlanCtas = 8;

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
CB_D int find_row(const long long *start, int n, long long e) {
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

__global__ void __launch_bounds__(kPlanThreads) kv4_plan_kernel(const cb_kv4_plan_args a, const int ctas) {
  __shared__ long long start[kPlanThreads + 1], base[kPlanThreads], warp_sums[kPlanThreads / 32];
  __shared__ int len_s[kPlanThreads], held_s[kPlanThreads];  // held_s: -1 for a refused row
  const int tid = threadIdx.x;
  const int rank = ctas > 1 ? (int)cg::this_cluster().block_rank() : 0;
  const int ps = a.page_size;
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
      for (long long e = (long long)rank * kPlanThreads + tid; e < total; e += (long long)ctas * kPlanThreads) {
        const int i = find_row(start, kPlanThreads, e);
        const int page = a.block_table[(r0 + i) * a.table_stride + held_s[i] + (e - start[i])];
        const long long to = count + back + e;
        if (to < a.num_pages) a.free[to] = page;
        else kv4_error(a.errors, kErrBounds);  // more pages came back than there are
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
    start[tid] = at;
    base[tid] = first;
    len_s[tid] = (int)len;
    held_s[tid] = ok ? held : -1;
    if (rank == 0 && r < a.requests) {
      a.q_start[r] = (int)min(at, 0x7fffffffll);
      a.status[r] = ok ? CB_PUT_STORED : CB_PUT_FAILED;
    }
    __syncthreads();
    const long long end = min(tokens + total, (long long)a.tokens);
    for (long long n = tokens + (long long)rank * kPlanThreads + tid; n < end;
         n += (long long)ctas * kPlanThreads) {
      const int i = find_row(start, kPlanThreads, n);
      const long long pos = len_s[i] + (n - start[i]);
      long long slot = -1;
      if (held_s[i] >= 0) {
        const long long col = pos / ps;
        int32_t *entry = a.block_table + (r0 + i) * a.table_stride + col;
        int page;
        if (col < held_s[i]) {
          page = *entry;
        } else {
          page = a.free[count - 1 - (base[i] + col - held_s[i])];
          if (pos == col * ps) *entry = page;  // the first token of a new page
        }
        if (page >= 0 && page < a.num_pages) slot = (long long)page * ps + (pos - col * ps);
        else kv4_error(a.errors, kErrBounds);
      }
      a.slots[n] = slot;
      a.positions[n] = (int)min(pos, 0x7fffffffll);
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
// A thread holds 8 adjacent dimensions of one token's keys or values of one
// head, so a row of D values is D/8 adjacent lanes: the group's minimum and
// maximum are shuffles among group/8 of them, and the word of codes of K is
// one lane's own. A 16-bit word of V collects a nibble from each of four
// adjacent lanes (dims 8 apart), which they exchange by shuffles.

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

struct TokenStrides {
  int64_t k_token, k_head, v_token, v_head;
};

constexpr int kTokenThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kTokenThreads)
    kv4_append_kernel(const Kv4View c, const int group, const T *__restrict__ k, const T *__restrict__ v,
                      const TokenStrides st, const bool vec, const int64_t *__restrict__ slots, const int n) {
  constexpr int kLanes = D / 8, kWords = (D < 128 ? D : 128) / 32;
  const int64_t rows = (int64_t)n * 2 * c.kv_heads;
  const int64_t id = (int64_t)blockIdx.x * kTokenThreads + threadIdx.x;
  int64_t row = id / kLanes;
  const int lane = (int)(id % kLanes);
  const bool there = row < rows;
  if (!there) row = rows - 1;  // every lane of a warp takes part in the shuffles
  const int head = (int)(row % c.kv_heads);
  const int64_t tk = row / c.kv_heads;
  const bool is_v = tk & 1;
  const int64_t token = tk >> 1;

  float x[8];
  const T *src = is_v ? v + token * st.v_token + head * st.v_head : k + token * st.k_token + head * st.k_head;
  load8(src + lane * 8, vec, x);
  // fmin/fmax drop a NaN; a sum that is NaN keeps it (the values are finite otherwise)
  float lo = INFINITY, hi = -INFINITY, nan = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (x[i] != x[i]) nan = x[i];
    x[i] = fminf(fmaxf(x[i], -kKv4Most), kKv4Most);
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
  for (int o = 1; o < group / 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    nan += __shfl_xor_sync(0xffffffffu, nan, o);
  }
  const __half scale_h = __float2half_rn(__fadd_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f), nan));
  const float s = __half2float(scale_h);
  const __half offset_h = __float2half_rn(__fadd_rn(lo, __fmul_rn(8.0f, s)));
  const float o = __half2float(offset_h);
  const float step = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
  uint32_t code[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = s > 0.0f ? rintf(__fmul_rn(__fsub_rn(x[i], o), step)) : 0.0f;
    code[i] = (uint32_t)((int)fminf(fmaxf(t, -8.0f), 7.0f) + 8);
  }

  const int64_t slot = there ? __ldg(slots + token) : -1;
  const int64_t page = slot >> c.page_log2;
  const bool ok = slot >= 0 && page < c.num_pages;
  if (slot >= 0 && !ok) kv4_error(c.errors, kErrBounds);
  const int in_page = (int)(slot & (c.page_size - 1)), tok = in_page % kKv4Tile;
  const int ng = D / group;
  uint8_t *tile = c.base + (ok ? page : 0) * c.page_stride + head * c.head_bytes +
                  (uint64_t)(in_page / kKv4Tile) * kv4_tile_bytes(D, group);
  const int slab = lane / (kWords * 4), i = lane % (kWords * 4) / 4, t = lane % 4;
  uint32_t word = 0;
  if (!is_v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) word |= code[e] << (4 * ((e & 1) * 4 + e / 2));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) word |= code[e] << (4 * e);
  }
  // V: nibbles g = 2t and 2t + 1 of the four lanes (dims 8 k + g)
  uint32_t p0 = 0, p1 = 0;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    const uint32_t w = __shfl_sync(0xffffffffu, word, (threadIdx.x & 28) + kk) >> (8 * t);
    p0 |= (w & 15u) << (4 * kk);
    p1 |= (w >> 4 & 15u) << (4 * kk);
  }
  if (!ok) return;
  if (!is_v) {
    *reinterpret_cast<uint32_t *>(tile + 4 * (((slab * 16 + tok) * 4 + t) * kWords + i)) = word;
  } else {
    const int p = tok / 8, vt = tok % 8 / 2, b = tok % 2;
    uint16_t *at = reinterpret_cast<uint16_t *>(tile + 8 * D) + (((slab * 2 + p) * 8 * 4 + vt) * kWords + i) * 2 + b;
    at[(2 * t) * 4 * kWords * 2] = (uint16_t)p0;
    at[(2 * t + 1) * 4 * kWords * 2] = (uint16_t)p1;
  }
  if (lane % (group / 8) == 0)
    reinterpret_cast<uint32_t *>(tile + 16 * D + (is_v ? 64 * ng : 0))[tok * ng + lane / (group / 8)] =
        (uint32_t)__half_as_ushort(scale_h) | (uint32_t)__half_as_ushort(offset_h) << 16;
}

template <typename T, int D>
__global__ void __launch_bounds__(kTokenThreads)
    kv4_read_kernel(const Kv4View c, const int group, T *__restrict__ k, T *__restrict__ v, const bool vec,
                    const int64_t *__restrict__ slots, const int n) {
  constexpr int kLanes = D / 8, kWords = (D < 128 ? D : 128) / 32;
  const int64_t rows = (int64_t)n * 2 * c.kv_heads;
  const int64_t id = (int64_t)blockIdx.x * kTokenThreads + threadIdx.x;
  int64_t row = id / kLanes;
  const int lane = (int)(id % kLanes);
  const bool there = row < rows;
  if (!there) row = rows - 1;
  const int head = (int)(row % c.kv_heads);
  const int64_t tk = row / c.kv_heads;
  const bool is_v = tk & 1;
  const int64_t token = tk >> 1;
  const int64_t slot = __ldg(slots + token);
  const int64_t page = slot >> c.page_log2;
  const bool ok = slot >= 0 && page < c.num_pages;
  if (there && slot >= 0 && !ok) kv4_error(c.errors, kErrBounds);
  const int in_page = (int)(slot & (c.page_size - 1)), tok = in_page % kKv4Tile;
  const int ng = D / group;
  const uint8_t *tile = c.base + (ok ? page : 0) * c.page_stride + head * c.head_bytes +
                        (uint64_t)(ok ? in_page / kKv4Tile : 0) * kv4_tile_bytes(D, group);
  const int slab = lane / (kWords * 4), i = lane % (kWords * 4) / 4, t = lane % 4;
  uint32_t word = 0, p0 = 0, p1 = 0;
  if (!is_v) {
    word = *reinterpret_cast<const uint32_t *>(tile + 4 * (((slab * 16 + tok) * 4 + t) * kWords + i));
  } else {
    const int p = tok / 8, vt = tok % 8 / 2, b = tok % 2;
    const uint16_t *at =
        reinterpret_cast<const uint16_t *>(tile + 8 * D) + (((slab * 2 + p) * 8 * 4 + vt) * kWords + i) * 2 + b;
    p0 = at[(2 * t) * 4 * kWords * 2];
    p1 = at[(2 * t + 1) * 4 * kWords * 2];
  }
  const uint32_t par = reinterpret_cast<const uint32_t *>(tile + 16 * D + (is_v ? 64 * ng : 0))[tok * ng + lane / (group / 8)];
  const float s = kv4_scale(par), o = kv4_offset(par);
  // V: lane t of the four holds nibbles of g = 2t, 2t + 1; it wants nibble t of every g
#pragma unroll
  for (int g2 = 0; g2 < 4; ++g2) {
    const uint32_t a = __shfl_sync(0xffffffffu, p0, (threadIdx.x & 28) + g2);
    const uint32_t b = __shfl_sync(0xffffffffu, p1, (threadIdx.x & 28) + g2);
    if (is_v) word |= (a >> (4 * t) & 15u) << (8 * g2) | (b >> (4 * t) & 15u) << (8 * g2 + 4);
  }
  if (!there) return;
  T y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int nib = is_v ? e : (e & 1) * 4 + e / 2;
    y[e] = ok ? kv4_round<T>(kv4_value(word >> (4 * nib) & 15u, s, o)) : kv4_round<T>(0.0f);
  }
  T *dst = (is_v ? v : k) + (token * c.kv_heads + head) * D + lane * 8;
  if (vec) {
#pragma unroll
    for (int w = 0; w < (int)sizeof(T) / 2; ++w)
      reinterpret_cast<uint4 *>(dst)[w] = *reinterpret_cast<const uint4 *>(y + w * (16 / sizeof(T)));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) dst[e] = y[e];
  }
}

template <typename T, int D>
cudaError_t launch_append(const Kv4View &c, int group, const void *k, const void *v, const TokenStrides &st,
                          const int64_t *slots, int n, cudaStream_t stream) {
  const uint64_t threads = (uint64_t)n * 2 * c.kv_heads * (D / 8);
  const uint64_t unit = 16 / sizeof(T);
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 &&
                   ((st.k_token | st.k_head | st.v_token | st.v_head) & (int64_t)(unit - 1)) == 0;
  kv4_append_kernel<T, D><<<(unsigned)((threads + kTokenThreads - 1) / kTokenThreads), kTokenThreads, 0, stream>>>(
      c, group, static_cast<const T *>(k), static_cast<const T *>(v), st, vec, slots, n);
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t launch_read(const Kv4View &c, int group, void *k, void *v, const int64_t *slots, int n,
                        cudaStream_t stream) {
  const uint64_t threads = (uint64_t)n * 2 * c.kv_heads * (D / 8);
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  kv4_read_kernel<T, D><<<(unsigned)((threads + kTokenThreads - 1) / kTokenThreads), kTokenThreads, 0, stream>>>(
      c, group, static_cast<T *>(k), static_cast<T *>(v), vec, slots, n);
  return cudaGetLastError();
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

// The last grid index of a launch over n tokens has to stay inside 31 bits.
bool tokens_fit(const cb_kv4_cache *c, int32_t n) {
  return (uint64_t)n * 2 * c->kv_heads * (c->head_dim / 8) / kTokenThreads < 0x7fffffffull;
}

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
  while (ctas < kPlanCtas && a->tokens > ctas * 2 * kPlanThreads) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_plan_kernel, *a, ctas);
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
  if (!tokens_fit(cache, n)) return kv4_fail(CB_ERR_ARG, "cb_kv4_append: too many tokens in one call");
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
  if (!tokens_fit(cache, n)) return kv4_fail(CB_ERR_ARG, "cb_kv4_read: too many tokens in one call");
  if (n == 0) return CB_OK;
  Kv4Device dev(cache->device);
  if (dev.err != cudaSuccess) return kv4_fail(CB_ERR_CUDA, "cb_kv4_read: device", dev.err);
  const cudaError_t e = by_form(dtype, cache->head_dim, [&](auto t, auto d) {
    return launch_read<decltype(t), decltype(d)::value>(c, cache->group, k_out, v_out, slots, n,
                                                        static_cast<cudaStream_t>(stream));
  });
  return e == cudaSuccess ? CB_OK : kv4_fail(CB_ERR_CUDA, "cb_kv4_read: launch", e);
}
