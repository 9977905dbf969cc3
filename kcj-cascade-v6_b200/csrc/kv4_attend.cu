// Attention over a paged KV cache held in 4 bits (cb_kv4_attend). Format:
// kv4.cuh.
//
//   out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q.k_t - max)
//
// in one pass over a row's tokens with the running maximum and sum.
#include "kv4.cuh"

namespace cb {

namespace {

struct AttendArgs {
  const void *q;
  void *out;
  float *lse;
  const int32_t *block_table, *kv_lens, *q_start;
  int64_t table_stride, q_token_stride, q_head_stride;
  float scale;
  int32_t requests, columns, total_q, q_heads, causal, group;
};

// The rows [q0, q1) of request r, inside [0, total_q).
CB_D void request_rows(const AttendArgs &a, int r, int &q0, int &q1) {
  if (!a.q_start) {
    q0 = r;
    q1 = r + 1;
  } else {
    q0 = min(max(a.q_start[r], 0), a.total_q);
    q1 = min(max(a.q_start[r + 1], q0), a.total_q);
  }
}

// One warp per (row, head): 32 tokens at a time, a lane for each while scores
// are taken, then a share of the dimensions for each while values are summed.
template <typename T, int D>
__global__ void __launch_bounds__(128) attend_kernel(const Kv4View c, const AttendArgs a) {
  constexpr int kWords = (D < 128 ? D : 128) / 32, kMine = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int row = (int)(id / a.q_heads), head = (int)(id % a.q_heads);
  if (row >= a.total_q) return;
  int r = 0, q0 = 0, q1 = 0;
  for (; r < a.requests; ++r) {
    request_rows(a, r, q0, q1);
    if (row >= q0 && row < q1) break;
  }
  if (r == a.requests) return;
  const int kvh = head / (a.q_heads / c.kv_heads), ng = D / a.group;
  const int64_t most = (int64_t)a.columns * c.page_size;
  int64_t len = a.kv_lens[r];
  if (len < 0 || len > most) {
    kv4_error(c.errors, kErrBounds);
    len = len < 0 ? 0 : most;
  }
  const int64_t limit = a.causal ? len - (q1 - 1 - row) : len;
  const T *q = static_cast<const T *>(a.q) + row * a.q_token_stride + head * a.q_head_stride;
  float m = -INFINITY, l = 0.0f, o[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) o[i] = 0.0f;
  for (int64_t t0 = 0; t0 < limit; t0 += 32) {
    const int64_t pos = t0 + lane;
    const uint8_t *tile = nullptr;
    if (pos < limit) {
      const int page = a.block_table[r * a.table_stride + (pos >> c.page_log2)];
      if (page >= 0 && page < c.num_pages)
        tile = c.base + page * c.page_stride + kvh * c.head_bytes +
               (uint64_t)((pos & (c.page_size - 1)) / kKv4Tile) * kv4_tile_bytes(D, a.group);
      else
        kv4_error(c.errors, kErrBounds);
    }
    const int tok = (int)(pos % kKv4Tile);
    float s = -INFINITY;
    if (tile) {
      s = 0.0f;
      const uint32_t *kw = reinterpret_cast<const uint32_t *>(tile);
      const uint32_t *par = reinterpret_cast<const uint32_t *>(tile + 16 * D) + tok * ng;
      for (int d = 0; d < D; ++d) {
        const int slab = d / 128, x = d % 128, i = x / 32, t = x % 32 / 8, n = x % 8;
        const uint32_t w = kw[((slab * 16 + tok) * 4 + t) * kWords + i];
        const uint32_t pr = par[d / a.group];
        s = fmaf(kv4_load1(q + d), kv4_value(w >> (4 * ((n & 1) * 4 + n / 2)) & 15u, kv4_scale(pr), kv4_offset(pr)), s);
      }
      s *= a.scale * 1.4426950408889634f;
    }
    float top = s;
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    // a NaN score makes the row NaN (fmaxf drops it)
    const float m2 = __any_sync(0xffffffffu, s != s) ? NAN : fmaxf(m, top);
    if (m2 == -INFINITY) continue;
    const float f = exp2f(m - m2);
    const float p = tile ? exp2f(s - m2) : 0.0f;
    m = m2;
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < kMine; ++i) o[i] *= f;
    for (int j = 0; j < 32; ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j);
      const uint64_t at = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(tile), j);
      if (!at) continue;
      const int tj = (int)((t0 + j) % kKv4Tile);
      const uint16_t *vw = reinterpret_cast<const uint16_t *>(at + 8 * D);
      const uint32_t *par = reinterpret_cast<const uint32_t *>(at + 16 * D + 64 * ng) + tj * ng;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int d = i * 32 + lane, slab = d / 128, x = d % 128;
        const uint32_t w = vw[((((slab * 2 + tj / 8) * 8 + x % 8) * 4 + tj % 8 / 2) * kWords + x / 32) * 2 + tj % 2];
        const uint32_t pr = par[d / a.group];
        o[i] = fmaf(pj, kv4_value(w >> (4 * (x % 32 / 8)) & 15u, kv4_scale(pr), kv4_offset(pr)), o[i]);
      }
    }
  }
  for (int x = 16; x; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  T *out = static_cast<T *>(a.out) + ((int64_t)row * a.q_heads + head) * D;
#pragma unroll
  for (int i = 0; i < kMine; ++i) out[i * 32 + lane] = kv4_round<T>(l > 0.0f ? o[i] / l : (l == 0.0f ? 0.0f : l));
  if (a.lse && lane == 0)
    a.lse[(int64_t)row * a.q_heads + head] = l == 0.0f ? -INFINITY : m * 0.6931471805599453f + logf(l);
}

int check(const cb_kv4_cache *cache, const cb_kv4_attend_args *a, Kv4View *c) {
  if (!a) return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: no arguments");
  if (int rc = kv4_check_cache(cache, a->layer, "cb_kv4_attend: no cache", c)) return rc;
  if (a->dtype != CB_KV4_F16 && a->dtype != CB_KV4_BF16)
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: q must be fp16 or bf16");
  if (a->requests < 0 || a->columns <= 0 || a->total_q < 0 || a->q_heads <= 0 || a->table_stride < a->columns)
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: bad sizes");
  if (a->q_heads % cache->kv_heads) return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: q_heads is not a multiple of kv_heads");
  if (!a->q_start && a->total_q != a->requests)
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: without q_start there is one row for each request");
  if ((long long)a->columns * cache->page_size > 0x7fffffffll)
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: a row may not hold more than 2^31 - 1 tokens");
  if (a->requests > 0 && a->total_q > 0 && (!a->q || !a->out || !a->block_table || !a->kv_lens))
    return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: missing array");
  return CB_OK;
}

}  // namespace

}  // namespace cb

extern "C" uint64_t cb_kv4_attend_workspace(const cb_kv4_cache *cache, const cb_kv4_attend_args *a) {
  (void)cache;
  (void)a;
  return 0;
}

extern "C" int cb_kv4_attend(const cb_kv4_cache *cache, const cb_kv4_attend_args *args, void *stream) {
  using namespace cb;
  Kv4View c;
  if (int rc = check(cache, args, &c)) return rc;
  if (args->requests == 0 || args->total_q == 0) return CB_OK;
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
  a.causal = args->causal;
  a.group = cache->group;
  const int64_t warps = (int64_t)a.total_q * a.q_heads;
  if ((warps + 3) / 4 > 0x7fffffff) return kv4_fail(CB_ERR_ARG, "cb_kv4_attend: too many rows");
  const unsigned grid = (unsigned)((warps + 3) / 4);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool half = args->dtype == CB_KV4_F16;
  if (cache->head_dim == 64) {
    if (half) attend_kernel<__half, 64><<<grid, 128, 0, st>>>(c, a);
    else attend_kernel<__nv_bfloat16, 64><<<grid, 128, 0, st>>>(c, a);
  } else if (cache->head_dim == 128) {
    if (half) attend_kernel<__half, 128><<<grid, 128, 0, st>>>(c, a);
    else attend_kernel<__nv_bfloat16, 128><<<grid, 128, 0, st>>>(c, a);
  } else {
    if (half) attend_kernel<__half, 256><<<grid, 128, 0, st>>>(c, a);
    else attend_kernel<__nv_bfloat16, 256><<<grid, 128, 0, st>>>(c, a);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? CB_OK : kv4_fail(CB_ERR_CUDA, "cb_kv4_attend: launch", e);
}
