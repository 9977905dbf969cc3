// What the attention kernels over 4-bit pages share: their arguments, the line of
// work that they cut into equal pieces, and barriers with bounded waits.
//
// An item is (request, row tile, KV head): L::kRows rows (query row x query head of
// the KV head) against the request's tokens in tiles of L::kTokens. The tiles of all
// items, in that order, are one long line, on which every item takes L::kCost more
// than its tiles, for what it costs beside them. Pieces of equal length go to the
// warps or blocks (L::kBlock) of a launch, whatever the lengths of the requests are,
// which only the device knows.
#pragma once

#include <atomic>
#include <type_traits>

#include "kv4.cuh"

namespace cb {

constexpr float kSlack = 8.0f;  // p may reach 2^8 before a running maximum is raised
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint64_t kWaitNs = 2000000000ull;  // the longest wait on a barrier
// How an item's parts are joined: not at all, a warp for 16 dims, a block for them.
constexpr int kJoinNone = 0, kJoinFew = 1, kJoinMany = 2;

struct AttendArgs {
  const void *q;
  void *out;
  float *lse;
  const int32_t *block_table, *kv_lens, *q_start;
  int64_t table_stride, q_token_stride, q_head_stride;
  float *parts;  // partial sums: two per piece
  // Of the item that a piece begins and does not end: its first query row, row
  // tile, head and rows; twice its number of parts, plus the place of its first;
  // and how its parts are joined (kJoin*).
  int4 *joins;
  int *join_n;
  uint8_t *join_how;
  float scale;
  int32_t requests, columns, total_q, q_heads, ratio, causal, bf16, q_vec;
  int32_t rows_above, rows_most;  // a kernel takes the requests with rows_above < rows <= rows_most
  int32_t min_share;              // of the line, for a piece
  int32_t fill;                   // CB_KV4_FILL_*
};

// What an item is: request b, row tile rt, KV head h, and its token tiles.
struct Item {
  int b, rt, h;
  int q0, qn, len;  // the request's rows and tokens
  int tiles;        // at least 1: a row tile that sees nothing still writes zeros
};

// Grid and workspace of a launch.
struct Launch {
  int rows;  // of a row tile
  int sms, pieces;
  int part;  // floats of a partial result
};

// Lets a kernel use `bytes` of shared memory on the current device, once for each.
template <typename K>
cudaError_t allow_shared(K kernel, int bytes, std::atomic<uint64_t> &ready) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (ready.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

inline uint64_t launch_bytes(const Launch &l) {
  return ((uint64_t)l.pieces * (sizeof(int4) + 2ull * sizeof(float) * l.part + sizeof(int) + 1) + 16 + 15) / 16 * 16;
}

inline void launch_arrays(const Launch &l, void *at, AttendArgs &a) {
  a.joins = static_cast<int4 *>(at);
  a.parts = reinterpret_cast<float *>(a.joins + l.pieces);
  a.join_n = reinterpret_cast<int *>(a.parts + (uint64_t)l.pieces * 2 * l.part);
  a.join_how = reinterpret_cast<uint8_t *>(a.join_n + l.pieces);
}

// Prompt chunks: more rows of a request than the few-row kernel takes (kv4_prompt.cu).
Launch prompt_launch(int head_dim, int sms);
cudaError_t run_prompt(const Kv4View &c, const AttendArgs &a, int head_dim, int group, const Launch &l,
                       cudaStream_t stream);

CB_D uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

CB_D void bar_init(uint32_t bar, uint32_t n) { asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(bar), "r"(n)); }

// Waits for a phase, two seconds at most; false if it did not come.
CB_D bool bar_wait(uint32_t bar, uint32_t parity) {
  uint64_t since = 0;
  for (uint32_t i = 0;; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((i & 63) == 63) {
      uint64_t now;
      asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
      if (!since) since = now;
      else if (now - since > kWaitNs) return false;
    }
  }
}

CB_D float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int N>
CB_D void load_words(const uint8_t *p, uint32_t *w) {
  if constexpr (N == 1) w[0] = *reinterpret_cast<const uint32_t *>(p);
  if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x, w[1] = v.y;
  }
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4 *>(p + 16 * i);
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  }
}

// The rows [q0, q0 + qn) of request b, inside [0, total_q), and its tokens.
CB_D void load_request(const AttendArgs &a, int most, int b, int &q0, int &qn, int &len) {
  if (!a.q_start) {
    q0 = b;
    qn = 1;
  } else {
    q0 = min(max(__ldg(a.q_start + b), 0), a.total_q);
    qn = min(max(__ldg(a.q_start + b + 1), q0), a.total_q) - q0;
  }
  if (qn * a.ratio <= a.rows_above || qn * a.ratio > a.rows_most) qn = 0;
  len = min(max(__ldg(a.kv_lens + b), 0), most);
}

// Tokens that row r (of qn * ratio) of a request sees.
CB_D int row_limit(const AttendArgs &a, const Item &it, int r) {
  return a.causal ? it.len - (it.qn - 1 - r / a.ratio) : it.len;
}

// The row of out (and lse) of a request's row r.
CB_D int64_t out_row(const AttendArgs &a, const Item &it, int r) {
  return (int64_t)(it.q0 + r / a.ratio) * a.q_heads + it.h * a.ratio + r % a.ratio;
}

CB_D uint32_t pack2(int bf16, float lo, float hi) {
  if (bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

template <typename L>
CB_D void item_tiles(const AttendArgs &a, Item &it) {
  const int last = min((it.rt + 1) * L::kRows, it.qn * a.ratio) - 1;
  it.tiles = max(1, (row_limit(a, it, last) + L::kTokens - 1) / L::kTokens);
}

// What all items of request b take of the line.
template <typename L>
CB_D long long request_tiles(const AttendArgs &a, int heads, int most, int b) {
  Item it;
  load_request(a, most, b, it.q0, it.qn, it.len);
  long long n = 0;
  const int rts = (it.qn * a.ratio + L::kRows - 1) / L::kRows;
  for (it.rt = 0; it.rt < rts; ++it.rt) {
    item_tiles<L>(a, it);
    n += it.tiles + L::kCost;
  }
  return n * heads;
}

// The item behind `it`; false behind the last.
template <typename L>
CB_D bool next_item(const AttendArgs &a, int heads, int most, Item &it) {
  if (++it.h < heads) return true;
  it.h = 0;
  ++it.rt;
  while (it.rt * L::kRows >= it.qn * a.ratio) {
    it.rt = 0;
    if (++it.b >= a.requests) return false;
    load_request(a, most, it.b, it.q0, it.qn, it.len);
  }
  item_tiles<L>(a, it);
  return true;
}

// a / b for b > 0, a >= 0, without the long division where both are short.
CB_D long long quotient(long long a, int b) {
  return a >> 31 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}

// Inclusive prefix sum over the block, and the block's sum. `sums` has an entry
// for each warp and may not be in use.
template <int WARPS>
CB_D long long block_scan(long long v, long long *sums, long long &all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) v += sums[w];
    all += sums[w];
  }
  return v;
}

// find_piece for more requests than a warp has lanes: prefix sums over the block.
template <typename L>
CB_D void find_among_many(const AttendArgs &a, const Kv4View &c, int most, long long *sums, long long *ends, int pieces,
                          long long place, long long &share, long long &f0, long long &f1, long long &first, Item &it,
                          bool &found) {
  constexpr int kWarps = L::kWarps, kThreads = kWarps * 32;
  const int lane = threadIdx.x & 31;
  long long total = 0, mine = 0;
  for (int b = threadIdx.x; b < a.requests; b += kThreads) {
    mine = request_tiles<L>(a, c.kv_heads, most, b);
    total += mine;
    const int len = __ldg(a.kv_lens + b);
    if (blockIdx.x == 0 && (len < 0 || len > most)) kv4_error(c.errors, kErrBounds);
  }
  const bool once = a.requests <= kThreads;  // a thread has a request at most
  long long chunk, v = block_scan<kWarps>(total, sums, chunk);
  total = chunk;
  share = max(quotient(total + pieces - 1, pieces), (long long)a.min_share);
  f0 = place * share;
  f1 = min(f0 + share, total);
  long long before = 0;
  for (int b0 = 0; b0 < a.requests; b0 += kThreads) {
    if (!once) {
      const int b = b0 + threadIdx.x;
      v = before + block_scan<kWarps>(b < a.requests ? request_tiles<L>(a, c.kv_heads, most, b) : 0,
                                      sums + (b0 / kThreads + 1 & 1) * kWarps, chunk);
    }
    ends[threadIdx.x] = v;
    __syncthreads();
    if (!found && f0 < before + chunk) {  // the first request that ends behind f0
      int n = 0;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) n += ends[i * 32 + lane] <= f0;
      n = __reduce_add_sync(0xffffffffu, n);
      it.b = b0 + n;
      first = n ? ends[n - 1] : before;
      found = true;
    }
    before += chunk;
    if (!once) __syncthreads();
  }
}

// Finds the warp's piece [f0, f1) of the line (the block's, if L::kBlock) and the
// item that holds f0, which begins at `first`; false if there is nothing left for
// it. Neighbouring pieces are on different SMs, so that a short line is spread
// over all of them. All threads of the block call; `sums` has two entries for
// each warp, `ends` one for each thread, in shared memory.
template <typename L>
CB_D bool find_piece(const AttendArgs &a, const Kv4View &c, int most, long long *sums, long long *ends,
                     long long &share, long long &f0, long long &f1, long long &first, Item &it) {
  constexpr int kWarps = L::kWarps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pieces = gridDim.x * (L::kBlock ? 1 : kWarps);
  const long long place = (L::kBlock ? 0 : warp * gridDim.x) + blockIdx.x;
  bool found = false;
  if (a.requests <= 32) {  // every warp for itself, a lane to a request: no barriers
    long long v = 0;
    if (lane < a.requests) {
      v = request_tiles<L>(a, c.kv_heads, most, lane);
      const int len = __ldg(a.kv_lens + lane);
      if (blockIdx.x == 0 && warp == 0 && (len < 0 || len > most)) kv4_error(c.errors, kErrBounds);
    }
    for (int o = 1; o < a.requests; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += y;
    }
    const long long total = __shfl_sync(0xffffffffu, v, a.requests - 1);
    share = max(quotient(total + pieces - 1, pieces), (long long)a.min_share);
    f0 = place * share;
    f1 = min(f0 + share, total);
    const int n = __popc(__ballot_sync(0xffffffffu, lane < a.requests && v <= f0));
    it.b = n;
    first = __shfl_sync(0xffffffffu, v, max(n - 1, 0));
    if (n == 0) first = 0;
    found = f0 < total;
  } else {
    find_among_many<L>(a, c, most, sums, ends, pieces, place, share, f0, f1, first, it, found);
  }
  if (!found || f0 >= f1) return false;
  load_request(a, most, it.b, it.q0, it.qn, it.len);
  for (it.rt = 0;; ++it.rt) {
    item_tiles<L>(a, it);
    const long long n = (long long)(it.tiles + L::kCost) * c.kv_heads;
    if (f0 < first + n) break;
    first += n;
  }
  it.h = (int)quotient(f0 - first, it.tiles + L::kCost);
  first += (long long)it.h * (it.tiles + L::kCost);
  return true;
}

// A piece of the line, item by item: the item and its tiles [t0, t1) in the
// piece. Positions count from the piece's beginning.
struct Walk {
  Item it;
  int at;  // of the item's first tile; not positive if it began in an earlier piece
  int t0, t1;
  CB_D void cut(int units) {
    t0 = max(0, -at);
    t1 = min(it.tiles, units - at);
  }
};

// The next item of the piece that has tiles in it; false behind the last.
template <typename L>
CB_D bool next_in_piece(const AttendArgs &a, int heads, int most, int units, Walk &w) {
  do {
    w.at += w.it.tiles + L::kCost;
    if (w.at >= units || !next_item<L>(a, heads, most, w.it)) return false;
    w.cut(units);
  } while (w.t1 <= w.t0);
  return true;
}

}  // namespace cb
