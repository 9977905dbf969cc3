// The 4-bit page format of a paged KV cache (cb_kv4_*), device side.
//
// Every (page, layer, KV head) is a run of tiles of 16 tokens; a tile holds
//   K codes 8*D bytes | V codes 8*D | K params 64*D/group | V params 64*D/group
// with one fp16 pair (scale, offset) per token and group of dimensions:
//   x = offset + scale * (code - 8),  code in 0..15.
// Codes of a token depend on nothing but its own values, so equal tokens give
// equal page bytes whatever calls wrote them, and pages deduplicate by content.
//
// The order of the codes inside a tile is that of the operands of a 16x8x16
// matrix product, so that a lane reads its share with 16-byte loads and turns a
// word into operands with one shift and four ANDs (dims are split into slabs of
// SD = min(D, 128), and a nibble read as the low mantissa bits of an fp16 is the
// subnormal number code * 2^-24, or code * 2^-20 for the second nibble of a byte):
//   K (token, slab, dim 32 i + 8 t + 2 k + h): nibble 4 h + k of the 32-bit word
//     ((slab*16 + token)*4 + t)*(SD/32) + i   -- pairs of adjacent dims, the axis
//     that q.k sums over;
//   V (token 8 p + 2 t + b, slab, dim 32 j + 8 k + g): nibble k of the 16-bit word
//     ((((slab*2 + p)*8 + g)*4 + t)*(SD/32) + j)*2 + b   -- pairs of adjacent
//     tokens, the axis that p.v sums over.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace cb {

constexpr int kKv4Tile = 16;             // tokens of a tile
constexpr float kKv4Most = 65000.0f;     // larger values are stored as this one
constexpr long long kKv4MostTokens = 1 << 30;  // of a row of a block table: positions stay clear of 2^31

CB_HD int kv4_slab(int d) { return d < 128 ? d : 128; }
CB_HD int kv4_tile_bytes(int d, int group) { return 16 * d + 128 * (d / group); }
CB_HD uint64_t kv4_head_bytes(int d, int group, int page_size) {
  return (uint64_t)(page_size / kKv4Tile) * kv4_tile_bytes(d, group);
}

// A cache as the kernels see it: one layer of it.
struct Kv4View {
  uint8_t *base;         // first byte of the layer in page 0
  uint64_t page_stride;  // bytes from page to page
  uint64_t head_bytes;   // bytes from head to head inside a page
  unsigned *errors;      // device error word (kErr* bits), or NULL
  int32_t num_pages, kv_heads, page_size, page_log2;
};

CB_D void kv4_error(unsigned *errors, unsigned bit) {
  if (errors) atomicOr(errors, bit);
}

CB_D float kv4_scale(uint32_t par) { return __half2float(__ushort_as_half((unsigned short)(par & 0xffffu))); }
CB_D float kv4_offset(uint32_t par) { return __half2float(__ushort_as_half((unsigned short)(par >> 16))); }

// The value of a code. scale * (code - 8) is exact in fp32 (11 + 4 bits), so the
// fused form rounds once, as the separate one does. (2^23 | code is 2^23 + code.)
CB_D float kv4_value(uint32_t code, float scale, float offset) {
  return fmaf(scale, __uint_as_float(0x4b000000u | code) - 8388616.0f, offset);
}

template <typename T>
CB_D float kv4_load1(const T *p);
template <>
CB_D float kv4_load1(const float *p) { return __ldg(p); }
template <>
CB_D float kv4_load1(const __half *p) { return __half2float(__ldg(p)); }
template <>
CB_D float kv4_load1(const __nv_bfloat16 *p) { return __bfloat162float(__ldg(p)); }

template <typename T>
CB_D T kv4_round(float x);
template <>
CB_D float kv4_round(float x) { return x; }
template <>
CB_D __half kv4_round(float x) { return __float2half_rn(x); }
template <>
CB_D __nv_bfloat16 kv4_round(float x) { return __float2bfloat16_rn(x); }

// Host side shared by the entry points (kv4.cu).
int kv4_fail(int code, const char *msg, cudaError_t e = cudaSuccess);
int kv4_check_cache(const cb_kv4_cache *c, int32_t layer, const char *who, Kv4View *out);

// Launches a kernel and says how that launch went, whatever failed before it. `early`:
// it may begin before the kernel in front of it has ended, and waits for it itself.
template <typename... P, typename... A>
cudaError_t kv4_launch(void (*kernel)(P...), dim3 grid, int threads, size_t shared, cudaStream_t stream, bool early,
                       A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Makes `device` current for the life of the object.
struct Kv4Device {
  int prev = -1, want;
  cudaError_t err;
  explicit Kv4Device(int device) : want(device) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess && prev != want) err = cudaSetDevice(want);
  }
  ~Kv4Device() {
    if (prev >= 0 && prev != want) cudaSetDevice(prev);
  }
};

}  // namespace cb
