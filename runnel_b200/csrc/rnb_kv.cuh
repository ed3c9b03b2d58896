// rnb_kv.cuh -- what the attention-side units (page plan, rotary append,
// paged attention) share: checks of a cache descriptor and the 16-bit types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "rnb_common.cuh"
#include "rnb_internal.h"
#include "rnb_moe.h"

namespace rnb {

// RNB_OK, or an error with its message: shapes, strides and alignment of a
// paged cache.
inline int check_cache(const rnb_kv_cache* c, const char* fn) {
  const std::string f = std::string(fn) + ": ";
  if (!c) return fail(RNB_ERR_INVALID, f + "the cache must be non-NULL");
  if (c->dtype != RNB_DTYPE_BF16 && c->dtype != RNB_DTYPE_F16)
    return fail(RNB_ERR_INVALID, f + "the cache's dtype must be RNB_DTYPE_BF16 or RNB_DTYPE_F16");
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(RNB_ERR_INVALID, f + "head_dim must be 64, 128 or 256");
  const int P = c->page_size;
  if (P < 16 || P > 256 || (P & (P - 1)))
    return fail(RNB_ERR_INVALID, f + "page_size must be 16, 32, 64, 128 or 256");
  if (c->num_pages <= 0 || c->n_kv_heads <= 0 || c->n_kv_heads > 65535)
    return fail(RNB_ERR_INVALID, f + "num_pages must be positive and n_kv_heads in [1, 65535]");
  if (static_cast<int64_t>(c->num_pages) * P > INT32_MAX)
    return fail(RNB_ERR_INVALID, f + "num_pages * page_size must be below 2^31");
  if (!c->k || !c->v) return fail(RNB_ERR_INVALID, f + "cache k and v must be non-NULL");
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(RNB_ERR_ALIGN, f + "cache k and v must be 16-byte aligned");
  const int64_t st[4] = {c->k_page_stride, c->k_head_stride, c->v_page_stride, c->v_head_stride};
  for (int64_t v : st)
    if (v < 0 || v % 8) return fail(RNB_ERR_INVALID, f + "cache strides must be multiples of 8 elements");
  return RNB_OK;
}

// Whether a packed output [T][H][D] of 16-bit elements shares memory with rows
// (T tokens, `heads` heads of D elements, strides >= 0 in elements).  Row by row
// where the ranges as a whole overlap: an output may lie in the gaps.
inline bool shares_memory(const void* out, int64_t T, int64_t H, int64_t D, const void* rows, int64_t token_stride,
                          int64_t head_stride, int64_t heads) {
  const uintptr_t o0 = reinterpret_cast<uintptr_t>(out), o1 = o0 + 2 * T * H * D;
  auto meets = [&](int64_t from, int64_t n) {  // n elements from `from` on
    const uintptr_t r0 = reinterpret_cast<uintptr_t>(rows) + 2 * from;
    return r0 < o1 && r0 + 2 * n > o0;
  };
  const int64_t token = (heads - 1) * head_stride + D;
  if (!rows || T == 0 || heads == 0 || !meets(0, (T - 1) * token_stride + token)) return false;
  for (int64_t t = 0; t < T; ++t)
    if (meets(t * token_stride, token))
      for (int64_t h = 0; h < heads; ++h)
        if (meets(t * token_stride + h * head_stride, D)) return true;
  return false;
}

// A launch whose grid may come up while the kernel before it in the stream ends
// (programmatic dependent launch; 1 us less between two small kernels).  Every
// kernel launched so waits for that one (griddep_wait) before anything else, its
// early returns included, so that "this grid is done" still means that all before
// it are.
template <typename... P, typename... A>
inline int launch(const char* what, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                  const A&... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return fail(RNB_ERR_CUDA, std::string(what) + " launch: " + cudaGetErrorString(e));
  return RNB_OK;
}

// First thing in such a kernel.
__device__ __forceinline__ void after_previous() {
  griddep_wait();
  griddep_launch_dependents();
}

// The address on the current device of each unit's status word, which its kernels
// set bits of (atomicOr) and rnb_kv_status takes.
cudaError_t rope_status_word(uint32_t** p);
cudaError_t attn_status_word(uint32_t** p);
cudaError_t prompt_status_word(uint32_t** p);
// The many-row kernel's word for the call that gave up, which a status read clears.
cudaError_t prompt_gave_up_word(uint32_t** p);

template <typename Sym>
inline cudaError_t status_word(Sym& word, uint32_t** p) {
  return cudaGetSymbolAddress(reinterpret_cast<void**>(p), word);
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
        "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}

// The two 16-bit types: packing (round to nearest even) and unpacking of pairs.
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
};
template <>
struct Pair<__half> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
};

}  // namespace rnb
