// rnb_attn.cuh -- arguments and the output epilogue of the paged-attention kernels.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "rnb_kv.cuh"

namespace rnb {

struct AttnArgs {
  const void *q, *gate, *kc, *vc;
  const int32_t *table, *seq, *cu;
  void* out;
  float* lse;
  char* ws;
  size_t ml_off, o_off;
  int64_t q_ts, q_hs, g_ts, g_hs, kc_ps, kc_hs, vc_ps, vc_hs;
  float scale_log2;  // scale * log2(e): softmax in powers of two
  uint32_t group_magic;  // for by_group
  int B, T, W, Hq, Hkv, group, group_shift, log2p, num_pages, window, max_kv;
  int direct;    // few-row kernel: whole tiles by number (one row a request)
  int split;     // many-row kernel: CTAs over which the tiles' positions are split (0: not)
  int few_rows;  // requests with rows * group below this are the few-row kernel's
  uint32_t call;  // many-row kernel: the call's number, not 0
};

// The many-row kernel (rnb_attn_prompt.cu): TMA maps of the call's tensors, and
// a launch for the requests with rows * group >= a.few_rows.  prepare_prompt is
// false where the kernel or the encoder does not take the layout.
struct PromptMaps {
  CUtensorMap k, v, q, gate, out;
  int k_box, v_box;  // cache rows a copy
  int tokens;        // tokens a row tile
};
int plan_split(AttnArgs* a, int D, int sms, size_t* bytes);
bool prepare_prompt(const AttnArgs& a, const rnb_kv_cache* c, PromptMaps* p);
int run_prompt(const AttnArgs& a, const rnb_kv_cache* c, const PromptMaps& p, cudaStream_t st);

template <typename T>
__device__ __forceinline__ const T* attn_gate(const AttnArgs& a, int t, int head) {
  return static_cast<const T*>(a.gate) + t * a.g_ts + head * a.g_hs;
}

// row / group for 0 <= row < 2^31 by a multiplication (an integer division is 35
// instructions, and these stand all over a short tile's start): with
// l = ceil(log2 group) and m = ceil(2^(31+l) / group) < 2^32 it is row m >> (31 + l),
// since m group exceeds 2^(31+l) by less than 2^l and row is below 2^31.
inline void set_group(AttnArgs* a, int group) {
  a->group = group;
  a->group_shift = 0;
  while ((1 << a->group_shift) < group) ++a->group_shift;
  a->group_magic = static_cast<uint32_t>(((1ull << (31 + a->group_shift)) + group - 1) / group);
}
__device__ __forceinline__ int by_group(const AttnArgs& a, int row) {
  return static_cast<int>(__umulhi(static_cast<uint32_t>(row) << 1, a.group_magic) >> a.group_shift);
}

// Four consecutive elements of one output row, times sigmoid(gate) (gw: the four
// gate elements) where there are gates, rounded once.
template <typename T, int D>
__device__ __forceinline__ void attn_write_four(const AttnArgs& a, int t, int head, int d, float4 o, uint2 gw) {
  if (a.gate) {
    const float2 g0 = Pair<T>::unpack(gw.x), g1 = Pair<T>::unpack(gw.y);
    o.x = __fdividef(o.x, 1.f + __expf(-g0.x)), o.y = __fdividef(o.y, 1.f + __expf(-g0.y));
    o.z = __fdividef(o.z, 1.f + __expf(-g1.x)), o.w = __fdividef(o.w, 1.f + __expf(-g1.y));
  }
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (static_cast<int64_t>(t) * a.Hq + head) * D + d) =
      make_uint2(Pair<T>::pack(o.x, o.y), Pair<T>::pack(o.z, o.w));
}

__device__ __forceinline__ void attn_write_lse(const AttnArgs& a, int t, int head, float m, float l) {
  if (a.lse)
    a.lse[static_cast<int64_t>(t) * a.Hq + head] = l > 0.f ? 0.6931471805599453f * (m + log2f(l)) : -INFINITY;
}

// The same for parts already summed: o / l, and the row's lse from the thread with d == 0.
template <typename T, int D>
__device__ __forceinline__ void attn_write_row(const AttnArgs& a, int t, int head, int d, float4 o, float m, float l,
                                               uint2 gw) {
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  attn_write_four<T, D>(a, t, head, d, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), gw);
  if (d == 0) attn_write_lse(a, t, head, m, l);
}

}  // namespace rnb
