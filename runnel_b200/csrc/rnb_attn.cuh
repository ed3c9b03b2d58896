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
  int B, T, W, Hq, Hkv, group, log2p, num_pages, window, max_kv;
  int direct;    // few-row kernel: whole tiles by number (one row a request)
  int split;     // many-row kernel: CTAs over which the tiles' positions are split (0: not)
  int few_rows;  // requests with rows * group below this are the few-row kernel's
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

// Four consecutive elements of one output row: o / l, times sigmoid(gate) (gw:
// the four gate elements), rounded once; the row's lse = ln 2 (m + log2 l) from
// the thread with d == 0.
template <typename T, int D>
__device__ __forceinline__ void attn_write_row(const AttnArgs& a, int t, int head, int d, float4 o, float m, float l,
                                               uint2 gw) {
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  float v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  if (a.gate) {
    const float2 g0 = Pair<T>::unpack(gw.x), g1 = Pair<T>::unpack(gw.y);
    v[0] = __fdividef(v[0], 1.f + __expf(-g0.x)), v[1] = __fdividef(v[1], 1.f + __expf(-g0.y));
    v[2] = __fdividef(v[2], 1.f + __expf(-g1.x)), v[3] = __fdividef(v[3], 1.f + __expf(-g1.y));
  }
  const int64_t row = static_cast<int64_t>(t) * a.Hq + head;
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + row * D + d) =
      make_uint2(Pair<T>::pack(v[0], v[1]), Pair<T>::pack(v[2], v[3]));
  if (a.lse && d == 0) a.lse[row] = l > 0.f ? 0.6931471805599453f * (m + log2f(l)) : -INFINITY;
}

}  // namespace rnb
