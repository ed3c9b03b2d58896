// rnb_rope.cu -- per-head RMSNorm, rotary positions with several axes, and
// the append of a step's keys and values to the paged cache (rnb_rope_append).
//
// One pass: a head's row is read once with 16-byte loads (D/8 lanes hold it,
// so the norm's sum is a few shuffles and the partner of element i, i +- rot/2,
// is 8 elements in another lane), turned in fp32 and written once, rounded
// once.  HBM bounds it: 4 (Hq + 2 Hkv) D bytes a token.
//
// Angles: fp32 loses far positions (position 10^5 at frequency 1 is off by
// 2^-8 rad), so position * frequency and its reduction to half turns are fp64,
// and sincospif works on the small remainder.  That is rot/2 evaluations a
// token for all its heads: a CTA computes those of its tokens once into shared
// memory and serves all heads from there.
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "rnb_kv.cuh"

namespace rnb {
namespace {

constexpr int kRopeThreads = 256;

__device__ uint32_t g_rope_status;

struct RopeArgs {
  const void *q, *k, *v, *qw, *kw;
  const int32_t* pos;
  const float* inv_freq;
  const int32_t* slots;
  void *q_out, *kc, *vc;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, kc_ps, kc_hs, vc_ps, vc_hs;
  float eps;
  int T, Hq, Hkv, half, tok, log2p, heads_per_cta;
  int n_axes, interleaved, sec[4];
  uint32_t num_slots;
};

__device__ __forceinline__ int axis_of(const RopeArgs& a, int i) {
  int ax = 0;
  if (a.interleaved) {
    const int r = i % a.n_axes;
    if (r && i < a.n_axes * a.sec[r]) ax = r;
  } else {
    int end = a.sec[0];
    while (ax + 1 < a.n_axes && i >= end) end += a.sec[++ax];
  }
  return ax;
}

// Heads are numbered queries first, then keys, then values.  CTA (x, y) takes
// tokens [x tok, (x + 1) tok) and heads [y heads_per_cta, ...) of each.
template <typename T, int D>
__global__ void __launch_bounds__(kRopeThreads) k_rope_append(const RopeArgs a) {
  constexpr int kLanes = D / 8;                      // lanes holding one head's row
  constexpr int kGroups = kRopeThreads / kLanes;     // rows in flight in the CTA
  __shared__ float2 cs[kRopeThreads];                // [tok][half] cos, sin
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * a.tok;
  const int nt = min(a.tok, a.T - t0);
  for (int i = tid; i < nt * a.half; i += kRopeThreads) {
    const int t = i / a.half, f = i - t * a.half;
    const double p = static_cast<double>(a.pos[static_cast<int64_t>(axis_of(a, f)) * a.T + t0 + t]);
    // in half turns; the fp64 remainder of whole turns is exact to 2^-52 of the angle
    double turns = p * static_cast<double>(a.inv_freq[f]) * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif(static_cast<float>(2.0 * turns), &s, &c);
    cs[i] = make_float2(c, s);
  }
  __syncthreads();

  const int lane = tid % kLanes, e0 = lane * 8;
  const int heads = a.Hq + 2 * a.Hkv;
  const int h0 = blockIdx.y * a.heads_per_cta, nh = min(a.heads_per_cta, heads - h0);
  // a warp's lanes all run the same number of rounds (shuffles below)
  const int rows = nt * nh;
  const int rounds = (rows + kGroups - 1) / kGroups;
  // where this lane's pairs are: the lane that holds elements e0 +- half
  const bool lo = e0 < a.half, turned = e0 < 2 * a.half;
  const int partner = turned ? (lo ? lane + a.half / 8 : lane - a.half / 8) : lane;
  const int src = (tid & 31) - lane + partner;
  for (int r = 0; r < rounds; ++r) {
    const int row = r * kGroups + tid / kLanes;
    const bool in = row < rows;
    const int tl = in ? row / nh : 0, h = h0 + (in ? row - tl * nh : 0), t = t0 + tl;
    const int slot = a.slots ? a.slots[t] : 0;
    const bool is_q = h < a.Hq, is_k = !is_q && h < a.Hq + a.Hkv;
    const int hk = is_q ? h : (h - a.Hq) - (is_k ? 0 : a.Hkv);
    const T* from = is_q   ? static_cast<const T*>(a.q) + t * a.q_ts + h * a.q_hs
                    : is_k ? static_cast<const T*>(a.k) + t * a.k_ts + hk * a.k_hs
                           : static_cast<const T*>(a.v) + t * a.v_ts + hk * a.v_hs;
    const bool live = in && slot >= 0 && (is_q || static_cast<uint32_t>(slot) < a.num_slots);
    if (in && slot >= 0 && !is_q && !live && lane == 0) atomicOr(&g_rope_status, RNB_STATUS_BAD_INDEX);
    uint4 w = make_uint4(0, 0, 0, 0);
    if (live) w = __ldcs(reinterpret_cast<const uint4*>(from + e0));  // coherent: q_out may be q
    uint32_t u[4] = {w.x, w.y, w.z, w.w};
    const T* nw = static_cast<const T*>(is_q ? a.qw : a.kw);
    const bool is_v = !is_q && !is_k;
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Pair<T>::unpack(u[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (nw && !is_v) {
      const float sc = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
      const uint4 g = __ldg(reinterpret_cast<const uint4*>(nw + e0));
      const uint32_t gu[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Pair<T>::unpack(gu[i]);
        x[2 * i] *= sc * f.x;
        x[2 * i + 1] *= sc * f.y;
      }
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], src);
    if (!is_v && turned) {
      const float2* c = cs + tl * a.half + (lo ? e0 : e0 - a.half);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 v = c[i];
        x[i] = lo ? x[i] * v.x - y[i] * v.y : x[i] * v.x + y[i] * v.y;
      }
    }
    if (live) {
      uint4 o = w;
      if (!is_v)
        o = make_uint4(Pair<T>::pack(x[0], x[1]), Pair<T>::pack(x[2], x[3]), Pair<T>::pack(x[4], x[5]),
                       Pair<T>::pack(x[6], x[7]));
      T* to;
      if (is_q) {
        to = static_cast<T*>(a.q_out) + (static_cast<int64_t>(t) * a.Hq + h) * D;
      } else {
        const int64_t page = slot >> a.log2p, off = (slot & ((1 << a.log2p) - 1)) * D;
        to = is_k ? static_cast<T*>(a.kc) + page * a.kc_ps + hk * a.kc_hs + off
                  : static_cast<T*>(a.vc) + page * a.vc_ps + hk * a.vc_hs + off;
      }
      *reinterpret_cast<uint4*>(to + e0) = o;
    }
  }
}

int check_rope(const rnb_rope_desc* d) {
  if (!d) return fail(RNB_ERR_INVALID, "rnb_rope_append: descriptor is NULL");
  if (d->dtype != RNB_DTYPE_BF16 && d->dtype != RNB_DTYPE_F16)
    return fail(RNB_ERR_INVALID, "rnb_rope_append: dtype must be RNB_DTYPE_BF16 or RNB_DTYPE_F16");
  if (d->T < 0) return fail(RNB_ERR_INVALID, "rnb_rope_append: T must be >= 0");
  if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
    return fail(RNB_ERR_INVALID, "rnb_rope_append: head_dim must be 64, 128 or 256");
  if (d->rot <= 0 || d->rot % 16 || d->rot > d->head_dim)
    return fail(RNB_ERR_INVALID, "rnb_rope_append: rot must be a positive multiple of 16, at most head_dim");
  if (d->n_q_heads <= 0 || d->n_q_heads > 65535 || d->n_kv_heads < 0 || d->n_kv_heads > 65535)
    return fail(RNB_ERR_INVALID, "rnb_rope_append: n_q_heads must be in [1, 65535], n_kv_heads in [0, 65535]");
  const int n = d->rot / 2;
  if (d->n_axes < 1 || d->n_axes > 4) return fail(RNB_ERR_INVALID, "rnb_rope_append: n_axes must be in [1, 4]");
  int64_t sum = 0;
  for (int i = 0; i < d->n_axes; ++i) {
    if (d->sections[i] < 0) return fail(RNB_ERR_INVALID, "rnb_rope_append: sections must be >= 0");
    sum += d->sections[i];
    if (d->interleaved && i && d->sections[i] && i + static_cast<int64_t>(d->n_axes) * (d->sections[i] - 1) >= n)
      return fail(RNB_ERR_INVALID, "rnb_rope_append: an interleaved section runs past rot/2");
  }
  if (sum != n) return fail(RNB_ERR_INVALID, "rnb_rope_append: sections must sum to rot/2");
  const int64_t st[6] = {d->q_token_stride, d->q_head_stride, d->k_token_stride,
                         d->k_head_stride,  d->v_token_stride, d->v_head_stride};
  for (int64_t v : st)
    if (v < 0 || v % 8) return fail(RNB_ERR_INVALID, "rnb_rope_append: strides must be multiples of 8 elements");
  return RNB_OK;
}

template <typename T>
void launch_rope(const RopeArgs& a, int D, dim3 grid, cudaStream_t st) {
  if (D == 64)
    k_rope_append<T, 64><<<grid, kRopeThreads, 0, st>>>(a);
  else if (D == 128)
    k_rope_append<T, 128><<<grid, kRopeThreads, 0, st>>>(a);
  else
    k_rope_append<T, 256><<<grid, kRopeThreads, 0, st>>>(a);
}

}  // namespace

int rope_status_take(uint32_t* bits, cudaStream_t st) { return status_take(g_rope_status, bits, st); }

}  // namespace rnb

extern "C" int rnb_rope_append(const rnb_rope_desc* d, const void* q, const void* k, const void* v,
                               const void* q_norm_w, const void* k_norm_w, const int32_t* positions,
                               const float* inv_freq, const int32_t* slots, const rnb_kv_cache* cache, void* q_out,
                               void* stream) {
  using namespace rnb;
  int rc = check_rope(d);
  if (rc) return rc;
  const int given = (k != nullptr) + (v != nullptr) + (slots != nullptr) + (cache != nullptr);
  if (given != 0 && given != 4)
    return fail(RNB_ERR_INVALID, "rnb_rope_append: k, v, slots and cache must be given together or all be NULL");
  if ((given == 4) != (d->n_kv_heads > 0))
    return fail(RNB_ERR_INVALID, "rnb_rope_append: n_kv_heads must be positive with a cache and 0 without one");
  if (cache) {
    if ((rc = check_cache(cache, "rnb_rope_append"))) return rc;
    if (cache->dtype != d->dtype || cache->head_dim != d->head_dim || cache->n_kv_heads != d->n_kv_heads)
      return fail(RNB_ERR_INVALID, "rnb_rope_append: the cache's dtype, head_dim and n_kv_heads must match");
  }
  if (d->T == 0) return RNB_OK;
  if (!q || !q_out || !positions || !inv_freq)
    return fail(RNB_ERR_INVALID, "rnb_rope_append: q, q_out, positions and inv_freq must be non-NULL");
  if (!aligned16(q) || !aligned16(q_out) || !aligned16(k) || !aligned16(v) || !aligned16(q_norm_w) ||
      !aligned16(k_norm_w))
    return fail(RNB_ERR_ALIGN, "rnb_rope_append: q, k, v, q_out and the norm weights must be 16-byte aligned");
  const int64_t D = d->head_dim;
  if (q == q_out && (d->q_head_stride != D || d->q_token_stride != D * d->n_q_heads))
    return fail(RNB_ERR_INVALID, "rnb_rope_append: q_out may be q only if q is packed [T][n_q_heads][head_dim]");
  if ((rc = check_device())) return rc;

  RopeArgs a{};
  a.q = q, a.k = k, a.v = v, a.qw = q_norm_w, a.kw = k_norm_w;
  a.pos = positions, a.inv_freq = inv_freq, a.slots = slots, a.q_out = q_out;
  a.q_ts = d->q_token_stride, a.q_hs = d->q_head_stride;
  a.k_ts = d->k_token_stride, a.k_hs = d->k_head_stride;
  a.v_ts = d->v_token_stride, a.v_hs = d->v_head_stride;
  if (cache) {
    a.kc = cache->k, a.vc = cache->v;
    a.kc_ps = cache->k_page_stride, a.kc_hs = cache->k_head_stride;
    a.vc_ps = cache->v_page_stride, a.vc_hs = cache->v_head_stride;
    a.num_slots = static_cast<uint32_t>(cache->num_pages) * cache->page_size;
    while ((1 << a.log2p) < cache->page_size) ++a.log2p;
  }
  a.eps = d->eps;
  a.T = d->T, a.Hq = d->n_q_heads, a.Hkv = d->n_kv_heads, a.half = d->rot / 2;
  a.n_axes = d->n_axes, a.interleaved = d->interleaved;
  for (int i = 0; i < 4; ++i) a.sec[i] = d->sections[i];

  // Many tokens: as many a CTA as give each thread one angle, all heads from
  // them.  Few: one token a CTA, its heads dealt over CTAs until the SMs are
  // covered (each repeats the token's angles, rot/2 of them).
  const int heads = a.Hq + 2 * a.Hkv, sms = dev_info().sms;
  const int groups = kRopeThreads / static_cast<int>(D / 8);
  int tok = kRopeThreads / a.half;
  while (tok > 1 && (a.T + tok - 1) / tok < 2 * sms) tok /= 2;
  a.tok = tok;
  const int ctas = (a.T + tok - 1) / tok;
  int split = 1;
  while (split < heads && ctas * split < sms && (heads + split - 1) / split > groups) ++split;
  a.heads_per_cta = (heads + split - 1) / split;
  const dim3 grid(ctas, (heads + a.heads_per_cta - 1) / a.heads_per_cta);
  if (d->dtype == RNB_DTYPE_BF16)
    launch_rope<__nv_bfloat16>(a, static_cast<int>(D), grid, static_cast<cudaStream_t>(stream));
  else
    launch_rope<__half>(a, static_cast<int>(D), grid, static_cast<cudaStream_t>(stream));
  return launch_status("rnb_rope_append");
}
