// rnb_rope.cu -- per-head RMSNorm, rotary positions with several axes, and
// the append of a step's keys and values to the paged cache (rnb_rope_append).
//
// One pass: a head's row is read once with 16-byte loads (D/8 lanes hold it,
// so the norm's sum is a few shuffles, and the partner of element i, i +- rot/2,
// is in another lane), turned in fp32 and written once, rounded once.  HBM
// bounds it: 4 (Hq + 2 Hkv) D bytes a token; what has to be kept small is the
// instructions a row.  So a group of D/8 lanes stays with one token and walks its
// heads, four rows under way, with the token's cosines and the norm's weights in
// registers; the partner comes as raw 16-bit pairs, four shuffles a row.  With
// few tokens a token's heads are dealt over several groups.
//
// Angles: fp32 loses far positions (position 10^5 at frequency 1 is off by
// 2^-8 rad), so position * frequency and its reduction to turns are fp64, and
// sincospif works on the small remainder.  That is rot/2 evaluations a token for
// all its heads: the CTA's threads share them through shared memory.
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "rnb_kv.cuh"

namespace rnb {
namespace {

constexpr int kRopeThreads = 64;  // small CTAs: no SM is left with the last large one
constexpr int kRopeCtas = 12;     // resident on an SM

__device__ uint32_t g_rope_status;

struct RopeArgs {
  const void *q, *k, *v, *qw, *kw;
  const int32_t* pos;
  const float* inv_freq;
  const int32_t* slots;
  void *q_out, *kc, *vc;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, kc_ps, kc_hs, vc_ps, vc_hs;
  float eps;
  int T, Hq, Hkv, half, log2p;
  int heads_a_chunk;
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

// Where a lane's elements and their partners are.
struct Lane {
  const float2* cs;  // cosine and sine of its 8 pairs (only where they turn)
  int e0, partner_e0;  // first elements, its own and its partner's
  int partner;         // the partner's lane in the warp
  bool turned, lo;     // its elements turn; they are the pairs' first elements
};

// Up to n rows of one token at a stride in elements.
template <typename T>
struct Rows {
  const T* from;
  int64_t stride;
  int n;
  // rows r .. r + 3 (coherent loads: q_out may be q)
  __device__ __forceinline__ void load(int r, uint4 (&v)[4]) const {
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (r + y < n) v[y] = __ldcs(reinterpret_cast<const uint4*>(from + (r + y) * stride));
  }
};

// The rows of `rows`, turned, to `to`; every lane of the warp calls it with the
// same n_max >= rows.n, for the shuffles.  `in` holds the first four and, after
// it, the first four of `next`: four rows are always under way.
template <typename T, int D>
__device__ __forceinline__ void turn_rows(uint4 (&in)[4], const Rows<T>& rows, T* to, int64_t to_stride, int n_max,
                                          const Rows<T>& next, const T* weight, float eps, const Lane& ln) {
  constexpr int kLanes = D / 8;
  // y = x w + z wp with z the partners: cosines and signed sines, times the norm's weights
  float2 w[4], wp[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float4 c = make_float4(1.f, 0.f, 1.f, 0.f);
    if (ln.turned) c = *reinterpret_cast<const float4*>(ln.cs + 2 * i);
    w[i] = make_float2(c.x, c.z);
    wp[i] = ln.lo ? make_float2(-c.y, -c.w) : make_float2(c.y, c.w);
  }
  if (weight) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(weight + ln.e0));
    const uint4 b = __ldg(reinterpret_cast<const uint4*>(weight + ln.partner_e0));
    const uint32_t au[4] = {a.x, a.y, a.z, a.w}, bu[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = mul2(w[i], Pair<T>::unpack(au[i])), wp[i] = mul2(wp[i], Pair<T>::unpack(bu[i]));
  }
  for (int r = 0; r < n_max; r += 4) {
    uint4 ahead[4] = {};
    if (r + 4 < n_max)
      rows.load(r + 4, ahead);
    else
      next.load(0, ahead);
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      if (r + y >= n_max) break;
      const uint32_t u[4] = {in[y].x, in[y].y, in[y].z, in[y].w};
      float2 x[4];
      float2 ss = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t z = __shfl_sync(0xffffffffu, u[i], ln.partner);
        const float2 f = Pair<T>::unpack(u[i]);
        ss = fma2(f, f, ss);
        x[i] = fma2(Pair<T>::unpack(ln.turned ? z : 0u), wp[i], mul2(f, w[i]));  // (0: what does not turn passes any bits)
      }
      if (weight) {
        float sum = ss.x + ss.y;
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float sc = rsqrtf(fmaf(sum, 1.0f / D, eps));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = mul2(x[i], make_float2(sc, sc));
      }
      if (r + y < rows.n)
        *reinterpret_cast<uint4*>(to + (r + y) * to_stride) =
            make_uint4(Pair<T>::pack(x[0].x, x[0].y), Pair<T>::pack(x[1].x, x[1].y), Pair<T>::pack(x[2].x, x[2].y),
                       Pair<T>::pack(x[3].x, x[3].y));
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) in[y] = ahead[y];
  }
}

// Heads are numbered queries first, then keys, then values; the groups of CTA
// (x, y) take heads [y heads_a_chunk, ...) of a token each.  (Groups of a warp
// have the same heads: a warp walks as many as its longest group.)
template <typename T, int D>
__global__ void __launch_bounds__(kRopeThreads, kRopeCtas) k_rope_append(const RopeArgs a) {
  constexpr int kLanes = D / 8;                   // lanes holding one head's row
  constexpr int kGroups = kRopeThreads / kLanes;  // rows in flight in the CTA
  __shared__ __align__(16) float2 cs[kGroups * D / 2];  // [token][half] cos, sin
  after_previous();
  const int tid = threadIdx.x, lane = tid % kLanes, e0 = lane * 8;
  const int t_first = blockIdx.x * kGroups, t_last = min(t_first + kGroups, a.T) - 1;

  // this group's token and heads; its first rows are under way before the angles
  const bool in = t_first + tid / kLanes < a.T;
  const int t = in ? t_first + tid / kLanes : t_first, h0 = blockIdx.y * a.heads_a_chunk;
  const int slot = !in ? -1 : a.slots ? a.slots[t] : 0;
  const int h1 = slot < 0 ? h0 : min(h0 + a.heads_a_chunk, a.Hq + 2 * a.Hkv);  // (no heads: a row left alone)
  const bool inside = a.slots && static_cast<uint32_t>(slot) < a.num_slots;
  const int64_t tt = t;
  const int qb = h0, kb = max(h0 - a.Hq, 0), vb = max(h0 - a.Hq - a.Hkv, 0);
  const Rows<T> q{static_cast<const T*>(a.q) + tt * a.q_ts + qb * a.q_hs + e0, a.q_hs, max(0, min(h1, a.Hq) - qb)};
  const Rows<T> k{static_cast<const T*>(a.k) + tt * a.k_ts + kb * a.k_hs + e0, a.k_hs,
                  inside ? max(0, min(h1 - a.Hq, a.Hkv) - kb) : 0};
  const Rows<T> v{static_cast<const T*>(a.v) + tt * a.v_ts + vb * a.v_hs + e0, a.v_hs,
                  inside ? max(0, h1 - a.Hq - a.Hkv - vb) : 0};
  // a warp's groups run the same number of rounds of each kind
  const int nq = __reduce_max_sync(0xffffffffu, q.n), nk = __reduce_max_sync(0xffffffffu, k.n);
  uint4 rows[4] = {};
  if (nq > 0)
    q.load(0, rows);
  else if (nk > 0)
    k.load(0, rows);
  else
    v.load(0, rows);

  for (int i = tid; i < (t_last - t_first + 1) * a.half; i += kRopeThreads) {
    const int tl = i / a.half, f = i - tl * a.half;
    const double p = static_cast<double>(a.pos[static_cast<int64_t>(axis_of(a, f)) * a.T + t_first + tl]);
    // the fp64 remainder of whole turns is exact to 2^-52 of the angle
    double turns = p * static_cast<double>(a.inv_freq[f]) * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif(static_cast<float>(2.0 * turns), &s, &c);
    cs[i] = make_float2(c, s);
  }
  __syncthreads();

  Lane ln;
  ln.e0 = e0, ln.lo = e0 < a.half, ln.turned = e0 < 2 * a.half;
  const int pl = ln.turned ? (ln.lo ? lane + a.half / 8 : lane - a.half / 8) : lane;
  ln.partner = (tid & 31) - lane + pl, ln.partner_e0 = pl * 8;
  ln.cs = cs + (t - t_first) * a.half + (ln.turned ? (ln.lo ? e0 : e0 - a.half) : 0);
  if (nq > 0)
    turn_rows<T, D>(rows, q, static_cast<T*>(a.q_out) + (tt * a.Hq + qb) * D + e0, D, nq, nk > 0 ? k : v,
                    static_cast<const T*>(a.qw), a.eps, ln);
  if (!a.slots) return;
  if (in && slot >= 0 && !inside && lane == 0 && h1 > a.Hq) atomicOr(&g_rope_status, RNB_STATUS_BAD_INDEX);
  const int64_t page = inside ? slot >> a.log2p : 0, off = inside ? (slot & ((1 << a.log2p) - 1)) * D : 0;
  if (nk > 0)
    turn_rows<T, D>(rows, k, static_cast<T*>(a.kc) + page * a.kc_ps + kb * a.kc_hs + off + e0, a.kc_hs, nk, v,
                    static_cast<const T*>(a.kw), a.eps, ln);
  T* to = static_cast<T*>(a.vc) + page * a.vc_ps + vb * a.vc_hs + off + e0;
  for (int r = 0; r < v.n; r += 4) {
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (r + y < v.n) *reinterpret_cast<uint4*>(to + (r + y) * a.vc_hs) = rows[y];
    v.load(r + 4, rows);
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
int launch_rope(const RopeArgs& a, int D, dim3 grid, cudaStream_t st) {
  return launch("rnb_rope_append", D == 64 ? k_rope_append<T, 64> : D == 128 ? k_rope_append<T, 128> : k_rope_append<T, 256>,
                grid, kRopeThreads, 0, st, a);
}

}  // namespace

cudaError_t rope_status_word(uint32_t** p) { return status_word(g_rope_status, p); }

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
  // groups write rows of q_out while others still read theirs
  if ((q != q_out &&
       shares_memory(q_out, d->T, d->n_q_heads, D, q, d->q_token_stride, d->q_head_stride, d->n_q_heads)) ||
      shares_memory(q_out, d->T, d->n_q_heads, D, k, d->k_token_stride, d->k_head_stride, d->n_kv_heads) ||
      shares_memory(q_out, d->T, d->n_q_heads, D, v, d->v_token_stride, d->v_head_stride, d->n_kv_heads))
    return fail(RNB_ERR_INVALID, "rnb_rope_append: q_out must not share memory with q (unless it is q), k or v");

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

  // Many tokens: a group a token.  Few: a token's heads over as many groups as
  // the SMs hold at once, four rows a group or more.
  const int heads = a.Hq + 2 * a.Hkv, groups = kRopeThreads / static_cast<int>(D / 8);
  const int64_t hold = static_cast<int64_t>(dev_info().sms) * kRopeCtas * groups;
  int64_t chunks = hold / a.T;  // (rounded up, 4097 tokens of 48 heads took 27 us instead of 25)
  if (chunks < 1) chunks = 1;
  if (chunks > (heads + 3) / 4) chunks = (heads + 3) / 4;
  a.heads_a_chunk = static_cast<int>((heads + chunks - 1) / chunks);
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(a.T) + groups - 1) / groups),
                  static_cast<unsigned>((heads + a.heads_a_chunk - 1) / a.heads_a_chunk));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return d->dtype == RNB_DTYPE_BF16 ? launch_rope<__nv_bfloat16>(a, static_cast<int>(D), grid, st)
                                    : launch_rope<__half>(a, static_cast<int>(D), grid, st);
}
