// rnb_attn.cu -- attention over the paged cache for few query rows a request
// (one new token, a few drafted ones), split over the cache's length and joined
// (rnb_paged_attention).
//
// For the R <= 16 query rows that share a key head (one token's group of query
// heads, or several tokens'), with s = scale q.k and running m = max s,
// l = sum e^(s-m), o = sum e^(s-m) v, one pass over K and V gives o/l.  Every
// cached token is 4 D bytes for 4 R D flops: HBM bounds it, so what counts is
// bytes in flight, an even split, and few instructions a byte.
//
// * Orientation.  S^T = K Q^T and O^T = V^T P^T: the 16 tokens of a subtile are
//   the m rows of mma m16n8k16 and the query rows its 8 columns, so a group of
//   up to 8 rows fills the instruction, and O takes D/4 registers a lane for 8
//   rows (D/2 the other way around).
// * No staging.  The contraction order is free, so K enters the A operand as
//   loaded: lane (g, c) reads 16 bytes, 8 consecutive elements, of token g and
//   of token g + 8, and the queries are read in the same order.  For V a lane
//   reads 16 bytes of four tokens and interleaves pairs of tokens with byte
//   permutes; which element of the head is which m row is free again.  Each
//   load instruction covers whole 64-byte (K) or 128-byte (V) pieces of rows,
//   shared memory holds nothing but the join of the warps, and a warp has up
//   to 16 KB in flight.  P^T leaves the S accumulators by one 8x8 transpose
//   (movmatrix) an operand register.
// * Split.  A unit is 64 positions of one (request, key head, row tile).  Every
//   CTA sums the units of all requests from the lengths on the device, takes an
//   equal contiguous share, and so has at most two tiles that it does not
//   cover alone; those leave (m, l, o) in the workspace, and a second kernel
//   adds a tile's parts in order.
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include <string>

#include "rnb_attn.cuh"

namespace rnb {

__device__ uint32_t g_attn_status;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kUnit = 64;  // positions
constexpr int kManyRows = 64;  // rows * group from which a request is the many-row kernel's

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 8x8 transpose of 16-bit elements across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename T>
__device__ __forceinline__ void mma_t(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1);
template <>
__device__ __forceinline__ void mma_t<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  mma_f16(d, a0, a1, a2, a3, b0, b1);
}
template <>
__device__ __forceinline__ void mma_t<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                     uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ceil(a / b) without the 64-bit division wherever 32 bits do (100 cycles on
// the way to the first load).
__device__ __forceinline__ int64_t share_of(int64_t a, uint32_t b) {
  return a < INT_MAX ? (static_cast<uint32_t>(a) + b - 1) / b : (a + b - 1) / b;
}

// One request's share of the work.
struct Request {
  int q0, rows, len;      // first query row, rows, cached positions
  int blk0, nblk, ntile;  // first unit of positions, units, row tiles
};

template <int R>
__device__ __forceinline__ Request request_of(const AttnArgs& a, int c0, int c1, int len) {
  Request r;
  r.q0 = min(max(c0, 0), a.T);
  r.rows = min(max(c1, r.q0), a.T) - r.q0;
  r.len = min(max(len, 0), a.max_kv);
  const int work = r.rows * a.group < a.few_rows ? r.rows * a.group : 0;
  r.ntile = (work + R - 1) / R;
  const int lo = a.window > 0 ? max(0, r.len - r.rows - a.window + 1) : 0;
  r.blk0 = lo / kUnit;
  r.nblk = max(1, (r.len + kUnit - 1) / kUnit - r.blk0);  // a row that sees nothing is written too
  return r;
}

__device__ __forceinline__ void read_request(const AttnArgs& a, int b, int& c0, int& c1, int& len) {
  c0 = c1 = len = 0;
  if (b < a.B) {
    c0 = a.cu ? a.cu[b] : b;
    c1 = a.cu ? a.cu[b + 1] : b + 1;
    len = a.seq[b];
  }
}

// The tile that CTA i began and others end.
struct Begun {
  int last;  // the CTA that ends it; -1: none
  int q0, work, h, tile;
};

// A tile's part that one CTA covers: units [blk, blk + n) of the tile's nblk.
struct Segment {
  int b, q0, rows, len, blk0, nblk;  // its request
  int h, tile, blk, n;               // n 0: none
};

template <typename T, int D, int NT>
struct __align__(16) Smem {
  float m[kWarps][8 * NT], l[kWarps][8 * NT];
  float o[kWarps][8 * NT][D + 4];
  T q[2][8 * NT][D + 32];  // queries of this segment and the next; rows 64 bytes off in the banks
  Segment seg[3];          // this one and the two behind it
};

// What a warp loads for one step: NS subtiles of 16 positions, 64 registers of K
// and 64 of V a lane (half as many where 16 rows leave no more).
template <int D, int NT>
struct Steps {
  static constexpr int NS = D == 64 && NT == 2 ? 2 : 256 / D;
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, 2) k_attn_few(const AttnArgs a) {
  after_previous();
  constexpr int R = 8 * NT, NS = Steps<D, NT>::NS, KC = D / 32, VC = D / 64;
  constexpr int kStep = 16 * NS, kStride = kWarps * kStep;
  constexpr int kTile = 512 / D;  // what starting and joining a tile costs, in units (without it
  // ragged batches left half of the SMs idle: 204 instead of 117 us, 63 instead of 35)
  __shared__ Smem<T, D, NT> sm;
  __shared__ int64_t wsum[kWarps], total;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  Begun* begun = reinterpret_cast<Begun*>(a.ws);
  if (tid == 0) begun[blockIdx.x].last = -1;

  // ---- this CTA's share.  The warp whose requests hold its first unit deals the
  // segments from there, two ahead of the one in work: it stands at cost p_at of row
  // tile tile_at of key head h_at of request `at`, whose numbers are c0, c1, len.
  bool dealer = false;
  int64_t start_rem = 0;
  int at = 0, h_at = 0, tile_at = 0, p_at = 0, c0 = 0, c1 = 0, len = 0;
  if (!a.direct) {
    const int per = (a.B + kThreads - 1) / kThreads;
    const int lo = min(tid * per, a.B), hi = min(lo + per, a.B);
    auto units = [&](int b) {
      read_request(a, b, c0, c1, len);
      if (blockIdx.x == 0 && (len < 0 || len > a.max_kv || c0 < 0 || c1 < c0 || c1 > a.T))
        atomicOr(&g_attn_status, RNB_STATUS_BAD_INDEX);
      const Request r = request_of<R>(a, c0, c1, len);
      return static_cast<int64_t>(r.ntile) * (r.nblk + kTile) * a.Hkv;
    };
    int64_t sum = 0;
    for (int b = lo; b < hi; ++b) sum += units(b);
    int64_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int64_t base = inc - sum;
    for (int w = 0; w < warp; ++w) base += wsum[w];
    if (tid == kThreads - 1) total = base + sum;
    __syncthreads();
    const int64_t share = share_of(total, gridDim.x), u0 = share * blockIdx.x;
    const bool here = u0 >= base && u0 < base + sum;
    if (here) {
      start_rem = u0 - base;
      at = lo;
      for (int64_t n = per == 1 ? sum : units(at); start_rem >= n && at + 1 < hi; n = units(at)) {
        start_rem -= n;
        ++at;
      }
    }
    const uint32_t who = __ballot_sync(0xffffffffu, here);
    dealer = who != 0;
    if (dealer) {
      const int from = __ffs(who) - 1;
      start_rem = __shfl_sync(0xffffffffu, start_rem, from), at = __shfl_sync(0xffffffffu, at, from);
      c0 = __shfl_sync(0xffffffffu, c0, from), c1 = __shfl_sync(0xffffffffu, c1, from);
      len = __shfl_sync(0xffffffffu, len, from);
    }
  }
  // (direct: every request has one row, so tile i is known without the lengths;
  // this CTA takes whole tiles, gridDim.x apart)
  const int tiles_a_head = (a.group + R - 1) / R, tiles_a_request = tiles_a_head * a.Hkv;
  const int64_t share = a.direct ? gridDim.x : share_of(total, gridDim.x);
  const int64_t u0 = a.direct ? blockIdx.x : share * blockIdx.x;
  const int64_t u1 = a.direct ? static_cast<int64_t>(a.B) * tiles_a_request : min(u0 + share, total);
  if (u0 >= u1) return;

  int64_t u_at = u0;
  // From an idle request to the next one that has tiles here: 32 are read at once, so
  // that a batch's empty places cost little (4092 of 4096 places idle: 331 -> 68 us).
  auto skip_idle = [&]() {
    for (uint32_t live = 0; live == 0 && at < a.B;) {
      const int left = a.B - 1 - at;
      read_request(a, lane < left ? at + 1 + lane : a.B, c0, c1, len);
      live = __ballot_sync(0xffffffffu, lane < left && request_of<R>(a, c0, c1, len).ntile > 0);
      const int i = live ? __ffs(live) - 1 : min(left, 31);
      at += i + 1;  // (nothing left: B)
      c0 = __shfl_sync(0xffffffffu, c0, i), c1 = __shfl_sync(0xffffffffu, c1, i);
      len = __shfl_sync(0xffffffffu, len, i);
    }
  };
  auto deal = [&](Segment& sg) {
    sg.n = 0;
    if (a.direct) {
      if (u_at < u1) {
        const int i = static_cast<int>(u_at);  // (T n_q_heads fits)
        u_at += share;
        sg.b = i / tiles_a_request;
        const int j = i - sg.b * tiles_a_request;
        sg.h = j / tiles_a_head, sg.tile = j - sg.h * tiles_a_head;
        read_request(a, sg.b, c0, c1, len);
        if (j == 0 && (len < 0 || len > a.max_kv)) atomicOr(&g_attn_status, RNB_STATUS_BAD_INDEX);
        const Request rq = request_of<R>(a, c0, c1, len);
        sg.q0 = rq.q0, sg.rows = rq.rows, sg.len = rq.len, sg.blk0 = rq.blk0, sg.nblk = sg.n = rq.nblk;
        sg.blk = 0;
      }
      return;
    }
    while (u_at < u1 && at < a.B) {  // (the second: lengths that change under way must not hang it)
      const Request rq = request_of<R>(a, c0, c1, len);
      if (h_at < a.Hkv && rq.ntile > 0) {
        const int cost = kTile + rq.nblk;
        const int take = static_cast<int>(min(static_cast<int64_t>(cost - p_at), u1 - u_at));
        const int first = max(p_at - kTile, 0), end = max(p_at + take - kTile, 0);
        sg.b = at, sg.q0 = rq.q0, sg.rows = rq.rows, sg.len = rq.len, sg.blk0 = rq.blk0, sg.nblk = rq.nblk;
        sg.h = h_at, sg.tile = tile_at, sg.blk = first, sg.n = end - first;
        u_at += take;
        p_at += take;
        if (p_at == cost) {
          p_at = 0;
          if (++tile_at == rq.ntile) tile_at = 0, ++h_at;
        }
      }
      if (rq.ntile == 0) {
        skip_idle();
        h_at = tile_at = p_at = 0;
      } else if (h_at == a.Hkv) {  // the next request's numbers are on their way when they are asked for
        h_at = tile_at = p_at = 0;
        read_request(a, ++at, c0, c1, len);
      }
      if (sg.n > 0) return;
    }
  };
  if (a.direct) {
    dealer = warp == 0;
    if (dealer) {
      deal(sm.seg[0]);
      deal(sm.seg[1]);
    }
  } else if (dealer) {
    const Request rq = request_of<R>(a, c0, c1, len);
    const int cost = rq.nblk + kTile;
    const int64_t tile_of = start_rem < INT_MAX ? static_cast<int>(start_rem) / cost : start_rem / cost;
    p_at = static_cast<int>(start_rem - tile_of * cost);
    const int nt = max(rq.ntile, 1);
    h_at = static_cast<int>(tile_of < INT_MAX ? static_cast<int>(tile_of) / nt : tile_of / nt);
    tile_at = static_cast<int>(tile_of - static_cast<int64_t>(h_at) * rq.ntile);
    deal(sm.seg[0]);
    deal(sm.seg[1]);
  }
  __syncthreads();

  // ---- what a warp's loads go by
  const T *kh = nullptr, *vh = nullptr;
  const int32_t* row_table = nullptr;
  int s = 0, s_end = 0;  // positions: the step whose K and V are (being) loaded, the segment's end
  const int pmask = (1 << a.log2p) - 1;
  auto positions_end = [&](const Segment& sg) {
    const int last = sg.len - sg.rows + by_group(a, min(sg.tile * R + R - 1, sg.rows * a.group - 1));
    return min((sg.blk0 + sg.blk + sg.n) * kUnit, last + 1);
  };
  auto enter = [&](const Segment& sg) {
    s = s_end = 0;
    if (sg.n > 0) {
      kh = static_cast<const T*>(a.kc) + sg.h * a.kc_hs + g * D + 8 * c;
      vh = static_cast<const T*>(a.vc) + sg.h * a.vc_hs + 2 * c * D + 8 * g;
      row_table = a.table + static_cast<int64_t>(sg.b) * a.W;
      s = (sg.blk0 + sg.blk) * kUnit + warp * kStep;
      s_end = positions_end(sg);
    }
  };
  auto pages_of = [&](const int32_t* tab, int from, int end, int (&pid)[NS]) {
#pragma unroll
    for (int ns = 0; ns < NS; ++ns) {
      const int st = from + 16 * ns;
      pid[ns] = st < end ? __ldg(tab + (st >> a.log2p)) : -1;
    }
  };
  uint4 kr[NS][KC][2], vr[NS][VC][4];
  auto load_k = [&](const int (&pid)[NS]) {
#pragma unroll
    for (int ns = 0; ns < NS; ++ns) {
      const bool ok = static_cast<uint32_t>(pid[ns]) < static_cast<uint32_t>(a.num_pages);
      const T* p = kh + (ok ? pid[ns] : 0) * a.kc_ps + ((s + 16 * ns) & pmask) * D;
#pragma unroll
      for (int i = 0; i < KC; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          kr[ns][i][e] = make_uint4(0, 0, 0, 0);
          if (ok) kr[ns][i][e] = ld_stream_v4(p + 32 * i + 8 * e * D);
        }
    }
  };
  auto load_v = [&](const int (&pid)[NS]) {
#pragma unroll
    for (int ns = 0; ns < NS; ++ns) {
      const bool ok = static_cast<uint32_t>(pid[ns]) < static_cast<uint32_t>(a.num_pages);
      const T* p = vh + (ok ? pid[ns] : 0) * a.vc_ps + ((s + 16 * ns) & pmask) * D;
#pragma unroll
      for (int i = 0; i < VC; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          vr[ns][i][e] = make_uint4(0, 0, 0, 0);
          if (ok) vr[ns][i][e] = ld_stream_v4(p + 64 * i + ((e & 1) + 8 * (e >> 1)) * D);
        }
    }
  };
  auto load_q = [&](const Segment& sg, int buf) {
    constexpr int kPer = D / 8;
    for (int x = tid; x < R * kPer; x += kThreads) {
      const int r = x / kPer, e = (x - r * kPer) * 8, row = sg.tile * R + r, i = by_group(a, row), j = row - i * a.group;
      if (row < sg.rows * a.group)
        cp_async16(&sm.q[buf][r][e],
                   static_cast<const T*>(a.q) + (sg.q0 + i) * a.q_ts + (sg.h * a.group + j) * a.q_hs + e);
      else
        *reinterpret_cast<uint4*>(&sm.q[buf][r][e]) = make_uint4(0, 0, 0, 0);
    }
  };

  int pid[NS], nxt[NS], first_pid[NS];
  load_q(sm.seg[0], 0);
  enter(sm.seg[0]);
  pages_of(row_table, s, s_end, pid);
  load_k(pid);
  load_v(pid);
  pages_of(row_table, s + kStride, s_end, nxt);
  cp_async_wait_all();
  __syncthreads();

  for (int x = 0;; ++x) {
    const Segment sg = sm.seg[x % 3];
    if (sg.n == 0) break;
    const int work = sg.rows * a.group, row0 = sg.tile * R, seg_end = s_end;
    {
      // the next segment: its queries, and the pages of this warp's first step in it
      const Segment& ns = sm.seg[(x + 1) % 3];
#pragma unroll
      for (int y = 0; y < NS; ++y) first_pid[y] = -1;
      if (ns.n > 0) {
        load_q(ns, (x + 1) & 1);
        pages_of(a.table + static_cast<int64_t>(ns.b) * a.W, (ns.blk0 + ns.blk) * kUnit + warp * kStep,
                 positions_end(ns), first_pid);
      }
    }
    const int p0 = sg.len - sg.rows;  // position of the request's first row
    int seen_hi[NT][2], seen_lo[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = min(row0 + nt * 8 + 2 * c + e, work - 1), p = p0 + by_group(a, row);
        seen_hi[nt][e] = p;
        seen_lo[nt][e] = a.window > 0 ? p - a.window + 1 : INT_MIN;
      }
    const int first_p = p0 + by_group(a, row0), last_p = p0 + by_group(a, min(row0 + R - 1, work - 1));
    const int all_lo = a.window > 0 ? last_p - a.window + 1 : INT_MIN;   // from here every row sees, up to first_p
    const int any_lo = a.window > 0 ? first_p - a.window + 1 : INT_MIN;  // before here none does

    float o[NT][VC][4][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) m[nt][e] = -INFINITY, l[nt][e] = 0.f;
#pragma unroll
      for (int i = 0; i < VC; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][i][j][e] = 0.f;
    }

    bool more = s < seg_end;
    bool entered = false;  // the loads are at the next segment
    auto advance = [&]() {  // to the next step, here or in the next segment
      s += kStride;
      more = s < seg_end;
      if (more) {
#pragma unroll
        for (int y = 0; y < NS; ++y) pid[y] = nxt[y];
      } else {
        enter(sm.seg[(x + 1) % 3]);
        entered = true;
#pragma unroll
        for (int y = 0; y < NS; ++y) pid[y] = first_pid[y];
      }
    };
    while (more) {
      // S^T
      float sc[NS][NT][4], sd[NS][NT][4];  // two chains of products
#pragma unroll
      for (int ns = 0; ns < NS; ++ns)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[ns][nt][e] = sd[ns][nt][e] = 0.f;
#pragma unroll
      for (int i = 0; i < KC; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 qf = *reinterpret_cast<const uint4*>(&sm.q[x & 1][nt * 8 + g][32 * i + 8 * c]);
#pragma unroll
          for (int ns = 0; ns < NS; ++ns) {
            const uint4 y = kr[ns][i][0], z = kr[ns][i][1];
            mma_t<T>(sc[ns][nt], y.x, z.x, y.y, z.y, qf.x, qf.y);
            mma_t<T>(NS * NT <= 2 ? sd[ns][nt] : sc[ns][nt], y.z, z.z, y.w, z.w, qf.z, qf.w);
          }
        }
      const int s_cur = s;
      int cur[NS];
      bool whole = s + kStep - 1 <= first_p && s >= all_lo;
#pragma unroll
      for (int ns = 0; ns < NS; ++ns) {
        cur[ns] = pid[ns];
        whole = whole && static_cast<uint32_t>(cur[ns]) < static_cast<uint32_t>(a.num_pages);
      }
      advance();
      load_k(pid);
      pages_of(row_table, s + kStride, s_end, nxt);
#pragma unroll
      for (int ns = 0; ns < NS; ++ns)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sc[ns][nt][e] = (NS * NT <= 2 ? sc[ns][nt][e] + sd[ns][nt][e] : sc[ns][nt][e]) * a.scale_log2;
      if (!whole) {
#pragma unroll
        for (int ns = 0; ns < NS; ++ns) {
          const int st = s_cur + 16 * ns;
          const bool ok = static_cast<uint32_t>(cur[ns]) < static_cast<uint32_t>(a.num_pages);
          if (!ok && st < seg_end && st + 15 >= any_lo && lane == 0) atomicOr(&g_attn_status, RNB_STATUS_BAD_INDEX);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = st + g + 8 * (e >> 1);
              if (!ok || t >= seg_end || t > seen_hi[nt][e & 1] || t < seen_lo[nt][e & 1]) sc[ns][nt][e] = -INFINITY;
            }
          // values that no row of the tile sees: their bits must not count
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = st + 2 * c + (e & 1) + 8 * (e >> 1);
            if (t >= seg_end || t < any_lo) {
#pragma unroll
              for (int i = 0; i < VC; ++i) vr[ns][i][e] = make_uint4(0, 0, 0, 0);
            }
          }
        }
      }
      // running maximum and sum
      bool grew = false;
      float f[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = m[nt][e];
#pragma unroll
          for (int ns = 0; ns < NS; ++ns) mx = fmaxf(mx, fmaxf(sc[ns][nt][e], sc[ns][nt][e + 2]));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float use = mx == -INFINITY ? 0.f : mx;
          f[nt][e] = ex2(m[nt][e] - use);
          grew = grew || mx > m[nt][e];
          m[nt][e] = mx;
          float add = 0.f;
#pragma unroll
          for (int ns = 0; ns < NS; ++ns) {
            sc[ns][nt][e] = ex2(sc[ns][nt][e] - use);
            sc[ns][nt][e + 2] = ex2(sc[ns][nt][e + 2] - use);
            add += sc[ns][nt][e] + sc[ns][nt][e + 2];
          }
          l[nt][e] = l[nt][e] * f[nt][e] + add;
        }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < VC; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][i][j][e] *= f[nt][e & 1];
      }
      // O^T += V^T P^T
#pragma unroll
      for (int ns = 0; ns < NS; ++ns) {
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          pb[nt][0] = transpose8(Pair<T>::pack(sc[ns][nt][0], sc[ns][nt][1]));
          pb[nt][1] = transpose8(Pair<T>::pack(sc[ns][nt][2], sc[ns][nt][3]));
        }
#pragma unroll
        for (int i = 0; i < VC; ++i) {
          const uint32_t* v0 = &vr[ns][i][0].x;
          const uint32_t* v1 = &vr[ns][i][1].x;
          const uint32_t* v2 = &vr[ns][i][2].x;
          const uint32_t* v3 = &vr[ns][i][3].x;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a0 = __byte_perm(v0[j], v1[j], 0x5410), a1 = __byte_perm(v0[j], v1[j], 0x7632);
            const uint32_t a2 = __byte_perm(v2[j], v3[j], 0x5410), a3 = __byte_perm(v2[j], v3[j], 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_t<T>(o[nt][i][j], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
        }
      }
      load_v(pid);
    }
    if (!entered) {  // this warp had no step here
      s = seg_end;
      advance();
      load_k(pid);
      load_v(pid);
      pages_of(row_table, s + kStride, s_end, nxt);
    }
    cp_async_wait_all();
    if (dealer) deal(sm.seg[(x + 2) % 3]);

    // ---- join the four warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], d);
        if (g == 0) {
          sm.m[warp][nt * 8 + 2 * c + e] = m[nt][e];
          sm.l[warp][nt * 8 + 2 * c + e] = l[nt][e];
        }
#pragma unroll
        for (int i = 0; i < VC; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float2*>(&sm.o[warp][nt * 8 + 2 * c + e][64 * i + 8 * g + 2 * j]) =
                make_float2(o[nt][i][j][e], o[nt][i][j][e + 2]);
      }
    __syncthreads();
    const bool begins = sg.blk == 0, ends = sg.blk + sg.n == sg.nblk;
    const int part = 2 * blockIdx.x + (begins ? 1 : 0);
    float* part_ml = reinterpret_cast<float*>(a.ws + a.ml_off) + static_cast<int64_t>(part) * R * 2;
    float* part_o = reinterpret_cast<float*>(a.ws + a.o_off) + static_cast<int64_t>(part) * R * D;
    // a thread has kPieces pieces of four elements of one row
    constexpr int kLanes = kThreads / R, kPieces = D / 4 / kLanes;
    const bool done = begins && ends;
    const int r = tid / kLanes, d0 = (tid % kLanes) * 4, row = row0 + r;
    if (row < work) {
      const int i = by_group(a, row), t = sg.q0 + i, head = sg.h * a.group + row - i * a.group;
      uint2 gw[kPieces];
      if (done && a.gate) {
#pragma unroll
        for (int y = 0; y < kPieces; ++y)
          gw[y] = __ldg(reinterpret_cast<const uint2*>(attn_gate<T>(a, t, head) + d0 + 4 * kLanes * y));
      }
      float mx = sm.m[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, sm.m[w][r]);
      const float use = mx == -INFINITY ? 0.f : mx;
      float wf[kWarps], ls = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        wf[w] = ex2(sm.m[w][r] - use);
        ls = fmaf(sm.l[w][r], wf[w], ls);
      }
      if (d0 == 0) {
        if (done)
          attn_write_lse(a, t, head, mx, ls);
        else
          part_ml[2 * r] = mx, part_ml[2 * r + 1] = ls;
      }
      if (done) {
        const float inv = ls > 0.f ? 1.0f / ls : 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) wf[w] *= inv;
      }
#pragma unroll
      for (int y = 0; y < kPieces; ++y) {
        const int d = d0 + 4 * kLanes * y;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(&sm.o[w][r][d]);
          acc.x = fmaf(v.x, wf[w], acc.x), acc.y = fmaf(v.y, wf[w], acc.y);
          acc.z = fmaf(v.z, wf[w], acc.z), acc.w = fmaf(v.w, wf[w], acc.w);
        }
        if (done)
          attn_write_four<T, D>(a, t, head, d, acc, gw[y]);
        else
          *reinterpret_cast<float4*>(part_o + r * D + d) = acc;
      }
    }
    if (begins && !ends && tid == 0) {
      // (a tile that is begun and not ended is the CTA's last: its units end
      // nblk - n behind the CTA's own)
      Begun bg;
      bg.last = static_cast<int>((u1 + (sg.nblk - sg.n) - 1) / share);
      bg.q0 = sg.q0, bg.work = work, bg.h = sg.h, bg.tile = sg.tile;
      begun[blockIdx.x] = bg;
    }
    __syncthreads();  // the join's shared memory is free again
  }
}

// Block (i, r): row r of the tile that CTA i of the kernel above began, from the
// parts of CTAs i .. last, in order.
template <typename T, int D, int R>
__global__ void __launch_bounds__(256) k_attn_join(const AttnArgs a) {
  constexpr int kCols = D / 4, kWays = 256 / kCols;
  __shared__ float4 acc_s[kWays][kCols];
  __shared__ float red[8], lred[kWays];
  after_previous();
  const Begun bg = reinterpret_cast<const Begun*>(a.ws)[blockIdx.x];
  const int r = blockIdx.y, row = bg.tile * R + r;
  if (bg.last < 0 || row >= bg.work) return;
  const int tid = threadIdx.x, n = bg.last - static_cast<int>(blockIdx.x) + 1;
  const float* ml = reinterpret_cast<const float*>(a.ws + a.ml_off);
  const float* po = reinterpret_cast<const float*>(a.ws + a.o_off);
  auto part = [&](int i) { return static_cast<int64_t>(2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * R + r; };
  const int col = tid % kCols, way = tid / kCols;
  const int i = by_group(a, row), t = bg.q0 + i, head = bg.h * a.group + row - i * a.group;
  uint2 gw = make_uint2(0, 0);
  if (a.gate && way == 0) gw = __ldg(reinterpret_cast<const uint2*>(attn_gate<T>(a, t, head) + 4 * col));
  float mx = -INFINITY;
  for (int i = tid; i < n; i += 256) mx = fmaxf(mx, ml[2 * part(i)]);
  mx = warp_max(mx);
  if ((tid & 31) == 0) red[tid >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) mx = fmaxf(mx, red[w]);
  const float use = mx == -INFINITY ? 0.f : mx;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float ls = 0.f;
#pragma unroll 4
  for (int i = way; i < n; i += kWays) {
    const int64_t p = part(i);
    const float f = ex2(ml[2 * p] - use);
    const float4 v = *reinterpret_cast<const float4*>(po + p * D + 4 * col);
    acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y);
    acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
    ls = fmaf(ml[2 * p + 1], f, ls);
  }
  acc_s[way][col] = acc;
  if (col == 0) lred[way] = ls;
  __syncthreads();
  if (way == 0) {
#pragma unroll
    for (int w = 1; w < kWays; ++w) {
      const float4 v = acc_s[w][col];
      acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
    }
    ls = lred[0];
#pragma unroll
    for (int w = 1; w < kWays; ++w) ls += lred[w];
    attn_write_row<T, D>(a, t, head, 4 * col, acc, mx, ls, gw);
  }
}

struct Plan {
  int R, grid, rows;  // rows a tile, CTAs, rows that a tile can have in use
  size_t ml_off, o_off, bytes;
  bool many;       // the many-row kernel may have work
  AttnArgs split;  // its split of tiles (the fields that plan_split sets)
};

int max_kv_of(const rnb_attn_desc* d, const rnb_kv_cache* c) {
  const int64_t kv = static_cast<int64_t>(d->table_cols) * c->page_size;
  return static_cast<int>(kv < INT32_MAX - 4096 ? kv : INT32_MAX - 4096);  // steps ahead stay in 31 bits
}

Plan plan_of(const rnb_attn_desc* d, const rnb_kv_cache* c, int sms, bool cu_given) {
  Plan p;
  const int64_t group = d->n_q_heads / c->n_kv_heads;
  // rows of one request, as far as they are known
  const int64_t most = !cu_given ? 1 : d->max_q > 0 ? d->max_q : d->T > d->B ? d->T : 1;
  // 8 rows where all fit (half the registers and products of 16); heads of 256
  // always, since 16 of them do not fit the registers
  p.R = c->head_dim == 256 || most * group <= 8 ? 8 : 16;
  p.rows = static_cast<int>(!cu_given && group < p.R ? group : p.R);
  p.grid = 2 * sms;
  p.ml_off = (sizeof(Begun) * p.grid + 255) & ~size_t(255);
  p.o_off = (p.ml_off + 2u * p.grid * p.R * 2 * sizeof(float) + 255) & ~size_t(255);
  p.bytes = p.o_off + 2u * p.grid * p.R * static_cast<size_t>(c->head_dim) * sizeof(float);
  p.many = cu_given && (d->max_q > 0 ? d->max_q : d->T) * group >= kManyRows;
  p.split = AttnArgs{};
  if (p.many) {
    // (the two kernels' parts follow each other in one workspace)
    size_t bytes = 0;
    p.split.T = d->T, p.split.B = d->B, p.split.Hkv = c->n_kv_heads, p.split.group = static_cast<int>(group);
    p.split.max_kv = max_kv_of(d, c);
    plan_split(&p.split, c->head_dim, sms, &bytes);
    if (bytes > p.bytes) p.bytes = bytes;
  }
  return p;
}

template <typename T, int D, int NT>
int run_few(const AttnArgs& a, int grid, int rows, cudaStream_t st) {
  const int64_t tiles = static_cast<int64_t>(a.B) * a.Hkv * ((a.group + 8 * NT - 1) / (8 * NT));
  const unsigned ctas = static_cast<unsigned>(a.direct && tiles < grid ? tiles : grid);
  const int rc = launch("rnb_paged_attention", k_attn_few<T, D, NT>, ctas, kThreads, 0, st, a);
  if (rc || a.direct) return rc;
  return launch("rnb_paged_attention join", k_attn_join<T, D, 8 * NT>, dim3(grid, rows), 256, 0, st, a);
}

template <typename T>
int run_few_typed(const AttnArgs& a, int D, const Plan& p, cudaStream_t st) {
  if (D == 256) return run_few<T, 256, 1>(a, p.grid, p.rows, st);
  if (D == 128) return p.R == 8 ? run_few<T, 128, 1>(a, p.grid, p.rows, st) : run_few<T, 128, 2>(a, p.grid, p.rows, st);
  return p.R == 8 ? run_few<T, 64, 1>(a, p.grid, p.rows, st) : run_few<T, 64, 2>(a, p.grid, p.rows, st);
}

int check_attn(const rnb_attn_desc* d, const rnb_kv_cache* c) {
  if (!d) return fail(RNB_ERR_INVALID, "rnb_paged_attention: descriptor is NULL");
  int rc = check_cache(c, "rnb_paged_attention");
  if (rc) return rc;
  if (d->B < 0 || d->T < 0) return fail(RNB_ERR_INVALID, "rnb_paged_attention: B and T must be >= 0");
  if (d->n_q_heads <= 0 || d->n_q_heads % c->n_kv_heads)
    return fail(RNB_ERR_INVALID, "rnb_paged_attention: n_q_heads must be a positive multiple of n_kv_heads");
  if (static_cast<int64_t>(d->T) * d->n_q_heads > INT32_MAX)
    return fail(RNB_ERR_INVALID, "rnb_paged_attention: T * n_q_heads must be below 2^31");
  if (d->table_cols <= 0) return fail(RNB_ERR_INVALID, "rnb_paged_attention: table_cols must be positive");
  if (d->max_q < 0 || d->window < 0)
    return fail(RNB_ERR_INVALID, "rnb_paged_attention: max_q and window must be >= 0");
  if (!(d->scale > 0.f) || !(d->scale < INFINITY))
    return fail(RNB_ERR_INVALID, "rnb_paged_attention: scale must be positive and finite");
  const int64_t st[4] = {d->q_token_stride, d->q_head_stride, d->gate_token_stride, d->gate_head_stride};
  for (int64_t v : st)
    if (v < 0 || v % 8) return fail(RNB_ERR_INVALID, "rnb_paged_attention: strides must be multiples of 8 elements");
  return RNB_OK;
}

}  // namespace

cudaError_t attn_status_word(uint32_t** p) { return status_word(g_attn_status, p); }

}  // namespace rnb

extern "C" {

int rnb_paged_attention_workspace_size(const rnb_attn_desc* d, const rnb_kv_cache* cache, size_t* bytes) {
  using namespace rnb;
  if (!bytes) return fail(RNB_ERR_INVALID, "bytes must be non-NULL");
  int rc = check_attn(d, cache);
  if (rc) return rc;
  const int sms = dev_info().sms;
  *bytes = plan_of(d, cache, sms > 0 ? sms : 148, true).bytes;
  return RNB_OK;
}

int rnb_paged_attention(const rnb_attn_desc* d, const rnb_kv_cache* cache, const void* q, const void* gate,
                        const int32_t* table, const int32_t* seq_lens, const int32_t* cu_q, void* out, float* lse,
                        void* ws, size_t ws_bytes, void* stream) {
  using namespace rnb;
  int rc = check_attn(d, cache);
  if (rc) return rc;
  if (!cu_q && d->T != d->B)
    return fail(RNB_ERR_INVALID, "rnb_paged_attention: without cu_q every request has one row (T == B)");
  if (d->B == 0 || d->T == 0) return RNB_OK;
  if (!q || !out || !table || !seq_lens)
    return fail(RNB_ERR_INVALID, "rnb_paged_attention: q, out, table and seq_lens must be non-NULL");
  if (!aligned16(q) || !aligned16(gate) || !aligned16(out) || !aligned16(ws))
    return fail(RNB_ERR_ALIGN, "rnb_paged_attention: q, gate, out and the workspace must be 16-byte aligned");
  // CTAs write rows of out while others still read theirs of q and gate
  const int64_t D = cache->head_dim;
  const bool in_place = out == q && (d->T == 1 || d->q_token_stride == D * d->n_q_heads) &&
                        (d->n_q_heads == 1 || d->q_head_stride == D);
  if (!in_place && shares_memory(out, d->T, d->n_q_heads, D, q, d->q_token_stride, d->q_head_stride, d->n_q_heads))
    return fail(RNB_ERR_INVALID,
                "rnb_paged_attention: out may be q where q is packed [T][n_q_heads][head_dim]; otherwise they must not "
                "share memory");
  if (shares_memory(out, d->T, d->n_q_heads, D, gate, d->gate_token_stride, d->gate_head_stride, d->n_q_heads))
    return fail(RNB_ERR_INVALID, "rnb_paged_attention: out and gate must not share memory");
  if ((rc = check_device())) return rc;
  const Plan p = plan_of(d, cache, dev_info().sms, cu_q != nullptr);
  if (!ws || ws_bytes < p.bytes)
    return fail(RNB_ERR_WORKSPACE, "rnb_paged_attention: the workspace needs " + std::to_string(p.bytes) + " bytes");

  AttnArgs a{};
  a.q = q, a.gate = gate, a.out = out, a.lse = lse;
  a.kc = cache->k, a.vc = cache->v;
  a.table = table, a.seq = seq_lens, a.cu = cu_q;
  a.ws = static_cast<char*>(ws), a.ml_off = p.ml_off, a.o_off = p.o_off;
  a.q_ts = d->q_token_stride, a.q_hs = d->q_head_stride;
  a.g_ts = d->gate_token_stride, a.g_hs = d->gate_head_stride;
  a.kc_ps = cache->k_page_stride, a.kc_hs = cache->k_head_stride;
  a.vc_ps = cache->v_page_stride, a.vc_hs = cache->v_head_stride;
  a.B = d->B, a.T = d->T, a.W = d->table_cols;
  a.Hq = d->n_q_heads, a.Hkv = cache->n_kv_heads;
  set_group(&a, a.Hq / a.Hkv);
  while ((1 << a.log2p) < cache->page_size) ++a.log2p;
  a.num_pages = cache->num_pages;
  a.max_kv = max_kv_of(d, cache);
  a.window = d->window < a.max_kv ? d->window : 0;
  a.few_rows = INT32_MAX;
  a.scale_log2 = d->scale * 1.4426950408889634f;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // One row a request and short tables: whole tiles, without the sums over the
  // requests and without the join (one request at head_dim 128: 256 positions 8.8 ->
  // 6.6 us, 64 at head_dim 256 10.2 -> 6.4).  A CTA walks a tile at 1.3 us a 64 KB of keys
  // and values, so longer ones are split; at this border (224 positions of 256, 448 of
  // 128) both take the same.
  a.direct = !cu_q && static_cast<int64_t>(a.max_kv) * cache->head_dim <= 224 * 256;
  if (p.many) {
    PromptMaps maps;
    if (prepare_prompt(a, cache, &maps)) {
      // (a single request is wholly the many-row kernel's, however few its rows are)
      a.few_rows = d->B == 1 ? 1 : kManyRows;
      AttnArgs m = a;
      m.split = p.split.split, m.ml_off = p.split.ml_off, m.o_off = p.split.o_off;
      if ((rc = run_prompt(m, cache, maps, st))) return rc;
      if (d->B == 1) return RNB_OK;
    }
  }
  return cache->dtype == RNB_DTYPE_BF16 ? run_few_typed<__nv_bfloat16>(a, cache->head_dim, p, st)
                                        : run_few_typed<__half>(a, cache->head_dim, p, st);
}

}  // extern "C"
