// rnb_attn_prompt.cu -- attention over the paged cache for requests with many
// query rows (prompts), on the 5th-generation tensor cores.
//
// One CTA takes 128 (head_dim 256) or 256 query rows of one key head: rows are
// (token, query head of the group) pairs, so the group's heads share every key
// and value that is loaded.  Over blocks of 128 positions
//     S = Q K^T,  P = 2^(scale log2e S - m),  O += P V,  l += rowsum P
// with S, P and O in tensor memory: S is 128 fp32 columns, P overwrites it as
// 16-bit pairs and is the A operand of the second product from there, so no
// probability passes through shared memory.  A thread owns a row: its maximum
// and sum need no exchange.
//
// * The maximum is lazy: m only moves when a row's maximum exceeds it by more
//   than 8 (P stays below 2^8, in range of both types), so O is hardly ever
//   rescaled after the first blocks.
// * Two S slots keep the tensor cores fed: while the softmax of one slot runs,
//   the products of the other do.  With head_dim <= 128 the slots are two row
//   tiles with a softmax warpgroup each; with 256, where one O fills half the tensor
//   memory, they are two successive blocks of one tile.
// * Keys and values come by TMA page by page into a ring of 128-byte-swizzled
//   units, K as the K-major and V as the MN-major operand, both as they lie in the
//   cache.  Pages behind the request's end (and ids out of range) are fetched at
//   a page coordinate behind the cache, which reads as zeros.
// * Every wait is bounded; one that gives up ends the CTA with RNB_STATUS_TIMEOUT.
//
// The tensor cores bound it for head_dim 256 (4 D flops a row and position
// against one exponential), with head_dim 64 the exponentials do.
#include <cuda.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include <string>

#include "rnb_attn.cuh"
#include "rnb_umma.cuh"

namespace rnb {
namespace {

__device__ uint32_t g_prompt_status;

constexpr int kBlk = 128;  // positions a block
constexpr uint64_t kWaitNs = 1000000000ull;

template <int D>
struct Cfg {
  static constexpr int NQ = D == 256 ? 1 : 2;              // row tiles a CTA
  static constexpr int kRows = 128 * NQ;
  static constexpr int kThreads = 128 + 128 * NQ;          // loader, issuer, two idle warps; softmax warpgroups
  static constexpr int UPT = D == 256 ? 2 : 1;             // ring units a K or V block
  static constexpr int kUnit = kBlk * D * 2 / UPT;         // bytes
  static constexpr int VR = kBlk / UPT;                    // V rows a unit (all of D)
  static constexpr int KD = D / UPT;                       // K elements a unit (all rows)
  static constexpr int NST = D == 64 ? 8 : 5;
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kSmem = kQBytes + NST * kUnit + 1024;
  static constexpr int kTmemO = 256;                       // S slots at columns 0 and 128
};

// D[tmem] (+)= A[tmem] * B[smem]; issued by one thread.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0)
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// MN-major SWIZZLE_128B operand: 64 elements of the M/N side are a 128-byte
// row, rows are the contraction index; 8-row atoms every 1024 bytes, 64-element
// columns every `lead` bytes.
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t saddr, uint32_t lead) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((lead >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// A whole warp waits: true for all its lanes or for none.  The clock is only
// read where the first try did not do.
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity) {
  bool ok = mbar_try(bar, parity);
  if (!ok) ok = mbar_wait(bar, parity, kWaitNs);
  return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Bars {
  uint64_t full[8], empty[8];   // ring units
  uint64_t q_full;              // Q in shared memory
  uint64_t s_full[2], p_full[2];  // slots: S written, P written (S read)
  uint64_t o_done[2];           // row tiles: a P V product done
  uint64_t o_last[2];           // row tiles: the last one done
  uint64_t drained;             // every product of the CTA done
};

template <typename T, int D>
__global__ void __launch_bounds__(Cfg<D>::kThreads, 1)
    k_attn_prompt(const AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                  int k_box, int v_box) {
  using C = Cfg<D>;
  extern __shared__ char raw[];
  __shared__ Bars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ int64_t wsum[C::kThreads / 32];
  __shared__ int found_b, found_tile;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  char* ring = smem + C::kQBytes;

  // ---- which request and tile: tiles of a request from its end (the longest first)
  const int h = blockIdx.x % a.Hkv;
  const int64_t want = blockIdx.x / a.Hkv;
  {
    if (tid == 0) found_b = -1;
    const int per = (a.B + C::kThreads - 1) / C::kThreads;
    const int lo = min(tid * per, a.B), hi = min(lo + per, a.B);
    auto tiles = [&](int b) {
      const int c0 = min(max(a.cu[b], 0), a.T), c1 = min(max(a.cu[b + 1], c0), a.T);
      const int work = (c1 - c0) * a.group;
      return work >= a.few_rows ? (work + C::kRows - 1) / C::kRows : 0;
    };
    int64_t sum = 0;
    for (int b = lo; b < hi; ++b) sum += tiles(b);
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
    if (want >= base && want < base + sum) {
      int64_t rem = want - base;
      int b = lo;
      int n = tiles(b);
      while (rem >= n) {
        rem -= n;
        n = tiles(++b);
      }
      found_b = b;
      found_tile = n - 1 - static_cast<int>(rem);
    }
    __syncthreads();
  }
  const int b = found_b, tile = found_tile;
  // (after a wait that gave up, until the status is read: a grid of CTAs that
  // each wait their second would hold the device for minutes)
  if (b < 0 || (*const_cast<volatile uint32_t*>(&g_prompt_status) & RNB_STATUS_TIMEOUT)) return;
  const int q0 = min(max(a.cu[b], 0), a.T), rows = min(max(a.cu[b + 1], q0), a.T) - q0;
  const int len_raw = a.seq[b], len = min(max(len_raw, 0), a.max_kv);
  const int work = rows * a.group, p0 = len - rows;
  const int row0 = tile * C::kRows, row_end = min(row0 + C::kRows, work);
  const int first_p = p0 + row0 / a.group, last_p = p0 + (row_end - 1) / a.group;
  const int any_lo = a.window > 0 ? max(first_p - a.window + 1, 0) : 0;
  const int kv_end = max(last_p + 1, 0);
  const int blk0 = any_lo / kBlk;
  const int nblk = max((kv_end + kBlk - 1) / kBlk - blk0, 0);
  const int32_t* row_table = a.table + static_cast<int64_t>(b) * a.W;

  // page ids out of range in this tile's positions: their masks need the table
  int bad = 0;
  for (int j = (any_lo >> a.log2p) + tid; j < (kv_end + (1 << a.log2p) - 1) >> a.log2p; j += C::kThreads)
    bad |= static_cast<uint32_t>(__ldg(row_table + j)) >= static_cast<uint32_t>(a.num_pages);

  if (tid == 0) {
    for (int i = 0; i < C::NST; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    mbar_init(&bars.q_full, 4 * C::NQ);
    mbar_init(&bars.drained, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 4);
      mbar_init(&bars.o_done[i], 1);
      mbar_init(&bars.o_last[i], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (len_raw != len) atomicOr(&g_prompt_status, RNB_STATUS_BAD_INDEX);
  }
  if (warp == 2) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  bad = __syncthreads_or(bad);
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  if (bad && tid == 0) atomicOr(&g_prompt_status, RNB_STATUS_BAD_INDEX);
  bool alive = true;
  const int jobs = nblk * C::NQ;  // job k: slot k & 1; two row tiles a block, or a block a job

  if (warp == 0) {
    // ---- loader: units in the order in which the issuer uses them
    const uint32_t rbase = smem_u32(ring);
    const int pmask = (1 << a.log2p) - 1;
    int u = 0;
    auto ids = [&](int blk) {  // lane l: the page of the block's subtile l of 16 positions
      const int t = blk * kBlk + 16 * lane;
      int id = a.num_pages;
      if (lane < kBlk / 16 && t < kv_end && (t | pmask) >= any_lo) {  // its page holds seen positions
        const int p = __ldg(row_table + (t >> a.log2p));
        if (static_cast<uint32_t>(p) < static_cast<uint32_t>(a.num_pages)) id = p;
      }
      return id;
    };
    auto load = [&](bool is_k, int blk, int id) {
      for (int part = 0; part < C::UPT && alive; ++part, ++u) {
        const int st = u % C::NST;
        alive = wait_on(&bars.empty[st], ((u / C::NST) & 1) ^ 1);
        if (!alive) break;
        const uint32_t bar = smem_u32(&bars.full[st]), dst = rbase + st * C::kUnit;
        if (lane == 0) mbar_arrive_expect_tx(&bars.full[st], C::kUnit);
        __syncwarp();
        const int box = is_k ? k_box : v_box;
        const int rows_u = is_k ? kBlk : C::VR, skip = is_k ? 0 : part * C::VR;
        const int nbox = rows_u / box;
        const int page = __shfl_sync(0xffffffffu, id, ((skip + lane * box) >> 4) & 31);
        if (lane < nbox) {
          const int t = blk * kBlk + skip + lane * box;
          const int nch = is_k ? C::KD / 64 : D / 64, ch0 = is_k ? part * (C::KD / 64) : 0;
          for (int c = 0; c < nch; ++c)
            tma_load_4d(dst + (c * rows_u + lane * box) * 128, is_k ? static_cast<const void*>(&kmap) : &vmap,
                        (ch0 + c) * 64, t & pmask, h, page, bar);
        }
        __syncwarp();
      }
    };
    if (nblk > 0) {
      if (C::NQ == 2) {
        int id = ids(blk0);
        for (int i = 0; i < nblk && alive; ++i) {
          const int next = i + 1 < nblk ? ids(blk0 + i + 1) : 0;
          load(true, blk0 + i, id);
          load(false, blk0 + i, id);
          id = next;
        }
      } else {
        int id = ids(blk0), next = nblk > 1 ? ids(blk0 + 1) : 0;
        load(true, blk0, id);
        for (int i = 0; i < nblk && alive; ++i) {
          const int ahead = i + 2 < nblk ? ids(blk0 + i + 2) : 0;
          if (i + 1 < nblk) load(true, blk0 + i + 1, next);
          load(false, blk0 + i, id);
          id = next;
          next = ahead;
        }
      }
    }
    // no copy may be in flight when the CTA ends
    for (int v = max(u - C::NST, 0); v < u; ++v) wait_on(&bars.full[v % C::NST], (v / C::NST) & 1);
  } else if (warp == 1) {
    // ---- issuer
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    const uint32_t id_s = umma_idesc_f16(128, kBlk, kBf16);
    const uint32_t id_o = umma_idesc_f16(128, D, kBf16) | (1u << 16);  // B is MN-major
    const uint32_t rbase = smem_u32(ring), qbase = smem_u32(smem);
    // ring units of block i: with two row tiles K0 V0 K1 V1 ..., else K0 K1 V0 K2 V1 ...
    auto unit_k = [&](int i) { return (C::NQ == 2 ? 2 * i : i == 0 ? 0 : 2 * i - 1) * C::UPT; };
    auto unit_v = [&](int i) { return (C::NQ == 2 ? 2 * i + 1 : min(2 + 2 * i, 2 * nblk - 1)) * C::UPT; };
    auto issue_s = [&](int k) {
      const int i = C::NQ == 2 ? k >> 1 : k, q = C::NQ == 2 ? k & 1 : 0;
      for (int part = 0; part < C::UPT && alive; ++part) {
        const int u = unit_k(i) + part, st = u % C::NST;
        alive = wait_on(&bars.full[st], (u / C::NST) & 1);
        if (!alive) return;
        tc_fence_after();
        if (lane == 0) {
#pragma unroll
          for (int c = 0; c < C::KD / 64; ++c)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              const int ch = part * (C::KD / 64) + c;
              const uint32_t qa = qbase + (q * (D / 64) + ch) * 128 * 128 + 32 * s;
              const uint32_t ka = rbase + st * C::kUnit + c * kBlk * 128 + 32 * s;
              umma_f16(tmem + (k & 1) * 128, umma_desc_sw128(qa), umma_desc_sw128(ka), id_s, (ch | s) != 0);
            }
          if (C::NQ == 1 || q == 1) umma_commit(smem_u32(&bars.empty[st]));
          if (part == C::UPT - 1) umma_commit(smem_u32(&bars.s_full[k & 1]));
        }
        __syncwarp();
      }
    };
    auto issue_o = [&](int k) {
      const int i = C::NQ == 2 ? k >> 1 : k, q = C::NQ == 2 ? k & 1 : 0;
      for (int part = 0; part < C::UPT && alive; ++part) {
        const int u = unit_v(i) + part, st = u % C::NST;
        alive = wait_on(&bars.full[st], (u / C::NST) & 1);
        if (!alive) return;
        const int t0 = (blk0 + i) * kBlk + part * C::VR;
        if (q == 0 && (t0 + C::VR > kv_end || t0 < any_lo)) {
          // rows that no query row of the tile sees may hold any bits: 0 * NaN must not count
          for (int r = 0; r < C::VR; ++r)
            if (t0 + r >= kv_end || t0 + r < any_lo)
              for (int x = lane; x < D / 8; x += 32)
                *reinterpret_cast<uint4*>(ring + st * C::kUnit + ((x >> 3) * C::VR + r) * 128 + (x & 7) * 16) =
                    make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (part == 0) {
          alive = wait_on(&bars.p_full[k & 1], (k >> 1) & 1);
          if (!alive) return;
        }
        tc_fence_after();
        if (lane == 0) {
#pragma unroll
          for (int s = 0; s < C::VR / 16; ++s) {
            const uint32_t va = rbase + st * C::kUnit + s * 16 * 128;
            umma_f16_ts(tmem + C::kTmemO + q * D, tmem + (k & 1) * 128 + (part * C::VR + s * 16) / 2,
                        umma_desc_mn(va, C::VR * 128), id_o, i != 0 || part != 0 || s != 0);
          }
          if (C::NQ == 1 || q == 1) umma_commit(smem_u32(&bars.empty[st]));
          if (part == C::UPT - 1) umma_commit(smem_u32(i + 1 < nblk ? &bars.o_done[q] : &bars.o_last[q]));
        }
        __syncwarp();
      }
    };
    if (jobs > 0) {
      alive = wait_on(&bars.q_full, 0);
      tc_fence_after();
      if (alive) issue_s(0);
      if (alive && jobs > 1) issue_s(1);
      for (int k = 0; k < jobs && alive; ++k) {
        issue_o(k);
        if (alive && k + 2 < jobs) issue_s(k + 2);
      }
      // no product may be in flight when the tensor memory is given back
      if (lane == 0) umma_commit(smem_u32(&bars.drained));
      __syncwarp();
      wait_on(&bars.drained, 0);
    }
  } else if (warp >= 4) {
    // ---- softmax: a thread is a row of tile wg
    const int wg = (warp - 4) >> 2, r = tid - 128 - 128 * wg;
    const int row = row0 + wg * 128 + r;
    // Q into the K-major layout, coalesced over the rows' elements
    for (int x = r; x < 128 * (D / 8); x += 128) {
      const int qr = x / (D / 8), e = (x - qr * (D / 8)) * 8, rr = row0 + wg * 128 + qr;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (rr < work) {
        const int i = rr / a.group, j = rr - i * a.group;
        v = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (q0 + i) * a.q_ts +
                                                 (h * a.group + j) * a.q_hs + e));
      }
      *reinterpret_cast<uint4*>(smem + (wg * (D / 64) + (e >> 6)) * 128 * 128 + sw128_offset(qr, e & 63)) = v;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.q_full);

    const int pos = p0 + min(row, work - 1) / a.group;
    const int see_lo = a.window > 0 ? pos - a.window + 1 : INT_MIN;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_o = tmem + C::kTmemO + wg * D + lane_base;
    // positions that all rows of this warpgroup's tile see
    const int wg_first = p0 + min(row0 + wg * 128, work - 1) / a.group;
    const int wg_last = p0 + min(row0 + wg * 128 + 127, work - 1) / a.group;
    const int all_lo = a.window > 0 ? wg_last - a.window + 1 : INT_MIN;
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < nblk && alive; ++i) {
      const int k = C::NQ == 2 ? 2 * i + wg : i, slot = k & 1;
      const uint32_t t_s = tmem + slot * 128 + lane_base;
      alive = wait_on(&bars.s_full[slot], (k >> 1) & 1);
      if (!alive) break;
      tc_fence_after();
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(t_s + 32 * c, v[c]);
      tmem_wait_ld();
      const int t0 = (blk0 + i) * kBlk;
      if (bad || t0 + kBlk - 1 > wg_first || t0 < all_lo) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int t = t0 + 32 * c + e;
            if (t > pos || t < see_lo) v[c][e] = __float_as_uint(-INFINITY);
          }
        if (bad) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 16) {
              const int t = t0 + 32 * c + e;
              if (t < kv_end && static_cast<uint32_t>(__ldg(row_table + (t >> a.log2p))) >=
                                    static_cast<uint32_t>(a.num_pages)) {
#pragma unroll
                for (int f = 0; f < 16; ++f) v[c][e + f] = __float_as_uint(-INFINITY);
              }
            }
        }
      }
      float mx = __uint_as_float(v[0][0]);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 32; ++e) mx = fmaxf(mx, __uint_as_float(v[c][e]));
      mx *= a.scale_log2;
      if (__any_sync(0xffffffffu, mx > m + 8.f)) {
        const float to = fmaxf(m, mx);
        const float f = ex2(m - (to == -INFINITY ? 0.f : to));
        m = to;
        l *= f;
        if (i > 0) {
          // the product before this one has to be in O (the one before that is:
          // S of this block was issued behind it)
          alive = wait_on(&bars.o_done[wg], (i - 1) & 1);
          if (!alive) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(t_o + 32 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st32(t_o + 32 * c, o);
          }
        }
      }
      const float use = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = ex2(fmaf(__uint_as_float(v[c][2 * e]), a.scale_log2, -use));
          const float y = ex2(fmaf(__uint_as_float(v[c][2 * e + 1]), a.scale_log2, -use));
          l += x + y;
          p[e] = Pair<T>::pack(x, y);
        }
        tmem_st16(t_s + 16 * c, p);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.p_full[slot]);
    }
    // ---- O / l
    // (o_done would not do: the last two products may both be under way, and a
    // parity only tells neighbouring phases apart)
    if (alive && nblk > 0) alive = wait_on(&bars.o_last[wg], 0);
    tc_fence_after();
    if (alive) {
      const int t = q0 + row / a.group, head = h * a.group + row % a.group;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (nblk > 0) {
          tmem_ld32(t_o + 32 * c, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        if (row < work) {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            attn_write_row<T, D>(a, t, head, 32 * c + e,
                                 make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]),
                                             __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3])),
                                 m, l);
        }
      }
    }
  }
  if (!alive && lane == 0) atomicOr(&g_prompt_status, RNB_STATUS_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

template <typename T, int D>
int launch_prompt(const AttnArgs& a, const rnb_kv_cache* cache, const CUtensorMap& km, const CUtensorMap& vm, int kbox,
                  int vbox, cudaStream_t st) {
  using C = Cfg<D>;
  const cudaError_t e = cudaFuncSetAttribute(k_attn_prompt<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return fail(RNB_ERR_CUDA, std::string("rnb_paged_attention: ") + cudaGetErrorString(e));
  // as many tiles as there can be: CTAs without one end at once
  const int64_t most = (static_cast<int64_t>(a.T) * a.group + C::kRows - 1) / C::kRows;
  const int64_t tiles = most + (a.B < static_cast<int64_t>(a.T) ? a.B : a.T);
  if (tiles * a.Hkv > INT32_MAX) return fail(RNB_ERR_INVALID, "rnb_paged_attention: too many rows");
  k_attn_prompt<T, D><<<static_cast<unsigned>(tiles * a.Hkv), C::kThreads, C::kSmem, st>>>(a, km, vm, kbox, vbox);
  return launch_status("rnb_paged_attention");
}

bool encode_cache(CUtensorMap* m, const rnb_kv_cache* c, const void* base, int64_t page_stride, int64_t head_stride,
                  int box_rows) {
  const uint64_t D = c->head_dim, P = c->page_size;
  const uint64_t dims[4] = {D, P, static_cast<uint64_t>(c->n_kv_heads), static_cast<uint64_t>(c->num_pages)};
  // (a stride over an extent of one is never used, but has to be one that the encoder takes)
  const uint64_t str[3] = {2 * D, c->n_kv_heads > 1 ? 2u * static_cast<uint64_t>(head_stride) : 2 * D * P,
                           c->num_pages > 1 ? 2u * static_cast<uint64_t>(page_stride) : 2 * D * P};
  const uint32_t box[4] = {64, static_cast<uint32_t>(box_rows), 1, 1};
  return encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, base, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

int prompt_status_take(uint32_t* bits, cudaStream_t st) { return status_take(g_prompt_status, bits, st); }

bool prepare_prompt(const rnb_kv_cache* c, PromptMaps* p) {
  const int D = c->head_dim, P = c->page_size;
  p->k_box = P < kBlk ? P : kBlk;
  const int vr = D == 256 ? Cfg<256>::VR : kBlk;
  p->v_box = P < vr ? P : vr;
  return encode_cache(&p->k, c, c->k, c->k_page_stride, c->k_head_stride, p->k_box) &&
         encode_cache(&p->v, c, c->v, c->v_page_stride, c->v_head_stride, p->v_box);
}

int run_prompt(const AttnArgs& a, const rnb_kv_cache* c, const PromptMaps& p, cudaStream_t st) {
  const int D = c->head_dim;
  if (c->dtype == RNB_DTYPE_BF16) {
    if (D == 64) return launch_prompt<__nv_bfloat16, 64>(a, c, p.k, p.v, p.k_box, p.v_box, st);
    if (D == 128) return launch_prompt<__nv_bfloat16, 128>(a, c, p.k, p.v, p.k_box, p.v_box, st);
    return launch_prompt<__nv_bfloat16, 256>(a, c, p.k, p.v, p.k_box, p.v_box, st);
  }
  if (D == 64) return launch_prompt<__half, 64>(a, c, p.k, p.v, p.k_box, p.v_box, st);
  if (D == 128) return launch_prompt<__half, 128>(a, c, p.k, p.v, p.k_box, p.v_box, st);
  return launch_prompt<__half, 256>(a, c, p.k, p.v, p.k_box, p.v_box, st);
}

}  // namespace rnb
