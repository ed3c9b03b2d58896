// rnb_attn_prompt.cu -- attention over the paged cache for requests with many
// query rows (prompts), on the 5th-generation tensor cores.
//
// One CTA takes one (head_dim 256) or two tiles of up to 128 query rows of one
// key head: a tile is floor(128 / group) tokens with the group's query heads, so
// that the heads share every key and value that is loaded, and queries, gates
// and outputs are boxes of (tokens, heads, elements) that TMA moves.  Over blocks of positions
//     S = Q K^T,  P = 2^(scale log2e S - m),  O += P V,  l += rowsum P
// with S, P and O in tensor memory: S is a column a position, P overwrites it as
// 16-bit pairs and is the A operand of the second product from there, so no
// probability passes through shared memory.  A thread owns a row: its maximum
// and sum need no exchange.
//
// * The maximum is lazy: m only moves when a row's maximum exceeds it by more
//   than 8 (P stays below 2^8, in range of both types), so O is hardly ever
//   rescaled after the first blocks.
// * Two slots of S, a block of 128 positions each, keep the tensor cores and the
//   softmax apart.  With head_dim <= 128 there are two row tiles with a softmax
//   warpgroup and one slot each: one tile's products run under the other's softmax,
//   but a tile's own chain softmax, P V, next Q K is in series, since P lies in the
//   slot (3900 cycles a block, of which the products take 2048).  Two slots of 64 a
//   tile were slower: products of N = 64 read shared memory at its limit (8192 rows at
//   128: 626 instead of 534 us).  With 256, where one O fills half the tensor memory,
//   one tile has both slots, and S of a block is computed before P of the one before
//   it is done.
// * Keys and values come by TMA page by page into a ring of 128-byte-swizzled
//   units, K as the K-major and V as the MN-major operand, both as they lie in the
//   cache.  Pages behind the request's end (and ids out of range) are fetched at
//   a page coordinate behind the cache, which reads as zeros.
// * Where a call has so few tiles that SMs would stay idle (a few drafted tokens
//   of large groups, a prompt's end on a long cache), the positions of a tile are split
//   over CTAs: each leaves its (m, l, O) in the workspace and k_attn_join_tiles adds
//   a tile's parts in order.
// * Every wait is bounded; one that gives up ends the CTA with RNB_STATUS_TIMEOUT.
//
// The tensor cores bound it for head_dim 256 (4 D flops a row and position
// against one exponential), with head_dim 64 the exponentials do.
#include <cuda.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include <atomic>
#include <string>

#include "rnb_attn.cuh"
#include "rnb_umma.cuh"

namespace rnb {
namespace {

__device__ uint32_t g_prompt_status;
// The call whose wait gave up last (0: none).  A grid of CTAs that each wait their
// second would hold the device for minutes, so the rest of that call does nothing;
// other calls, on whatever stream, go on.
__device__ uint32_t g_gave_up;

constexpr uint64_t kWaitNs = 1000000000ull;

template <int D>
struct Cfg {
  static constexpr int NQ = D == 256 ? 1 : 2;              // row tiles a CTA
  static constexpr int BN = 128;                           // positions a block
  static constexpr int NS = 256 / BN;                      // S slots, of BN columns, in 256
  static constexpr int kThreads = 128 + 128 * NQ;          // loader, issuer, two idle warps; softmax warpgroups
  static constexpr int UPT = D == 256 ? 2 : 1;             // ring units a K or V block
  static constexpr int kUnit = BN * D * 2 / UPT;           // bytes
  static constexpr int VR = BN / UPT;                      // V rows a unit (all of D)
  static constexpr int KD = D / UPT;                       // K elements a unit (all rows)
  static constexpr int NST = D == 64 ? 8 : 5;              // ring units
  static constexpr int kQBytes = 128 * NQ * D * 2;
  static constexpr int kSmem = kQBytes + NST * kUnit + 1024;
  static constexpr int kTmemO = 256;
};

// D[tmem] (+)= A * B, A from shared memory (ss) or tensor memory (ts).  The
// whole warp executes these with one lane's predicate set: in a branch of one
// lane the operands would have to be moved to uniform registers one by one,
// which cost 115 cycles a product.
__device__ __forceinline__ void umma_ss(uint32_t leader, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}

__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, e;\n\t}"
      : "=r"(r));
  return r;
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

// 3-D tiled TMA store of a box in shared memory; its group is committed and
// waited for (until the box is read) by the issuing thread.
__device__ __forceinline__ void tma_store_3d(const void* tmap, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(tmap),
               "r"(x), "r"(y), "r"(z), "r"(src)
               : "memory");
}
__device__ __forceinline__ void bulk_commit_and_wait_read() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// A barrier of 128 threads: whether `ok` holds for all of them.
__device__ __forceinline__ bool all_of_128(int id, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(static_cast<uint32_t>(ok))
      : "memory");
  return r != 0;
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

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// A tile whose positions are split, for the join.
struct SplitTile {
  int parts;  // 0: no tile, or one that its CTA wrote
  int n;      // tiles of the call: part p is CTA p n + i's
  int q0, tok0, rows, h;
};

struct Bars {
  uint64_t full[10], empty[10];   // ring units
  uint64_t q_full;              // Q in shared memory
  uint64_t q_done;              // every product with Q done
  uint64_t g_full;              // the gates where Q was
  uint64_t s_full[2];           // slots: S written
  uint64_t p_full[2][2];        // slots: each half of P written (S read)
  uint64_t o_done[2];           // row tiles: a P V product done
  uint64_t o_last[2];           // row tiles: the last one done
  uint64_t drained;             // every product of the CTA done
};

template <typename T, int D>
__global__ void __launch_bounds__(Cfg<D>::kThreads, 1)
    k_attn_prompt(const AttnArgs a, const __grid_constant__ PromptMaps maps) {
  after_previous();
  using C = Cfg<D>;
  extern __shared__ char raw[];
  __shared__ Bars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ int64_t wsum[C::kThreads / 32];
  __shared__ int found[5];  // request, tile, first row, rows, length
  __shared__ bool gave_up;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  char* ring = smem + C::kQBytes;
  const int tt = maps.tokens;            // tokens a row tile
  const int cta_tokens = tt * C::NQ;

  // ---- which request and tokens: tiles of a request from its end (the longest first).
  // With a.split the grid's CTAs are dealt to the call's N tiles, the i-th of each N
  // to a tile's i-th part.
  SplitTile* split = reinterpret_cast<SplitTile*>(a.ws);
  int h = blockIdx.x % a.Hkv, part = 0, parts = 1, n_tiles = 0;
  int64_t want = blockIdx.x / a.Hkv;
  {
    if (tid == 0) {
      found[0] = -1;
      // (of several requests the few-row kernel tells)
      if (a.B == 1 && blockIdx.x == 0 && (a.cu[0] < 0 || a.cu[1] < a.cu[0] || a.cu[1] > a.T))
        atomicOr(&g_prompt_status, RNB_STATUS_BAD_INDEX);
      gave_up = *const_cast<volatile uint32_t*>(&g_gave_up) == a.call;
    }
    const int per = (a.B + C::kThreads - 1) / C::kThreads;
    const int lo = min(tid * per, a.B), hi = min(lo + per, a.B);
    int c0 = 0, c1 = 0, ln = 0;
    auto tiles = [&](int b) {
      c0 = min(max(a.cu[b], 0), a.T), c1 = min(max(a.cu[b + 1], c0), a.T);
      ln = a.seq[b];
      return (c1 - c0) * a.group >= a.few_rows ? (c1 - c0 + cta_tokens - 1) / cta_tokens : 0;
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
    if (a.split) {
      int64_t all = 0;
      for (int w = 0; w < C::kThreads / 32; ++w) all += wsum[w];
      n_tiles = static_cast<int>(all) * a.Hkv;  // at most the grid
      if (tid == 0) split[blockIdx.x].parts = 0;  // (until it is known)
      if (n_tiles > 0) {
        const int i = blockIdx.x % n_tiles;
        part = blockIdx.x / n_tiles, parts = gridDim.x / n_tiles;
        h = i % a.Hkv, want = part < parts ? i / a.Hkv : -1;
      }
    }
    if (want >= base && want < base + sum) {
      int64_t rem = want - base;
      int b = lo;
      int n = per == 1 ? static_cast<int>(sum) : tiles(b);
      while (rem >= n && b + 1 < hi) {  // (the second: row bounds that change under way must not lead out)
        rem -= n;
        n = tiles(++b);
      }
      found[0] = b, found[1] = n - 1 - static_cast<int>(rem);
      found[2] = c0, found[3] = c1 - c0, found[4] = ln;
    }
    __syncthreads();
  }
  const int b = found[0], tile = found[1], q0 = found[2], rows = found[3];
  if (b < 0 || gave_up) return;
  const int len = min(max(found[4], 0), a.max_kv);
  const int p0 = len - rows;                          // position of the request's first token
  const int tok0 = tile * cta_tokens, tok_end = min(tok0 + cta_tokens, rows);
  const int first_p = p0 + tok0, last_p = p0 + tok_end - 1;
  const int any_lo = a.window > 0 ? max(first_p - a.window + 1, 0) : 0;
  const int kv_end = max(last_p + 1, 0);
  int blk0 = any_lo / C::BN;
  int nblk = max((kv_end + C::BN - 1) / C::BN - blk0, 0);
  if (a.split) {
    // (two blocks a part or more: a part's start and end cost about two)
    parts = max(min(parts, nblk / 2), 1);
    if (tid == 0 && part == 0 && parts > 1) {
      SplitTile t;
      t.parts = parts, t.n = n_tiles;
      t.q0 = q0, t.tok0 = tok0, t.rows = rows, t.h = h;
      split[blockIdx.x] = t;
    }
    if (part >= parts) return;
    const int lo = static_cast<int>(static_cast<int64_t>(nblk) * part / parts);
    nblk = static_cast<int>(static_cast<int64_t>(nblk) * (part + 1) / parts) - lo;
    blk0 += lo;
  }
  const int32_t* row_table = a.table + static_cast<int64_t>(b) * a.W;
  // a row tile in shared memory: 64-element columns of 128 rows, 128-byte swizzle
  constexpr int kCol = 128 * 128;
  const uint32_t q_bytes = C::NQ * (D / 64) * static_cast<uint32_t>(tt * a.group) * 128;

  if (tid == 0) {
    for (int i = 0; i < C::NST; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_done, 1);
    mbar_init(&bars.g_full, 1);
    mbar_init(&bars.drained, 1);
    for (int i = 0; i < C::NS; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i][0], 4);
      mbar_init(&bars.p_full[i][1], 4);
    }
    for (int i = 0; i < C::NQ; ++i) {
      mbar_init(&bars.o_done[i], 1);
      mbar_init(&bars.o_last[i], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (found[4] != len) atomicOr(&g_prompt_status, RNB_STATUS_BAD_INDEX);
  }
  if (warp == 2) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  bool alive = true;
  // queries or gates of the CTA's tiles; tokens behind the last are read as
  // zeros or as another request's, whose rows are not used
  auto load_tiles = [&](const CUtensorMap* map, uint64_t* bar) {
    if (lane == 0) mbar_arrive_expect_tx(bar, q_bytes);
    __syncwarp();
    if (lane < C::NQ * (D / 64)) {
      const int q = lane / (D / 64), c = lane - q * (D / 64);
      tma_load_3d(smem_u32(smem) + lane * kCol, map, 64 * c, h * a.group, q0 + tok0 + q * tt, smem_u32(bar));
    }
    __syncwarp();
  };
  const int jobs = nblk * C::NQ;  // job k: block k / NQ of row tile k % NQ, in slot k % NS

  if (warp == 0) {
    // ---- loader: units in the order in which the issuer uses them
    const uint32_t rbase = smem_u32(ring);
    const int pmask = (1 << a.log2p) - 1;
    int u = 0;
    auto ids = [&](int blk) {  // lane l: the page of the block's subtile l of 16 positions
      const int t = blk * C::BN + 16 * lane;
      int id = a.num_pages;
      if (lane < C::BN / 16 && t < kv_end && (t | pmask) >= any_lo) {  // its page holds seen positions
        const int p = __ldg(row_table + (t >> a.log2p));
        if (static_cast<uint32_t>(p) < static_cast<uint32_t>(a.num_pages))
          id = p;
        else
          atomicOr(&g_prompt_status, RNB_STATUS_BAD_INDEX);
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
        const int box = is_k ? maps.k_box : maps.v_box;
        const int rows_u = is_k ? C::BN : C::VR, skip = is_k ? 0 : part * C::VR;
        const int nbox = rows_u / box;
        const int page = __shfl_sync(0xffffffffu, id, ((skip + lane * box) >> 4) & 31);
        if (lane < nbox) {
          const int t = blk * C::BN + skip + lane * box;
          const int nch = is_k ? C::KD / 64 : D / 64, ch0 = is_k ? part * (C::KD / 64) : 0;
          for (int c = 0; c < nch; ++c)
            tma_load_4d(dst + (c * rows_u + lane * box) * 128, is_k ? static_cast<const void*>(&maps.k) : &maps.v,
                        (ch0 + c) * 64, t & pmask, h, page, bar);
        }
        __syncwarp();
      }
    };
    if (nblk > 0) {
      load_tiles(&maps.q, &bars.q_full);
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
    const bool gates = a.gate && parts == 1;
    if (gates && alive && nblk > 0) alive = wait_on(&bars.q_done, 0);
    if (gates && alive) load_tiles(&maps.gate, &bars.g_full);
    // no copy may be in flight when the CTA ends
    if (nblk > 0) wait_on(&bars.q_full, 0);
    if (gates && alive) wait_on(&bars.g_full, 0);
    for (int v = max(u - C::NST, 0); v < u; ++v) wait_on(&bars.full[v % C::NST], (v / C::NST) & 1);
  } else if (warp == 1) {
    // ---- issuer
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    const uint32_t id_s = umma_idesc_f16(128, C::BN, kBf16);
    const uint32_t id_o = umma_idesc_f16(128, D, kBf16) | (1u << 16);  // B is MN-major
    const uint32_t rbase = smem_u32(ring);
    const uint64_t qdesc = umma_desc_sw128(smem_u32(smem));
    const uint32_t leader = elect_one();
    // ring units of block i: K0 K1 V0 K2 V1 ...
    auto unit_k = [&](int i) { return (i == 0 ? 0 : 2 * i - 1) * C::UPT; };
    auto unit_v = [&](int i) { return min(2 + 2 * i, 2 * nblk - 1) * C::UPT; };
    auto issue_s = [&](int k) {
      const int i = k / C::NQ, q = k % C::NQ;
      for (int part = 0; part < C::UPT && alive; ++part) {
        const int u = unit_k(i) + part, st = u % C::NST;
        alive = wait_on(&bars.full[st], (u / C::NST) & 1);
        if (!alive) return;
        tc_fence_after();
        const uint64_t qd = qdesc + ((q * (D / 64) + part * (C::KD / 64)) * (128 * 128 >> 4));
        const uint64_t kd = umma_desc_sw128(rbase + st * C::kUnit);
#pragma unroll
        for (int c = 0; c < C::KD / 64; ++c)
#pragma unroll
          for (int s = 0; s < 4; ++s)
            umma_ss(leader, tmem + (k % C::NS) * C::BN, qd + ((c * 128 * 128 + 32 * s) >> 4),
                    kd + ((c * C::BN * 128 + 32 * s) >> 4), id_s, part != 0 || (c | s) != 0);
        if (leader) {
          if (C::NQ == 1 || q == 1) umma_commit(smem_u32(&bars.empty[st]));
          if (part == C::UPT - 1) umma_commit(smem_u32(&bars.s_full[k % C::NS]));
        }
        __syncwarp();
      }
    };
    auto issue_o = [&](int k) {
      const int i = k / C::NQ, q = k % C::NQ;
      for (int part = 0; part < C::UPT && alive; ++part) {
        const int u = unit_v(i) + part, st = u % C::NST;
        alive = wait_on(&bars.full[st], (u / C::NST) & 1);
        if (!alive) return;
        const int t0 = (blk0 + i) * C::BN + part * C::VR;
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
        const uint64_t vd = umma_desc_mn(rbase + st * C::kUnit, C::VR * 128);
#pragma unroll
        for (int s = 0; s < C::VR / 16; ++s) {
          const int t = part * C::VR + s * 16;
          if (t % 64 == 0) {  // the first half's products run while the second half of P is computed
            alive = wait_on(&bars.p_full[k % C::NS][t / 64], (k / C::NS) & 1);
            if (!alive) return;
            tc_fence_after();
          }
          umma_ts(leader, tmem + C::kTmemO + q * D, tmem + (k % C::NS) * C::BN + t / 2, vd + (s * 16 * 128 >> 4), id_o,
                  i != 0 || t != 0);
        }
        if (leader) {
          if (C::NQ == 1 || q == 1) umma_commit(smem_u32(&bars.empty[st]));
          if (part == C::UPT - 1) umma_commit(smem_u32(i + 1 < nblk ? &bars.o_done[q] : &bars.o_last[q]));
        }
        __syncwarp();
      }
    };
    if (jobs > 0) {
      alive = wait_on(&bars.q_full, 0);
      tc_fence_after();
      for (int k = 0; k < min(C::NS, jobs) && alive; ++k) issue_s(k);
      for (int k = 0; k < jobs && alive; ++k) {
        issue_o(k);
        if (alive && k + C::NS < jobs) issue_s(k + C::NS);
        if (k + C::NS + 1 == jobs || (k == 0 && jobs <= C::NS)) {  // the last product with Q is issued
          if (leader) umma_commit(smem_u32(&bars.q_done));
          __syncwarp();
        }
      }
      // no product may be in flight when the tensor memory is given back
      if (leader) umma_commit(smem_u32(&bars.drained));
      __syncwarp();
      wait_on(&bars.drained, 0);
    }
  } else if (warp >= 4) {
    // ---- softmax: a thread is a row of tile wg
    const int wg = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;  // row tile and row in it
    const int wt0 = tok0 + wg * tt, wt_end = min(wt0 + tt, rows);  // its tokens (none: wt0 >= rows)
    const int tok = wt0 + r / a.group, head = h * a.group + r % a.group;
    const bool in = r < tt * a.group && tok < rows;
    const int pos = p0 + min(tok, tok_end - 1);
    const int see_lo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_o = tmem + C::kTmemO + wg * D + lane_base;
    // positions that all rows of this warpgroup's tile see
    const int wg_first = p0 + min(wt0, tok_end - 1);
    const int all_lo = a.window > 0 ? p0 + min(wt0 + tt, tok_end) - a.window : INT_MIN;
    // the first lanes watch the page ids of the next block's subtiles of 16 positions
    auto page_at = [&](int i) {
      const int t = (blk0 + i) * C::BN + 16 * lane;
      return lane < C::BN / 16 && t < kv_end ? __ldg(row_table + (t >> a.log2p)) : 0;
    };
    int page = nblk > 0 ? page_at(0) : 0;
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < nblk && alive; ++i) {
      const uint32_t bad =
          __ballot_sync(0xffffffffu, static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.num_pages));
      if (i + 1 < nblk) page = page_at(i + 1);
      const int k = C::NQ * i + wg, slot = k % C::NS;
      const uint32_t t_s = tmem + slot * C::BN + lane_base;
      alive = wait_on(&bars.s_full[slot], (k / C::NS) & 1);
      if (!alive) break;
      tc_fence_after();
      constexpr int NC = C::BN / 32;
      uint32_t v[NC][32];
#pragma unroll
      for (int c = 0; c < NC; ++c) tmem_ld32(t_s + 32 * c, v[c]);
      tmem_wait_ld();
      const int t0 = (blk0 + i) * C::BN;
      if (__builtin_expect(bad || t0 + C::BN - 1 > wg_first || t0 < all_lo, 0)) {
        const int hi = pos - t0, lo = see_lo - t0;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * c + e > hi) v[c][e] = __float_as_uint(-INFINITY);
        if (bad || t0 < all_lo) {
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * c + e < lo || (bad >> (2 * c + (e >> 4)) & 1)) v[c][e] = __float_as_uint(-INFINITY);
        }
      }
      float mc[NC][2];
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          mc[c][y] = __uint_as_float(v[c][16 * y]);
#pragma unroll
          for (int e = 1; e < 15; e += 2)
            mc[c][y] = max3(mc[c][y], __uint_as_float(v[c][16 * y + e]), __uint_as_float(v[c][16 * y + e + 1]));
          mc[c][y] = fmaxf(mc[c][y], __uint_as_float(v[c][16 * y + 15]));
        }
      float mx = fmaxf(mc[0][0], mc[0][1]);
#pragma unroll
      for (int c = 1; c < NC; ++c) mx = max3(mx, mc[c][0], mc[c][1]);
      mx *= a.scale_log2;
      if (__any_sync(0xffffffffu, in && mx > m + 8.f)) {  // (what rows out of use hold must not matter)
        const float to = fmaxf(m, mx);
        const float f = ex2(m - (to == -INFINITY ? 0.f : to));
        m = to;
        l *= f;
        if (i > 0) {
          // the product before this one has to be in O (with two slots a tile the one
          // before that is, since S of this block was issued behind it; with one
          // slot S was issued behind this very product)
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
      const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), use2 = make_float2(-use, -use);
      float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 x =
              fma2(make_float2(__uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1])), scale2, use2);
          const float2 y = make_float2(ex2(x.x), ex2(x.y));
          if (e & 1)
            sum1 = add2(sum1, y);
          else
            sum0 = add2(sum0, y);
          p[e] = Pair<T>::pack(y.x, y.y);
        }
        tmem_st16(t_s + 16 * c, p);
        if (c & 1) {  // a half of P
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.p_full[slot][c >> 1]);
        }
      }
      l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
    }
    // ---- O / l
    // (o_done would not do: with two slots a tile the last two products may both be
    // under way, and a parity only tells neighbouring phases apart)
    if (alive && nblk > 0) alive = wait_on(&bars.o_last[wg], 0);
    tc_fence_after();
    if (parts > 1) {
      // this part's row of O, m and l for the join
      const int64_t row = (static_cast<int64_t>(blockIdx.x) * C::NQ + wg) * 128 + r;
      float* po = reinterpret_cast<float*>(a.ws + a.o_off) + row * D;
      if (in && alive) {
        float* ml = reinterpret_cast<float*>(a.ws + a.ml_off) + 2 * row;
        ml[0] = m, ml[1] = l;
      }
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(t_o + 32 * c, o);
        tmem_wait_ld();
        if (in && alive) {
#pragma unroll
          for (int x = 0; x < 8; ++x)
            *reinterpret_cast<uint4*>(po + 32 * c + 4 * x) = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
        }
      }
    }
    const bool whole = alive && parts == 1;
    if (a.gate && whole) alive = wait_on(&bars.g_full, 0);
    if (whole && alive) {
      // in place of Q, or of the gates that have come there
      char* base = smem + wg * (D / 64) * kCol;
      const float inv = l > 0.f ? 1.0f / l : 0.f;
      if (a.lse && in)
        a.lse[static_cast<int64_t>(q0 + tok) * a.Hq + head] = l > 0.f ? 0.6931471805599453f * (m + log2f(l)) : -INFINITY;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0;
        if (nblk > 0) {
          tmem_ld32(t_o + 32 * c, o);
          tmem_wait_ld();
        }
        char* at = base + (c >> 1) * kCol;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint4* piece = reinterpret_cast<uint4*>(at + sw128_offset(r, (c & 1) * 32 + 8 * x));
          uint32_t w[4];
          uint4 gw = make_uint4(0, 0, 0, 0);
          if (a.gate) gw = *piece;
          const uint32_t gu[4] = {gw.x, gw.y, gw.z, gw.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float y0 = __uint_as_float(o[8 * x + 2 * e]) * inv, y1 = __uint_as_float(o[8 * x + 2 * e + 1]) * inv;
            if (a.gate) {
              const float2 gf = Pair<T>::unpack(gu[e]);
              y0 = __fdividef(y0, 1.f + __expf(-gf.x)), y1 = __fdividef(y1, 1.f + __expf(-gf.y));
            }
            w[e] = Pair<T>::pack(y0, y1);
          }
          *piece = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      fence_proxy_async_smem();
    }
    // the warpgroup's four warps, those that gave up among them
    if (all_of_128(1 + wg, whole && alive)) {
      const char* base = smem + wg * (D / 64) * kCol;
      if (wt0 + tt <= rows) {
        if (r == 0) {
          for (int c = 0; c < D / 64; ++c)
            tma_store_3d(&maps.out, smem_u32(base + c * kCol), 64 * c, h * a.group, q0 + wt0);
          bulk_commit_and_wait_read();
        }
      } else {
        // the request's last tile: only its own rows
        const int n = max(wt_end - wt0, 0) * a.group;
        for (int x = r; x < n * (D / 8); x += 128) {
          const int rr = x / (D / 8), e = (x - rr * (D / 8)) * 8, i = rr / a.group;
          *reinterpret_cast<uint4*>(static_cast<T*>(a.out) +
                                    (static_cast<int64_t>(q0 + wt0 + i) * a.Hq + h * a.group + rr - i * a.group) * D + e) =
              *reinterpret_cast<const uint4*>(base + (e >> 6) * kCol + sw128_offset(rr, e & 63));
        }
      }
    }
  }
  if (!alive && lane == 0) {
    atomicExch(&g_gave_up, a.call);
    atomicOr(&g_prompt_status, RNB_STATUS_TIMEOUT);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

// Block (i, y): rows [16 y, 16 y + 16) of split tile i.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_attn_join_tiles(const AttnArgs a, int tokens) {
  after_previous();
  using C = Cfg<D>;
  constexpr int kCols = D / 4, kRowsIt = 256 / kCols;
  const SplitTile* split = reinterpret_cast<const SplitTile*>(a.ws);
  const SplitTile tile = split[blockIdx.x];
  if (tile.parts < 2) return;
  const int col = threadIdx.x % kCols;
  for (int x = threadIdx.x / kCols; x < 16; x += kRowsIt) {
    const int rr = blockIdx.y * 16 + x, q = rr / 128, r = rr - 128 * q;
    const int tok = tile.tok0 + q * tokens + r / a.group, head = tile.h * a.group + r % a.group;
    if (r >= tokens * a.group || tok >= tile.rows) continue;
    const uint2 gw = a.gate ? __ldg(reinterpret_cast<const uint2*>(attn_gate<T>(a, tile.q0 + tok, head) + 4 * col))
                            : make_uint2(0, 0);
    const float* ml = reinterpret_cast<const float*>(a.ws + a.ml_off);
    const float* po = reinterpret_cast<const float*>(a.ws + a.o_off);
    auto row_of = [&](int p) {
      return (static_cast<int64_t>(p * tile.n + static_cast<int>(blockIdx.x)) * C::NQ + q) * 128 + r;
    };
    float mx = -INFINITY;
    for (int p = 0; p < tile.parts; ++p) mx = fmaxf(mx, ml[2 * row_of(p)]);
    const float use = mx == -INFINITY ? 0.f : mx;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll 4
    for (int p = 0; p < tile.parts; ++p) {
      const int64_t row = row_of(p);
      const float f = ex2(ml[2 * row] - use);
      const float4 v = *reinterpret_cast<const float4*>(po + row * D + 4 * col);
      acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y);
      acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
      l = fmaf(ml[2 * row + 1], f, l);
    }
    attn_write_row<T, D>(a, tile.q0 + tok, head, 4 * col, acc, mx, l, gw);
  }
}

template <int D>
int64_t tiles_at_most(const AttnArgs& a) {
  const int64_t per = static_cast<int64_t>(128 / a.group) * Cfg<D>::NQ;  // tokens a CTA
  return (a.T + per - 1) / per + (a.B < a.T ? a.B : a.T);
}

template <typename T, int D>
int launch_prompt(const AttnArgs& a, const PromptMaps& maps, cudaStream_t st) {
  using C = Cfg<D>;
  const cudaError_t e = cudaFuncSetAttribute(k_attn_prompt<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return fail(RNB_ERR_CUDA, std::string("rnb_paged_attention: ") + cudaGetErrorString(e));
  // as many tiles as there can be: CTAs without one end at once
  const int64_t ctas = tiles_at_most<D>(a) * a.Hkv;
  if (ctas > INT32_MAX) return fail(RNB_ERR_INVALID, "rnb_paged_attention: too many rows");
  const unsigned grid = static_cast<unsigned>(a.split ? a.split : ctas);
  const int rc = launch("rnb_paged_attention", k_attn_prompt<T, D>, grid, C::kThreads, C::kSmem, st, a, maps);
  if (rc || !a.split) return rc;
  return launch("rnb_paged_attention join", k_attn_join_tiles<T, D>, dim3(static_cast<unsigned>(ctas), C::NQ * 128 / 16),
                256, 0, st, a, maps.tokens);
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

// [T][n_q_heads][D] in boxes of (tokens, the group's heads, 64 elements)
bool encode_rows(CUtensorMap* m, const AttnArgs& a, const void* base, int D, int64_t ts, int64_t hs, int tokens) {
  const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a.Hq), static_cast<uint64_t>(a.T)};
  const uint64_t str[2] = {a.Hq > 1 ? 2u * static_cast<uint64_t>(hs) : 2u * D,
                           a.T > 1 ? 2u * static_cast<uint64_t>(ts) : 2u * D * a.Hq};
  const uint32_t box[3] = {64, static_cast<uint32_t>(a.group), static_cast<uint32_t>(tokens)};
  return encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, base, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

cudaError_t prompt_status_word(uint32_t** p) { return status_word(g_prompt_status, p); }
cudaError_t prompt_gave_up_word(uint32_t** p) { return status_word(g_gave_up, p); }

bool prepare_prompt(const AttnArgs& a, const rnb_kv_cache* c, PromptMaps* p) {
  if (a.group > 128) return false;
  const int D = c->head_dim, P = c->page_size;
  p->tokens = 128 / a.group;
  const int bn = D == 256 ? Cfg<256>::BN : Cfg<128>::BN;
  p->k_box = P < bn ? P : bn;
  const int vr = D == 256 ? Cfg<256>::VR : Cfg<128>::VR;
  p->v_box = P < vr ? P : vr;

  return encode_cache(&p->k, c, c->k, c->k_page_stride, c->k_head_stride, p->k_box) &&
         encode_cache(&p->v, c, c->v, c->v_page_stride, c->v_head_stride, p->v_box) &&
         encode_rows(&p->q, a, a.q, D, a.q_ts, a.q_hs, p->tokens) &&
         encode_rows(&p->out, a, a.out, D, static_cast<int64_t>(a.Hq) * D, D, p->tokens) &&
         (!a.gate || encode_rows(&p->gate, a, a.gate, D, a.g_ts, a.g_hs, p->tokens));
}

// CTAs of a call whose tiles are split (0: not split), and its workspace: where
// the tiles that there can be do not fill the SMs, and are long enough.
int plan_split(AttnArgs* a, int D, int sms, size_t* bytes) {
  a->split = 0;
  *bytes = 0;
  if (a->group > 128 || a->max_kv < 4 * Cfg<128>::BN) return 0;
  const int64_t tiles = D == 256 ? tiles_at_most<256>(*a) : D == 128 ? tiles_at_most<128>(*a) : tiles_at_most<64>(*a);
  if (tiles * a->Hkv > sms) return 0;
  const size_t rows = static_cast<size_t>(sms) * (D == 256 ? 1 : 2) * 128;
  a->split = sms;
  a->ml_off = (sizeof(SplitTile) * sms + 255) & ~size_t(255);
  a->o_off = a->ml_off + 2 * sizeof(float) * rows;
  *bytes = a->o_off + sizeof(float) * rows * D;
  return a->split;
}

int run_prompt(const AttnArgs& args, const rnb_kv_cache* c, const PromptMaps& p, cudaStream_t st) {
  static std::atomic<uint32_t> calls{0};
  AttnArgs a = args;
  do a.call = ++calls;
  while (a.call == 0);
  const int D = c->head_dim;
  if (c->dtype == RNB_DTYPE_BF16) {
    if (D == 64) return launch_prompt<__nv_bfloat16, 64>(a, p, st);
    if (D == 128) return launch_prompt<__nv_bfloat16, 128>(a, p, st);
    return launch_prompt<__nv_bfloat16, 256>(a, p, st);
  }
  if (D == 64) return launch_prompt<__half, 64>(a, p, st);
  if (D == 128) return launch_prompt<__half, 128>(a, p, st);
  return launch_prompt<__half, 256>(a, p, st);
}

}  // namespace rnb
