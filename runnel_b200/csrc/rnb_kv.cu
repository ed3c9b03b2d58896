// rnb_kv.cu -- pages, slots and positions of a serving step, from the
// requests' lengths, on the device (rnb_kv_plan, rnb_kv_release).
//
// With P rows a page, request b holds ceil(ctx/P) pages and needs
// need_b = ceil((ctx + new)/P) - ceil(ctx/P) more.  Exclusive sums over the
// requests of new_b (token rows) and need_b (pages off the free list's end)
// place everything:
//   table[b][held_b + j] = free[count - 1 - (base_b + j)]
//   slot(t) = page(pos) * P + pos % P,  pos = ctx_b + t - cu_b
// Bytes: 8 a request in, 8 out, 8 a token row, 8 a new page; the largest step
// here (2048 requests, 64 Ki rows) moves 0.5 MB, under 0.1 us of HBM time, so
// the launch and one trip of dependent loads bound it.  Hence one launch and
// no grid-wide exchange: every CTA computes both sums over all requests by
// itself (shared memory, 8 bytes a request) and looks at all ids that the step
// takes, so that all agree on whether the plan is void, then takes its share of
// the token rows and of the new pages and finds each one's request by binary
// search.  A row in a new page takes the id from the free list, not from the table
// entry that another CTA may be writing.
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>
#include <string>

#include "rnb_kv.cuh"

namespace rnb {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanMaxB = 16384;

__device__ uint32_t g_kv_status;

// The words are shared by all streams of the device, and a kernel may set a bit
// at any time: each is exchanged for zero, so that every bit is either in this
// read or in the next.
__device__ uint32_t g_status_taken;

struct StatusWords {
  uint32_t* word[4];
  uint32_t* gave_up;
};

__global__ void k_take_status(const StatusWords s) {
  uint32_t bits = 0;
  for (uint32_t* w : s.word) bits |= atomicExch(w, 0u);
  if (bits & RNB_STATUS_TIMEOUT) atomicExch(s.gave_up, 0u);  // (a captured call may run again)
  g_status_taken = bits;
}

// Exclusive sums, in place, over n values of two shared arrays (values >= 0,
// sums saturating at 2^31 - 1); totals in tot[0..1].  Every thread of the
// block calls it.
__device__ void block_sums(int32_t* a, int32_t* b, int n, int64_t (*wsum)[2], int64_t* tot) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = ((n + kPlanThreads - 1) / kPlanThreads) | 1;  // odd: no bank conflicts between the threads' parts
  const int lo = min(tid * per, n), hi = min(lo + per, n);
  int64_t sa = 0, sb = 0;
  for (int i = lo; i < hi; ++i) {
    sa += a[i];
    sb += b[i];
  }
  int64_t ia = sa, ib = sb;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t ua = __shfl_up_sync(0xffffffffu, ia, o), ub = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) {
      ia += ua;
      ib += ub;
    }
  }
  if (lane == 31) {
    wsum[warp][0] = ia;
    wsum[warp][1] = ib;
  }
  __syncthreads();
  int64_t ba = ia - sa, bb = ib - sb;
  for (int w = 0; w < warp; ++w) {
    ba += wsum[w][0];
    bb += wsum[w][1];
  }
  if (tid == kPlanThreads - 1) {
    tot[0] = ba + sa;
    tot[1] = bb + sb;
  }
  const int64_t top = INT32_MAX;
  for (int i = lo; i < hi; ++i) {
    const int32_t va = a[i], vb = b[i];
    a[i] = static_cast<int32_t>(ba < top ? ba : top);
    b[i] = static_cast<int32_t>(bb < top ? bb : top);
    ba += va;
    bb += vb;
  }
  __syncthreads();
}

// The last i in [0, n) with start[i] <= v (start[0] == 0, v >= 0, ascending):
// of requests with equal starts the last, which is the one that is not empty.
__device__ __forceinline__ int find_request(const int32_t* start, int n, int32_t v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= v)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

struct PlanArgs {
  int B, W, log2p, num_pages, max_tokens, free_capacity;
  int32_t* table;
  const int32_t *ctx, *fresh, *free_pages, *free_count;
  int32_t *seq, *cu, *pos, *slots, *free_out;
};

__global__ void __launch_bounds__(kPlanThreads) k_kv_plan(const PlanArgs a) {
  after_previous();
  extern __shared__ int32_t sh[];
  int32_t* cu = sh;           // [B] first token row of each request
  int32_t* base = sh + a.B;   // [B] first new page of each request
  __shared__ int64_t wsum[kPlanThreads / 32][2], tot[2];
  const int tid = threadIdx.x;
  const int P = 1 << a.log2p;
  const int fc = *a.free_count;
  // the ids that most steps take at most: under way before the sums (2048 requests
  // with 3869 new pages 7.7 -> 6.1 us)
  constexpr int kAhead = 16;
  const int32_t* next_free = a.free_pages + fc - 1;
  uint32_t ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int n = tid + i * kPlanThreads;
    ahead[i] = n < fc && fc <= a.free_capacity ? next_free[-n] : 0;
  }
  int bad = 0;
  for (int b = tid; b < a.B; b += kPlanThreads) {
    const int64_t c = a.ctx[b], n = a.fresh[b];
    const int64_t held = (c + P - 1) >> a.log2p, all = (c + n + P - 1) >> a.log2p;
    const bool wrong = c < 0 || n < 0 || c + n > INT32_MAX || all > a.W;
    bad |= wrong;
    cu[b] = wrong ? 0 : static_cast<int32_t>(n);
    base[b] = wrong ? 0 : static_cast<int32_t>(all - held);
  }
  bad = __syncthreads_or(bad);
  block_sums(cu, base, a.B, wsum, tot);
  bool ok = !bad && tot[0] <= a.max_tokens && fc >= 0 && fc <= a.free_capacity && tot[1] <= fc;
  // a taken id that is no page would lose its rows while the lengths go on
  uint32_t top = 0;
  if (ok) {
    const int need = static_cast<int>(tot[1]);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (tid + i * kPlanThreads < need) top = max(top, ahead[i]);
#pragma unroll 4
    for (uint32_t n = tid + kAhead * kPlanThreads; n < static_cast<uint32_t>(need); n += kPlanThreads)
      top = max(top, static_cast<uint32_t>(next_free[-static_cast<int64_t>(n)]));
  }
  const bool strange = __syncthreads_or(top >= static_cast<uint32_t>(a.num_pages));
  ok = ok && !strange;
  const int tokens = ok ? static_cast<int>(tot[0]) : 0, pages = ok ? static_cast<int>(tot[1]) : 0;

  // (unsigned: a step past the last of almost 2^31 rows or pages stays a number)
  const uint32_t stride = gridDim.x * kPlanThreads, at = blockIdx.x * kPlanThreads + tid;
  if (at == 0) {
    a.cu[a.B] = tokens;
    *a.free_out = fc - pages;
    if (!ok) atomicOr(&g_kv_status, RNB_STATUS_NO_PAGES | (strange ? RNB_STATUS_BAD_INDEX : 0));
  }
  for (uint32_t b = at; b < static_cast<uint32_t>(a.B); b += stride) {
    a.cu[b] = ok ? cu[b] : 0;
    a.seq[b] = a.ctx[b] + (ok ? a.fresh[b] : 0);
  }
  for (uint32_t i = at; i < static_cast<uint32_t>(pages); i += stride) {
    const int n = static_cast<int>(i), b = find_request(base, a.B, n);
    const int held = static_cast<int>((static_cast<int64_t>(a.ctx[b]) + P - 1) >> a.log2p);
    a.table[static_cast<int64_t>(b) * a.W + held + (n - base[b])] = a.free_pages[fc - 1 - n];
  }
  for (uint32_t i = at; i < static_cast<uint32_t>(a.max_tokens); i += stride) {
    const int t = static_cast<int>(i);
    int pos = 0, slot = -1;
    if (t < tokens) {
      const int b = find_request(cu, a.B, t);
      const int c = a.ctx[b], held = static_cast<int>((static_cast<int64_t>(c) + P - 1) >> a.log2p);
      pos = c + (t - cu[b]);
      const int j = pos >> a.log2p;
      const int page = j < held ? a.table[static_cast<int64_t>(b) * a.W + j] : a.free_pages[fc - 1 - (base[b] + j - held)];
      if (page >= 0 && page < a.num_pages)
        slot = (page << a.log2p) + (pos & (P - 1));
      else
        atomicOr(&g_kv_status, RNB_STATUS_BAD_INDEX);
    }
    a.pos[t] = pos;
    a.slots[t] = slot;
  }
}

struct ReleaseArgs {
  int B, W, log2p, num_pages, free_capacity;
  const int32_t *table, *lens, *finished;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t *lens_out, *free_out;
};

// One CTA (requests finish one at a time): the table entries of all finished
// requests as one flat range, each found by binary search, 256 at a time; those
// that are pages close up in order (a ballot a warp, the warps' counts summed).
__global__ void __launch_bounds__(kPlanThreads) k_kv_release(const ReleaseArgs a) {
  after_previous();
  extern __shared__ int32_t sh[];
  int32_t* base = sh;        // [B]
  int32_t* none = sh + a.B;  // [B] the second of block_sums' arrays
  __shared__ int64_t wsum[kPlanThreads / 32][2], tot[2];
  __shared__ int in_warp[2][kPlanThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int P = 1 << a.log2p;
  __shared__ int count;  // (one read: barriers below hang on it)
  if (tid == 0) count = *a.free_count;
  int bad = 0;
  for (int b = tid; b < a.B; b += kPlanThreads) {
    int32_t pages = 0;
    if (a.finished[b]) {
      const int64_t n = a.lens[b], held = (n + P - 1) >> a.log2p;
      const bool wrong = n < 0 || held > a.W;
      bad |= wrong;
      pages = wrong ? 0 : static_cast<int32_t>(held);
    }
    base[b] = pages;
    none[b] = 0;
  }
  bad = __syncthreads_or(bad);
  const int fc = count;
  block_sums(base, none, a.B, wsum, tot);
  bool ok = !bad && fc >= 0 && fc <= a.free_capacity && tot[0] < INT32_MAX;
  const int held = ok ? static_cast<int>(tot[0]) : 0;
  auto entry = [&](int n) {
    const int b = find_request(base, a.B, n);
    return a.table[static_cast<int64_t>(b) * a.W + (n - base[b])];
  };
  // entry n's place among the pages of its 256, and how many those are
  int round = 0;
  auto place = [&](bool page, int* all) {
    const uint32_t mask = __ballot_sync(0xffffffffu, page);
    int* n_in = in_warp[round++ & 1];  // (two in turns: one barrier a round)
    if (lane == 0) n_in[warp] = __popc(mask);
    __syncthreads();
    int at = __popc(mask & ((1u << lane) - 1));
    *all = 0;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      at += w < warp ? n_in[w] : 0;
      *all += n_in[w];
    }
    return at;
  };
  bool strange = false;
  int pages = 0;
  // entries that are no pages need no room: where not all entries fit, the pages are counted first
  for (int pass = held <= a.free_capacity - fc ? 1 : 0; pass < 2 && ok; ++pass) {
    pages = 0;
    for (uint32_t n0 = 0; n0 < static_cast<uint32_t>(held); n0 += kPlanThreads) {
      const uint32_t n = n0 + tid;
      const int id = n < static_cast<uint32_t>(held) ? entry(static_cast<int>(n)) : -1;
      const bool page = id >= 0 && id < a.num_pages;
      strange = strange || id >= a.num_pages;
      int all;
      const int at = place(page, &all);
      if (page && pass == 1) a.free_pages[fc + pages + at] = id;
      pages += all;
    }
    ok = pages <= a.free_capacity - fc;
  }
  if (!ok) pages = 0;
  for (int b = tid; b < a.B; b += kPlanThreads) a.lens_out[b] = ok && a.finished[b] ? 0 : a.lens[b];
  if (strange) atomicOr(&g_kv_status, RNB_STATUS_BAD_INDEX);
  if (tid == 0) {
    *a.free_out = fc + pages;
    if (!ok) atomicOr(&g_kv_status, RNB_STATUS_NO_PAGES);
  }
}

int check_plan(int B, int W, int page_size, const char* fn) {
  const std::string f = std::string(fn) + ": ";
  if (B < 0 || B > kPlanMaxB) return fail(RNB_ERR_INVALID, f + "B must be in [0, 16384]");
  if (W <= 0) return fail(RNB_ERR_INVALID, f + "table_cols must be positive");
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
    return fail(RNB_ERR_INVALID, f + "page_size must be 16, 32, 64, 128 or 256");
  return RNB_OK;
}

// Shared memory beyond 48 KB has to be asked for; the kernels' static arrays count
// too (under 1 KB: 6127 to 6144 requests were refused with the border at 48).
template <typename K>
int allow_smem(K kernel, size_t bytes) {
  if (bytes <= 47 * 1024) return RNB_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) return fail(RNB_ERR_CUDA, std::string("shared memory: ") + cudaGetErrorString(e));
  return RNB_OK;
}

int log2_of(int p) {
  int l = 0;
  while ((1 << l) < p) ++l;
  return l;
}

}  // namespace
}  // namespace rnb

extern "C" {

int rnb_kv_plan(int B, int table_cols, int page_size, int num_pages, int max_tokens, int32_t* table,
                const int32_t* ctx_lens, const int32_t* new_lens, const int32_t* free_pages, int free_capacity,
                const int32_t* free_count, int32_t* seq_lens, int32_t* cu_q, int32_t* positions, int32_t* slots,
                int32_t* free_count_out, void* stream) {
  using namespace rnb;
  int rc = check_plan(B, table_cols, page_size, "rnb_kv_plan");
  if (rc) return rc;
  if (max_tokens < 0 || free_capacity < 0)
    return fail(RNB_ERR_INVALID, "rnb_kv_plan: max_tokens and free_capacity must be >= 0");
  if (num_pages <= 0 || static_cast<int64_t>(num_pages) * page_size > INT32_MAX)
    return fail(RNB_ERR_INVALID, "rnb_kv_plan: num_pages must be positive and num_pages * page_size below 2^31");
  if ((B && (!table || !ctx_lens || !new_lens || !seq_lens)) || !free_count || !cu_q || !free_count_out ||
      (free_capacity && !free_pages) || (max_tokens && (!positions || !slots)))
    return fail(RNB_ERR_INVALID, "rnb_kv_plan: tensors must be non-NULL");
  if (free_count_out == free_count)
    return fail(RNB_ERR_INVALID, "rnb_kv_plan: free_count_out must not be free_count");
  if (B && (seq_lens == ctx_lens || seq_lens == new_lens))
    return fail(RNB_ERR_INVALID, "rnb_kv_plan: seq_lens must not be ctx_lens or new_lens");
  if ((rc = check_device())) return rc;
  const size_t smem = 8u * static_cast<size_t>(B);
  if ((rc = allow_smem(k_kv_plan, smem))) return rc;
  // one row or request a thread, at most one CTA per SM: every CTA repeats the
  // sums over the requests, so more CTAs would only repeat them again
  const int work = max_tokens > B ? max_tokens : B;
  const int sms = dev_info().sms;
  int grid = work / kPlanThreads + (work % kPlanThreads ? 1 : 0);
  grid = grid < 1 ? 1 : grid > sms ? sms : grid;
  const PlanArgs a{B, table_cols, log2_of(page_size), num_pages, max_tokens, free_capacity, table, ctx_lens, new_lens,
                   free_pages, free_count, seq_lens, cu_q, positions, slots, free_count_out};
  return launch("rnb_kv_plan", k_kv_plan, grid, kPlanThreads, smem, static_cast<cudaStream_t>(stream), a);
}

int rnb_kv_release_bounded(int B, int table_cols, int page_size, int num_pages, const int32_t* table,
                           const int32_t* lens, const int32_t* finished, int32_t* free_pages, int free_capacity,
                           const int32_t* free_count, int32_t* lens_out, int32_t* free_count_out, void* stream) {
  using namespace rnb;
  int rc = check_plan(B, table_cols, page_size, "rnb_kv_release");
  if (rc) return rc;
  if (num_pages <= 0) return fail(RNB_ERR_INVALID, "rnb_kv_release: num_pages must be positive");
  if (free_capacity < 0) return fail(RNB_ERR_INVALID, "rnb_kv_release: free_capacity must be >= 0");
  if ((B && (!table || !lens || !finished || !lens_out)) || !free_count || !free_count_out ||
      (free_capacity && !free_pages))
    return fail(RNB_ERR_INVALID, "rnb_kv_release: tensors must be non-NULL");
  if (free_count_out == free_count)
    return fail(RNB_ERR_INVALID, "rnb_kv_release: free_count_out must not be free_count");
  if ((rc = check_device())) return rc;
  const size_t smem = 8u * static_cast<size_t>(B);
  if ((rc = allow_smem(k_kv_release, smem))) return rc;
  const ReleaseArgs a{B, table_cols, log2_of(page_size), num_pages, free_capacity, table, lens, finished, free_pages,
                      free_count, lens_out, free_count_out};
  return launch("rnb_kv_release", k_kv_release, 1, kPlanThreads, smem, static_cast<cudaStream_t>(stream), a);
}

int rnb_kv_release(int B, int table_cols, int page_size, const int32_t* table, const int32_t* lens,
                   const int32_t* finished, int32_t* free_pages, int free_capacity, const int32_t* free_count,
                   int32_t* lens_out, int32_t* free_count_out, void* stream) {
  return rnb_kv_release_bounded(B, table_cols, page_size, INT32_MAX, table, lens, finished, free_pages, free_capacity,
                                free_count, lens_out, free_count_out, stream);
}

int rnb_kv_status(uint32_t* status, void* stream) {
  using namespace rnb;
  if (!status) return fail(RNB_ERR_INVALID, "status must be non-NULL");
  int rc = check_device();
  if (rc) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  static std::mutex one_reader;  // g_status_taken is one word
  const std::lock_guard<std::mutex> lock(one_reader);
  StatusWords words{};
  cudaError_t e = status_word(g_kv_status, &words.word[0]);
  if (e == cudaSuccess) e = rope_status_word(&words.word[1]);
  if (e == cudaSuccess) e = attn_status_word(&words.word[2]);
  if (e == cudaSuccess) e = prompt_status_word(&words.word[3]);
  if (e == cudaSuccess) e = prompt_gave_up_word(&words.gave_up);
  if (e == cudaSuccess) {
    k_take_status<<<1, 1, 0, st>>>(words);
    e = cudaGetLastError();
  }
  uint32_t bits = 0;
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(&bits, g_status_taken, sizeof bits, 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return fail(RNB_ERR_CUDA, std::string("rnb_kv_status: ") + cudaGetErrorString(e));
  *status = bits;
  return RNB_OK;
}

}  // extern "C"
