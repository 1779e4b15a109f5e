// One step of serving over a paged K/V cache, apart from its attention: the step's
// block tables, slot map and positions built on the GPU from the requests' lengths, and
// the new K/V rows written into their slots.
//
// Tables.  With c_b tokens in the cache and n_b new ones, request b holds
// have_b = ceil(c_b / P) pages and needs ceil((c_b + n_b) / P); two prefix sums over the
// requests (new tokens, new pages) say where its tokens start and which entries of the
// free list are its.  A few thousand lengths and some ten thousand tokens are far too
// few bytes to bound anything: the launch and the scans' latency do.  So one launch,
// and every CTA scans all the lengths itself (two 4-byte loads per request, from L2) instead of
// waiting for another one's sums; then each new token and each new page finds its
// request by bisection in shared memory, and computes its own page from the free list
// rather than read a table entry that another CTA writes.  3.6 us on the GPU for 8 requests
// of one token, launch included, in a captured graph; 1000 requests with 65313 tokens take
// 13.5 us a call, which is the host's side of it.
#include "paged.cuh"

namespace pa {
namespace {

constexpr int kStepThreads = 512;
constexpr int kMaxRequests = 16384;

// Inclusive scan of (a, b) over the CTA; sums of the whole CTA in (ta, tb).
__device__ __forceinline__ void block_scan2(int& a, int& b, int& ta, int& tb, int2* warp_sum) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
  __syncthreads();   // the previous round's readers are done with warp_sum
  if (lane == 31) warp_sum[w] = make_int2(a, b);
  __syncthreads();
  // every thread adds up the warps itself: 16 broadcast reads
  int pa_ = 0, pb = 0;
  ta = tb = 0;
#pragma unroll
  for (int i = 0; i < kStepThreads / 32; ++i) {
    const int2 s = warp_sum[i];
    if (i < w) {
      pa_ += s.x;
      pb += s.y;
    }
    ta += s.x;
    tb += s.y;
  }
  a += pa_;
  b += pb;
}

// Largest i in [0, n) with pre[i] <= x (pre ascending, pre[0] = 0).
__device__ __forceinline__ int find_request(const int2* pre, int n, int x, bool pages) {
  int lo = 0, hi = n;   // pre[lo] <= x < pre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    const int v = pages ? pre[mid].y : pre[mid].x;
    if (v <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kStepThreads) paged_step_kernel(pa_paged_step_args a) {
  extern __shared__ int2 pre[];          // [requests + 1]: (tokens, pages) before request b
  __shared__ int2 warp_sum[kStepThreads / 32];
  pdl_wait();
  pdl_begin_next();
  const int B = a.requests, P = a.page_size;
  const long long W = a.table_width;
  auto div_up = [P](long long x) { return (x + P - 1) / P; };
  int base_t = 0, base_p = 0;
  int over = 0;                          // pages that the table's width leaves out
  for (int b0 = 0; b0 < B; b0 += kStepThreads) {
    const int b = b0 + threadIdx.x;
    int n = 0, np = 0;
    if (b < B) {
      const int c = max(__ldg(a.old_lens + b), 0);
      n = max(__ldg(a.new_lens + b), 0);
      const long long have = div_up(c), need = div_up((long long)c + n);
      np = (int)(max(min(need, W), min(have, W)) - min(have, W));
      over += (int)(need - have) - np;
      if (blockIdx.x == 0) a.seq_lens[b] = (int)min((long long)c + n, 0x7fffffffll);
    }
    int st = n, sp = np, tt, tp;
    block_scan2(st, sp, tt, tp, warp_sum);
    if (b < B) {
      pre[b] = make_int2(base_t + st - n, base_p + sp - np);
      if (blockIdx.x == 0) a.q_start[b] = base_t + st - n;
    }
    base_t += tt;
    base_p += tp;
  }
  if (threadIdx.x == 0) pre[B] = make_int2(base_t, base_p);
  const int head = min(max(__ldg(a.free_head), 0), a.free_count);
  const int got = max(min(base_p, a.free_count - head), 0);
  if (blockIdx.x == 0) {
    const int left_out = __syncthreads_or(over != 0);
    __shared__ int sum_over;
    if (threadIdx.x == 0) {
      sum_over = 0;
      a.q_start[B] = base_t;
      *a.free_head_out = head + got;
    }
    __syncthreads();
    if (left_out && over) atomicAdd(&sum_over, over);
    __syncthreads();
    if (threadIdx.x == 0) *a.missing = base_p - got + sum_over;
  }
  __syncthreads();

  const int tid = blockIdx.x * kStepThreads + threadIdx.x;
  const int step = gridDim.x * kStepThreads;   // steps in 64 bits: the last one may pass 2^31
  // Columns are compared with the table's width, and entries of the free list with those to
  // be had, also where sums of absurd lengths have overflowed: nothing outside is touched.
  // page id for a slot, or -1 when the slot would not fit in 32 bits (no such page)
  auto page_ok = [P](int page) { return page >= 0 && (long long)(page + 1ll) * P <= 0x7fffffffll; };
  for (long long i = tid; i < a.tokens; i += step) {
    const int t = (int)i;
    int slot = -1, pos = -1;
    if (t < base_t) {
      const int b = find_request(pre, B, t, false);
      const int c = max(__ldg(a.old_lens + b), 0);
      const long long at = (long long)c + t - pre[b].x;
      if (at >= 0 && at <= 0x7fffffffll) {
        pos = (int)at;
        const long long have = div_up(c);
        const int col = pos / P;
        int page = -1;
        if (col < W) {
          if (col < have) {
            page = a.block_table[b * a.table_stride + col];   // not written by this launch
          } else {
            const long long x = pre[b].y + (col - have);
            if (x >= 0 && x < got) page = __ldg(a.free_pages + head + x);
          }
        }
        if (page_ok(page)) slot = page * P + (pos - col * P);
      }
    }
    a.slot_map[t] = slot;
    a.positions[t] = pos;
  }
  for (long long i = tid; i < base_p; i += step) {
    const int x = (int)i;
    const int b = find_request(pre, B, x, true);
    const long long col = div_up(max(__ldg(a.old_lens + b), 0)) + (x - pre[b].y);
    if (col >= 0 && col < W)
      a.block_table[b * a.table_stride + col] = x < got ? __ldg(a.free_pages + head + x) : -1;
  }
}

// Copy of the new rows into their slots.  HBM-bound: 2 x 2 x tokens x kv_heads x D x 2 bytes.
// A thread moves one 16-byte vector of K and of V for each of kAppendRows tokens, every
// load issued before the first store.  33680 tokens of 8 heads of 128 (276 MB): 45.7 us =
// 6.04 TB/s, 0.92 of a plain copy's rate; 61 tokens: 1.8 us on the GPU.
constexpr int kAppendThreads = 256;
constexpr int kAppendRows = 2;

__global__ void __launch_bounds__(kAppendThreads)
paged_append_kernel(pa_paged_append_args a, int vecs, int tpc) {
  pdl_wait();
  pdl_begin_next();
  // thread -> (token of the CTA's group, vector of the token's kv_heads * D elements)
  const int slots = a.pages * a.page_size;
  const int hv = a.D / 8;
  for (int c = threadIdx.x; c < vecs * tpc; c += kAppendThreads) {
    const int tk = c / vecs, x = c - tk * vecs;
    const int h = x / hv, d = (x - h * hv) * 8;
    const long long ks = h * a.k_head_stride + d, vs = h * a.v_head_stride + d;
    const long long kd = h * a.kc_head_stride + d, vd = h * a.vc_head_stride + d;
    uint4 kx[kAppendRows], vx[kAppendRows];
    int slot[kAppendRows];
#pragma unroll
    for (int r = 0; r < kAppendRows; ++r) {
      const long long t = ((long long)blockIdx.x * kAppendRows + r) * tpc + tk;
      slot[r] = t < a.tokens ? __ldg(a.slot_map + t) : -1;
      if ((unsigned)slot[r] >= (unsigned)slots) slot[r] = -1;
      if (slot[r] >= 0) {
        kx[r] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.k) +
                                                      t * a.k_token_stride + ks));
        vx[r] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.v) +
                                                      t * a.v_token_stride + vs));
      }
    }
#pragma unroll
    for (int r = 0; r < kAppendRows; ++r) {
      if (slot[r] < 0) continue;
      const long long page = slot[r] / a.page_size, row = slot[r] % a.page_size;
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.k_cache) + page * a.kc_page_stride +
                                row * a.kc_row_stride + kd) = kx[r];
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.v_cache) + page * a.vc_page_stride +
                                row * a.vc_row_stride + vd) = vx[r];
    }
  }
}

}  // namespace
}  // namespace pa

extern "C" int pa_paged_step(const pa_paged_step_args* a, pa_stream_t stream) {
  using namespace pa;
  PA_CHECK_ARG(a != nullptr, "pa_paged_step: null args");
  PA_CHECK_ARG(a->requests >= 1 && a->requests <= kMaxRequests,
               "pa_paged_step: requests=%d not in [1, %d]", a->requests, kMaxRequests);
  PA_CHECK_ARG(a->page_size >= 1 && a->table_width >= 1 && a->tokens >= 0 && a->free_count >= 0,
               "pa_paged_step: bad page_size=%d table_width=%d tokens=%d free_count=%d",
               a->page_size, a->table_width, a->tokens, a->free_count);
  PA_CHECK_ARG(a->table_stride >= a->table_width || a->requests == 1,
               "pa_paged_step: table_stride=%lld is below the table's width %d",
               (long long)a->table_stride, a->table_width);
  PA_CHECK_ARG(a->old_lens && a->new_lens && a->free_head && a->block_table && a->q_start &&
                   a->seq_lens && a->free_head_out && a->missing &&
                   (a->free_pages || a->free_count == 0) &&
                   ((a->slot_map && a->positions) || a->tokens == 0),
               "pa_paged_step: null pointer");
  PA_CHECK_ARG(a->free_head != a->free_head_out, "pa_paged_step: free_head_out is free_head");
  // every CTA reads the inputs while one of them writes the outputs
  struct Span {
    const int32_t* p;
    long long n;
  };
  const long long B = a->requests;
  const Span in[] = {{a->old_lens, B}, {a->new_lens, B}, {a->free_pages, a->free_count},
                     {a->free_head, 1}};
  const Span out[] = {{a->q_start, B + 1}, {a->seq_lens, B}, {a->slot_map, a->tokens},
                      {a->positions, a->tokens}, {a->free_head_out, 1}, {a->missing, 1},
                      {a->block_table, (B - 1) * a->table_stride + a->table_width}};
  for (const Span& x : in)
    for (const Span& y : out)
      PA_CHECK_ARG(x.n == 0 || y.n == 0 || x.p + x.n <= y.p || y.p + y.n <= x.p,
                   "pa_paged_step: an output overlaps old_lens, new_lens, free_pages or free_head");
  const int smem = (a->requests + 1) * (int)sizeof(int2);
  if (smem > 40 * 1024) {
    const int rc = paged::prepare_kernel<paged_step_kernel>(
        "pa_paged_step", (kMaxRequests + 1) * (int)sizeof(int2), 0);
    if (rc) return rc;
  }
  int sms = 0;
  const int rc = paged::sm_count(&sms, "pa_paged_step");
  if (rc) return rc;
  int grid = a->tokens / kStepThreads + (a->tokens % kStepThreads != 0);
  grid = grid < 1 ? 1 : grid > sms ? sms : grid;
  return launch_after("pa_paged_step", paged_step_kernel, grid, kStepThreads, smem,
                      (cudaStream_t)stream, *a);
}

extern "C" int pa_paged_append(const pa_paged_append_args* a, pa_stream_t stream) {
  using namespace pa;
  PA_CHECK_ARG(a != nullptr, "pa_paged_append: null args");
  PA_CHECK_ARG(a->tokens >= 0 && a->kv_heads >= 1 && a->pages >= 1 && a->page_size >= 1,
               "pa_paged_append: bad tokens=%d kv_heads=%d pages=%d page_size=%d", a->tokens,
               a->kv_heads, a->pages, a->page_size);
  PA_CHECK_ARG(a->D >= 8 && a->D % 8 == 0 && a->D <= 512 && a->kv_heads <= 1024,
               "pa_paged_append: D=%d must be a multiple of 8 in [8, 512], kv_heads=%d at most 1024",
               a->D, a->kv_heads);
  PA_CHECK_ARG((long long)a->pages * a->page_size <= 0x7fffffffll,
               "pa_paged_append: %d pages of %d rows: slots must fit in 32 bits", a->pages,
               a->page_size);
  if (a->tokens == 0) return PA_OK;
  PA_CHECK_ARG(a->k && a->v && a->k_cache && a->v_cache && a->slot_map,
               "pa_paged_append: null pointer");
  const long long strides[] = {a->k_token_stride, a->k_head_stride, a->v_token_stride,
                               a->v_head_stride, a->kc_page_stride, a->kc_row_stride,
                               a->kc_head_stride, a->vc_page_stride, a->vc_row_stride,
                               a->vc_head_stride};
  for (long long s : strides)
    PA_CHECK_ARG(s % 8 == 0, "pa_paged_append: strides must be multiples of 8 elements");
  PA_CHECK_ARG(aligned(a->k, 16) && aligned(a->v, 16) && aligned(a->k_cache, 16) &&
                   aligned(a->v_cache, 16),
               "pa_paged_append: pointers must be 16-byte aligned");
  const int vecs = a->kv_heads * a->D / 8;              // 16-byte vectors of a token
  const int tpc = vecs >= kAppendThreads ? 1 : kAppendThreads / vecs;
  const int per = tpc * kAppendRows;
  const int grid = a->tokens / per + (a->tokens % per != 0);
  return launch_after("pa_paged_append", paged_append_kernel, grid, kAppendThreads, 0,
                      (cudaStream_t)stream, *a, vecs, tpc);
}
