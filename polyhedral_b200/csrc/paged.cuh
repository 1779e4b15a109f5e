// Shared pieces of the attention over a paged K/V cache: the forward's parameters and
// the keys that a run of query positions can see.
#pragma once
#include <math.h>
#include <atomic>
#include "common.cuh"
#include "capi_util.h"

namespace pa {
namespace paged {

struct Params {
  uint32_t group_inv;   // (x * group_inv) >> 20 = x / group for 0 <= x < 512
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* lse;
  const int32_t* table;
  const int32_t* seq_lens;
  const int32_t* q_start;
  int requests, tokens, heads, kv_heads, group;
  int pages, page_shift, width;
  long long table_stride;
  long long q_t, q_h, k_p, k_r, k_h, v_p, v_r, v_h, o_t, o_h, lse_h;
  Pred pred;
  float scale_log2;
};

// x / group for 0 <= x < 512: group_inv = ceil(2^20 / group) is above 2^20 / group by less
// than 1, which shifts the product by less than 512 / 2^20 < 1 / (8 * 128).
__device__ __forceinline__ int div_group(const Params& P, int x) {
  return (int)(((uint32_t)x * P.group_inv) >> 20);
}

// A request as the kernels see it: its first row of q / o, its new tokens, the position of the
// first of them, and its tokens, all kept inside the buffers whatever the arrays say.
struct Request {
  int row0, n, pos0, len;
};
__device__ __forceinline__ Request get_request(const Params& P, int b) {
  Request r;
  const int s = __ldg(P.q_start + b), e = __ldg(P.q_start + b + 1);
  r.row0 = min(max(s, 0), P.tokens);
  r.n = max(min(e, P.tokens) - r.row0, 0);
  const int len = __ldg(P.seq_lens + b);
  // a token's position counts back from the request's last one, also where the table
  // is too narrow for all of them
  // (kept within 2^26, so that no sum with a mask's widths overflows)
  const long long pos = (long long)len - ((long long)e - s) + ((long long)r.row0 - s);
  r.pos0 = (int)max(min(pos, 1ll << 26), -(1ll << 26));
  r.len = min(max(len, 0), P.width << P.page_shift);
  return r;
}

// Keys that positions [i0, i1] of a request of `len` tokens can see: [a0, b0) and
// [a1, b1), ascending and not touching (empty: a == b).  Exact for the bands; a lattice
// counts as everything between its ends.
struct KeyRanges {
  int a0, b0, a1, b1;
};
__device__ __forceinline__ KeyRanges key_ranges(const Pred& p, int i0, int i1, int len) {
  const int hi = min(i1 + 1, len);
  int a = 0, b = hi, c = 0, d = 0;   // near [a, b), far [c, d)
  switch (p.kind) {
    case PA_WINDOW:
      a = i0 - p.p0 + 1;
      break;
    case PA_SINKS:
      a = i0 - p.p0 + 1;
      d = p.p1;
      break;
    case PA_TWOBAND:
      a = i0 - p.p0 + 1;
      c = i0 - p.p1 - p.p2 + 1;
      d = i1 - p.p1 + 1;
      break;
    case PA_FAR_STRIDED:
      b = i1 - p.p0 + 1;
      break;
    default:
      break;
  }
  a = max(a, 0);
  c = max(c, 0);
  b = min(b, hi);
  d = min(d, hi);
  KeyRanges r{0, 0, 0, 0};
  if (a >= b) a = b = 0;
  if (c >= d) c = d = 0;
  if (a < b && c < d) {
    if (c > a) {
      int t = a; a = c; c = t;
      t = b; b = d; d = t;
    }
    if (d >= a) {       // they touch: one range
      b = max(b, d);
      a = c;
      c = d = 0;
    }
  }
  if (c < d) {
    r.a0 = c;
    r.b0 = d;
    r.a1 = a;
    r.b1 = b;
  } else {
    r.a0 = a;
    r.b0 = b;
  }
  return r;
}

// Multiprocessors of the current device.
inline int sm_count(int* sms, const char* who) {
  int dev = 0;
  PA_CUDA(cudaGetDevice(&dev), who);
  PA_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev), who);
  return PA_OK;
}

// Allows kernel kKernel `smem` bytes of shared memory, once per device and always the same
// (the limit belongs to the function: a smaller one set by another thread's call would make a
// launch fail); with `min_regs`, refuses a build with fewer registers per thread (a register
// split that they do not cover would never complete).
template <auto kKernel>
int prepare_kernel(const char* who, int smem, int min_regs) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  PA_CUDA(cudaGetDevice(&dev), who);
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return PA_OK;
  PA_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), who);
  if (min_regs > 0) {
    cudaFuncAttributes fa;
    PA_CUDA(cudaFuncGetAttributes(&fa, kKernel), who);
    if (fa.numRegs < min_regs)
      return fail(PA_ERR_UNSUPPORTED, "%s: kernel built with %d registers per thread, below its "
                  "register split", who, fa.numRegs);
  }
  done.fetch_or(bit, std::memory_order_relaxed);
  return PA_OK;
}

// ------------------------------------------------------------- shares of work
// A unit is kRows query rows (token-major, the query heads of one key head inside) of
// one request and key head; its keys come in blocks.  The plan lines all units up,
// request by request, key head by key head, and cuts the line into equal shares, one per
// worker, wherever the cut falls: a unit that a cut divides is worked on by several
// workers, whose partial results (sum, running maximum and unnormalised O of every row,
// 32-bit) are joined by a second kernel in the order of the keys.  No counters, no order
// that depends on timing: the same call gives the same bits.
struct __align__(16) Share {
  int b, h, t, blk;   // request, key head, unit of them, first block
  Request R;          // the request, so that a worker starts without a chain of loads
};
// A divided unit: the worker that begins it, its pieces, and where its rows are.
struct __align__(16) Cut {
  int worker, pieces, h, t;
  Request R;
};

// Whether the plan was built from other lengths than the arrays hold now, as far as shares
// w0, w0 + step, ... and requests in the same steps can tell.  A worker takes the request that
// its share begins in from the plan and all others from the arrays, so a result can only be
// wrong where such a request has changed, or where one has rows now that lies before the
// first share (or any, if the plan has no share).
__device__ __forceinline__ bool other_lengths(const Params& P, const Share* shares, int used, int w0,
                                              int step) {
  bool other = false;
  for (int w = w0; w < used; w += step) {
    const Share s = shares[w];
    if (s.b >= P.requests) break;
    const Request R = get_request(P, s.b);
    other |= R.row0 != s.R.row0 || R.n != s.R.n || R.pos0 != s.R.pos0 ||
             R.len != min(s.R.len, P.width << P.page_shift);
  }
  const int idle = used > 0 ? min(shares[0].b, P.requests) : P.requests;
  for (int b = w0; b < idle; b += step) other |= get_request(P, b).n > 0;
  return other;
}

// What the host chooses from the sizes and hints alone, alike for plan and forward.
struct Config {
  int unit_rows;      // query rows per unit
  int half_tokens;    // chunk kernel: tokens per half of a unit; few-rows kernel: 0
  int workers;        // most shares
  int min_share;      // blocks below which a share is not worth a worker
  int min_piece;      // blocks of a piece below which a unit is not cut there
  int split;          // units may be cut
};

// Blocks that a unit costs beside its own (loading q, writing o): 24 ragged requests took 97
// us with 2 or 3, 101 us with 1.
constexpr int kUnitCost = 2;

struct PlanView {
  int32_t* status;
  int32_t* meta;      // shares in use, divided units, most rows of a unit
  Share* shares;      // [workers + 1]; the entry behind those in use is past all requests
  Cut* cuts;          // [workers] divided units
  long long* before;  // [requests + 1] cost before a request
};
inline __host__ size_t plan_bytes(const Config& c, int requests) {
  return 256 + sizeof(Share) * (c.workers + 1) + sizeof(Cut) * c.workers + 8 * (size_t)(requests + 1);
}
inline __host__ PlanView plan_view(void* p, const Config& c) {
  char* b = static_cast<char*>(p);
  PlanView v;
  v.status = reinterpret_cast<int32_t*>(b);
  v.meta = reinterpret_cast<int32_t*>(b + 64);
  v.shares = reinterpret_cast<Share*>(b + 256);
  v.cuts = reinterpret_cast<Cut*>(b + 256 + sizeof(Share) * (c.workers + 1));
  v.before = reinterpret_cast<long long*>(v.cuts + c.workers);
  return v;
}

// Partial result of a divided unit: worker w's piece of a unit that it does not begin
// goes to slot 2 w, of one that it begins and does not end to slot 2 w + 1.
template <int D>
__host__ __device__ constexpr size_t slot_floats(int unit_rows) {
  return (size_t)unit_rows * (D + 2);
}

// Keys of a unit whose rows sit at positions [i0, i1]: two runs of `cnt` keys a, a + step,
// ..., of which those before `lo` are only there because a run with step 1 starts at a
// multiple of `align` (a power of two, the rows that are copied together).  A single position's lattice keys are listed one by one (step = the
// modulus), so that only they are read (not if kDense).  `exact`: every listed key from
// lo on is live for every row.
struct Runs {
  int a[2], cnt[2], step[2], lo[2];
  bool exact;
};
template <int kBlock, bool kDense>
__device__ __forceinline__ Runs unit_runs(const Pred& p, int i0, int i1, int len, int align) {
  Runs r;
  r.step[0] = r.step[1] = 1;
  r.exact = i0 == i1;
  if (p.mod > 1 && i0 == i1 && !kDense) {
    // run 0: the lattice from the band (if any) down; run 1: the band
    const int top = min(i0, len - 1);
    const int near = p.kind == PA_LOCAL_STRIDED ? min(max(p.p0, 0), i0 + 1) : 0;   // band's keys
    const int far0 = p.kind == PA_FAR_STRIDED ? max(p.p0, 0) : near;
    const int last = min(top, i0 - far0);
    const int first = i0 >= 0 ? i0 % p.mod : 0;
    r.a[0] = r.lo[0] = first;
    r.step[0] = p.mod;
    r.cnt[0] = i0 >= 0 && last >= first ? (last - first) / p.mod + 1 : 0;
    r.lo[1] = max(i0 - near + 1, 0);
    r.a[1] = r.lo[1] & ~(align - 1);
    r.cnt[1] = near > 0 ? max(top + 1 - r.a[1], 0) : 0;
    return r;
  }
  if (p.mod > 1) r.exact = false;
  const KeyRanges k = key_ranges(p, i0, i1, len);
  r.lo[0] = k.a0;
  r.lo[1] = k.a1;
  r.a[0] = k.a0 & ~(align - 1);
  r.a[1] = k.a1 & ~(align - 1);
  r.cnt[0] = k.b0 > k.a0 ? k.b0 - r.a[0] : 0;
  r.cnt[1] = k.b1 > k.a1 ? k.b1 - r.a[1] : 0;
  // the first run's last block reaches into the second: one run
  if (r.cnt[0] > 0 && r.cnt[1] > 0 && r.a[1] < r.a[0] + (r.cnt[0] + kBlock - 1) / kBlock * kBlock) {
    r.cnt[0] = k.b1 - r.a[0];
    r.cnt[1] = 0;
    r.exact = false;
  }
  return r;
}
template <int kBlock>
__device__ __forceinline__ int run_blocks(const Runs& r) {
  return (r.cnt[0] + kBlock - 1) / kBlock + (r.cnt[1] + kBlock - 1) / kBlock;
}

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The few-rows kernel: units of 16 rows, blocks of 16 keys, a warp per share.
constexpr int kFewRows = 16;
constexpr int kFewBlock = 16;
constexpr int kFewWarps = 8;

// Rows of a unit: few-rows kernel -- 16 of the request's n * group, which may begin and end
// inside a token; chunk kernel -- two halves of 128, the first half_tokens * group of which
// are whole tokens' (row r of half x: token x * half_tokens + r / group, head r % group).
int launch_few(const Params& P, bool bf16, int D, const PlanView& pv, const Config& c,
               float* scratch, int sms, cudaStream_t stream);
int launch_plan(const Params& P, const Config& c, const PlanView& pv, cudaStream_t stream);
// Joins the partial results of divided units; runs behind the forward on `stream`.
int launch_join(const Params& P, bool bf16, int D, const PlanView& pv, const Config& c,
                const float* scratch, int sms, cudaStream_t stream);

template <bool kBf16>
__device__ __forceinline__ float2 unpack_pair(uint32_t u) {
  if constexpr (kBf16)
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (kBf16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

// Keys of block `blk` of a unit: runs[0]'s blocks, then runs[1]'s.  Place x holds key
// j0 + x * step; those with x in [lo, hi) are listed.
struct BlockKeys {
  int j0, step, lo, hi;
};
template <int kBlock>
__device__ __forceinline__ BlockKeys block_keys(const Runs& r, int blk) {
  const int n0 = (r.cnt[0] + kBlock - 1) / kBlock;
  const int part = blk >= n0;
  const int base = (blk - (part ? n0 : 0)) * kBlock;
  BlockKeys k;
  k.step = part ? r.step[1] : r.step[0];
  k.j0 = (part ? r.a[1] : r.a[0]) + base * k.step;
  k.lo = 0;
  k.hi = min((part ? r.cnt[1] : r.cnt[0]) - base, kBlock);
  if (k.step == 1) k.lo = max((part ? r.lo[1] : r.lo[0]) - k.j0, 0);
  return k;
}

// One row (token t of q, query head h * group + g, position i) over blocks [blk0, blk1), one
// key at a time, skipping masked keys instead of weighing their values by 0: the way out
// when a masked key's value is not finite (0 times it is not 0).  All lanes take part;
// lane x ends with columns [D / 32 x, D / 32 (x + 1)) of the unnormalised O.
template <int D, bool kBf16, int kBlock>
__device__ __noinline__ void row_by_key(const Params& P, int b, int h, int t, int g, int i,
                                        const Runs& runs, int blk0, int blk1, float& m_out,
                                        float& l_out, float (&acc)[D / 32]) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int a = h * P.group + g;
  const uint16_t* qp = static_cast<const uint16_t*>(P.q) + (long long)t * P.q_t +
                       (long long)a * P.q_h + lane * E;
  float q[E];
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    const float2 x = unpack_pair<kBf16>(*reinterpret_cast<const uint32_t*>(qp + e));
    q[e] = x.x;
    q[e + 1] = x.y;
    acc[e] = acc[e + 1] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int mask = (1 << P.page_shift) - 1;
  const uint16_t* kh = static_cast<const uint16_t*>(P.k) + (long long)h * P.k_h;
  const uint16_t* vh = static_cast<const uint16_t*>(P.v) + (long long)h * P.v_h + lane * E;
#pragma unroll 1
  for (int blk = blk0; blk < blk1; ++blk) {
    const BlockKeys bk = block_keys<kBlock>(runs, blk);
#pragma unroll 1
    for (int x0 = 0; x0 < kBlock; x0 += 32) {        // a key per lane
      const int x = x0 + lane, j = bk.j0 + x * bk.step;
      bool live = x >= bk.lo && x < bk.hi && pred_live(P.pred, i, j);
      int page = -1;
      if (live) page = __ldg(P.table + (long long)b * P.table_stride + (j >> P.page_shift));
      live = live && (unsigned)page < (unsigned)P.pages;
      const long long vo = live ? page * P.v_p + (j & mask) * P.v_r : 0;
      const uint16_t* kp = kh + (live ? page * P.k_p + (j & mask) * P.k_r : 0);
      float s = 0.f;
#pragma unroll 1
      for (int d = 0; d < 32; ++d) {                  // lane d's columns of q
        float2 y[E / 2];
#pragma unroll
        for (int e = 0; e < E; e += 2)
          y[e / 2] = unpack_pair<kBf16>(*reinterpret_cast<const uint32_t*>(kp + d * E + e));
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          s = fmaf(__shfl_sync(0xffffffffu, q[e], d), y[e / 2].x, s);
          s = fmaf(__shfl_sync(0xffffffffu, q[e + 1], d), y[e / 2].y, s);
        }
      }
      s = live ? s * P.scale_log2 : -INFINITY;
      float mn = s;
#pragma unroll
      for (int o = 16; o; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mn = fmaxf(m, mn);
      const float base = mn == -INFINITY ? 0.f : mn;
      const float f = ex2f(m - base), p = live ? ex2f(s - base) : 0.f;
      m = mn;
      float sum = p;
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l = l * f + sum;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= f;
#pragma unroll 1
      for (uint32_t todo = __ballot_sync(0xffffffffu, live); todo; todo &= todo - 1) {
        const int y = __ffs(todo) - 1;
        const float py = __shfl_sync(0xffffffffu, p, y);
        const uint16_t* vp = vh + __shfl_sync(0xffffffffu, vo, y);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 z = unpack_pair<kBf16>(*reinterpret_cast<const uint32_t*>(vp + e));
          acc[e] = fmaf(py, z.x, acc[e]);
          acc[e + 1] = fmaf(py, z.y, acc[e + 1]);
        }
      }
    }
  }
  m_out = m;
  l_out = l;
}

}  // namespace paged
}  // namespace pa
