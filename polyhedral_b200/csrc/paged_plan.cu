// The plan of a step's paged attention (equal shares of its key blocks) and the kernel that
// joins the partial results of divided units.
#include "paged.cuh"

namespace pa {
namespace paged {
namespace {

constexpr int kPlanThreads = 1024;

// Units of a request per key head, and what unit t costs in blocks.
__device__ __forceinline__ int unit_count(const Params& P, const Config& c, const Request& R) {
  if (c.half_tokens) return (R.n + 2 * c.half_tokens - 1) / (2 * c.half_tokens);
  return (R.n * P.group + kFewRows - 1) / kFewRows;
}
__device__ __forceinline__ int unit_cost(const Params& P, const Config& c, const Request& R, int t) {
  if (c.half_tokens) {
    const int t0 = t * 2 * c.half_tokens;
    return kUnitCost + run_blocks<128>(unit_runs<128, true>(
                           P.pred, R.pos0 + t0, R.pos0 + min(R.n, t0 + 2 * c.half_tokens) - 1, R.len,
                           min(1 << P.page_shift, 128)));
  }
  const int row0 = t * kFewRows, rows = min(R.n * P.group - row0, kFewRows);
  return kUnitCost + run_blocks<kFewBlock>(unit_runs<kFewBlock, false>(
                         P.pred, R.pos0 + row0 / P.group, R.pos0 + (row0 + rows - 1) / P.group, R.len,
                         kFewBlock));
}
// Rows of a request's largest unit that hold a token.
__device__ __forceinline__ int unit_rows_used(const Params& P, const Config& c, const Request& R) {
  if (c.half_tokens) return R.n > c.half_tokens ? 256 : R.n * P.group;
  return min(R.n * P.group, kFewRows);
}

// One CTA: the cost of every request, their running sum, and for each share the unit and
// block where it begins.  A request of many units is added up, and searched, by a whole
// warp.  Once per step, not per layer: 5.4-6.1 us for one token of one request, 9.1-10.8 us of
// 32 to 500, 25 us for 8 chunks of 1000 tokens and 28-36 us for one of 4096 (128 units a key
// head, gone through by the warps of their shares once more each); latency of dependent steps
// bounds it (lengths, sums, searches), not what it reads.
__global__ void __launch_bounds__(kPlanThreads)
paged_plan_kernel(const __grid_constant__ Params P, Config c, PlanView pv) {
  __shared__ long long warp_sum[kPlanThreads / 32];
  __shared__ long long s_before[kPlanThreads + 1];   // `before`, where it fits
  __shared__ int4 s_shares[kPlanThreads + 1];        // b, h, t, blk of a round's shares
  __shared__ int s_rows, s_cuts;
  pdl_wait();
  pdl_begin_next();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int B = P.requests;
  long long* pre = B <= kPlanThreads ? s_before : pv.before;
  if (threadIdx.x == 0) {
    s_rows = s_cuts = 0;
    *pv.status = 0;
  }
  __syncthreads();
  int rows = 0;
  long long base = 0;
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    Request R{0, 0, 0, 0};
    if (b < B) R = get_request(P, b);
    const int n = unit_count(P, c, R);
    rows = max(rows, unit_rows_used(P, c, R));
    long long cost = 0;
    if (n <= 4) {
      for (int t = 0; t < n; ++t) cost += unit_cost(P, c, R, t);
    }
    for (uint32_t big = __ballot_sync(0xffffffffu, n > 4); big; big &= big - 1) {
      const int src = __ffs(big) - 1;
      Request Q;
      Q.row0 = __shfl_sync(0xffffffffu, R.row0, src);
      Q.n = __shfl_sync(0xffffffffu, R.n, src);
      Q.pos0 = __shfl_sync(0xffffffffu, R.pos0, src);
      Q.len = __shfl_sync(0xffffffffu, R.len, src);
      const int m = unit_count(P, c, Q);
      long long sum = 0;
      for (int t = lane; t < m; t += 32) sum += unit_cost(P, c, Q, t);
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == src) cost = sum;
    }
    cost *= P.kv_heads;
    long long x = cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    long long before = base, all = 0;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 32; ++i) {
      const long long s = warp_sum[i];
      if (i < warp) before += s;
      all += s;
    }
    if (b < B) pre[b] = before + x - cost;
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) pre[B] = base;
#pragma unroll
  for (int o = 16; o; o >>= 1) rows = max(rows, __shfl_xor_sync(0xffffffffu, rows, o));
  if (lane == 0) atomicMax(&s_rows, rows);
  __syncthreads();
  const long long total = base;
  long long share;
  int used;
  if (total <= 0x7fff0000ll) {
    const uint32_t t32 = (uint32_t)total;
    const uint32_t s32 = max((t32 + c.workers - 1) / c.workers, (uint32_t)c.min_share);
    share = s32;
    used = (int)((t32 + s32 - 1) / s32);
  } else {
    share = (total + c.workers - 1) / c.workers;
    used = (int)((total + share - 1) / share);
  }

  // Rounds of shares, of which each knows the next round's first too.  Divided units are
  // entered by the worker of their last piece: the worker that begins one is the nearest
  // earlier one whose share ends inside a unit that it has begun (a running maximum).
  __shared__ int warp_max[kPlanThreads / 32];
  int carry = -1;
  constexpr int kRound = kPlanThreads - 1;
  for (int wb = 0; wb < used; wb += kRound) {
    const int w = wb + threadIdx.x;
    Share sh{B, 0, 0, 0, {0, 0, 0, 0}};
    long long rem = 0;
    Request R{0, 0, 0, 0};
    int n = 0;
    const bool in = w < used;
    if (in) {
      const long long x = w * share;
      int lo = 0, hi = B;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= x) lo = mid; else hi = mid;
      }
      sh.b = lo;
      const long long all = pre[lo + 1] - pre[lo], in_b = x - pre[lo];
      if (all <= 0x7fffffffll) {                      // the usual case, in 32 bits
        const uint32_t per_head = (uint32_t)all / (uint32_t)P.kv_heads;
        sh.h = (int)((uint32_t)in_b / per_head);
        rem = (uint32_t)in_b - sh.h * per_head;
      } else {
        const long long per_head = all / P.kv_heads;
        sh.h = (int)(in_b / per_head);
        rem = in_b - sh.h * per_head;
      }
      R = get_request(P, lo);
      n = unit_count(P, c, R);
      if (n <= 4) {
        int t = 0, cost = unit_cost(P, c, R, 0);
        while (rem >= cost && t + 1 < n) {
          rem -= cost;
          cost = unit_cost(P, c, R, ++t);
        }
        sh.t = t;
      }
    }
    for (uint32_t big = __ballot_sync(0xffffffffu, in && n > 4); big; big &= big - 1) {
      const int src = __ffs(big) - 1;
      Request Q;
      Q.row0 = __shfl_sync(0xffffffffu, R.row0, src);
      Q.n = __shfl_sync(0xffffffffu, R.n, src);
      Q.pos0 = __shfl_sync(0xffffffffu, R.pos0, src);
      Q.len = __shfl_sync(0xffffffffu, R.len, src);
      long long left = __shfl_sync(0xffffffffu, rem, src);
      const int m = unit_count(P, c, Q);
      int t0 = 0, found = m - 1;
      for (; t0 < m; t0 += 32) {
        const int cost = t0 + lane < m ? unit_cost(P, c, Q, t0 + lane) : 0;
        long long sum = cost;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long y = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += y;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, sum > left);
        if (past) {
          const int at = __ffs(past) - 1;
          found = t0 + at;
          left -= __shfl_sync(0xffffffffu, sum - cost, at);
          break;
        }
        left -= __shfl_sync(0xffffffffu, sum, 31);
      }
      if (lane == src) {
        sh.t = found;
        rem = left;
      }
    }
    if (in) {
      // A cut inside the unit's own cost, or so early that the piece before it would be short,
      // falls on the unit's begin; one that would leave a short piece behind it, or any
      // inside a unit where units stay whole, on the next unit's.
      sh.blk = max((int)rem - kUnitCost, 0);
      if (sh.blk < c.min_piece) sh.blk = 0;
      const int left = unit_cost(P, c, R, sh.t) - kUnitCost - sh.blk;
      if (c.split ? sh.blk > 0 && left < c.min_piece : rem > 0) {
        sh.blk = 0;
        if (++sh.t >= n) {
          sh.t = 0;
          if (++sh.h == P.kv_heads) {
            sh.h = 0;
            R = ++sh.b < B ? get_request(P, sh.b) : Request{0, 0, 0, 0};
          }
        }
      }
      sh.R = R;
    }
    if (w <= used) pv.shares[w] = sh;
    s_shares[threadIdx.x] = make_int4(sh.b, sh.h, sh.t, sh.blk);
    __syncthreads();
    const Share& s = sh;
    const bool mine = w < used && (int)threadIdx.x < kRound;
    const int4 en = s_shares[mine ? threadIdx.x + 1 : threadIdx.x];
    const Share e{en.x, en.y, en.z, en.w, {0, 0, 0, 0}};
    const bool same = s.b == e.b && s.h == e.h && s.t == e.t;
    const bool begins = mine && e.blk > 0 && (!same || s.blk == 0);
    int x = begins ? w : -1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x = max(x, y);
    }
    __syncthreads();
    if (lane == 31) warp_max[warp] = x;
    __syncthreads();
    int before = carry;
    for (int i = 0; i < warp; ++i) before = max(before, warp_max[i]);
    int all = carry;
    for (int i = 0; i < kPlanThreads / 32; ++i) all = max(all, warp_max[i]);
    // the running maximum before this worker
    int w0 = __shfl_up_sync(0xffffffffu, x, 1);
    w0 = max(lane == 0 ? -1 : w0, before);
    carry = all;
    if (mine && s.blk > 0 && !same)
      pv.cuts[atomicAdd(&s_cuts, 1)] = Cut{w0, w - w0 + 1, s.h, s.t, s.R};
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (used == 0) pv.shares[0] = Share{B, 0, 0, 0, {0, 0, 0, 0}};
    pv.meta[0] = used;
    pv.meta[1] = s_cuts;
    pv.meta[2] = s_rows;
  }
}

// One divided unit's row: O = sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i over its pieces, m
// the largest m_i.  Reading the pieces bounds it (they are in L2).  Three ways, by how many
// rows and pieces there are: of the chunk kernel's large units a warp takes 8 rows, 4 at a time
// so that their loads overlap and the unit's addresses are worked out once (a row per warp
// was bound by those instructions: 24 ragged requests took 104 us in all instead of 96); of
// the few-rows kernel's small ones a warp takes one row, four pieces at a time (8 rows as
// above: 64 requests' decode took 163 us instead of 158); and where units have many pieces
// the warps of a CTA share a row's.  (The order of `cuts` is that of an atomic counter; it
// decides only which warp joins which row.)
constexpr int kJoinWarps = 8;
__host__ __device__ inline int check_ctas(const Config& c) {   // a thread per share
  return (c.workers + kJoinWarps * 32 - 1) / (kJoinWarps * 32);
}

// 3 CTAs a multiprocessor: 78 registers a thread, which the loads of 4 rows at once need (with
// 64 at D = 64, 24 ragged requests took 96.2 us instead of 94.8).
template <int D, bool kBf16>
__global__ void __launch_bounds__(kJoinWarps * 32, 3)
paged_join_kernel(const __grid_constant__ Params P, Config c, PlanView pv,
                  const float* __restrict__ scratch) {
  constexpr int E = D / 32;
  __shared__ float s_acc[kJoinWarps][D];
  __shared__ float2 s_ml[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_begin_next();
  const int used = pv.meta[0], cuts = pv.meta[1], rows = pv.meta[2];
  // the first CTAs compare the plan's lengths instead of joining (a joining one would begin later)
  const int checks = check_ctas(c), ctas = gridDim.x - checks, cta = (int)blockIdx.x - checks;
  if (cta < 0) {
    if (other_lengths(P, pv.shares, used, blockIdx.x * (kJoinWarps * 32) + threadIdx.x,
                      checks * (kJoinWarps * 32)))
      atomicExch(pv.status, (int32_t)DEV_OTHER_LENGTHS);
    return;
  }
  const bool many = used > kJoinWarps * cuts;   // pieces per unit, on average
  const int unit_rows = c.unit_rows;
  const size_t slot = slot_floats<D>(unit_rows);
  const float* ml0 = scratch + (size_t)unit_rows * D;
  // row r of a unit: its token of the request (-1: none) and head of the group
  auto place = [&](const Cut& cut, int r, int& g) -> int {
    int t;
    if (c.half_tokens) {
      const int x = r & 127, y = div_group(P, x);
      g = x - y * P.group;
      t = y < c.half_tokens ? (cut.t * 2 + (r >> 7)) * c.half_tokens + y : -1;
    } else {
      const int row = cut.t * kFewRows + r;
      t = row / P.group;
      g = row - t * P.group;
    }
    return t < cut.R.n ? t : -1;
  };
  auto write = [&](const Cut& cut, int tok, int g, float m, float l, const float (&acc)[E]) {
    const int t = cut.R.row0 + tok, a = cut.h * P.group + g;
    const float inv = l == 0.f ? 0.f : 1.f / l;   // a sum that is no number stays one
    uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(P.o) + (long long)t * P.o_t +
                                              (long long)a * P.o_h + lane * E);
    if constexpr (E == 4)
      *reinterpret_cast<uint2*>(o) = make_uint2(pack_pair<kBf16>(acc[0] * inv, acc[1] * inv),
                                                pack_pair<kBf16>(acc[2] * inv, acc[3] * inv));
    else
      o[0] = pack_pair<kBf16>(acc[0] * inv, acc[1] * inv);
    if (P.lse && lane == 0)
      P.lse[a * P.lse_h + t] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
  };
  auto load = [&](size_t at, int r, float2& ml, float (&x)[E]) {
    ml = *reinterpret_cast<const float2*>(ml0 + at + 2 * r);
    if constexpr (E == 4) {
      const float4 v = *reinterpret_cast<const float4*>(scratch + at + (size_t)r * D + lane * 4);
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(scratch + at + (size_t)r * D + lane * 2);
      x[0] = v.x; x[1] = v.y;
    }
  };
  constexpr int U = 4;

  if (!many && c.half_tokens) {
    constexpr int kGroup = 8;
    const int groups = (rows + kGroup - 1) / kGroup;
    for (int it = cta * kJoinWarps + warp; it < cuts * groups; it += ctas * kJoinWarps) {
      const int k = it / groups;
      const Cut cut = pv.cuts[k];
      const int r0 = (it - k * groups) * kGroup;
#pragma unroll 1
      for (int r1 = r0; r1 < r0 + kGroup; r1 += U) {
        int tok[U], g[U];
        float m[U], l[U], acc[U][E];
        bool some = false;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          tok[u] = r1 + u < unit_rows ? place(cut, r1 + u, g[u]) : -1;
          some |= tok[u] >= 0;
          m[u] = -INFINITY;
          l[u] = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[u][e] = 0.f;
        }
        if (!some) continue;
#pragma unroll 1
        for (int p = 0; p < cut.pieces; ++p) {
          const size_t at = (size_t)(p == 0 ? 2 * cut.worker + 1 : 2 * (cut.worker + p)) * slot;
          float2 ml[U];
          float x[U][E];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (tok[u] >= 0) load(at, r1 + u, ml[u], x[u]);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (tok[u] < 0) continue;
            const float mn = fmaxf(m[u], ml[u].x), z = mn == -INFINITY ? 0.f : mn;
            const float f = ex2f(m[u] - z), h = ex2f(ml[u].x - z);
            m[u] = mn;
            l[u] = fmaf(h, ml[u].y, l[u] * f);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[u][e] = fmaf(h, x[u][e], acc[u][e] * f);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (tok[u] >= 0) write(cut, tok[u], g[u], m[u], l[u], acc[u]);
      }
    }
    return;
  }

  const int it0 = many ? cta : cta * kJoinWarps + warp;
  for (int it = it0; it < cuts * rows; it += many ? ctas : ctas * kJoinWarps) {
    const int k = it / rows, r = it - k * rows;
    const Cut cut = pv.cuts[k];
    int g;
    const int tok = place(cut, r, g);
    if (tok < 0) continue;                       // alike for the whole CTA, where it shares a row
    float m = -INFINITY, l = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    const int dp = many ? kJoinWarps : 1;
    for (int p = many ? warp : 0; p < cut.pieces; p += dp * U) {
      float2 ml[U];
      float x[U][E];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int q = p + u * dp;
        ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = 0.f;
        if (q < cut.pieces)
          load((size_t)(q == 0 ? 2 * cut.worker + 1 : 2 * (cut.worker + q)) * slot, r, ml[u], x[u]);
      }
      float mn = m;
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, ml[u].x);
      const float z = mn == -INFINITY ? 0.f : mn;
      const float f = ex2f(m - z);
      m = mn;
      l *= f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float h = ex2f(ml[u].x - z);
        l = fmaf(h, ml[u].y, l);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(h, x[u][e], acc[e]);
      }
    }
    if (many) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) s_acc[warp][lane * E + e] = acc[e];
      if (lane == 0) s_ml[warp] = make_float2(m, l);
      __syncthreads();
      if (warp > 0) continue;
      float mn = -INFINITY;
#pragma unroll
      for (int i = 0; i < kJoinWarps; ++i) mn = fmaxf(mn, s_ml[i].x);
      const float z = mn == -INFINITY ? 0.f : mn;
      l = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
      for (int i = 0; i < kJoinWarps; ++i) {
        const float h = ex2f(s_ml[i].x - z);
        l = fmaf(h, s_ml[i].y, l);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(h, s_acc[i][lane * E + e], acc[e]);
      }
      m = mn;
    }
    write(cut, tok, g, m, l, acc);
  }
}

}  // namespace

int launch_plan(const Params& P, const Config& c, const PlanView& pv, cudaStream_t stream) {
  return launch_after("pa_paged_plan", paged_plan_kernel, 1, kPlanThreads, 0, stream, P, c, pv);
}

int launch_join(const Params& P, bool bf16, int D, const PlanView& pv, const Config& c,
                const float* scratch, int sms, cudaStream_t stream) {
  auto go = [&](auto kernel) {
    return launch_after("pa_paged_attn", kernel, sms * 4, kJoinWarps * 32, 0, stream, P, c, pv, scratch);
  };
  if (D == 128) return bf16 ? go(paged_join_kernel<128, true>) : go(paged_join_kernel<128, false>);
  return bf16 ? go(paged_join_kernel<64, true>) : go(paged_join_kernel<64, false>);
}

}  // namespace paged
}  // namespace pa
