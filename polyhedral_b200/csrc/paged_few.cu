// Attention of few new tokens (one, as a rule) over a paged K/V cache, and of any where the
// keys are few in all.
//
// With at most 16 query rows per key head the work is reading the cache: 4 D bytes per
// key against 4 D FLOP per key and row, at most 16 FLOP per byte where the GPU has 250.  So HBM
// bounds it, and what counts is bytes in flight.  Every warp works alone: it has an
// equal share of the step's key blocks (16 keys each), its own ring of blocks in shared
// memory that it fills with 16-byte asynchronous copies several blocks ahead, and its own
// running maximum, sum and O in registers; no barrier ties it to another warp.  The products run on
// the warp's matrix instructions (16 rows x 16 keys): idle rows cost nothing that
// is short here, and the 5th-generation tensor path would bring tensor memory and
// CTA-wide barriers to a kernel that issues in 30 % of its cycles.
//
// Blocks of 16 keys and 192 KB of ring per multiprocessor (8 warps x 3 blocks x 8 KB at D =
// 128) keep some 128 KB in flight.  Measured (the least and the most of several GPUs): 64
// requests of up to 8000 tokens (998 MB) 158-168 us = 5.9-6.3 TB/s, 0.91-0.97 of a plain copy's
// rate; 4 of up to 131071 tokens (1.89 GB) 279-291 us = 6.5-6.8 TB/s; 128 requests under a window
// of 1024 and 4 sinks (541 MB) 93-101 us = 5.3-5.8 TB/s: 65 blocks a unit, and 2300 cycles to
// begin one and as many to fill its ring.  That is what bounds units of few blocks: the ring
// drains at every unit's end, and the next one's lengths, table entries, q and first blocks
// are read one after another (500 requests of 20-200 tokens 51 us, of D = 64 47 us, where their
// bytes take 36 and 18 us).  A single request of 1000 tokens: 8.7 us on the GPU with the join; the
// chain share -> table -> keys -> partial result -> join bounds it.
#include "paged.cuh"

namespace pa {
namespace paged {
namespace {

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;"
               ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3},"
                 " {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3},"
                 " {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D>
struct Few {
  static constexpr int kRowBytes = D * 2;
  static constexpr int kTile = kFewBlock * kRowBytes;       // 16 rows of K or of V
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kWarpBytes = kStages * 2 * kTile;
  static constexpr int kMetaOff = kFewWarps * kWarpBytes;
  static constexpr int kBytes = kMetaOff + kFewWarps * kStages * 4;
};

// A piece of a unit: its blocks [blk0, blk1), and where its rows go.
struct Piece {
  Request R;
  Runs runs;
  int b, h, row0, rows, blk0, blk1;
  float* slot;        // partial result, or null: o and lse
};

template <int D, bool kBf16>
__device__ __noinline__ void piece_by_key(const Params& P, const Piece& c) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int r = 0; r < c.rows; ++r) {
    float m, l, acc[E];
    const int row = c.row0 + r;
    row_by_key<D, kBf16, kFewBlock>(P, c.b, c.h, c.R.row0 + row / P.group, row % P.group,
                                   c.R.pos0 + row / P.group, c.runs, c.blk0, c.blk1, m, l, acc);
    if (c.slot) {
#pragma unroll
      for (int e = 0; e < E; ++e) c.slot[r * D + lane * E + e] = acc[e];
      if (lane == 0) {
        c.slot[kFewRows * D + 2 * r] = m;
        c.slot[kFewRows * D + 2 * r + 1] = l;
      }
    } else {
      const int t = c.R.row0 + row / P.group, a = c.h * P.group + row % P.group;
      const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
      uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(P.o) + (long long)t * P.o_t +
                                                a * P.o_h + lane * E);
#pragma unroll
      for (int e = 0; e < E; e += 2) o[e / 2] = pack_pair<kBf16>(acc[e] * inv, acc[e + 1] * inv);
      if (P.lse && lane == 0)
        P.lse[a * P.lse_h + t] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
    }
  }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kFewWarps * 32, 1)
paged_few_kernel(const __grid_constant__ Params P, const Share* __restrict__ shares,
                 const int32_t* __restrict__ meta, float* __restrict__ scratch, int32_t* status) {
  using F = Few<D>;
  constexpr int S = F::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait();
  pdl_begin_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // neighbouring shares go to different multiprocessors, so that little work spreads
  const int w = warp * gridDim.x + blockIdx.x;
  const uint32_t ring = smem_u32(smem) + warp * F::kWarpBytes;
  uint32_t* s_live = reinterpret_cast<uint32_t*>(smem + F::kMetaOff) + warp * S;
  const int used = __ldg(meta);
  const Share first = shares[w], end = shares[w + 1];   // inside the plan for every worker
  // the plan's lengths, where no join compares them: by the last workers, which have no share
  // where the work is little
  if (status && warp == kFewWarps - 1 &&
      other_lengths(P, shares, used, (gridDim.x - 1 - blockIdx.x) * 32 + lane, gridDim.x * 32))
    atomicExch(status, (int32_t)DEV_OTHER_LENGTHS);
  if (w >= used) return;
  const int G = P.group;
  const int mask = (1 << P.page_shift) - 1;
  const int g = lane >> 2, tq = lane & 3;      // fragment row and column pair of this lane

  Share at = first;
  bool fresh = true;                           // first piece of this worker
  while (true) {
    // past the last unit of the share
    if (at.b >= P.requests || at.b > end.b ||
        (at.b == end.b && (at.h > end.h || (at.h == end.h && at.t > end.t))))
      break;
    Piece c;
    if (fresh && at.b == first.b) {
      c.R = first.R;
      c.R.len = min(c.R.len, P.width << P.page_shift);
    } else {
      c.R = get_request(P, at.b);
    }
    const int total = c.R.n * G;
    if (at.t * kFewRows >= total) {            // past the request's last unit
      at.t = 0;
      if (total == 0 || ++at.h == P.kv_heads) {
        at.h = 0;
        ++at.b;
      }
      continue;
    }
    const bool last = at.b == end.b && at.h == end.h && at.t == end.t;
    if (last && end.blk == 0) break;
    c.b = at.b;
    c.h = at.h;
    c.row0 = at.t * kFewRows;
    c.rows = min(total - c.row0, kFewRows);
    const int t0 = c.row0 / G, in0 = c.row0 - t0 * G;      // first token, head inside it
    auto token = [&](int r) { return t0 + div_group(P, in0 + r); };
    const int i0 = c.R.pos0 + t0, i1 = c.R.pos0 + token(c.rows - 1);
    c.runs = unit_runs<kFewBlock, false>(P.pred, i0, i1, c.R.len, kFewBlock);
    const int nblk = run_blocks<kFewBlock>(c.runs);
    c.blk0 = fresh ? min(first.blk, nblk) : 0;
    c.blk1 = last ? min(end.blk, nblk) : nblk;
    // an earlier worker has begun it, or a later one ends it: a partial result
    c.slot = nullptr;
    if (fresh && first.blk > 0) c.slot = scratch + (size_t)(2 * w) * slot_floats<D>(kFewRows);
    else if (last) c.slot = scratch + (size_t)(2 * w + 1) * slot_floats<D>(kFewRows);
    fresh = false;

    // q fragments: rows g and g + 8
    uint32_t qa[D / 16][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = min(g + half * 8, c.rows - 1), t = token(r);
      const uint16_t* qp = static_cast<const uint16_t*>(P.q) + (long long)(c.R.row0 + t) * P.q_t +
                           (long long)(c.h * G + c.row0 + r - t * G) * P.q_h + tq * 2;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qa[kk][half] = *reinterpret_cast<const uint32_t*>(qp + kk * 16);
        qa[kk][half + 2] = *reinterpret_cast<const uint32_t*>(qp + kk * 16 + 8);
      }
    }
    const int ig = c.R.pos0 + token(min(g, c.rows - 1));
    const int ig8 = c.R.pos0 + token(min(g + 8, c.rows - 1));

    const uint16_t* kh = static_cast<const uint16_t*>(P.k) + (long long)c.h * P.k_h;
    const uint16_t* vh = static_cast<const uint16_t*>(P.v) + (long long)c.h * P.v_h;
    const int32_t* trow = P.table + (long long)c.b * P.table_stride;

    // Page of block blk, read a block ahead of its rows: a block of consecutive keys starts
    // at a multiple of 16 and lies in one page; of a lattice every lane reads its own key's.
    auto page_of = [&](int blk) -> int {
      if (blk >= c.blk1) return -1;
      const BlockKeys k = block_keys<kFewBlock>(c.runs, blk);
      if (k.step == 1) return __ldg(trow + (k.j0 >> P.page_shift));
      const int x = lane & 15;
      return x < k.hi ? __ldg(trow + ((k.j0 + x * k.step) >> P.page_shift)) : -1;
    };
    // issue the copies of block blk into its stage; rows that are not listed become 0
    constexpr int kChunks = D / 8;                 // 16-byte chunks of a row
    constexpr int kPer = 32 / kChunks;             // rows per warp-wide copy
    const int cx = lane % kChunks, rx = lane / kChunks;
    auto load = [&](int blk, int page) {
      if (blk < c.blk1) {
        const int st = (blk - c.blk0) % S;
        const BlockKeys k = block_keys<kFewBlock>(c.runs, blk);
        const uint32_t dk = ring + st * 2 * F::kTile + rx * F::kRowBytes, dv = dk + F::kTile;
        const bool ok = (unsigned)page < (unsigned)P.pages;
        uint32_t live;
        if (k.step == 1) {
          live = ok ? ((1u << k.hi) - 1u) & ~((1u << k.lo) - 1u) : 0u;
          const int row = (k.j0 & mask) + rx;
          const uint16_t* kp = kh + (ok ? page * P.k_p + row * P.k_r : 0) + cx * 8;
          const uint16_t* vp = vh + (ok ? page * P.v_p + row * P.v_r : 0) + cx * 8;
#pragma unroll
          for (int i = 0; i < kFewBlock / kPer; ++i) {
            const int r = i * kPer + rx;
            const int bytes = (live >> r) & 1 ? 16 : 0;
            const uint32_t d = i * kPer * F::kRowBytes + ((cx ^ (r & 7)) << 4);
            cp16(dk + d, kp, bytes);
            cp16(dv + d, vp, bytes);
            kp += kPer * P.k_r;
            vp += kPer * P.v_r;
          }
        } else {
          live = __ballot_sync(0xffffffffu, ok) & 0xffffu;
          const int j = k.j0 + (lane & 15) * k.step;
          const long long ko = ok ? page * P.k_p + (j & mask) * P.k_r : 0;
          const long long vo = ok ? page * P.v_p + (j & mask) * P.v_r : 0;
#pragma unroll 2
          for (int i = 0; i < kFewBlock / kPer; ++i) {
            const int r = i * kPer + rx;
            const long long a = __shfl_sync(0xffffffffu, ko, r), b = __shfl_sync(0xffffffffu, vo, r);
            const int bytes = (live >> r) & 1 ? 16 : 0;
            const uint32_t d = i * kPer * F::kRowBytes + ((cx ^ (r & 7)) << 4);
            cp16(dk + d, kh + a + cx * 8, bytes);
            cp16(dv + d, vh + b + cx * 8, bytes);
          }
        }
        if (lane == 0) s_live[st] = live;
      }
      cp_commit();
    };

    float acc[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    int page = page_of(c.blk0);
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
      const int next = page_of(c.blk0 + s + 1);
      load(c.blk0 + s, page);
      page = next;
    }
#pragma unroll 1
    for (int blk = c.blk0; blk < c.blk1; ++blk) {
      const int next = page_of(blk + S);
      cp_wait<S - 2>();
      __syncwarp();
      const int st = (blk - c.blk0) % S;
      const uint32_t sk = ring + st * 2 * F::kTile, sv = sk + F::kTile;
      const uint32_t live = s_live[st];
      const BlockKeys k = block_keys<kFewBlock>(c.runs, blk);

      // two sums of D / 2 products each, so that half as many wait for one another
      float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
      float u0[4] = {0.f, 0.f, 0.f, 0.f}, u1[4] = {0.f, 0.f, 0.f, 0.f};
      {
        // matrices: keys 0-7 and 8-15 by the two 16-byte halves of 16 columns
        const int r = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
        const uint32_t base = sk + r * F::kRowBytes;
#pragma unroll
        for (int kk = 0; kk < D / 16; kk += 2) {
          uint32_t b[4], b2[4];
          ldm4(base + (((kk * 2 + half) ^ (r & 7)) << 4), b);
          ldm4(base + (((kk * 2 + 2 + half) ^ (r & 7)) << 4), b2);
          mma16816<kBf16>(s0, qa[kk], b[0], b[1]);
          mma16816<kBf16>(s1, qa[kk], b[2], b[3]);
          mma16816<kBf16>(u0, qa[kk + 1], b2[0], b2[1]);
          mma16816<kBf16>(u1, qa[kk + 1], b2[2], b2[3]);
        }
      }
      // the next copies go into the stage that the last round has read, while the products run
      load(blk + S - 1, page);
      page = next;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s0[e] += u0[e];
        s1[e] += u1[e];
      }
      // this lane's keys: places 2 tq, 2 tq + 1, 8 + 2 tq, 9 + 2 tq; rows g (0, 1) and g + 8 (2, 3)
      float x[2][4] = {{s0[0], s0[1], s1[0], s1[1]}, {s0[2], s0[3], s1[2], s1[3]}};
      const int jl = k.j0 + 15 * k.step;
      const bool all = live == 0xffffu &&
                       (c.runs.exact || (jl <= i0 && (P.pred.kind == PA_CAUSAL ||
                                                 ((P.pred.kind == PA_WINDOW || P.pred.kind == PA_SINKS) &&
                                                  i1 - k.j0 < P.pred.p0))));
      if (!all) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int place = 2 * tq + (e & 1) + (e >> 1) * 8;
          const bool listed = (live >> place) & 1;
          const int j = k.j0 + place * k.step;
          if (!(listed && (c.runs.exact || pred_live(P.pred, ig, j)))) x[0][e] = -INFINITY;
          if (!(listed && (c.runs.exact || pred_live(P.pred, ig8, j)))) x[1][e] = -INFINITY;
        }
      }
      float t0 = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3]));
      float t1 = fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3]));
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2)) * P.scale_log2;
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2)) * P.scale_log2;
      // the maximum that is subtracted moves only when it has grown by more than 2^8
      const bool up = t0 > m0 + 8.f || t1 > m1 + 8.f;
      if (__any_sync(0xffffffffu, up)) {
        const float n0 = t0 > m0 + 8.f ? t0 : m0, n1 = t1 > m1 + 8.f ? t1 : m1;
        const float f0 = n0 == m0 ? 1.f : ex2f(m0 - n0), f1 = n1 == m1 ? 1.f : ex2f(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          acc[n][0] *= f0;
          acc[n][1] *= f0;
          acc[n][2] *= f1;
          acc[n][3] *= f1;
        }
      }
      const float z0 = m0 == -INFINITY ? 0.f : m0, z1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[0][e] = ex2f(fmaf(x[0][e], P.scale_log2, -z0));
        x[1][e] = ex2f(fmaf(x[1][e], P.scale_log2, -z1));
      }
      l0 += (x[0][0] + x[0][1]) + (x[0][2] + x[0][3]);
      l1 += (x[1][0] + x[1][1]) + (x[1][2] + x[1][3]);
      const uint32_t pa_[4] = {pack_pair<kBf16>(x[0][0], x[0][1]), pack_pair<kBf16>(x[1][0], x[1][1]),
                               pack_pair<kBf16>(x[0][2], x[0][3]), pack_pair<kBf16>(x[1][2], x[1][3])};
      {
        const int r = lane & 15, half = lane >> 4;
        const uint32_t base = sv + r * F::kRowBytes;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          uint32_t b[4];
          ldm4t(base + (((n * 2 + half) ^ (r & 7)) << 4), b);
          mma16816<kBf16>(acc[2 * n], pa_, b[0], b[1]);
          mma16816<kBf16>(acc[2 * n + 1], pa_, b[2], b[3]);
        }
      }
      __syncwarp();                   // the stage may be filled again
    }
    cp_wait<0>();
    __syncwarp();

    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    // a value that is not finite, seen or weighed by 0: key by key instead
    float probe = 0.f;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      probe += (acc[n][0] - acc[n][0]) + (acc[n][1] - acc[n][1]) + (acc[n][2] - acc[n][2]) +
               (acc[n][3] - acc[n][3]);
    if (__any_sync(0xffffffffu, probe != 0.f)) {
      piece_by_key<D, kBf16>(P, c);
    } else {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = g + half * 8;
        if (r >= c.rows) continue;
        const float m = half ? m1 : m0, l = half ? l1 : l0;
        if (c.slot) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(c.slot + r * D + n * 8 + tq * 2) =
                make_float2(acc[n][2 * half], acc[n][2 * half + 1]);
          if (tq == 0)
            *reinterpret_cast<float2*>(c.slot + kFewRows * D + 2 * r) = make_float2(m, l);
        } else {
          const int tk = token(r), t = c.R.row0 + tk, a = c.h * G + c.row0 + r - tk * G;
          const float inv = l > 0.f ? 1.f / l : 0.f;
          uint16_t* o = static_cast<uint16_t*>(P.o) + (long long)t * P.o_t + (long long)a * P.o_h + tq * 2;
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<uint32_t*>(o + n * 8) =
                pack_pair<kBf16>(acc[n][2 * half] * inv, acc[n][2 * half + 1] * inv);
          if (P.lse && tq == 0)
            P.lse[a * P.lse_h + t] = l > 0.f ? (m + log2f(l)) * 0.69314718055994530942f : -INFINITY;
        }
      }
    }
    if (last) break;
    ++at.t;
  }
}

}  // namespace

namespace {
template <int D, bool kBf16>
int launch_few_body(const Params& P, const PlanView& pv, const Config& c, float* scratch, int sms,
                    cudaStream_t stream) {
  const int rc = prepare_kernel<paged_few_kernel<D, kBf16>>("pa_paged_attn", Few<D>::kBytes, 0);
  if (rc) return rc;
  return launch_after("pa_paged_attn", paged_few_kernel<D, kBf16>, sms, kFewWarps * 32, Few<D>::kBytes,
                      stream, P, pv.shares, pv.meta, scratch,
                      c.split ? nullptr : pv.status);
}
}  // namespace

int launch_few(const Params& P, bool bf16, int D, const PlanView& pv, const Config& c,
               float* scratch, int sms, cudaStream_t stream) {
  if (D == 128)
    return bf16 ? launch_few_body<128, true>(P, pv, c, scratch, sms, stream)
                : launch_few_body<128, false>(P, pv, c, scratch, sms, stream);
  return bf16 ? launch_few_body<64, true>(P, pv, c, scratch, sms, stream)
              : launch_few_body<64, false>(P, pv, c, scratch, sms, stream);
}

}  // namespace paged
}  // namespace pa
