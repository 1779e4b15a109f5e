// Attention of chunks of new tokens over a paged K/V cache, on the 5th-generation tensor
// cores.
//
// A unit is 256 query rows of one request and key head -- tokens in order, the query heads
// that share the key head inside a token -- as two halves of 128 rows that share one
// stream of 128-key super-tiles, so a row of K and V is read once for 256 / group tokens
// and the work is bound by the matrix products and the exponentials.  A CTA (one per
// multiprocessor) works through its share of the step's units and super-tiles:
//
//   warp 8       copies: Q tiles, and for each super-tile its pages of K and V, one TMA box
//                of min(page, 128) rows each, into a ring of 128-row slots;
//   warp 9       matrix products: S = Q K^T and O += P V of each half in turn, so that one
//                half's softmax runs under the other half's products;
//   warps 0-3    softmax of half 0 (a thread per row), warps 4-7 of half 1: S comes from
//                and P (16-bit) goes to tensor memory, two 64-key parts, the product of the
//                first running while the second is still exponentiated; the running
//                maximum is moved, and O rescaled, only when it has grown by more than 2^8;
//   warps 10-11  complete the third warpgroup, so that registers can move to the softmax.
//
// Masks cost nothing on super-tiles that every row of a half sees whole (a uniform test);
// on the others each row has its live bits from the framework's closed forms.  The cache
// rows behind a request's last token are never read: the page's box starts that many rows
// early, so they fall off its end and rows before the page (out of bounds: zeros) come in
// front, and the mask follows the shift.
#pragma once
#include "attn_kernel.cuh"
#include "paged.cuh"

namespace pa {
namespace paged {

constexpr int kChunkThreads = 384;
constexpr int kChunkLoadWarp = 8;
constexpr int kChunkMmaWarp = 9;
constexpr int kChunkSoftRegs = 200;    // 256 x 200 + 128 x 104 = 384 x 168 launch registers
constexpr int kChunkOtherRegs = 104;

struct ChunkParams {
  Params p;
  int tb;                 // tokens per half: 128 / group
  int seg, nseg;          // rows of a page's box, boxes per super-tile
  uint32_t idesc_qk, idesc_pv;
  ErrSink err;
};

// A piece of a unit, handed from the copying warp to the others.
struct ChunkUnit {
  int b, h;               // b < 0: no more
  int row0, n;            // first token's row of q, tokens of the unit
  int pos0, len;          // its position; tokens of the request
  int blk0, blk1;         // super-tiles of this piece
  int slot;               // partial result, or -1
  Runs runs;
};

template <int D>
struct ChunkSmem {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kSlots = D == 128 ? 4 : 8;
  static constexpr int kKVOff = 2 * kTile;
  static constexpr int kEpiOff = kKVOff + kSlots * kTile;            // 8 warps x 32 rows x 128 bytes
  static constexpr int kBarOff = kEpiOff + 8 * 32 * 128;
  // q_full[2] q_empty[2] s_full[2] pa_full[2] pb_full[2] o_full[2] drain unit_full[2]
  // unit_empty[2] kv_full[S] kv_empty[S]
  static constexpr int kNumBars = 17 + 2 * kSlots;
  static constexpr int kMiscOff = kBarOff + 8 * kNumBars;
  static constexpr int kUnitOff = (kMiscOff + 16 + 15) & ~15;
  static constexpr int kBytes = kUnitOff + 2 * (int)sizeof(ChunkUnit);
  static constexpr int kAlloc = kBytes + 1024;
  static_assert(kAlloc <= 232448, "shared memory of one CTA");
};

// 2^x for two values on the FMA and integer pipes: j = rint(x) by adding 1.5 * 2^23, 2^(x - j)
// by a degree-4 polynomial fitted for least maximum relative error on [-1/2, 1/2] (2.7e-6 in
// 32 bits), 2^j by its exponent field.  x <= 127; below -127, -inf too, the scale is 0.
__device__ __forceinline__ void exp2_poly(float x0, float x1, float& y0, float& y1) {
  constexpr float kRound = 12582912.0f;
  x0 = fmaxf(x0, -127.0f);
  x1 = fmaxf(x1, -127.0f);
  float t0, t1, j0, j1, f0, f1, p0, p1;
  attn::fma2v(t0, t1, x0, x1, 1.0f, 1.0f, kRound, kRound);
  attn::fma2v(j0, j1, t0, t1, 1.0f, 1.0f, -kRound, -kRound);
  attn::fma2v(f0, f1, j0, j1, -1.0f, -1.0f, x0, x1);
  attn::fma2v(p0, p1, f0, f1, 0.0095701022f, 0.0095701022f, 0.0559178629f, 0.0559178629f);
  attn::fma2v(p0, p1, p0, p1, f0, f1, 0.2402474433f, 0.2402474433f);
  attn::fma2v(p0, p1, p0, p1, f0, f1, 0.6931217909f, 0.6931217909f);
  attn::fma2v(p0, p1, p0, p1, f0, f1, 0.9999992847f, 0.9999992847f);
  const float s0 = __uint_as_float(__float_as_uint(t0) * 8388608u + 0x3F800000u);
  const float s1 = __uint_as_float(__float_as_uint(t1) * 8388608u + 0x3F800000u);
  attn::fma2v(y0, y1, p0, p1, s0, s1, 0.0f, 0.0f);
}

// Pairs, of the 16 of each 32 columns, whose exponentials run on the FMA pipe.
template <int D>
__device__ __forceinline__ constexpr bool on_fma(int pair) {
  return false;
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kChunkThreads, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ ChunkParams C,
                   const Share* __restrict__ shares, const int32_t* __restrict__ meta,
                   float* __restrict__ scratch) {
  using SM = ChunkSmem<D>;
  constexpr int NS = SM::kSlots;
  constexpr int kParts = D / 64;             // 128-byte columns of a row
  constexpr uint32_t kRegion = 128 * 128;    // one such column of a 128-row tile
  const Params& P = C.p;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + SM::kKVOff;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::kBarOff);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 2;
  uint64_t* s_full = bars + 4;
  uint64_t* pa_full = bars + 6;
  uint64_t* pb_full = bars + 8;
  uint64_t* o_full = bars + 10;
  uint64_t* drain = bars + 12;
  uint64_t* unit_full = bars + 13;
  uint64_t* unit_empty = bars + 15;
  uint64_t* kv_full = bars + 17;
  uint64_t* kv_empty = bars + 17 + NS;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + SM::kMiscOff);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + SM::kMiscOff + 4);
  int* s_slow = reinterpret_cast<int*>(smem + SM::kMiscOff + 8);   // warps going key by key
  ChunkUnit* s_unit = reinterpret_cast<ChunkUnit*>(smem + SM::kUnitOff);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const ErrSink& err = C.err;
  // A bounded wait (mbar_wait); the time in which a warp goes key by key does not count.
  auto wait_bar = [&](uint64_t* bar, uint32_t parity, int32_t code) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    uint64_t t0 = globaltimer();
    while (true) {
      if (mbar_try_wait(bar, parity)) return true;
      if (*s_abort) return false;
      if (globaltimer() - t0 > err.limit_ns) {
        if (*static_cast<volatile int*>(s_slow) > 0) {
          t0 = globaltimer();
          continue;
        }
        *s_abort = 1;
        err.record(code);
        return false;
      }
    }
  };
  asm volatile("griddepcontrol.launch_dependents;");
  if ((int)blockIdx.x >= __ldg(meta)) return;   // no share: the whole CTA leaves

  if (threadIdx.x == 0) {
    for (int h = 0; h < 2; ++h) {
      mbar_init(&q_full[h], 1);
      mbar_init(&q_empty[h], 1);
      mbar_init(&s_full[h], 1);
      mbar_init(&pa_full[h], 128);
      mbar_init(&pb_full[h], 128);
      mbar_init(&o_full[h], 1);
      mbar_init(&unit_full[h], 1);
      mbar_init(&unit_empty[h], 9);          // the issuing thread and a lane per softmax warp
    }
    mbar_init(drain, 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    *s_abort = 0;
    *s_slow = 0;
    fence_barrier_init();
  }
  // rows of the Q tiles that no box fills (128 is no multiple of the group) stay 0
  for (int x = threadIdx.x; x < 2 * SM::kTile / 16; x += kChunkThreads)
    reinterpret_cast<uint4*>(sQ)[x] = make_uint4(0u, 0u, 0u, 0u);
  fence_proxy_async_shared();
  if (warp == kChunkLoadWarp && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (warp == kChunkMmaWarp) {
    tmem_alloc(s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kChunkOtherRegs));
    if (warp == kChunkLoadWarp) {
      // ---------------------------------------------------------------- copies
      const int w = blockIdx.x;
      const Share first = shares[w], end = shares[w + 1];
      const int per = 2 * C.tb;              // tokens of a unit
      Share at = first;
      bool fresh = true;
      uint32_t ring = 0, kv_g = 0;
      int q_armed[2] = {0, 0};
      int ok = 1;
      while (ok) {
        // the next piece
        ChunkUnit u;
        u.b = -1;
        while (true) {
          if (at.b >= P.requests || at.b > end.b ||
              (at.b == end.b && (at.h > end.h || (at.h == end.h && at.t > end.t))))
            break;
          const Request R = get_request(P, at.b);
          if (at.t * per >= R.n) {
            at.t = 0;
            if (R.n == 0 || ++at.h == P.kv_heads) {
              at.h = 0;
              ++at.b;
            }
            continue;
          }
          const bool last = at.b == end.b && at.h == end.h && at.t == end.t;
          if (last && end.blk == 0) break;
          u.b = at.b;
          u.h = at.h;
          u.row0 = R.row0 + at.t * per;
          u.n = min(R.n - at.t * per, per);
          u.pos0 = R.pos0 + at.t * per;
          u.len = R.len;
          u.runs = unit_runs<128, true>(P.pred, u.pos0, u.pos0 + u.n - 1, u.len);
          const int nblk = run_blocks<128>(u.runs);
          u.blk0 = fresh ? min(first.blk, nblk) : 0;
          u.blk1 = last ? min(end.blk, nblk) : nblk;
          u.slot = fresh && first.blk > 0 ? 2 * w : last ? 2 * w + 1 : -1;
          fresh = false;
          ++at.t;
          break;
        }
        const uint32_t rs = ring & 1;
        if (lane == 0) {
          if (ring >= 2 && !wait_bar(&unit_empty[rs], ((ring >> 1) - 1) & 1, DEV_TIMEOUT_ITEM)) {
            ok = 0;
          } else {
            if (*s_abort) u.b = -1;
            s_unit[rs] = u;
            mbar_arrive(&unit_full[rs]);
          }
        }
        ++ring;
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok || __shfl_sync(0xffffffffu, u.b, 0) < 0) break;
        if (u.blk1 <= u.blk0) continue;
        const int halves = u.n > C.tb ? 2 : 1;
        if (lane == 0) {
          for (int h = 0; h < halves && ok; ++h) {
            if (q_armed[h] > 0 &&
                !wait_bar(&q_empty[h], (q_armed[h] - 1) & 1, DEV_TIMEOUT_Q)) {
              ok = 0;
              break;
            }
            mbar_arrive_expect_tx(&q_full[h], C.tb * P.group * D * 2);
            ++q_armed[h];
            for (int c = 0; c < kParts; ++c)
              tma_load_4d(sQ + h * SM::kTile + c * kRegion, &tm_q, &q_full[h], c * 64, 0, u.h,
                          u.row0 + h * C.tb);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        // lane x < nseg copies box x of every super-tile; its page is read one ahead
        const int32_t* trow = P.table + (long long)u.b * P.table_stride;
        const int n0 = (u.runs.cnt[0] + 127) / 128;
        auto key_of = [&](int blk) {
          const int part = blk >= n0;
          return u.runs.a[part] + (blk - (part ? n0 : 0)) * 128 + lane * C.seg;
        };
        auto page_of = [&](int blk) -> int {
          if (blk >= u.blk1 || lane >= C.nseg) return P.pages;
          const int j = key_of(blk);
          if (j >= u.len) return P.pages;              // out of bounds: the box reads zeros
          const int page = __ldg(trow + (j >> P.page_shift));
          return (unsigned)page < (unsigned)P.pages ? page : P.pages;
        };
        int page = page_of(u.blk0);
        for (int blk = u.blk0; blk < u.blk1 && ok; ++blk) {
          const int next = page_of(blk + 1);
          const int j = key_of(blk);
          int row = j & ((1 << P.page_shift) - 1);
          if (u.len - j < C.seg) row -= C.seg - max(u.len - j, 0);   // the last page's end
          if (page == P.pages) row = 0;
          for (int kv = 0; kv < 2; ++kv) {
            const uint32_t slot = kv_g % NS;
            if (lane == 0) {
              if (kv_g >= (uint32_t)NS &&
                  !wait_bar(&kv_empty[slot], ((kv_g / NS) - 1) & 1, DEV_TIMEOUT_KV))
                ok = 0;
              else
                mbar_arrive_expect_tx(&kv_full[slot], SM::kTile);
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            ++kv_g;
            if (lane < C.nseg) {
              uint8_t* dst = sKV + slot * SM::kTile + lane * C.seg * 128;
              const void* tm = kv == 0 ? (const void*)&tm_k : (const void*)&tm_v;
              for (int c = 0; c < kParts; ++c)
                tma_load_4d(dst + c * kRegion, tm, &kv_full[slot], c * 64, row, u.h, page);
            }
            __syncwarp();
          }
          page = next;
        }
      }
      // every copy issued lands before the CTA can exit
      if (lane == 0) {
        const uint64_t t0 = globaltimer();
        for (uint32_t s = 0; s < (uint32_t)NS && s < kv_g; ++s) {
          const uint32_t uses = (kv_g - s + NS - 1) / NS;
          while (!mbar_try_wait(&kv_full[s], (uses - 1) & 1)) {
            if (globaltimer() - t0 > attn::kDrainLimitNs) { err.record(DEV_TIMEOUT_DRAIN); break; }
          }
        }
        for (int h = 0; h < 2; ++h) {
          if (q_armed[h] == 0) continue;
          while (!mbar_try_wait(&q_full[h], (q_armed[h] - 1) & 1)) {
            if (globaltimer() - t0 > attn::kDrainLimitNs) { err.record(DEV_TIMEOUT_DRAIN); break; }
          }
        }
      }
    } else if (warp == kChunkMmaWarp) {
      // ------------------------------------------------------------ matrix products
      if (lane == 0) {
        uint32_t ring = 0, kv_c = 0, tp[2] = {0, 0}, tq[2] = {0, 0};
        bool ok = true;
        const uint32_t sQa = smem_u32(sQ), sKVa = smem_u32(sKV);
        const uint64_t q_desc[2] = {smem_desc_sw128(sQa, 16), smem_desc_sw128(sQa + SM::kTile, 16)};
        auto wait_kv = [&](uint32_t& slot) -> bool {
          slot = kv_c % NS;
          const bool r = wait_bar(&kv_full[slot], (kv_c / NS) & 1, DEV_TIMEOUT_KV);
          ++kv_c;
          tc_fence_after();
          return r;
        };
        auto issue_s = [&](int h, uint32_t kslot) {
          const uint64_t kd = smem_desc_sw128(sKVa + kslot * SM::kTile, 16);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t off = ((kk >> 2) * kRegion + (kk & 3) * 32) >> 4;
            mma_ss(tmem + h * 128, q_desc[h] + off, kd + off, C.idesc_qk, kk > 0);
          }
          tc_commit(&s_full[h]);
        };
        // O += P V of half h: the first 64 keys as soon as their P is there
        auto issue_pv = [&](int h, uint32_t vslot, bool acc) -> bool {
          const uint32_t d = tmem + 256 + h * D, p = tmem + h * 128 + 64;
          const uint64_t vd = smem_desc_sw128(sKVa + vslot * SM::kTile, kRegion);
          if (!wait_bar(&pa_full[h], tp[h] & 1, DEV_TIMEOUT_P)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ts(d, p + kk * 8, vd + (uint64_t)((kk * 16 * 128) >> 4), C.idesc_pv,
                   (acc || kk > 0) ? 1u : 0u);
          if (!wait_bar(&pb_full[h], tp[h] & 1, DEV_TIMEOUT_P)) return false;
          ++tp[h];
          tc_fence_after();
#pragma unroll
          for (int kk = 4; kk < 8; ++kk)
            mma_ts(d, p + kk * 8, vd + (uint64_t)((kk * 16 * 128) >> 4), C.idesc_pv, 1u);
          return true;
        };
        while (ok) {
          const uint32_t rs = ring & 1;
          if (!(ok = wait_bar(&unit_full[rs], (ring >> 1) & 1, DEV_TIMEOUT_ITEM)))
            break;
          const int b = s_unit[rs].b, n = s_unit[rs].n, tiles = s_unit[rs].blk1 - s_unit[rs].blk0;
          mbar_arrive(&unit_empty[rs]);
          ++ring;
          if (b < 0) break;
          if (tiles <= 0) continue;
          const int halves = n > C.tb ? 2 : 1;
          for (int h = 0; h < halves && ok; ++h)
            ok = wait_bar(&q_full[h], tq[h]++ & 1, DEV_TIMEOUT_Q);
          tc_fence_after();
          uint32_t ks, vs;
          if (!ok || !(ok = wait_kv(ks))) break;
          for (int h = 0; h < halves; ++h) issue_s(h, ks);
          tc_commit(&kv_empty[ks]);
          for (int u = 1; u < tiles && ok; ++u) {
            if (!(ok = wait_kv(vs)) || !(ok = wait_kv(ks))) break;
            for (int h = 0; h < halves; ++h) {
              if (!(ok = issue_pv(h, vs, u > 1))) break;
              issue_s(h, ks);
            }
            tc_commit(&kv_empty[vs]);
            tc_commit(&kv_empty[ks]);
          }
          if (!ok) break;
          for (int h = 0; h < halves; ++h) tc_commit(&q_empty[h]);
          if (!(ok = wait_kv(vs))) break;
          for (int h = 0; h < halves; ++h) {
            if (!(ok = issue_pv(h, vs, tiles > 1))) break;
            tc_commit(&o_full[h]);
          }
          tc_commit(&kv_empty[vs]);
        }
        // the commit lands once every product issued above has completed
        tc_commit(drain);
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(drain, 0)) {
          if (globaltimer() - t0 > attn::kDrainLimitNs) { err.record(DEV_TIMEOUT_DRAIN); break; }
        }
      }
    }
  } else {
    // -------------------------------------------------------------- softmax, results
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kChunkSoftRegs));
    const int h = warp >> 2, wq = warp & 3;
    const int r_in = wq * 32 + lane;                 // row of the half
    const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
    const uint32_t tS = tmem + lane_off + h * 128;
    const uint32_t tO = tmem + lane_off + 256 + h * D;
    uint8_t* stage = smem + SM::kEpiOff + warp * (32 * 128);
    const float c2 = P.scale_log2;
    const int tok = r_in / P.group;                  // token of the half
    const int qh = r_in - tok * P.group;             // query head of the group
    uint32_t ring = 0, ts = 0, to = 0;
    while (true) {
      const uint32_t rs = ring & 1;
      bool ok = wait_bar(&unit_full[rs], (ring >> 1) & 1, DEV_TIMEOUT_ITEM);
      if (!__all_sync(0xffffffffu, ok)) break;
      const ChunkUnit& u = s_unit[rs];                // held until the unit is done
      ++ring;
      if (u.b < 0) break;
      if (h * C.tb >= u.n) {                         // no row in this half
        __syncwarp();
        if (lane == 0) mbar_arrive(&unit_empty[rs]);
        continue;
      }
      const int t_in = h * C.tb + tok;               // token of the unit
      const bool valid = tok < C.tb && t_in < u.n;
      const int i = u.pos0 + t_in;
      const int i_lo = u.pos0 + h * C.tb, i_hi = u.pos0 + min(u.n, (h + 1) * C.tb) - 1;
      const int32_t* trow = P.table + (long long)u.b * P.table_stride;
      const int n0 = (u.runs.cnt[0] + 127) / 128;
      auto base_of = [&](int blk) {
        const int part = blk >= n0;
        return (part ? u.runs.a[1] : u.runs.a[0]) + (blk - (part ? n0 : 0)) * 128;
      };
      // bit x: box x of the super-tile has keys
      auto boxes_of = [&](int blk) -> bool {
        if (blk >= u.blk1 || lane >= C.nseg) return false;
        const int j = base_of(blk) + lane * C.seg;
        return j < u.len && (unsigned)__ldg(trow + (j >> P.page_shift)) < (unsigned)P.pages;
      };
      bool box = boxes_of(u.blk0);
      float m_used = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int blk = u.blk0; blk < u.blk1; ++blk) {
        const uint32_t boxes = __ballot_sync(0xffffffffu, box);
        box = boxes_of(blk + 1);
        const int kb = base_of(blk);
        const bool whole = kb + 128 <= u.len && boxes == (1u << C.nseg) - 1u;
        const bool full = whole && kb + 127 <= i_lo &&
                          (P.pred.kind == PA_CAUSAL ||
                           ((P.pred.kind == PA_WINDOW || P.pred.kind == PA_SINKS) &&
                            i_hi - kb < P.pred.p0));
        uint32_t mk[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (!full) {
          // live bits of this row, box by box (a word of 32 keys at most)
          const int width = min(C.seg, 32);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t word = 0;
#pragma unroll 1
            for (int c0 = k * 32; c0 < k * 32 + 32; c0 += width) {
              const int sg = c0 / C.seg, in = c0 - sg * C.seg;
              if (!((boxes >> sg) & 1u)) continue;
              const int j = kb + sg * C.seg;
              const int shift = max(C.seg - (u.len - j), 0);   // the last page's end
              uint32_t bits;
              if (!progression_bits(P.pred, i - (j - shift), j - shift, 1, 0, in, C.seg, bits))
                bits = element_bits(P.pred, i, nullptr, j - shift, 1, in, width);
              bits &= range_bits(shift, C.seg - 1, in);
              word |= bits << (c0 - k * 32);
            }
            mk[k] = word;
          }
        }
        ok = wait_bar(&s_full[h], ts & 1, DEV_TIMEOUT_S);
        ++ts;
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
        float s[128];
        {
          uint32_t r0[32], r1[32], r2[32], r3[32];
          tmem_ld32(tS + 0, r0);
          tmem_ld32(tS + 32, r1);
          tmem_ld32(tS + 64, r2);
          tmem_ld32(tS + 96, r3);
          tmem_wait_ld();
          tmem_regs_ready(r0);
          tmem_regs_ready(r1);
          tmem_regs_ready(r2);
          tmem_regs_ready(r3);
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            s[x] = __uint_as_float(r0[x]);
            s[32 + x] = __uint_as_float(r1[x]);
            s[64 + x] = __uint_as_float(r2[x]);
            s[96 + x] = __uint_as_float(r3[x]);
          }
        }
        if (!full) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (!((mk[k] >> x) & 1u)) s[k * 32 + x] = -INFINITY;
        }
        float mx;
        {
          float m8[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) m8[j] = fmaxf(s[2 * j], s[2 * j + 1]);
#pragma unroll
          for (int c = 16; c < 128; c += 16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) m8[j] = attn::fmax3(m8[j], s[c + 2 * j], s[c + 2 * j + 1]);
          }
          mx = attn::fmax3(attn::fmax3(m8[0], m8[1], m8[2]), attn::fmax3(m8[3], m8[4], m8[5]),
                           fmaxf(m8[6], m8[7]));
        }
        const float m_tile = mx * c2;
        const bool bump = m_tile > m_used + 8.0f;    // from -inf: the first live key
        float factor = 1.f;
        if (bump) {
          factor = ex2f(m_used - m_tile);
          m_used = m_tile;
          l *= factor;
        }
        if (__any_sync(0xffffffffu, bump && blk > u.blk0)) {
#pragma unroll 1
          for (int k = 0; k < D / 32; ++k) {
            uint32_t r[32];
            tmem_ld32(tO + k * 32, r);
            tmem_wait_ld();
            tmem_regs_ready(r);
#pragma unroll
            for (int x = 0; x < 32; ++x) r[x] = __float_as_uint(__uint_as_float(r[x]) * factor);
            tmem_st32(tO + k * 32, r);
          }
        }
        const float msub = m_used == -INFINITY ? 0.f : m_used;
        float r8[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r8[j] = 0.f;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          uint32_t pk[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const int c = q4 * 32 + 2 * x;
            float x0, x1, a, b;
            attn::ffma2(x0, x1, s[c], s[c + 1], c2, -msub);
            if (on_fma<D>(x)) {
              exp2_poly(x0, x1, a, b);
            } else {
              a = ex2f(x0);
              b = ex2f(x1);
            }
            const int j = (2 * x) & 7;
            attn::fadd2(r8[j], r8[j + 1], a, b);
            pk[x] = pack_pair<kBf16>(a, b);
          }
          tmem_st16(tS + 64 + q4 * 16, pk);
          if (q4 & 1) {
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(q4 == 1 ? &pa_full[h] : &pb_full[h]);
          }
        }
        l += ((r8[0] + r8[1]) + (r8[2] + r8[3])) + ((r8[4] + r8[5]) + (r8[6] + r8[7]));
      }
      if (!ok) break;

      // results: o and lse, or this piece's O, maximum and sum
      const bool any = u.blk1 > u.blk0;
      const int t = u.row0 + t_in, a = u.h * P.group + qh;
      float* part = u.slot >= 0 ? scratch + (size_t)u.slot * slot_floats<D>(256) : nullptr;
      const int rr = h * 128 + r_in;
      unsigned long long row_ptr = 0;
      if (valid)
        row_ptr = reinterpret_cast<unsigned long long>(
            part ? static_cast<void*>(part + (size_t)rr * D)
                 : static_cast<void*>(static_cast<uint16_t*>(P.o) + (long long)t * P.o_t +
                                      (long long)a * P.o_h));
      if (any) {
        ok = wait_bar(&o_full[h], to & 1, DEV_TIMEOUT_O);
        ++to;
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
      }
      const float inv_l = part ? 1.f : l > 0.f ? 1.f / l : 0.f;
      float probe = l - l;
      const int chunks = part ? D / 32 : D / 64;      // of 128 bytes of a row
#pragma unroll 1
      for (int c = 0; c < chunks; ++c) {
        __syncwarp();                                 // the last chunk has left the stage
        if (part) {
          uint32_t r[32];
          if (any) {
            tmem_ld32(tO + c * 32, r);
            tmem_wait_ld();
            tmem_regs_ready(r);
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) r[x] = 0u;
          }
#pragma unroll
          for (int x = 0; x < 32; ++x) probe += __uint_as_float(r[x]) - __uint_as_float(r[x]);
#pragma unroll
          for (int x = 0; x < 8; ++x)
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((x ^ (lane & 7)) << 4)) =
                make_uint4(r[4 * x], r[4 * x + 1], r[4 * x + 2], r[4 * x + 3]);
        } else {
          uint32_t r0[32], r1[32];
          if (any) {
            tmem_ld32(tO + c * 64, r0);
            tmem_ld32(tO + c * 64 + 32, r1);
            tmem_wait_ld();
            tmem_regs_ready(r0);
            tmem_regs_ready(r1);
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) r0[x] = r1[x] = 0u;
          }
#pragma unroll
          for (int x = 0; x < 32; ++x)
            probe += (__uint_as_float(r0[x]) - __uint_as_float(r0[x])) +
                     (__uint_as_float(r1[x]) - __uint_as_float(r1[x]));
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            uint32_t w4[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int col = 8 * (x & 3) + 2 * j;
              w4[j] = pack_pair<kBf16>(__uint_as_float(x < 4 ? r0[col] : r1[col]) * inv_l,
                                       __uint_as_float(x < 4 ? r0[col + 1] : r1[col + 1]) * inv_l);
            }
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((x ^ (lane & 7)) << 4)) =
                make_uint4(w4[0], w4[1], w4[2], w4[3]);
          }
        }
        __syncwarp();
        const int x = lane & 7;
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const int rw = it * 4 + (lane >> 3);
          const uint4 v = *reinterpret_cast<const uint4*>(stage + rw * 128 + ((x ^ (rw & 7)) << 4));
          const unsigned long long dst = __shfl_sync(0xffffffffu, row_ptr, rw);
          if (dst) *reinterpret_cast<uint4*>(reinterpret_cast<char*>(dst) + c * 128 + x * 16) = v;
        }
      }
      if (any) tc_fence_before();
      // a value that is not finite, seen or weighed by 0: those rows key by key instead
      uint32_t odd = __ballot_sync(0xffffffffu, valid && probe != 0.f);
      if (odd) {
        __syncwarp();
        if (lane == 0) atomicAdd(s_slow, 1);          // the other warps' waits hold on
      }
      const bool slow = odd != 0;
      for (; odd; odd &= odd - 1) {
        const int src = __ffs(odd) - 1;
        const int t2 = __shfl_sync(0xffffffffu, t, src), g2 = __shfl_sync(0xffffffffu, qh, src);
        const int i2 = __shfl_sync(0xffffffffu, i, src);
        const unsigned long long dst = __shfl_sync(0xffffffffu, row_ptr, src);
        float m2, l2, acc[D / 32];
        row_by_key<D, kBf16, 128>(P, u.b, u.h, t2, g2, i2, u.runs, u.blk0, u.blk1, m2, l2, acc);
        if (lane == src) {
          m_used = m2;
          l = l2;
        }
        const float inv = part ? 1.f : l2 == 0.f ? 0.f : 1.f / l2;
#pragma unroll
        for (int e = 0; e < D / 32; e += 2) {
          if (part) {
            float* d = reinterpret_cast<float*>(dst) + lane * (D / 32) + e;
            d[0] = acc[e];
            d[1] = acc[e + 1];
          } else {
            reinterpret_cast<uint32_t*>(dst)[lane * (D / 64) + e / 2] =
                pack_pair<kBf16>(acc[e] * inv, acc[e + 1] * inv);
          }
        }
      }
      if (slow && lane == 0) atomicSub(s_slow, 1);
      if (valid) {
        if (part)
          *reinterpret_cast<float2*>(part + (size_t)256 * D + 2 * rr) = make_float2(m_used, l);
        else if (P.lse)
          P.lse[a * P.lse_h + t] =
              l == 0.f ? -INFINITY : (m_used + log2f(l)) * 0.69314718055994530942f;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&unit_empty[rs]);
    }
  }

  // ------------------------------------------------------------------ teardown
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kChunkMmaWarp) tmem_dealloc(tmem, 512);
}

int launch_chunk_d128(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                      const ChunkParams& C, bool bf16, const PlanView& pv, float* scratch, int sms,
                      cudaStream_t stream);
int launch_chunk_d64(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                     const ChunkParams& C, bool bf16, const PlanView& pv, float* scratch, int sms,
                     cudaStream_t stream);

template <int D>
int launch_chunk_body(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                      const ChunkParams& C, bool bf16, const PlanView& pv, float* scratch, int sms,
                      cudaStream_t stream) {
  auto go = [&](auto kernel) -> int {
    PA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 ChunkSmem<D>::kAlloc), "pa_paged_attn");
    // the warpgroups' register shares must fit in the registers of the launch
    static std::atomic<int> regs_ok{0};
    cudaFuncAttributes fa;
    fa.numRegs = 1 << 20;
    if (!regs_ok.load(std::memory_order_relaxed))
      PA_CUDA(cudaFuncGetAttributes(&fa, kernel), "pa_paged_attn");
    if (fa.numRegs * kChunkThreads < 256 * kChunkSoftRegs + 128 * kChunkOtherRegs)
      return fail(PA_ERR_UNSUPPORTED, "pa_paged_attn: kernel built with %d registers per thread, "
                  "below its register split", fa.numRegs);
    regs_ok.store(1, std::memory_order_relaxed);
    kernel<<<sms, kChunkThreads, ChunkSmem<D>::kAlloc, stream>>>(tq, tk, tv, C, pv.shares, pv.meta,
                                                                 scratch);
    return check_launch("pa_paged_attn");
  };
  return bf16 ? go(paged_chunk_kernel<D, true>) : go(paged_chunk_kernel<D, false>);
}

}  // namespace paged
}  // namespace pa
