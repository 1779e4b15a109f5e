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
//                and P (16-bit) goes to tensor memory in two 64-key parts, the product of the
//                first running while the second is still exponentiated; the running
//                maximum is moved, and O rescaled, only when it has grown by more than 2^8;
//   warps 10-11  complete the third warpgroup, so that registers can move to the softmax.
//
// Masks cost nothing on super-tiles that every row of a half sees whole (a uniform test);
// on the others each row has its live bits from the framework's closed forms.  The cache
// rows behind a request's last token are never read: the page's box starts that many rows
// early, so they fall off its end and rows before the page (out of bounds: zeros) come in
// front, and the mask follows the shift.
//
// What bounds it: a half's chain per super-tile -- S read (100 cycles), its maximum (330),
// the exponentials and P (1400; 1024 are the exponential unit's alone), then P V of the
// second part and the next S (768 and the hand-overs) -- of which half runs under the other
// half's products.  4096 new tokens over 16384, 32 heads of 128 sharing 8 key heads: 1010-1060
// us in a short run, 1090-1140 in a long one = 1.09-1.22 PFLOP/s (of 1.64 measured for a
// library product in a burst, 1.40 sustained: like that one it runs into the power limit, at
// 1.55 GHz); tensor cores and exponential unit both 64 % busy.  8 chunks of 2000 under a window
// of 1024 and 4 sinks, a key head per query head: 450-501 us = 0.54-0.60 PFLOP/s of live products;
// a unit has 11 super-tiles, one of them for the 4 sinks, 4 of a half's 10 are partly masked
// and its first and last are the other half's, and between units nothing overlaps a half's
// last products, result and first scores (7 000 of its 45 000 cycles).  D = 64: no unit is
// saturated.  The same chain with half the products leaves 4096 over 16384 at 780 us = 0.79
// PFLOP/s (exponential unit 52 %, issue 53 %, tensor cores 35 % busy), and unit ends take their
// share where units are short: 8 chunks of 1000 over 2000 0.64 PFLOP/s, 24 ragged requests 96
// us = 0.48 PFLOP/s (43, 47 and 28 %).
#pragma once
#include <type_traits>
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
  int o32;                // rows of o are 32-byte aligned
  int check;              // compare the plan's lengths
  uint32_t idesc_qk, idesc_pv;
  int withhold_q;         // test hook: the Q tiles of half 0 are never loaded
  uint64_t q_limit_ns;    // limit of the waits for Q tiles
  ErrSink err;            // status word, limit of all other waits
};

// What decides, for one half of a unit, the kind of the super-tile at key kb: some row sees
// some of it when kb <= i_hi and (kb >= live_min or kb < sink_end); every row sees all of it
// when full_min <= kb <= full_max and all its boxes have keys.
struct __align__(16) HalfTiles {
  int i_hi, live_min, full_min, full_max;
};

// A piece of a unit, handed from the copying warp to the others.
struct __align__(16) ChunkUnit {
  HalfTiles half[2];
  int a0, a1, n0, sink_end;       // super-tile blk: a0 + 128 blk, from n0 on a1 + 128 (blk - n0)
  const int32_t* table;           // the request's row of the block table
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
  static constexpr int kSlots = D == 128 ? 5 : 10;
  static constexpr int kKVOff = 2 * kTile;
  static constexpr int kBarOff = kKVOff + kSlots * kTile;
  // q_full[2] q_empty[2] s_full[2] pa_full[2] pb_full[2] o_full[2] drain unit_full[2]
  // unit_empty[2] kv_full[S] kv_empty[S]
  static constexpr int kNumBars = 17 + 2 * kSlots;
  static constexpr int kMiscOff = kBarOff + 8 * kNumBars;
  static constexpr int kUnitOff = (kMiscOff + 16 + 15) & ~15;
  static constexpr int kBytes = kUnitOff + 2 * (int)sizeof(ChunkUnit);
  static constexpr int kAlloc = kBytes + 1024;
  static_assert(kAlloc <= 232448, "shared memory of one CTA");
};

__device__ __forceinline__ HalfTiles half_tiles(const Pred& p, int i_lo, int i_hi, int len) {
  const bool window = p.kind == PA_WINDOW || p.kind == PA_SINKS;
  HalfTiles t;
  t.i_hi = i_hi;
  t.live_min = window ? i_lo - p.p0 - 126 : INT32_MIN;
  t.full_min = window ? i_hi - p.p0 + 1 : p.kind == PA_CAUSAL ? 0 : INT32_MAX;
  t.full_max = min(i_lo - 127, len - 128);
  return t;
}
__device__ __forceinline__ bool tile_live(const HalfTiles& t, int kb, int sink_end) {
  return kb <= t.i_hi && (kb >= t.live_min || kb < sink_end);
}
// 16 bytes of shared memory, read where it is written and kept no longer: the softmax
// threads have no register to spare, and a spilled one costs a trip to L2 (their local
// memory does not fit what shared memory leaves of L1).
__device__ __forceinline__ int4 lds4(const void* p) {
  int4 v;
  asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem_u32(p)));
  return v;
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32"
      " {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// 32 bytes to global memory, at once where the address is a multiple of 32.
__device__ __forceinline__ void st32(void* p, bool whole, uint32_t a, uint32_t b, uint32_t c,
                                     uint32_t d, uint32_t e, uint32_t f, uint32_t g, uint32_t h) {
  if (whole) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e), "r"(f), "r"(g), "r"(h) : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(a, b, c, d);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(e, f, g, h);
  }
}

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(r));
  return r != 0;
}

// 2^x for two values on the FMA and integer pipes: j = rint(x) by adding 1.5 * 2^23, 2^(x - j)
// by a degree-4 polynomial fitted for least maximum relative error on [-1/2, 1/2] (2.7e-6 in
// 32 bits), 2^j by its exponent field.  x <= 127; below -127, -inf too, the scale is 0.  A
// NaN stays one (a clamp by fmaxf would make it -127, and the key that it comes from would
// drop out of the row).
__device__ __forceinline__ void exp2_poly(float x0, float x1, float& y0, float& y1) {
  constexpr float kRound = 12582912.0f;
  x0 = attn::max_or_nan(x0, -127.0f);
  x1 = attn::max_or_nan(x1, -127.0f);
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

// Pairs, of the 16 of each 32 columns, whose exponentials run on the FMA pipe.  At D = 64
// the products take half as long and the exponential unit is what both halves wait for: 4
// of 16 pairs moved, 24 ragged requests took 109 us instead of 114.  At D = 128 they leave
// the issue slots too few: 2 of 16 moved, 4096 new tokens over 16384 took 1086 us instead
// of 1076, 4 of 16 1127 us.
template <int D>
__device__ __forceinline__ constexpr bool on_fma(int pair) {
  return D == 64 && (pair & 3) == 3;
}

// kInPlace: o is q.  (A kernel of its own: the extra pass at a unit's end, tested at run time,
// cost every call: 24 ragged requests took 96.5 us instead of 94.8.)
template <int D, bool kBf16, bool kInPlace>
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

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const ErrSink& err = C.err;
  // A bounded wait (mbar_wait); the time in which a warp goes key by key does not count.
  auto wait_for = [&](uint64_t* bar, uint32_t parity, int32_t code, uint64_t limit_ns) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    uint64_t t0 = globaltimer();
    while (true) {
      if (mbar_try_wait(bar, parity)) return true;
      if (*s_abort) return false;
      if (globaltimer() - t0 > limit_ns) {
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
  auto wait_bar = [&](uint64_t* bar, uint32_t parity, int32_t code) -> bool {
    return wait_for(bar, parity, code, err.limit_ns);
  };
  pdl_wait();
  pdl_begin_next();
  // no share: the whole CTA leaves, but for the first, which may have lengths to compare
  if ((int)blockIdx.x >= max(__ldg(meta), 1)) return;

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
  const uint32_t tmem = __shfl_sync(0xffffffffu, *s_tmem, 0);

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
          Request R = first.R;
          if (fresh && at.b == first.b) R.len = min(R.len, P.width << P.page_shift);
          else R = get_request(P, at.b);
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
          u.runs = unit_runs<128, true>(P.pred, u.pos0, u.pos0 + u.n - 1, u.len, C.seg);
          const int nblk = run_blocks<128>(u.runs);
          u.blk0 = fresh ? min(first.blk, nblk) : 0;
          u.blk1 = last ? min(end.blk, nblk) : nblk;
          u.slot = fresh && first.blk > 0 ? 2 * w : last ? 2 * w + 1 : -1;
          for (int x = 0; x < 2; ++x)
            u.half[x] = half_tiles(P.pred, u.pos0 + x * C.tb,
                                   u.pos0 + min(u.n, (x + 1) * C.tb) - 1, u.len);
          u.a0 = u.runs.a[0];
          u.a1 = u.runs.a[1];
          u.n0 = (u.runs.cnt[0] + 127) >> 7;
          u.sink_end = P.pred.kind == PA_SINKS ? P.pred.p1 : 0;
          u.table = P.table + (long long)u.b * P.table_stride;
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
            if (h == 0 && C.withhold_q) continue;
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
      // the plan's lengths, where no join compares them, while the last copies are on their way
      // and used (in a warp of its own, or before the warps part, this made the D = 64 softmax
      // spill 44-96 bytes)
      if (C.check) {
        const int used = __ldg(meta);            // CTAs that are here: these, or the first alone
        if (other_lengths(P, shares, used, w * 32 + lane, max(used, 1) * 32))
          err.record(DEV_OTHER_LENGTHS);
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
      // The whole warp runs this code, one elected lane issues: then every address is the
      // same in all lanes for the compiler too and stays in uniform registers.  (With
      // one lane in the whole branch, a product took 97 cycles to issue where the tensor
      // cores take 64: 4096 new tokens over 16384 were 1215 us.)
      const bool leader = elect_one();
      uint32_t ring = 0, kv_c = 0, tp[2] = {0, 0}, tq[2] = {0, 0};
      bool ok = true;
      const uint32_t sQa = smem_u32(sQ), sKVa = smem_u32(sKV);
      auto wait_all = [&](uint64_t* bar, uint32_t parity, int32_t code) -> bool {
        const bool r = __all_sync(0xffffffffu, wait_bar(bar, parity, code));
        tc_fence_after();
        return r;
      };
      auto wait_kv = [&](uint32_t& slot) -> bool {
        slot = kv_c % NS;
        const bool r = wait_all(&kv_full[slot], (kv_c / NS) & 1, DEV_TIMEOUT_KV);
        ++kv_c;
        return r;
      };
      auto commit = [&](uint64_t* bar) {
        if (leader) tc_commit(bar);
      };
      auto issue_s = [&](int h, uint32_t kslot) {
        const uint64_t qd = smem_desc_sw128(sQa + h * SM::kTile, 16);
        const uint64_t kd = smem_desc_sw128(sKVa + kslot * SM::kTile, 16);
        const uint32_t d = tmem + h * 128;
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t off = ((kk >> 2) * kRegion + (kk & 3) * 32) >> 4;
            mma_ss(d, qd + off, kd + off, C.idesc_qk, kk > 0);
          }
          tc_commit(&s_full[h]);
        }
        __syncwarp();
      };
      // O += P V of half h: the first 64 keys as soon as their P is there
      auto issue_pv = [&](int h, uint32_t vslot, bool acc) -> bool {
        const uint32_t d = tmem + 256 + h * D, p = tmem + h * 128 + 64;
        const uint64_t vd = smem_desc_sw128(sKVa + vslot * SM::kTile, kRegion);
        if (!wait_all(&pa_full[h], tp[h] & 1, DEV_TIMEOUT_P)) return false;
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ts(d, p + kk * 8, vd + (uint64_t)((kk * 16 * 128) >> 4), C.idesc_pv,
                   (acc || kk > 0) ? 1u : 0u);
        }
        __syncwarp();
        if (!wait_all(&pb_full[h], tp[h] & 1, DEV_TIMEOUT_P)) return false;
        ++tp[h];
        if (leader) {
#pragma unroll
          for (int kk = 4; kk < 8; ++kk)
            mma_ts(d, p + kk * 8, vd + (uint64_t)((kk * 16 * 128) >> 4), C.idesc_pv, 1u);
        }
        __syncwarp();
        return true;
      };
      while (ok) {
        const uint32_t rs = ring & 1;
        if (!(ok = wait_all(&unit_full[rs], (ring >> 1) & 1, DEV_TIMEOUT_ITEM))) break;
        auto same = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
        const int b = same(s_unit[rs].b), n = same(s_unit[rs].n);
        const int blk0 = same(s_unit[rs].blk0), tiles = same(s_unit[rs].blk1) - blk0;
        const int a0 = same(s_unit[rs].a0), a1 = same(s_unit[rs].a1), n0 = same(s_unit[rs].n0);
        const int sink_end = same(s_unit[rs].sink_end);
        HalfTiles ht[2];
        for (int x = 0; x < 2; ++x) {
          ht[x].i_hi = same(s_unit[rs].half[x].i_hi);
          ht[x].live_min = same(s_unit[rs].half[x].live_min);
        }
        __syncwarp();
        if (leader) mbar_arrive(&unit_empty[rs]);
        ++ring;
        if (b < 0) break;
        if (tiles <= 0) continue;
        const int halves = n > C.tb ? 2 : 1;
        for (int h = 0; h < halves && ok; ++h) {
          ok = __all_sync(0xffffffffu, wait_for(&q_full[h], tq[h] & 1, DEV_TIMEOUT_Q, C.q_limit_ns));
          tc_fence_after();
          ++tq[h];
        }
        uint32_t ks = 0, vs = 0;
        // O begun; P V owed; no scores to come
        bool started[2] = {false, false}, held[2] = {false, false}, last[2] = {false, false};
        // step u: the products with V of super-tile u - 1, then S of super-tile u
        for (int u = 0; u <= tiles && ok; ++u) {
          if (u > 0 && !(ok = wait_kv(vs))) break;
          if (u < tiles && !(ok = wait_kv(ks))) break;
          const int blk = blk0 + u;
          const int kb = blk < n0 ? a0 + blk * 128 : a1 + (blk - n0) * 128;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h >= halves) break;
            if (held[h]) {
              if (!(ok = issue_pv(h, vs, started[h]))) break;
              started[h] = true;
              if (last[h]) commit(&o_full[h]);
            }
            // a piece may also end on super-tiles that the half skips for another reason
            // (they are before its window)
            if (u == tiles && started[h] && !last[h]) commit(&o_full[h]);
            held[h] = u < tiles && tile_live(ht[h], kb, sink_end);
            if (held[h]) {
              issue_s(h, ks);
              // a half whose last position is before the next super-tile is done with its
              // scores: it need not wait for the other's last ones to write its result
              last[h] = u == tiles - 1 || (blk + 1 < n0 ? kb + 128 : a1 + (blk + 1 - n0) * 128) > ht[h].i_hi;
            }
          }
          if (!ok) break;
          if (u > 0) commit(&kv_empty[vs]);
          if (u < tiles) commit(&kv_empty[ks]);
          if (u == tiles - 1)
            for (int h = 0; h < halves; ++h) commit(&q_empty[h]);
        }
      }
      // the commit lands once every product issued above has completed
      if (leader) {
        tc_commit(drain);
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(drain, 0)) {
          if (globaltimer() - t0 > attn::kDrainLimitNs) { err.record(DEV_TIMEOUT_DRAIN); break; }
        }
      }
      __syncwarp();
    }
  } else {
    // -------------------------------------------------------------- softmax, results
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kChunkSoftRegs));
    const int h = warp >> 2, wq = warp & 3;
    const int r_in = wq * 32 + lane;                 // row of the half
    const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
    const uint32_t tS = tmem + lane_off + h * 128;
    const uint32_t tO = tmem + lane_off + 256 + h * D;
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
      // page of box `lane` of a super-tile, read one ahead and looked at then
      auto page_of = [&](int blk) -> int {
        const int4 g = lds4(&u.a0);
        const int j = (blk < g.z ? g.x + blk * 128 : g.y + (blk - g.z) * 128) + lane * C.seg;
        return blk < u.blk1 && lane < C.nseg && j < u.len ? __ldg(u.table + (j >> P.page_shift)) : -1;
      };
      int blk = u.blk0;
      int page = page_of(blk);
      float m_used = -INFINITY, l = 0.f;
      bool any = false;                              // a product with V has been asked for
#pragma unroll 1
      for (; blk < *const_cast<volatile const int*>(&u.blk1); ++blk) {
        const int4 g = lds4(&u.a0), ht = lds4(&u.half[h]);
        const int kb = blk < g.z ? g.x + blk * 128 : g.y + (blk - g.z) * 128;
        // bit x: box x of the super-tile has keys
        const uint32_t boxes = __ballot_sync(0xffffffffu, (unsigned)page < (unsigned)P.pages);
        page = page_of(blk + 1);
        if (kb > ht.x || (kb < ht.y && kb >= g.w)) continue;
        const bool all_boxes = boxes == (1u << C.nseg) - 1u;
        const bool full = kb >= ht.z && kb <= ht.w && all_boxes;
        uint32_t mk[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (__builtin_expect(!full, 0)) {
          const int len = u.len;
          const bool whole = kb + 128 <= len && all_boxes;
          // Live bits of this row.  The bands are one or two ranges of columns, in closed form;
          // the columns of the box with the request's last token are shifted, those of
          // boxes without keys are dead.  The lattices go box by box.
          const int seg_shift = 31 - __clz(C.seg);
          const int tail0 = min(((len - kb) >> seg_shift) << seg_shift, 128);   // the shifted box
          const int shift = tail0 < 128 ? C.seg - (len - kb - tail0) : 0;       // C.seg: it is empty
          if (P.pred.mod <= 1) {
            const int c = i - kb;
            int a0 = 0, b0 = c, a1 = 0, b1 = -1;
            if (P.pred.kind == PA_WINDOW || P.pred.kind == PA_SINKS || P.pred.kind == PA_TWOBAND)
              a0 = max(c - P.pred.p0 + 1, 0);
            if (P.pred.kind == PA_SINKS) b1 = min(P.pred.p1 - 1 - kb, c);
            if (P.pred.kind == PA_TWOBAND) {
              a1 = max(c - P.pred.p1 - P.pred.p2 + 1, 0);
              b1 = min(c - P.pred.p1, c);
            }
            if (P.pred.kind == PA_LOCAL_STRIDED || P.pred.kind == PA_DILATED) a0 = 0;   // every key
            if (P.pred.kind == PA_FAR_STRIDED) b0 = min(c - P.pred.p0, c);
            if (whole && kb >= g.w && P.pred.kind != PA_TWOBAND) {   // one range
#pragma unroll
              for (int k = 0; k < 4; ++k) mk[k] = range_bits(a0, b0, k * 32);
            } else if (whole) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mk[k] = range_bits(a0, b0, k * 32) | range_bits(a1, b1, k * 32);
            } else {
              const int last = len - kb - 1;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mk[k] = range_bits(a0, min(b0, tail0 - 1), k * 32) |
                        range_bits(a1, min(b1, tail0 - 1), k * 32) |
                        range_bits(max(a0, tail0) + shift, min(b0, last) + shift, k * 32) |
                        range_bits(max(a1, tail0) + shift, min(b1, last) + shift, k * 32);
              for (uint32_t gone = ~boxes & ((1u << C.nseg) - 1u); gone; gone &= gone - 1) {
                const int c0 = (__ffs(gone) - 1) << seg_shift;
#pragma unroll
                for (int k = 0; k < 4; ++k) mk[k] &= ~range_bits(c0, c0 + C.seg - 1, k * 32);
              }
            }
          } else {
            const int width = min(C.seg, 32);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t word = 0;
#pragma unroll 1
              for (int c0 = k * 32; c0 < k * 32 + 32; c0 += width) {
                const int sg = c0 >> seg_shift, in = c0 & (C.seg - 1);
                if (!((boxes >> sg) & 1u)) continue;
                const int sh = sg << seg_shift == tail0 ? shift : 0;
                const int j = kb + (sg << seg_shift) - sh;
                uint32_t bits;
                if (!progression_bits(P.pred, i - j, j, 1, 0, in, C.seg, bits))
                  bits = element_bits(P.pred, i, nullptr, j, 1, in, width);
                bits &= range_bits(sh, C.seg - 1, in);
                word |= bits << (c0 - k * 32);
              }
              mk[k] = word;
            }
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
        if (__builtin_expect(!full, 0)) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (!((mk[k] >> x) & 1u)) s[k * 32 + x] = -INFINITY;
          }
        }
        float mx;
        {
          float m8[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) m8[j] = fmaxf(s[2 * j], s[2 * j + 1]);
#pragma unroll
          for (int c = 16; c < 128; c += 16)
#pragma unroll
            for (int j = 0; j < 8; ++j) m8[j] = attn::fmax3(m8[j], s[c + 2 * j], s[c + 2 * j + 1]);
          mx = attn::fmax3(attn::fmax3(m8[0], m8[1], m8[2]), attn::fmax3(m8[3], m8[4], m8[5]),
                           fmaxf(m8[6], m8[7]));
        }
        const float m_tile = mx * c2;
        const bool bump = m_tile > m_used + 8.0f;    // from -inf: the first live key
        if (__builtin_expect(__any_sync(0xffffffffu, bump), 0)) {
          float factor = 1.f;
          if (bump) {
            factor = ex2f(m_used - m_tile);
            m_used = m_tile;
            l *= factor;
          }
          if (any) {
#pragma unroll 1
            for (int k = 0; k < D / 16; ++k) {
              uint32_t r[16];
              tmem_ld16(tO + k * 16, r);
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < 16; ++x) asm volatile("" : "+r"(r[x]));
#pragma unroll
              for (int x = 0; x < 16; ++x) r[x] = __float_as_uint(__uint_as_float(r[x]) * factor);
              tmem_st16(tO + k * 16, r);
            }
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
            float x0, x1, e0, e1;
            attn::ffma2(x0, x1, s[c], s[c + 1], c2, -msub);
            if (on_fma<D>(x)) {
              exp2_poly(x0, x1, e0, e1);
            } else {
              e0 = ex2f(x0);
              e1 = ex2f(x1);
            }
            const int j = (2 * x) & 7;
            attn::fadd2(r8[j], r8[j + 1], e0, e1);
            pk[x] = pack_pair<kBf16>(e0, e1);
          }
          tmem_st16(tS + 64 + q4 * 16, pk);
          if (q4 & 1) {
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(q4 == 1 ? &pa_full[h] : &pb_full[h]);
          }
        }
        any = true;
        l += ((r8[0] + r8[1]) + (r8[2] + r8[3])) + ((r8[4] + r8[5]) + (r8[6] + r8[7]));
      }
      if (!ok) break;

      // results: o and lse, or this piece's O, maximum and sum
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
      // every thread writes its row, 32 bytes (a whole sector) at a time where rows are so
      // aligned
      const float inv_l = part ? 1.f : l > 0.f ? 1.f / l : 0.f;
      // where o is q, rows that are computed again from their q come first: a pass that only
      // looks for them
#pragma unroll 1
      for (int pass = kInPlace ? 0 : 1; pass < 2; ++pass) {
        float probe[4] = {l * 0.f, 0.f, 0.f, 0.f};        // 0 unless something is not finite
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
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
          for (int x = 0; x < 32; x += 4) {
            attn::fma2v(probe[0], probe[1], __uint_as_float(r[x]), __uint_as_float(r[x + 1]), 0.f, 0.f,
                        probe[0], probe[1]);
            attn::fma2v(probe[2], probe[3], __uint_as_float(r[x + 2]), __uint_as_float(r[x + 3]), 0.f,
                        0.f, probe[2], probe[3]);
          }
          if (row_ptr && pass > 0) {
            char* dst = reinterpret_cast<char*>(row_ptr);
            if (part) {
#pragma unroll
              for (int x = 0; x < 4; ++x)
                st32(dst + c * 128 + x * 32, true, r[8 * x], r[8 * x + 1], r[8 * x + 2], r[8 * x + 3],
                     r[8 * x + 4], r[8 * x + 5], r[8 * x + 6], r[8 * x + 7]);
            } else {
#pragma unroll
              for (int x = 0; x < 16; ++x)
                r[x] = pack_pair<kBf16>(__uint_as_float(r[2 * x]) * inv_l,
                                        __uint_as_float(r[2 * x + 1]) * inv_l);
#pragma unroll
              for (int x = 0; x < 2; ++x)
                st32(dst + c * 64 + x * 32, C.o32, r[8 * x], r[8 * x + 1], r[8 * x + 2], r[8 * x + 3],
                     r[8 * x + 4], r[8 * x + 5], r[8 * x + 6], r[8 * x + 7]);
            }
          }
        }
        if (any) tc_fence_before();
        // a value that is not finite, seen or weighed by 0: those rows key by key instead
        const bool mine = row_ptr && !((probe[0] + probe[1]) + (probe[2] + probe[3]) == 0.f);
        uint32_t odd = __ballot_sync(0xffffffffu, mine);
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
        if (kInPlace && mine) row_ptr = 0;             // its row is written
      }
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

template <int D, bool kBf16>
int launch_chunk_body(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                      const ChunkParams& C, const PlanView& pv, float* scratch, int sms,
                      cudaStream_t stream) {
  constexpr int kMinRegs = (256 * kChunkSoftRegs + 128 * kChunkOtherRegs) / kChunkThreads;
  auto go = [&](auto in_place) {
    constexpr auto kKernel = paged_chunk_kernel<D, kBf16, decltype(in_place)::value>;
    const int rc = prepare_kernel<kKernel>("pa_paged_attn", ChunkSmem<D>::kAlloc, kMinRegs);
    if (rc) return rc;
    return launch_after("pa_paged_attn", kKernel, sms, kChunkThreads, ChunkSmem<D>::kAlloc, stream, tq,
                        tk, tv, C, pv.shares, pv.meta, scratch);
  };
  return C.p.o == C.p.q ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace paged
}  // namespace pa
