// Shared pieces of the attention over a paged K/V cache: the forward's parameters and
// the keys that a run of query positions can see.
#pragma once
#include <math.h>
#include "common.cuh"
#include "capi_util.h"

namespace pa {
namespace paged {

struct Params {
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
  r.pos0 = len - (e - s) + (r.row0 - s);
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
  typedef long long ll;
  ll hi = min((ll)i1 + 1, (ll)len);
  ll a = 0, b = hi, c = 0, d = 0;   // near [a, b), far [c, d)
  switch (p.kind) {
    case PA_WINDOW:
      a = (ll)i0 - p.p0 + 1;
      break;
    case PA_SINKS:
      a = (ll)i0 - p.p0 + 1;
      d = p.p1;
      break;
    case PA_TWOBAND:
      a = (ll)i0 - p.p0 + 1;
      c = (ll)i0 - p.p1 - p.p2 + 1;
      d = (ll)i1 - p.p1 + 1;
      break;
    case PA_FAR_STRIDED:
      b = (ll)i1 - p.p0 + 1;
      break;
    default:
      break;
  }
  a = max(a, 0ll);
  c = max(c, 0ll);
  b = min(b, hi);
  d = min(d, hi);
  KeyRanges r{0, 0, 0, 0};
  if (a >= b) a = b = 0;
  if (c >= d) c = d = 0;
  if (a < b && c < d) {
    if (c > a) {
      ll t = a; a = c; c = t;
      t = b; b = d; d = t;
    }
    if (d >= a) {       // they touch: one range
      b = max(b, d);
      a = c;
      c = d = 0;
    }
  }
  if (c < d) {
    r.a0 = (int)c;
    r.b0 = (int)d;
    r.a1 = (int)a;
    r.b1 = (int)b;
  } else {
    r.a0 = (int)a;
    r.b0 = (int)b;
  }
  return r;
}

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

}  // namespace paged
}  // namespace pa
