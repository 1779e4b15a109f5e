// Attention over a paged K/V cache: argument checks, the plan and the C entry points.
#include "paged.cuh"

namespace pa {
namespace paged {
namespace {

// One warp per (new token, query head), one key at a time: lane x holds D / 32 columns of
// q, a key's score is a sum over the lanes, and the running maximum and sum of the
// softmax scale what has been added up so far.
template <int D, bool kBf16>
__global__ void __launch_bounds__(128) paged_rows_kernel(Params P) {
  constexpr int E = D / 64;      // 32-bit words of a row per lane
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(item / P.heads), a = (int)(item % P.heads);
  if (t >= P.tokens) return;
  // the request of row t: the last one that starts at or before it and is not empty
  int lo = 0, hi = P.requests;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(P.q_start + mid) <= t) lo = mid; else hi = mid;
  }
  const Request R = get_request(P, lo);
  if (t < R.row0 || t >= R.row0 + R.n) return;
  const int i = R.pos0 + (t - R.row0), h = a / P.group;
  const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(P.q) +
                                                        t * P.q_t + a * P.q_h) + lane * E;
  float2 qf[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qf[e] = unpack_pair<kBf16>(q[e]);
    acc[e] = make_float2(0.f, 0.f);
  }
  float m = -INFINITY, l = 0.f;
  const KeyRanges kr = key_ranges(P.pred, i, i, R.len);
  const int mask = (1 << P.page_shift) - 1;
  for (int part = 0; part < 2; ++part) {
    const int j1 = part ? kr.b1 : kr.b0;
    for (int j = part ? kr.a1 : kr.a0; j < j1; ++j) {
      if (!pred_live(P.pred, i, j)) continue;
      const int page = __ldg(P.table + lo * P.table_stride + (j >> P.page_shift));
      if ((unsigned)page >= (unsigned)P.pages) continue;
      const uint32_t* k = reinterpret_cast<const uint32_t*>(
          static_cast<const uint16_t*>(P.k) + page * P.k_p + (j & mask) * P.k_r + h * P.k_h) + lane * E;
      const uint32_t* v = reinterpret_cast<const uint32_t*>(
          static_cast<const uint16_t*>(P.v) + page * P.v_p + (j & mask) * P.v_r + h * P.v_h) + lane * E;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float2 x = unpack_pair<kBf16>(k[e]);
        s = fmaf(qf[e].x, x.x, fmaf(qf[e].y, x.y, s));
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      s *= P.scale_log2;
      const float mn = fmaxf(m, s);
      const float f = exp2f(m - (mn == -INFINITY ? 0.f : mn));
      const float p = exp2f(s - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l = l * f + p;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float2 x = unpack_pair<kBf16>(v[e]);
        acc[e].x = acc[e].x * f + p * x.x;
        acc[e].y = acc[e].y * f + p * x.y;
      }
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(P.o) + t * P.o_t + a * P.o_h) + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = pack_pair<kBf16>(acc[e].x * inv, acc[e].y * inv);
  if (P.lse && lane == 0)
    P.lse[a * P.lse_h + t] = l > 0.f ? (m + log2f(l)) * 0.69314718055994530942f : -INFINITY;
}

int check_sizes(const pa_paged_attn_args* a, const char* who) {
  PA_CHECK_ARG(a != nullptr, "%s: null args", who);
  PA_CHECK_ARG(a->requests >= 1 && a->requests <= 65536, "%s: requests=%d not in [1, 65536]", who,
               a->requests);
  PA_CHECK_ARG(a->tokens >= 0, "%s: tokens=%d < 0", who, a->tokens);
  PA_CHECK_ARG(a->kv_heads >= 1 && a->heads >= 1 && a->heads <= 65535 && a->heads % a->kv_heads == 0,
               "%s: heads=%d must be a multiple of kv_heads=%d", who, a->heads, a->kv_heads);
  PA_CHECK_ARG(a->heads / a->kv_heads <= 128, "%s: %d query heads per key head (at most 128)", who,
               a->heads / a->kv_heads);
  PA_CHECK_ARG(a->D == 64 || a->D == 128, "%s: D=%d unsupported (64 or 128)", who, a->D);
  PA_CHECK_ARG(a->dtype == PA_BF16 || a->dtype == PA_F16, "%s: bad dtype %d", who, a->dtype);
  PA_CHECK_ARG(a->page_size >= 16 && a->page_size <= 1024 && (a->page_size & (a->page_size - 1)) == 0,
               "%s: page_size=%d must be a power of two in [16, 1024]", who, a->page_size);
  PA_CHECK_ARG(a->max_new >= 0 && a->max_len >= 0, "%s: max_new=%d, max_len=%d must not be negative",
               who, a->max_new, a->max_len);
  PA_CHECK_ARG(a->seq_lens && a->q_start, "%s: null seq_lens / q_start", who);
  return PA_OK;
}

int check_args(const pa_paged_attn_args* a, const char* who) {
  PA_CHECK_ARG(a->pages >= 1 && (long long)a->pages * a->page_size <= 0x7fffffffll,
               "%s: pages=%d of %d rows: slots must fit in 32 bits", who, a->pages, a->page_size);
  PA_CHECK_ARG(a->table_width >= 1 && (long long)a->table_width * a->page_size <= (1 << 24),
               "%s: table_width=%d pages of %d rows: at most 2^24 tokens per request", who,
               a->table_width, a->page_size);
  PA_CHECK_ARG(a->q && a->k_cache && a->v_cache && a->o && a->block_table, "%s: null pointer", who);
  PA_CHECK_ARG(aligned(a->q, 16) && aligned(a->k_cache, 16) && aligned(a->v_cache, 16) &&
                   aligned(a->o, 16),
               "%s: q, o and the caches must be 16-byte aligned", who);
  const long long strides[] = {a->q_token_stride, a->q_head_stride, a->k_page_stride,
                               a->k_row_stride, a->k_head_stride, a->v_page_stride,
                               a->v_row_stride, a->v_head_stride, a->o_token_stride,
                               a->o_head_stride};
  for (long long s : strides)
    PA_CHECK_ARG(s >= 0 && s % 8 == 0, "%s: strides must be multiples of 8 elements", who);
  return PA_OK;
}

int make_params(const pa_paged_attn_args* a, Params* P, const char* who) {
  P->q = a->q;
  P->k = a->k_cache;
  P->v = a->v_cache;
  P->o = a->o;
  P->lse = a->lse;
  P->table = a->block_table;
  P->seq_lens = a->seq_lens;
  P->q_start = a->q_start;
  P->requests = a->requests;
  P->tokens = a->tokens;
  P->heads = a->heads;
  P->kv_heads = a->kv_heads;
  P->group = a->heads / a->kv_heads;
  P->pages = a->pages;
  P->page_shift = __builtin_ctz(a->page_size);
  P->width = a->table_width;
  P->table_stride = a->table_stride;
  P->q_t = a->q_token_stride;
  P->q_h = a->q_head_stride;
  P->k_p = a->k_page_stride;
  P->k_r = a->k_row_stride;
  P->k_h = a->k_head_stride;
  P->v_p = a->v_page_stride;
  P->v_r = a->v_row_stride;
  P->v_h = a->v_head_stride;
  P->o_t = a->o_token_stride;
  P->o_h = a->o_head_stride;
  P->lse_h = a->lse_head_stride;
  const float scale = a->scale > 0.f ? a->scale : 1.0f / sqrtf((float)a->D);
  P->scale_log2 = scale * 1.4426950408889634f;
  return make_pred(&a->pred, &P->pred, who);
}

}  // namespace
}  // namespace paged
}  // namespace pa

extern "C" size_t pa_paged_plan_size(const pa_paged_attn_args* a) { return a ? 256 : 0; }

extern "C" size_t pa_paged_scratch_size(const pa_paged_attn_args*) { return 0; }

extern "C" int pa_paged_plan(const pa_paged_attn_args* a, void* plan, size_t plan_bytes,
                             pa_stream_t stream) {
  using namespace pa;
  const int rc = paged::check_sizes(a, "pa_paged_plan");
  if (rc) return rc;
  Pred p;
  const int rp = make_pred(&a->pred, &p, "pa_paged_plan");
  if (rp) return rp;
  PA_CHECK_ARG(plan && plan_bytes >= pa_paged_plan_size(a) && aligned(plan, 256),
               "pa_paged_plan: plan must be 256-byte aligned and >= %zu bytes",
               pa_paged_plan_size(a));
  PA_CUDA(cudaMemsetAsync(plan, 0, 256, (cudaStream_t)stream), "pa_paged_plan");
  return PA_OK;
}

extern "C" int pa_paged_attn(const pa_paged_attn_args* a, void* plan, size_t plan_bytes,
                             void* scratch, size_t scratch_bytes, pa_stream_t stream) {
  using namespace pa;
  using namespace pa::paged;
  int rc = check_sizes(a, "pa_paged_attn");
  if (rc) return rc;
  if (a->tokens == 0) return PA_OK;
  if ((rc = check_args(a, "pa_paged_attn"))) return rc;
  PA_CHECK_ARG(plan && plan_bytes >= pa_paged_plan_size(a) && aligned(plan, 256),
               "pa_paged_attn: plan must be 256-byte aligned and >= %zu bytes",
               pa_paged_plan_size(a));
  (void)scratch;
  (void)scratch_bytes;
  Params P;
  if ((rc = make_params(a, &P, "pa_paged_attn"))) return rc;
  const long long items = (long long)a->tokens * a->heads;
  const long long grid = (items + 3) / 4;
  PA_CHECK_ARG(grid <= 0x7fffffffll, "pa_paged_attn: tokens=%d x heads=%d are too many", a->tokens,
               a->heads);
  const cudaStream_t s = (cudaStream_t)stream;
  const bool bf = a->dtype == PA_BF16;
  if (a->D == 128)
    bf ? paged_rows_kernel<128, true><<<(int)grid, 128, 0, s>>>(P)
       : paged_rows_kernel<128, false><<<(int)grid, 128, 0, s>>>(P);
  else
    bf ? paged_rows_kernel<64, true><<<(int)grid, 128, 0, s>>>(P)
       : paged_rows_kernel<64, false><<<(int)grid, 128, 0, s>>>(P);
  return check_launch("pa_paged_attn");
}

extern "C" int pa_paged_status(const void* plan, int32_t* status_host, pa_stream_t stream) {
  PA_CHECK_ARG(plan && status_host, "pa_paged_status: null pointer");
  PA_CUDA(cudaMemcpyAsync(status_host, plan, sizeof(int32_t), cudaMemcpyDeviceToHost,
                          (cudaStream_t)stream), "pa_paged_status");
  PA_CUDA(cudaStreamSynchronize((cudaStream_t)stream), "pa_paged_status");
  return *status_host ? PA_ERR_DEVICE : PA_OK;
}
