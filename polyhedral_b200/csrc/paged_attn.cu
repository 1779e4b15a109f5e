// Attention over a paged K/V cache: argument checks, the plan and the C entry points.
#include <mutex>
#include "paged_chunk.cuh"

namespace pa {
namespace paged {
namespace {

int check_sizes(const pa_paged_attn_args* a, const char* who) {
  PA_CHECK_ARG(a != nullptr, "%s: null args", who);
  PA_CHECK_ARG(a->requests >= 1 && a->requests <= 65536, "%s: requests=%d not in [1, 65536]", who,
               a->requests);
  PA_CHECK_ARG(a->tokens >= 0 && (long long)a->tokens * a->heads <= 0x7fffffffll,
               "%s: tokens=%d x heads=%d must be in [0, 2^31)", who, a->tokens, a->heads);
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
  // a row's o is written when its q is read no more, and nothing else is then where o is q
  PA_CHECK_ARG(a->o != a->q || (a->o_token_stride == a->q_token_stride &&
                                a->o_head_stride == a->q_head_stride),
               "%s: o lies over q with other strides", who);
  PA_CHECK_ARG(a->o != a->k_cache && a->o != a->v_cache, "%s: o lies over a cache", who);
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
  P->group_inv = ((1u << 20) + P->group - 1) / P->group;
  P->pages = a->pages;
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
  P->page_shift = a->page_size > 0 ? __builtin_ctz(a->page_size) : 0;
  const float scale = a->scale > 0.f ? a->scale : 1.0f / sqrtf((float)a->D);
  P->scale_log2 = scale * 1.4426950408889634f;
  // positions stay below 2^24, so larger widths mean the same and would overflow sums
  pa_pred pr = a->pred;
  pr.p0 = pr.p0 < (1 << 25) ? pr.p0 : 1 << 25;
  pr.p1 = pr.p1 < (1 << 25) ? pr.p1 : 1 << 25;
  pr.p2 = pr.p2 < (1 << 25) ? pr.p2 : 1 << 25;
  return make_pred(&pr, &P->pred, who);
}

// Kernel and shares for these sizes and hints.
Config choose(const pa_paged_attn_args* a, int sms) {
  Config c;
  const int group = a->heads / a->kv_heads;
  const long long most = a->max_new > 0 && a->max_new < a->tokens ? a->max_new : a->tokens;
  // Few rows: the keys are read once and bound the work (64 requests' decode: 165 us; through
  // the chunk kernel 226 us; with 32 rows per key head, read twice, 331 us against 249 us).
  // Few keys in all, at most 4 blocks a worker: latency bounds it, and the chunk kernel's is
  // longer (64 tokens of one request: 13 us on the GPU against 20 us; 4 tokens after 999, 64
  // query heads: 15 against 32 us; 16 requests of 16 after 500, 14 blocks a worker: 32
  // against 24 us).
  const long long units = (most * group + kFewRows - 1) / kFewRows * a->requests * a->kv_heads;
  const long long each = (a->max_len + kFewBlock - 1ll) / kFewBlock;
  const bool few_keys = a->max_len > 0 && units <= 4ll * sms * kFewWarps / each;
  if (most * group <= kFewRows || few_keys) {
    c.unit_rows = kFewRows;
    c.half_tokens = 0;
    c.workers = sms * kFewWarps;
    // one block: a single request of 1000 tokens took 8.9 us on the GPU with shares of one
    // block, 9.1 us with two, 10.5 us with four
    c.min_share = 1 + kUnitCost;
    c.min_piece = 1;
  } else {
    c.unit_rows = 256;
    c.half_tokens = 128 / group;
    c.workers = sms;
    c.min_share = 2 + kUnitCost;
    // small units stay whole: 3 requests of 300 new tokens under a window of 27, 36 us cut
    // anywhere, 24 us with pieces of 3; 22 requests of 356, 39 and 31 us
    c.min_piece = 3;
  }
  // Requests of at most 128 tokens stay whole, which spares the join's launch: 14.1 us a call
  // instead of 18.2-18.5 us wherever the host bounds it.  On the GPU alone (captured) chunks gain
  // too: 5 of 32 new tokens 7.1 us instead of 9.7, 8 of 60-100 16.5 instead of 18.0, 64 of them
  // 48.4 instead of 52.1; decode by how many warps it fills: 500 of 20-126 tokens 42.2 instead of
  // 42.8, 64 of 60-120 11.5 instead of 11.4, 8 of 100-120 10.6 instead of 9.3, one of 120 10.3
  // instead of 8.1.
  c.split = !(a->max_len > 0 && a->max_len <= 128);
  return c;
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                             CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(p);
  });
  return fn;
}

// 16-bit tensor (D, n1, n2, n3) by element strides s1..s3, in boxes of 64 x b1 x 1 x b3, 128-byte
// swizzle, zeros outside.
int make_map(CUtensorMap* m, const void* base, int dtype, int D, const long long (&n)[3],
             const long long (&s)[3], int b1, int b3, const char* name) {
  EncodeFn enc = encode_fn();
  if (!enc) return fail(PA_ERR_CUDA, "pa_paged_attn: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[4] = {(cuuint64_t)D, 0, 0, 0}, strides[3];
  const cuuint32_t box[4] = {64, (cuuint32_t)b1, 1, (cuuint32_t)b3}, one[4] = {1, 1, 1, 1};
  for (int i = 0; i < 3; ++i) {
    dims[i + 1] = (cuuint64_t)n[i];
    strides[i] = n[i] > 1 ? (cuuint64_t)s[i] * 2 : (cuuint64_t)D * 2;   // unused where there is one
  }
  const CUresult r =
      enc(m, dtype == PA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
          const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(PA_ERR_ARG, "pa_paged_attn: tensor map for %s rejected (CUresult %d): check its strides",
                name, (int)r);
  return PA_OK;
}

int launch_chunk(const pa_paged_attn_args* a, const Params& P, const Config& c, const PlanView& pv,
                 float* scratch, int sms, cudaStream_t stream, uint64_t wait_ns, int withhold_q) {
  CUtensorMap tq, tk, tv;
  int rc;
  ChunkParams C;
  C.p = P;
  C.tb = c.half_tokens;
  C.seg = a->page_size < 128 ? a->page_size : 128;
  C.nseg = 128 / C.seg;
  if ((rc = make_map(&tq, a->q, a->dtype, a->D, {P.group, a->kv_heads, a->tokens},
                     {a->q_head_stride, a->q_head_stride * P.group, a->q_token_stride}, P.group, C.tb,
                     "q")))
    return rc;
  if ((rc = make_map(&tk, a->k_cache, a->dtype, a->D, {a->page_size, a->kv_heads, a->pages},
                     {a->k_row_stride, a->k_head_stride, a->k_page_stride}, C.seg, 1, "k_cache")))
    return rc;
  if ((rc = make_map(&tv, a->v_cache, a->dtype, a->D, {a->page_size, a->kv_heads, a->pages},
                     {a->v_row_stride, a->v_head_stride, a->v_page_stride}, C.seg, 1, "v_cache")))
    return rc;
  C.check = !c.split;
  C.o32 = aligned(a->o, 32) && a->o_token_stride % 16 == 0 && a->o_head_stride % 16 == 0;
  const uint32_t fmt = a->dtype == PA_BF16 ? 1u : 0u;
  C.idesc_qk = make_idesc_f16(fmt, 128, 128, 0, 0);
  C.idesc_pv = make_idesc_f16(fmt, 128, a->D, 0, 1);
  C.err.word = pv.status;
  C.err.epoch = 0;
  C.err.limit_ns = wait_ns;
  C.q_limit_ns = withhold_q ? wait_ns / 4 : wait_ns;
  C.withhold_q = withhold_q;
  return a->D == 128 ? launch_chunk_d128(tq, tk, tv, C, fmt != 0, pv, scratch, sms, stream)
                     : launch_chunk_d64(tq, tk, tv, C, fmt != 0, pv, scratch, sms, stream);
}

size_t scratch_bytes_of(const pa_paged_attn_args* a, const Config& c) {
  if (!c.split) return 0;
  const size_t f = a->D == 128 ? slot_floats<128>(c.unit_rows) : slot_floats<64>(c.unit_rows);
  return 2 * (size_t)c.workers * f * sizeof(float);
}

// The forward, with the limit of its bounded waits; withhold_q: pa_paged_attn_withheld.
int forward(const pa_paged_attn_args* a, void* plan, size_t plan_size, void* scratch,
            size_t scratch_bytes, cudaStream_t stream, uint64_t wait_ns, int withhold_q,
            const char* who) {
  int rc = check_sizes(a, who), sms = 0;
  if (rc) return rc;
  if (a->tokens == 0) return PA_OK;
  if ((rc = check_args(a, who))) return rc;
  Params P;
  if ((rc = make_params(a, &P, who))) return rc;
  if ((rc = sm_count(&sms, who))) return rc;
  const Config c = choose(a, sms);
  PA_CHECK_ARG(plan && plan_size >= plan_bytes(c, a->requests) && aligned(plan, 256),
               "%s: plan must be 256-byte aligned and >= %zu bytes", who, plan_bytes(c, a->requests));
  const size_t need = scratch_bytes_of(a, c);
  PA_CHECK_ARG(need == 0 || (scratch && scratch_bytes >= need && aligned(scratch, 256)),
               "%s: scratch must be 256-byte aligned and >= %zu bytes", who, need);
  if (withhold_q && !c.half_tokens)
    return fail(PA_ERR_UNSUPPORTED, "%s: these sizes run the few-rows kernel, which waits for no barrier",
                who);
  const PlanView pv = plan_view(plan, c);
  const bool bf = a->dtype == PA_BF16;
  float* part = static_cast<float*>(scratch);
  rc = c.half_tokens ? launch_chunk(a, P, c, pv, part, sms, stream, wait_ns, withhold_q)
                     : launch_few(P, bf, a->D, pv, c, part, sms, stream);
  if (rc) return rc;
  return c.split ? launch_join(P, bf, a->D, pv, c, part, sms, stream) : PA_OK;
}

}  // namespace
}  // namespace paged
}  // namespace pa

extern "C" size_t pa_paged_plan_size(const pa_paged_attn_args* a) {
  using namespace pa::paged;
  int sms = 0;
  if (check_sizes(a, "pa_paged_plan_size") || sm_count(&sms, "pa_paged_plan_size")) return 0;
  return plan_bytes(choose(a, sms), a->requests);
}

extern "C" size_t pa_paged_scratch_size(const pa_paged_attn_args* a) {
  using namespace pa::paged;
  int sms = 0;
  if (check_sizes(a, "pa_paged_scratch_size") || sm_count(&sms, "pa_paged_scratch_size")) return 0;
  return scratch_bytes_of(a, choose(a, sms));
}

extern "C" int pa_paged_plan(const pa_paged_attn_args* a, void* plan, size_t plan_size,
                             pa_stream_t stream) {
  using namespace pa;
  using namespace pa::paged;
  int rc = check_sizes(a, "pa_paged_plan"), sms = 0;
  if (rc) return rc;
  PA_CHECK_ARG(a->table_width >= 1 && (long long)a->table_width * a->page_size <= (1 << 24),
               "pa_paged_plan: table_width=%d pages of %d rows: at most 2^24 tokens per request",
               a->table_width, a->page_size);
  Params P;
  if ((rc = make_params(a, &P, "pa_paged_plan"))) return rc;
  if ((rc = sm_count(&sms, "pa_paged_plan"))) return rc;
  const Config c = choose(a, sms);
  PA_CHECK_ARG(plan && plan_size >= plan_bytes(c, a->requests) && aligned(plan, 256),
               "pa_paged_plan: plan must be 256-byte aligned and >= %zu bytes",
               plan_bytes(c, a->requests));
  return launch_plan(P, c, plan_view(plan, c), (cudaStream_t)stream);
}

extern "C" int pa_paged_attn(const pa_paged_attn_args* a, void* plan, size_t plan_size,
                             void* scratch, size_t scratch_bytes, pa_stream_t stream) {
  return pa::paged::forward(a, plan, plan_size, scratch, scratch_bytes, (cudaStream_t)stream,
                            pa::kWaitLimitNs, 0, "pa_paged_attn");
}

extern "C" int pa_paged_attn_withheld(const pa_paged_attn_args* a, void* plan, size_t plan_size,
                                      void* scratch, size_t scratch_bytes, int64_t wait_limit_ns,
                                      pa_stream_t stream) {
  using namespace pa;
  PA_CHECK_ARG(wait_limit_ns >= 1000 && wait_limit_ns <= (int64_t)kWaitLimitNs,
               "pa_paged_attn_withheld: wait_limit_ns=%lld outside [1 us, 1 s]",
               (long long)wait_limit_ns);
  return paged::forward(a, plan, plan_size, scratch, scratch_bytes, (cudaStream_t)stream,
                        (uint64_t)wait_limit_ns, 1, "pa_paged_attn_withheld");
}

extern "C" int pa_paged_status(const void* plan, int32_t* status_host, pa_stream_t stream) {
  PA_CHECK_ARG(plan && status_host, "pa_paged_status: null pointer");
  PA_CUDA(cudaMemcpyAsync(status_host, plan, sizeof(int32_t), cudaMemcpyDeviceToHost,
                          (cudaStream_t)stream), "pa_paged_status");
  PA_CUDA(cudaStreamSynchronize((cudaStream_t)stream), "pa_paged_status");
  return *status_host ? PA_ERR_DEVICE : PA_OK;
}
