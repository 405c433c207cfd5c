// C entries of the packed attention: descriptor checks, workspace, choice of the kernels.
#include "attention.h"

namespace {

int fill_params(const sempyr_attention_desc* d, attn::Params& p, const char* who) {
    if (!d) SEMPYR_FAIL("%s: null descriptor", who);
    if (!dtype_ok(d->dtype)) SEMPYR_FAIL("%s: unknown element type %d", who, d->dtype);
    const int sz = dtype_size(d->dtype);
    if (d->dim < 1 || d->dim > 128 || d->dim * sz % 16) SEMPYR_FAIL("%s: head dim must be at most 128 and whole 16-byte vectors, got %d", who, d->dim);
    if (d->heads_q < 1 || d->heads_k < 1 || d->heads_q > 65536 || d->heads_q % d->heads_k) SEMPYR_FAIL("%s: %d query heads over %d key heads", who, d->heads_q, d->heads_k);
    if (d->total_q < 0 || d->total_k < 0 || d->total_q > 1 << 30 || d->total_k > 1 << 30) SEMPYR_FAIL("%s: %lld / %lld rows", who, (long long)d->total_q, (long long)d->total_k);
    if (d->nseq < 0 || d->nseq > 1 << 24) SEMPYR_FAIL("%s: %d sequences", who, d->nseq);
    // (the kernels multiply by scale log2(e))
    if (!(d->scale > 0.f) || !(d->scale * 1.4426950408889634f < INFINITY)) SEMPYR_FAIL("%s: scale must be positive and below 2e38", who);
    const int64_t strides[] = {d->q_stride_token, d->k_stride_token, d->v_stride_token, d->q_stride_head, d->k_stride_head, d->v_stride_head};
    for (int i = 0; i < 6; ++i) {
        if (strides[i] < 0 || strides[i] * sz % 16) SEMPYR_FAIL("%s: strides must be whole 16-byte vectors", who);
        if (i < 3 && (strides[i] < d->dim || strides[i] > (int64_t)1 << 23)) SEMPYR_FAIL("%s: token strides from dim to 2^23 elements, got %lld", who, (long long)strides[i]);
    }
    p = attn::Params{};
    p.q_tok = d->q_stride_token; p.q_head = d->q_stride_head;
    p.k_tok = d->k_stride_token; p.k_head = d->k_stride_head;
    p.v_tok = d->v_stride_token; p.v_head = d->v_stride_head;
    p.total_q = (int)d->total_q; p.total_k = (int)d->total_k; p.nseq = d->nseq;
    p.heads_q = d->heads_q; p.heads_k = d->heads_k; p.group = d->heads_q / d->heads_k;
    p.dim = d->dim; p.causal = d->causal != 0;
    p.scale = d->scale; p.scale_log2 = d->scale * 1.4426950408889634f;
    return 0;
}

}  // namespace

static int64_t workspace_floats(const attn::Params& p, const attn::SplitPlan& plan) {
    return plan.splits > 1 ? (int64_t)plan.splits * p.total_q * p.heads_q * (p.dim + 2) : 0;
}

extern "C" int sempyr_attention_workspace(const sempyr_attention_desc* d, int64_t* floats)
{
    attn::Params p;
    if (int rc = fill_params(d, p, "attention_workspace")) return rc;
    if (!floats) SEMPYR_FAIL("attention_workspace: null pointer");
    *floats = workspace_floats(p, attn::plan_split(p));
    return 0;
}

extern "C" int sempyr_attention_fwd(const sempyr_attention_desc* d, const void* q, const void* k, const void* v, const int32_t* cu_q,
                                    const int32_t* cu_k, const int32_t* len_k, void* o, void* o_low, float* stats, float* workspace,
                                    int64_t workspace_size, void* stream)
{
    attn::Params p;
    if (int rc = fill_params(d, p, "attention_fwd")) return rc;
    if (p.total_q == 0) return 0;
    if (!q || !o || (p.total_k > 0 && (!k || !v)) || !cu_q || !cu_k) SEMPYR_FAIL("attention_fwd: null pointer");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(o_low)) SEMPYR_FAIL("attention_fwd: tensors must be 16-byte aligned");
    p.q = q; p.k = k; p.v = v; p.cu_q = cu_q; p.cu_k = cu_k; p.len_k = len_k; p.o = o; p.o_low = o_low; p.stats = stats;
    const attn::SplitPlan plan = attn::plan_split(p);
    if (plan.splits == 0) return attn::launch_fwd(d->dtype, p, (hipStream_t)stream);
    const int64_t need = workspace_floats(p, plan);
    if (need > 0 && (!workspace || workspace_size < need || !aligned16(workspace)))
        SEMPYR_FAIL("attention_fwd: %lld floats of 16-byte aligned workspace expected, got %lld", (long long)need, (long long)workspace_size);
    return attn::launch_split(d->dtype, p, plan, workspace, (hipStream_t)stream);
}

extern "C" int sempyr_attention_bwd(const sempyr_attention_desc* d, const void* q, const void* k, const void* v, const void* o,
                                    const void* o_low, const float* stats, const void* go, const int32_t* cu_q, const int32_t* cu_k, const int32_t* len_k,
                                    void* dq, void* dk, void* dv, float* delta, void* stream)
{
    attn::Params p;
    if (int rc = fill_params(d, p, "attention_bwd")) return rc;
    if (p.total_q == 0 && p.total_k == 0) return 0;
    if ((p.total_q > 0 && (!q || !o || !stats || !go || !dq || !delta)) || (p.total_k > 0 && (!k || !v || !dk || !dv)) || !cu_q || !cu_k)
        SEMPYR_FAIL("attention_bwd: null pointer");
    const void* ptrs[] = {q, k, v, o, o_low, go, dq, dk, dv};
    for (const void* x : ptrs)
        if (!aligned16(x)) SEMPYR_FAIL("attention_bwd: tensors must be 16-byte aligned");
    if ((int64_t)d->heads_q * d->dim > (int64_t)1 << 23) SEMPYR_FAIL("attention_bwd: rows of more than 2^23 elements");
    p.q = q; p.k = k; p.v = v; p.cu_q = cu_q; p.cu_k = cu_k; p.len_k = len_k;
    p.o = const_cast<void*>(o); p.o_low = const_cast<void*>(o_low); p.stats = const_cast<float*>(stats); p.go = go; p.delta = delta; p.dq = dq; p.dk = dk; p.dv = dv;
    return attn::launch_bwd(d->dtype, p, (hipStream_t)stream);
}
