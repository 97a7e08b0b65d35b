// C entry points of the transformer training operators (see include/megray/c_api.h).
#include "kernels/adamw.cuh"
#include "kernels/attention.cuh"
#include "kernels/balance.cuh"
#include "megray/c_api.h"
#include "megray/types.h"

namespace {
constexpr int kInvalid = 6;
int rc(cudaError_t e) { return e == cudaSuccess ? 0 : -static_cast<int>(e); }
cudaStream_t S(void* s) { return static_cast<cudaStream_t>(s); }
bool f32_or_bf16(int dtype) { return dtype == MegRay::MEGRAY_FLOAT32 || dtype == MegRay::MEGRAY_BFLOAT16; }
bool is_bf16(int dtype) { return dtype == MegRay::MEGRAY_BFLOAT16; }

bool to_router(const megray_router* r, mgk::balance::Router* to) {
    if (r == nullptr || !f32_or_bf16(r->dtype))
        return false;
    *to = {r->logits, is_bf16(r->dtype), r->ld, r->idx, r->idx64 != 0, r->mask, r->tokens, r->experts, r->top};
    return true;
}
bool to_result(const megray_balance_out* o, mgk::balance::Result* to) {
    if (o == nullptr || (o->dlogits != nullptr && !f32_or_bf16(o->dtype)))
        return false;
    *to = {o->coef, o->loss, o->counts, o->dlogits, is_bf16(o->dtype), o->ldd, o->accumulate != 0};
    return true;
}
bool to_problem(const megray_attn_args* a, mgk::attn::Problem* to) {
    if (a == nullptr || (a->dtype != MegRay::MEGRAY_BFLOAT16 && a->dtype != MegRay::MEGRAY_FLOAT16))
        return false;
    *to = {a->dtype == MegRay::MEGRAY_FLOAT16, a->tokens, a->heads, a->kv_heads, a->dim, a->cu, a->seqs,
           a->causal != 0, a->scale, a->error_flag};
    return true;
}
mgk::attn::Tensor T(const megray_attn_tensor* t) {
    return t != nullptr ? mgk::attn::Tensor{t->p, t->row, t->head} : mgk::attn::Tensor{};
}
}  // namespace

extern "C" {

int megray_attention(const megray_attn_args* a, const megray_attn_tensor* q, const megray_attn_tensor* k,
                     const megray_attn_tensor* v, const megray_attn_tensor* out, float* lse, void* stream) {
    mgk::attn::Problem p;
    if (!to_problem(a, &p))
        return kInvalid;
    return rc(mgk::attn::launch_forward(p, T(q), T(k), T(v), T(out), lse, S(stream)));
}
size_t megray_attention_bwd_workspace(const megray_attn_args* a) {
    mgk::attn::Problem p;
    return to_problem(a, &p) ? mgk::attn::backward_workspace(p) : 0;
}
int megray_attention_bwd(const megray_attn_args* a, const megray_attn_tensor* dout, const megray_attn_tensor* q,
                         const megray_attn_tensor* k, const megray_attn_tensor* v, const megray_attn_tensor* out,
                         const float* lse, const megray_attn_tensor* dq, const megray_attn_tensor* dk,
                         const megray_attn_tensor* dv, void* workspace, void* stream) {
    mgk::attn::Problem p;
    if (!to_problem(a, &p))
        return kInvalid;
    return rc(mgk::attn::launch_backward(p, T(dout), T(q), T(k), T(v), T(out), lse, T(dq), T(dk), T(dv), workspace, S(stream)));
}

int megray_adamw(const megray_adamw_tensor* tensors, int count, const megray_adamw_args* a, void* stream) {
    if (a == nullptr || !f32_or_bf16(a->p_dtype) || !f32_or_bf16(a->g_dtype))
        return kInvalid;
    static_assert(sizeof(megray_adamw_tensor) == sizeof(mgk::adamw::Tensor), "the list is passed on as it is");
    mgk::adamw::Step s{};
    s.p_bf16 = is_bf16(a->p_dtype);
    s.g_bf16 = is_bf16(a->g_dtype);
    s.bits = a->bits;
    s.m = a->m;
    s.v = a->v;
    s.m_scale = a->m_scale;
    s.v_scale = a->v_scale;
    s.lr = a->lr;
    s.beta1 = a->beta1;
    s.beta2 = a->beta2;
    s.eps = a->eps;
    s.weight_decay = a->weight_decay;
    s.grad_scale = a->grad_scale;
    s.step = a->step;
    s.lr_dev = a->lr_dev;
    s.grad_scale_dev = a->grad_scale_dev;
    s.step_dev = a->step_dev;
    return rc(mgk::adamw::launch(reinterpret_cast<const mgk::adamw::Tensor*>(tensors), count, s, S(stream)));
}

int megray_balance_partials(int tokens, int experts) { return mgk::balance::partials(tokens, experts); }
size_t megray_balance_record(int experts) { return static_cast<size_t>(mgk::balance::partial_words(experts)) * 4; }
size_t megray_balance_workspace(int tokens, int experts) { return mgk::balance::workspace_bytes(tokens, experts); }
int megray_balance_stats(const megray_router* r, void* workspace, void* stream) {
    mgk::balance::Router router;
    if (!to_router(r, &router))
        return kInvalid;
    return rc(mgk::balance::launch_stats(router, workspace, S(stream)));
}
int megray_balance_grad(const megray_router* r, const void* partials, int n_partials, const void* workspace,
                        const megray_balance_out* out, void* stream) {
    mgk::balance::Router router;
    mgk::balance::Result result;
    if (!to_router(r, &router) || !to_result(out, &result))
        return kInvalid;
    return rc(mgk::balance::launch_grad(router, partials, n_partials, workspace, result, false, S(stream)));
}
int megray_balance(const megray_router* r, const megray_balance_out* out, void* workspace, void* stream) {
    mgk::balance::Router router;
    mgk::balance::Result result;
    if (!to_router(r, &router) || !to_result(out, &result))
        return kInvalid;
    if (mgk::balance::is_small(router.tokens, router.experts))
        return rc(mgk::balance::launch_small(router, workspace, result, S(stream)));
    const cudaError_t e = mgk::balance::launch_stats(router, workspace, S(stream));
    if (e != cudaSuccess)
        return rc(e);
    return rc(mgk::balance::launch_grad(router, workspace, mgk::balance::partials(router.tokens, router.experts), workspace,
                                        result, true, S(stream)));
}

}  // extern "C"
